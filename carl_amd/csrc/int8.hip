// int8.hip - products of 8-bit codes on the matrix cores, with scales for each
// row and column, a bias, or the gate of a feed-forward block.
//
//   acc = x w^T, exact in 32 bits          y = (acc x_scale) w_scale + bias
// A product of two codes is at most 2^14 and a sum has at most 2^16 of them.
// Sums are whole numbers, so neither tiles nor the order change a result.
//
// `product` multiplies panels that it copies straight into LDS; rows that do not
// lie in whole 16-byte pieces go there through registers.  A row's last piece
// may hold bytes that are not its own: they are zeros in one of the operands.
// `thin` is the product of a few rows, from memory to registers.
#include <algorithm>

#include "../../include/carl_amd_ops.h"
#include "ffn_kernel.h"

using namespace carl;

namespace {

struct Args {
    const int8_t *x, *w[2];
    int64_t xRow, wRow[2], rows;
    const float *xScale, *wScale[2];
    const void* bias;
    void* y;
    int32_t width, columns, activation;
};

__device__ inline i32x4 mma(uint4 a, uint4 b, i32x4 c)
{
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, a), __builtin_bit_cast(i32x4, b), c, 0, 0, 0);
}

// The first `have` of 16 bytes, zeros after them.
__device__ inline uint4 firstBytes(uint4 x, int have)
{
    i32x4 v = __builtin_bit_cast(i32x4, x);
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int bytes = have - i * 4;
        v[i] = bytes >= 4 ? v[i] : bytes <= 0 ? 0 : v[i] & (int)((1u << (bytes * 8)) - 1u);
    }
    return __builtin_bit_cast(uint4, v);
}

__device__ inline uint4 loadBytes(const int8_t* p, int have)
{
    uint4 r;
    if (have >= 16) __builtin_memcpy(&r, p, 16);
    else {
        vec<int8_t, 16> b;
#pragma unroll
        for (int j = 0; j < 16; j++) b[j] = j < have ? p[j] : (int8_t)0;
        r = __builtin_bit_cast(uint4, b);
    }
    return r;
}

// kActivation: of the gated form, or kNone.
constexpr int kNone = -1;

// The gate is not multiplied by log2(e) in its column's scale, which is a product less for each value (131,072 x 512 to two of
// 1,408 255 us, so 261): past 2.36e38 that would leave float32's range, to an infinity or, of a negative gate, a NaN.
template <int kActivation> __device__ inline float valueOf(int acc, int up, float xScale, float scale, float upScale)
{
    const float y = (float)acc * xScale * scale;
    if constexpr (kActivation == kNone) return y;
    // (the gate first: of a large negative one it is 0 whatever u is, where y u may be an infinity)
    return activate(y, kActivation) * ((float)up * xScale * upScale);
}

// kRun neighbouring values of a row, of which `have` are the result's.
template <typename T, int kRun> __device__ inline void storeRun(T* to, const float (&x)[kRun], int have)
{
    constexpr int kE = 16 / sizeof(T), kPiece = kRun < kE ? kRun : kE;
    if (have >= kRun) {
#pragma unroll
        for (int e = 0; e < kRun; e += kPiece) {
            vec<float, kPiece> v;
#pragma unroll
            for (int i = 0; i < kPiece; i++) v[i] = x[e + i];
            const auto r = fromFloat<T, kPiece>(v);
            __builtin_memcpy(to + e, &r, sizeof(r));
        }
    } else {
#pragma unroll
        for (int e = 0; e < kRun; e++)
            if (e < have) to[e] = (T)x[e];
    }
}

// ---- product -------------------------------------------------------------------

constexpr int kRowBytes = 128, kPieces = kRowBytes / 16;     // of a row in a stage

// 4 bytes a lane from memory to 4 x lane bytes past `lds`, as copyToLds.
__device__ inline void copyWordToLds(i32x4 from, int offset, uint32_t lds)
{
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dword %1, %2, 0 offen lds" : : "s"(lds), "v"(offset), "s"(from) : "memory");
}

template <int kYounger> __device__ inline void waitAllBut()
{
    static_assert(kYounger < 64, "what vmcnt counts");
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kYounger) : "memory");
}

// What is computed from it is computed where it is used: the largest tiles have
// no register left to keep it in.
__device__ inline int anew(int x)
{
    asm volatile("" : "+v"(x));
    return x;
}

// A tile of kBM rows by kBN columns (of the gated form: of both weights) that
// kWM x kWN waves compute from stages of 128 bytes of every row in LDS.
//
// The tiles of b that a wave multiplies are dealt to the columns so that a
// lane's results are runs of 8 neighbours, and the four quads' runs lie next to
// each other: element e of tile j and quad q is column 32 (j / 2) + 8 q +
// 4 (j % 2) + e.  Rows in LDS have their eight 16-byte pieces permuted by the
// number, mod 8, of the lane that reads them, so that eight lanes meet all
// banks: x's by the row's, w's by what wReader says.
template <typename T, bool kGated, int kBM, int kBN, int kWM, int kWN> struct Tile {
    static constexpr int kNB = kGated ? 2 : 1, kThreads = kWM * kWN * 64;
    static constexpr int kTM = kBM / kWM / 16, kTN = kBN / kWN / 16, kRun = 8;
    static constexpr int kRows = kBM + kNB * kBN, kStage = kRows * kRowBytes;
    static constexpr int kCopyRows = kThreads / kPieces, kCopies = kRows / kCopyRows;
    // words of scales: of the rows, of the columns, and the bias
    static constexpr int kBiasWords = kGated ? 0 : (kBN * (int)sizeof(T) / 4 + 63) / 64 * 64, kWords = kBM + kNB * kBN + kBiasWords;
    static constexpr int kScales = kWords * 4;
    static constexpr int kStores = kTM * (kTN / 2) * (int)sizeof(T) / 2;       // of a whole tile
    static_assert(kBM % kCopyRows == 0 && kBN % kCopyRows == 0, "whole copies");
    static_assert(kCopyRows % 16 == 0 && kTN % 2 == 0, "one permutation for a thread's pieces, runs of two tiles");
    static_assert(kBM % 64 == 0 && kBN % 64 == 0, "a wave's words are of one kind");

    i32x4 acc[kNB][kTN][kTM];
    int wm, wn;

    __device__ Tile()
    {
        const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        wm = wave / kWN;
        wn = wave % kWN;
    }

    __device__ void clear()
    {
#pragma unroll
        for (int b = 0; b < kNB; b++)
#pragma unroll
            for (int j = 0; j < kTN; j++)
#pragma unroll
                for (int i = 0; i < kTM; i++) acc[b][j][i] = i32x4{ 0, 0, 0, 0 };
    }

    // What a thread copies of x's rows (or w's): a piece of every kCopyRows-th, at this byte of their 128.
    static __device__ int wReader(int row) { return (row & 3) | (row >> 3 & 1) << 2; }
    static __device__ int pieceOf(int thread, bool weights)
    {
        const int row = thread / kPieces;
        return (thread % kPieces ^ (weights ? wReader(row) : row & 7)) * 16;
    }

    // What a wave multiplies of half a stage.
    struct Fragments {
        uint4 x[kTM], w[kNB][kTN];
    };

    __device__ void load(Fragments& f, const char* lds, int half) const
    {
        const int lane = anew(threadIdx.x) & 63, col = lane & 15, quad = lane >> 4, piece = (half * 4 + quad ^ col & 7) * 16;
        const char* const x = lds + (wm * kTM * 16 + col) * kRowBytes + piece;
        const char* const w = lds + (kBM + wn * kTN * 16 + (col >> 2) * 8 + (col & 3)) * kRowBytes + piece;
#pragma unroll
        for (int i = 0; i < kTM; i++) f.x[i] = *reinterpret_cast<const uint4*>(x + i * 16 * kRowBytes);
#pragma unroll
        for (int b = 0; b < kNB; b++)
#pragma unroll
            for (int j = 0; j < kTN; j++) f.w[b][j] = *reinterpret_cast<const uint4*>(w + (b * kBN + j / 2 * 32 + j % 2 * 4) * kRowBytes);
    }

    // have: bytes of the rows from this half on; what lies past them counts as zeros.
    __device__ void multiply(Fragments& f, int have)
    {
        if (have < 64) {
            const int quad = (anew(threadIdx.x) & 63) >> 4;
#pragma unroll
            for (int i = 0; i < kTM; i++) f.x[i] = firstBytes(f.x[i], have - quad * 16);
        }
#pragma unroll
        for (int b = 0; b < kNB; b++)
#pragma unroll
            for (int j = 0; j < kTN; j++)
#pragma unroll
                for (int i = 0; i < kTM; i++) acc[b][j][i] = mma(f.w[b][j], f.x[i], acc[b][j][i]);
    }

    template <int kActivation, bool kWhole> __device__ void finish(const Args& args, const float* scales, int64_t m0, int n0) const
    {
        const int lane = anew(threadIdx.x) & 63, n = wn * kTN * 16 + (lane >> 4) * 8, m = wm * kTM * 16 + (lane & 15);
        T* const y = static_cast<T*>(args.y) + (m0 + m) * args.columns + n0 + n;
        float xScale[kTM];
#pragma unroll
        for (int i = 0; i < kTM; i++) xScale[i] = scales[m + i * 16];
#pragma unroll
        for (int r = 0; r < kTN / 2; r++) {
            f32x4 scale[kNB][2];
            vec<T, kRun> bias;
#pragma unroll
            for (int b = 0; b < kNB; b++)
#pragma unroll
                for (int h = 0; h < 2; h++) scale[b][h] = *reinterpret_cast<const f32x4*>(scales + kBM + b * kBN + n + r * 32 + h * 4);
            if (!kGated && args.bias) bias = *reinterpret_cast<const vec<T, kRun>*>(reinterpret_cast<const T*>(scales + kBM + kBN) + n + r * 32);
#pragma unroll
            for (int i = 0; i < kTM; i++) {
                if (!kWhole && m0 + m + i * 16 >= args.rows) continue;
                float value[kRun];
#pragma unroll
                for (int e = 0; e < kRun; e++) {
                    const int j = r * 2 + e / 4;
                    value[e] = valueOf<kActivation>(acc[0][j][i][e % 4], acc[kNB - 1][j][i][e % 4], xScale[i], scale[0][e / 4][e % 4],
                                                    scale[kNB - 1][e / 4][e % 4]);
                    if (!kGated && args.bias) value[e] += (float)bias[e];
                }
                storeRun<T, kRun>(y + (int64_t)i * 16 * args.columns + r * 32, value, kWhole ? kRun : args.columns - n0 - n - r * 32);
            }
        }
    }

    // Whether all of the tile was stored, with kStores stores.
    __device__ bool finish(const Args& args, const float* scales, int64_t m0, int n0) const
    {
        const bool whole = m0 + kBM <= args.rows && n0 + kBN <= args.columns;
        const auto with = [&](auto activation) {
            if (whole) finish<activation(), true>(args, scales, m0, n0);
            else finish<activation(), false>(args, scales, m0, n0);
        };
        if constexpr (!kGated) with(std::integral_constant<int, kNone>());
        else if (args.activation == CARL_SILU) with(std::integral_constant<int, CARL_SILU>());
        else with(std::integral_constant<int, CARL_GELU>());
        return whole;
    }
};

// Each of the 8 dies (blocks are dealt to them in turn) takes every eighth row of
// tiles, so that x's rows are read from memory once, and an eighth of the tiles of
// the rows that are left (512 rows of 4,096 to 8,192, four rows of tiles, 29 us;
// by four dies alone 43).  Rows far apart for each die would not do: 131,072 x 512
// to 1,408, where they lie 2^23 bytes apart, 174 us, so 168.
struct Places {
    int die, tilesN, own, rest, restBegin, count;        // of the die's tiles, in order

    __device__ Places(const Args& args, int bm, int bn) : die(blockIdx.x % 8), tilesN((args.columns + bn - 1) / bn)
    {
        const int tilesM = (int)((args.rows + bm - 1) / bm), left = tilesM % 8 * tilesN;
        own = tilesM / 8 * tilesN;
        rest = tilesM / 8 * 8;
        restBegin = left * die / 8;
        count = own + left * (die + 1) / 8 - restBegin;
    }
    __device__ int row(int place) const { return place < own ? place / tilesN * 8 + die : rest + (restBegin + place - own) / tilesN; }
    __device__ int column(int place) const { return (place < own ? place : restBegin + place - own) % tilesN; }
};

// Workgroups stay and take every so-many-th tile of their die.  While half a
// stage is multiplied from registers, the next half is read from LDS, and the
// stages after it are on their way there, across the ends of tiles, so that the
// next tile's first ones (and its scales) arrive while a tile's results are
// computed and written.  Between the halves a step waits for the next stage's
// copies, the younger ones (and the last results' stores) stay outstanding; the
// one barrier after it hands that stage over and frees this one, which is in
// registers by then.
template <typename T, bool kGated, int kBM, int kBN, int kWM, int kWN, int kStages, int kBlocks>
__global__ __launch_bounds__(kWM* kWN * 64, kWM* kWN * kBlocks / 4) void int8ProductKernel(const Args args)
{
    using Tile = Tile<T, kGated, kBM, kBN, kWM, kWN>;
    constexpr int kNB = Tile::kNB, kThreads = Tile::kThreads, kStage = Tile::kStage, kCopyRows = Tile::kCopyRows;
    constexpr int kCopies = Tile::kCopies, kYounger = kCopies * (kStages - 2);
    // stages, the scales of a tile and of those that copies may be ahead by
    __shared__ __align__(1024) char stages[kStages * kStage + (kStages + 1) * Tile::kScales];
    const Places places(args, kBM, kBN);
    const int stride = gridDim.x / 8, first = blockIdx.x / 8;
    if (first >= places.count) return;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int steps = (args.width + kRowBytes - 1) / kRowBytes;
    const uint32_t lds = ldsAddress(stages);

    // Rows past an operand's end lie past its descriptor's, pieces past a row's
    // width are sent there: both arrive as zeros.  (A piece with a byte of a
    // row in it is read whole: it lies in one page with that byte.)
    i32x4 from[1 + kNB];
    int at[1 + kNB];
    at[0] = (int)threadIdx.x / kPieces * (int)args.xRow + Tile::pieceOf(threadIdx.x, false);
#pragma unroll
    for (int b = 0; b < kNB; b++) at[1 + b] = (int)threadIdx.x / kPieces * (int)args.wRow[b] + Tile::pieceOf(threadIdx.x, true);
    int copyPlace = first, copyStep = 0, copyScales = 0;
    const auto copyNext = [&](int slot) {
        if (copyStep == 0) {        // another tile: its rows, and its scales
            const bool any = copyPlace < places.count;
            const int64_t m0 = (int64_t)places.row(copyPlace) * kBM;
            const int n0 = places.column(copyPlace) * kBN;
            const int rows = !any ? 0 : args.rows - m0 < kBM ? (int)(args.rows - m0) : kBM;
            const int columns = !any ? 0 : args.columns - n0 < kBN ? args.columns - n0 : kBN;
            from[0] = descriptor(args.x + m0 * args.xRow, rows * (int)args.xRow);
#pragma unroll
            for (int b = 0; b < kNB; b++) from[1 + b] = descriptor(args.w[b] + n0 * args.wRow[b], columns * (int)args.wRow[b]);
            for (int word = wave * 64; word < Tile::kWords; word += kThreads) {
                const void* of = args.xScale + m0 + word;
                int bytes = (rows - word) * 4;
                if (word >= kBM + kNB * kBN) {
                    // (a last column's odd half is read with the one before it)
                    const int c = (word - kBM - kNB * kBN) * 4 / (int)sizeof(T);
                    of = static_cast<const T*>(args.bias) + n0 + c;
                    bytes = args.bias ? ((columns - c) * (int)sizeof(T) + 3) / 4 * 4 : 0;
                } else if (word >= kBM) {
                    const int b = (word - kBM) / kBN, c = (word - kBM) % kBN;
                    of = args.wScale[b] + n0 + c;
                    bytes = (columns - c) * 4;
                }
                copyWordToLds(descriptor(of, bytes > 0 ? bytes : 0), (int)(threadIdx.x & 63) * 4,
                              lds + kStages * kStage + copyScales * Tile::kScales + word * 4);
            }
            copyScales = copyScales == kStages ? 0 : copyScales + 1;
            copyPlace += stride;
        }
        const int k0 = copyStep * kRowBytes, thread = anew(threadIdx.x);
#pragma unroll
        for (int p = 0; p < 1 + kNB; p++) {
            const bool within = k0 + Tile::pieceOf(thread, p > 0) < args.width;
            const int apart = kCopyRows * (int)(p == 0 ? args.xRow : args.wRow[p == 2 ? 1 : 0]);
#pragma unroll
            for (int i = 0; i < (p == 0 ? kBM : kBN) / kCopyRows; i++)
                copyToLds(from[p], within ? at[p] + i * apart : kOutside, k0,
                          lds + slot * kStage + (p == 0 ? 0 : kBM + (p - 1) * kBN) * kRowBytes + i * kThreads * 16 + wave * 1024);
        }
        copyStep = copyStep + 1 == steps ? 0 : copyStep + 1;
    };

#pragma unroll
    for (int i = 0; i < kStages; i++) copyNext(i);
    Tile tile;
    typename Tile::Fragments even, odd;
    waitAllBut<kCopies*(kStages - 1)>();
    __syncthreads();
    tile.load(even, stages, 0);
    int slot = 0, scales = 0, storesLeft = 0;
    for (int place = first; place < places.count; place += stride) {
        tile.clear();
        for (int i = 0; i < steps; i++) {
            const int have = args.width - i * kRowBytes;
            tile.load(odd, stages + slot * kStage, 1);
            tile.multiply(even, have);
            if (storesLeft > 0) {
                waitAllBut<kYounger + Tile::kStores>();
                storesLeft--;
            } else waitAllBut<kYounger>();
            __syncthreads();
            copyNext(slot);
            slot = slot + 1 == kStages ? 0 : slot + 1;
            tile.load(even, stages + slot * kStage, 0);
            if (have > 64) tile.multiply(odd, have - 64);
        }
        const float* const own = reinterpret_cast<const float*>(stages + kStages * kStage + scales * Tile::kScales);
        const bool whole = tile.finish(args, own, (int64_t)places.row(place) * kBM, places.column(place) * kBN);
        scales = scales == kStages ? 0 : scales + 1;
        // the stores are younger than the copies of the next kStages stages; a part of a tile has fewer, so that they are waited for
        if (!whole) waitCopies();
        storesLeft = whole ? kStages - 1 : 0;
    }
    waitCopies();          // none outlives its workgroup's LDS
}

// The same of rows that do not lie in whole pieces, or scales and biases that
// do not begin at words: through registers, a tile a workgroup.
template <typename T, bool kGated, int kBM, int kBN, int kWM, int kWN>
__global__ __launch_bounds__(kWM* kWN * 64) void int8LooseKernel(const Args args)
{
    using Tile = Tile<T, kGated, kBM, kBN, kWM, kWN>;
    constexpr int kNB = Tile::kNB, kThreads = Tile::kThreads, kStage = Tile::kStage, kCopyRows = Tile::kCopyRows;
    __shared__ __align__(1024) char stages[2 * kStage + Tile::kScales];
    const Places places(args, kBM, kBN);
    const int place = blockIdx.x / 8;
    if (place >= places.count) return;
    const int64_t m0 = (int64_t)places.row(place) * kBM;
    const int n0 = places.column(place) * kBN;

    float* const scales = reinterpret_cast<float*>(stages + 2 * kStage);
    for (int i = threadIdx.x; i < kBM; i += kThreads) scales[i] = m0 + i < args.rows ? args.xScale[m0 + i] : 0.0f;
    for (int i = threadIdx.x; i < kNB * kBN; i += kThreads) scales[kBM + i] = n0 + i % kBN < args.columns ? args.wScale[i / kBN][n0 + i % kBN] : 0.0f;
    if (!kGated && args.bias)
        for (int i = threadIdx.x; i < kBN; i += kThreads)
            reinterpret_cast<T*>(scales + kBM + kBN)[i] = n0 + i < args.columns ? static_cast<const T*>(args.bias)[n0 + i] : T(0);

    uint4 held[Tile::kCopies];
    const auto load = [&](int k0) {
#pragma unroll
        for (int n = 0; n < Tile::kCopies; n++) {
            const int panel = n * kCopyRows < kBM ? 0 : (n * kCopyRows - kBM) / kBN + 1;
            const int row = n * kCopyRows - (panel == 0 ? 0 : kBM + (panel - 1) * kBN) + (int)threadIdx.x / kPieces, c = k0 + Tile::pieceOf(threadIdx.x, panel > 0);
            const int64_t at = (panel == 0 ? m0 : n0) + row, stride = panel == 0 ? args.xRow : args.wRow[panel - 1];
            const bool have = at < (panel == 0 ? args.rows : args.columns);
            held[n] = loadBytes((panel == 0 ? args.x : args.w[panel - 1]) + at * stride + c, have ? args.width - c : 0);
        }
    };
    const auto put = [&](int slot) {
#pragma unroll
        for (int n = 0; n < Tile::kCopies; n++) *reinterpret_cast<uint4*>(stages + slot * kStage + (n * kThreads + threadIdx.x) * 16) = held[n];
    };
    Tile tile;
    tile.clear();
    load(0);
    put(0);
    const int steps = (args.width + kRowBytes - 1) / kRowBytes;
    for (int i = 0; i < steps; i++) {
        __syncthreads();
        if (i + 1 < steps) load((i + 1) * kRowBytes);
#pragma unroll
        for (int half = 0; half < 2; half++) {
            typename Tile::Fragments now;
            tile.load(now, stages + (i & 1) * kStage, half);
            tile.multiply(now, args.width - i * kRowBytes - half * 64);
        }
        if (i + 1 < steps) put((i + 1) & 1);
    }
    tile.finish(args, scales, m0, n0);
}

// ---- thin ----------------------------------------------------------------------

// A product of at most 64 rows a workgroup, which is a matter of latency: 16
// columns a workgroup, its eight waves taking the sum's blocks in turn,
// fragments straight from memory, whatever its alignment, to registers, one
// exchange at the end.
template <typename T, bool kGated, int kTM> __global__ __launch_bounds__(512) void int8ThinKernel(const Args args)
{
    constexpr int kWaves = 8, kNB = kGated ? 2 : 1;
    __shared__ i32x4 parts[kWaves][kNB][kTM][64];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, col = lane & 15, quad = lane >> 4;
    const int n0 = blockIdx.x * 16, m0 = blockIdx.y * 16 * kTM;
    // rows past the end are the last one again; their results are not stored
    const int own = n0 + col < args.columns ? n0 + col : args.columns - 1;
    const int8_t* w[kNB];
#pragma unroll
    for (int p = 0; p < kNB; p++) w[p] = args.w[p] + own * args.wRow[p];
    const int8_t* x[kTM];
#pragma unroll
    for (int i = 0; i < kTM; i++) {
        const int64_t m = m0 + i * 16 + col;
        x[i] = args.x + (m < args.rows ? m : args.rows - 1) * args.xRow;
    }
    i32x4 acc[kNB][kTM];
#pragma unroll
    for (int p = 0; p < kNB; p++)
#pragma unroll
        for (int i = 0; i < kTM; i++) acc[p][i] = i32x4{ 0, 0, 0, 0 };
#pragma unroll(kTM == 4 ? 2 : 4)
    for (int k = wave * 64 + quad * 16; k - quad * 16 < args.width; k += kWaves * 64) {
        const int have = args.width - k;
        uint4 b[kNB];
#pragma unroll
        for (int p = 0; p < kNB; p++) b[p] = loadBytes(w[p] + k, have);
#pragma unroll
        for (int i = 0; i < kTM; i++) {
            const uint4 a = loadBytes(x[i] + k, have);
#pragma unroll
            for (int p = 0; p < kNB; p++) acc[p][i] = mma(b[p], a, acc[p][i]);
        }
    }
#pragma unroll
    for (int p = 0; p < kNB; p++)
#pragma unroll
        for (int i = 0; i < kTM; i++) parts[wave][p][i][lane] = acc[p][i];
    __syncthreads();
    if (wave >= kTM) return;
    i32x4 sum[kNB];
#pragma unroll
    for (int p = 0; p < kNB; p++) {
        sum[p] = parts[0][p][wave][lane];
        for (int i = 1; i < kWaves; i++) sum[p] += parts[i][p][wave][lane];
    }
    const int64_t m = m0 + wave * 16 + col;
    if (m >= args.rows) return;
    const int n = n0 + quad * 4;
    const float xScale = args.xScale[m];
    float y[4];
#pragma unroll
    for (int e = 0; e < 4; e++) {
        const int at = n + e < args.columns ? n + e : args.columns - 1;
        const float scale = args.wScale[0][at], second = kGated ? args.wScale[1][at] : 0.0f;
        const auto value = [&](auto activation) {
            return valueOf<activation()>(sum[0][e], sum[kNB - 1][e], xScale, scale, second);
        };
        if constexpr (!kGated) {
            y[e] = value(std::integral_constant<int, kNone>());
            if (args.bias) y[e] += (float)static_cast<const T*>(args.bias)[at];
        } else if (args.activation == CARL_SILU) y[e] = value(std::integral_constant<int, CARL_SILU>());
        else y[e] = value(std::integral_constant<int, CARL_GELU>());
    }
    storeRun<T, 4>(static_cast<T*>(args.y) + m * args.columns + n, y, args.columns - n);
}

// ---- launches ------------------------------------------------------------------

constexpr int64_t kThinRows = 16;

// kBlocks workgroups a compute unit.
template <typename T, bool kGated, int kBM, int kBN, int kWM, int kWN, int kStages, int kBlocks> void launchTile(const Args& a, hipStream_t stream)
{
    const int64_t tiles = (a.rows + kBM - 1) / kBM * ((a.columns + kBN - 1) / kBN);
    const dim3 grid((unsigned)std::min<int64_t>((tiles + 7) / 8 * 8, 256 * kBlocks));
    int8ProductKernel<T, kGated, kBM, kBN, kWM, kWN, kStages, kBlocks><<<grid, kWM * kWN * 64, 0, stream>>>(a);
}

// Rows that a descriptor can take: whole 16-byte pieces, one row after another.
bool inPieces(const void* p, int64_t stride, int width)
{
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride % 16 == 0 && stride >= width && stride <= (int64_t)1 << 22;
}

bool inWords(const void* p) { return reinterpret_cast<uintptr_t>(p) % 4 == 0; }

// By sweeps from 1 to 131,072 rows (us):
//   few rows      1,408 to 512, 512 rows   thin 5.6   64 x 64 7.1     1,024 rows  9.0 and 7.4
//                 4,096 to 8,192, 1 row   7.0 and 16.2     32 rows  13.4 and 16.4     64 rows  21.2 and 16.5
//                 1,024 to 20,000, 16 rows   7.0 and 7.5     32 rows  9.5 and 7.8     128 rows  32.4 and 11.6
//                 (one row of 4,096 to 65,536 53 us: 5.0 TB/s of weights)
//   small tiles   1,024 to 2,816, 512 rows   64 x 64 7.5   128 x 128 9.3     1,024 rows  9.7 and 9.4     8,192 rows  44.8 and 34.0
//                 gated, 512 rows   64 x 64 9.4   128 x 64 12.5      2,001 rows  20.6 and 18.8
//   large tiles   1,408 to 512, 32,768 rows (256 tiles)   128 x 128 29.9   256 x 256 28.7      131,072 rows  139 and 107
//                 512 to 1,408, 16,384 rows (384 tiles, a round and a half)  22.8 and 26.5
// so the largest tiles are taken where they leave no more than a fifth of
// their rounds empty.  Of whole matrices at 8,192 cubed they reach 2,330 TOP/s
// (the library's 8-bit product, without scales: 2,420; 131,072 x 1,408 to 512
// 1,730 against 940).  They are bound by their copies into LDS (which alone
// take 0.6 of the time, in stages of 64 bytes a row 0.75) beside the matrix
// instructions (0.75); the gated form then by the operations on its results:
// some 113 of 261 us of 131,072 x 512 to 1,408, which no other tile's products hide.
// Few columns pay for whole tiles: 131,072 x 512 to 1, 18 and 64 columns 27, 27 and
// 28 us, 2.5 TB/s of x.
template <typename T, bool kGated> void launchAll(const Args& a, hipStream_t stream)
{
    const auto tiles = [&](int rows, int columns) { return (a.rows + rows - 1) / rows * ((a.columns + columns - 1) / columns); };
    if (a.rows <= kThinRows || tiles(16, 16) <= 1024) {
        const unsigned columns = (unsigned)((a.columns + 15) / 16);
        const auto thin = [&](auto tiles) {
            int8ThinKernel<T, kGated, tiles()><<<dim3(columns, (unsigned)((a.rows + 16 * tiles() - 1) / (16 * tiles()))), 512, 0, stream>>>(a);
        };
        // as few rows a workgroup as there are, or as keep the GPU from more than one round or so (4,096 to 64, 1,006 rows: 16 rows
        // 5.8 us, 64 rows 11.0; 1,408 to 512, 512 rows: 7.4 and 5.7; 4,096 to 8,192, one row: 7.0 and 11.8)
        if (a.rows <= 16 || tiles(16, 16) <= 256) thin(std::integral_constant<int, 1>());
        else if (a.rows <= 32 || tiles(32, 16) <= 384) thin(std::integral_constant<int, 2>());
        else thin(std::integral_constant<int, 4>());
        return;
    }
    const bool direct = inPieces(a.x, a.xRow, a.width) && inPieces(a.w[0], a.wRow[0], a.width)
                     && (!kGated || inPieces(a.w[1], a.wRow[1], a.width)) && inWords(a.bias);
    const auto fills = [](int64_t tiles) { return 5 * tiles >= 4 * ((tiles + 255) / 256 * 256); };
    if (!direct) {
        // (683 to 257, 2,001 rows: tiles of 128 x 128 24.8 us, of 64 x 64 15.6; 257 to 512, 16,384 rows: 14.4 and 19.0)
        constexpr int kBN = kGated ? 64 : 128;
        const auto loose = [&](auto bm, auto bn) {
            int8LooseKernel<T, kGated, bm(), bn(), 2, 2><<<dim3((unsigned)((tiles(bm(), bn()) + 7) / 8 * 8)), 256, 0, stream>>>(a);
        };
        if (tiles(128, kBN) >= 256) loose(std::integral_constant<int, 128>(), std::integral_constant<int, kBN>());
        else loose(std::integral_constant<int, 64>(), std::integral_constant<int, 64>());
    } else if constexpr (kGated) {
        if (fills(tiles(256, 128))) launchTile<T, kGated, 256, 128, 4, 2, 2, 1>(a, stream);
        else if (tiles(128, 64) >= 256) launchTile<T, kGated, 128, 64, 2, 2, 2, 2>(a, stream);
        else launchTile<T, kGated, 64, 64, 2, 2, 2, 3>(a, stream);
    } else {
        if (fills(tiles(256, 256))) launchTile<T, kGated, 256, 256, 4, 2, 2, 1>(a, stream);
        else if (tiles(128, 128) >= 176) launchTile<T, kGated, 128, 128, 4, 2, 2, 2>(a, stream);
        else launchTile<T, kGated, 64, 64, 2, 2, 3, 3>(a, stream);
    }
}

template <typename T> void launchFor(const Args& a, hipStream_t stream)
{
    if (a.w[1]) launchAll<T, true>(a, stream);
    else launchAll<T, false>(a, stream);
}

}  // namespace

extern "C" int carl_int8_linear_forward(const carl_int8_linear* p, void* stream)
{
    if (!p) return fail(CARL_ERR_VALUE, "null product argument");
    if (p->type != CARL_OP_F32 && p->type != CARL_OP_BF16 && p->type != CARL_OP_F16) return fail(CARL_ERR_TYPE, "unknown element type");
    const bool gated = p->w_up != nullptr;
    if (gated && p->activation != CARL_SILU && p->activation != CARL_GELU) return fail(CARL_ERR_VALUE, "unknown activation");
    if (p->width < 1 || p->width > CARL_INT8_MAX_DIM) return fail(CARL_ERR_VALUE, "width must be in [1, 65536]");
    if (p->columns < 1 || p->columns > CARL_INT8_MAX_DIM) return fail(CARL_ERR_VALUE, "columns must be in [1, 65536]");
    const int64_t tiles = (p->rows + 127) / 128 * ((p->columns + 127) / 128);
    if (p->rows < 0 || p->rows > CARL_INT8_MAX_ROWS || tiles > CARL_INT8_MAX_TILES) return fail(CARL_ERR_VALUE, "rows are out of range");
    if (gated && p->bias) return fail(CARL_ERR_VALUE, "the gated product has no bias");
    if (p->rows == 0) return CARL_OK;
    if (!p->x || !p->x_scale || !p->w || !p->w_scale || (gated && !p->w_up_scale) || !p->y) return fail(CARL_ERR_VALUE, "null product tensor");
    const Args a{ p->x, { p->w, p->w_up }, p->x_row, { p->w_row, p->w_up_row }, p->rows, p->x_scale, { p->w_scale, p->w_up_scale },
                  p->bias, p->y, p->width, p->columns, p->activation };
    if (p->type == CARL_OP_F32) launchFor<float>(a, (hipStream_t)stream);
    else if (p->type == CARL_OP_BF16) launchFor<bf16>(a, (hipStream_t)stream);
    else launchFor<f16>(a, (hipStream_t)stream);
    return launched("8-bit product");
}
