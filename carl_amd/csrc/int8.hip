// int8.hip - products of 8-bit codes on the matrix cores, with scales for each
// row and column, a bias, or the gate of a feed-forward block.
//
//   acc = x w^T, exact in 32 bits          y = (acc x_scale) w_scale + bias
// A product of two codes is at most 2^14 and a sum has at most 2^16 of them.
// Sums are whole numbers, so neither tiles nor the order change a result.
//
// `product` copies panels of both operands straight into LDS, two stages of 128
// bytes a row, one barrier a stage; rows that do not lie in whole 16-byte pieces
// go there through registers.  A row's last piece may hold bytes that are not
// its own: they are zeros in one of the operands.  `thin` is the product of a
// few rows, from memory to registers.
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
    int32_t width, columns, type, activation;
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

__device__ inline float biasOf(const Args& a, int n)
{
    if (a.type == CARL_OP_F32) return static_cast<const float*>(a.bias)[n];
    if (a.type == CARL_OP_BF16) return (float)static_cast<const bf16*>(a.bias)[n];
    return (float)static_cast<const f16*>(a.bias)[n];
}

template <bool kGated> __device__ inline float valueOf(const Args& a, int acc, int up, float xScale, const float (&scale)[2], float bias)
{
    const float y = (float)acc * xScale * scale[0];
    if constexpr (kGated) return activate(y, a.activation) * ((float)up * xScale * scale[1]);
    return a.bias ? y + bias : y;
}

// kRun neighbouring values of a row from column n on.
template <typename T, int kRun> __device__ inline void storeRun(const Args& a, int64_t row, int n, const float (&x)[kRun])
{
    constexpr int kE = 16 / sizeof(T), kPiece = kRun < kE ? kRun : kE;
    T* const to = static_cast<T*>(a.y) + row * a.columns + n;
    if (n + kRun <= a.columns) {
#pragma unroll
        for (int e = 0; e < kRun; e += kPiece) {
            vec<T, kPiece> v;
#pragma unroll
            for (int i = 0; i < kPiece; i++) v[i] = (T)x[e + i];
            __builtin_memcpy(to + e, &v, sizeof(v));
        }
    } else {
#pragma unroll
        for (int e = 0; e < kRun; e++)
            if (n + e < a.columns) to[e] = (T)x[e];
    }
}

// ---- product -------------------------------------------------------------------

constexpr int kRowBytes = 128, kPieces = kRowBytes / 16;

// Rows in LDS have their pieces permuted by the number of the lane that reads
// them, as in the block's products: a's rows by the row mod 8, b's by what
// bReader() says.
template <bool kGated, bool kDirect, int kBM, int kBN, int kWM, int kWN>
__global__ __launch_bounds__(kWM* kWN * 64) void int8ProductKernel(const Args args)
{
    constexpr int kNB = kGated ? 2 : 1, kThreads = kWM * kWN * 64;
    constexpr int kTM = kBM / kWM / 16, kTN = kBN / kWN / 16, kRun = 4 * kTN;
    constexpr int kStage = (kBM + kNB * kBN) * kRowBytes, kCopyRows = kThreads / kPieces;
    static_assert(kBM % kCopyRows == 0 && kBN % kCopyRows == 0, "whole copies");
    static_assert(kCopyRows % 8 == 0 && kCopyRows % (2 * kRun) == 0, "one permutation for a thread's pieces");
    __shared__ __align__(1024) char stages[2 * kStage];

    // the tiles of one row of tiles run next to each other on one of the 8 dies
    const int tilesN = (args.columns + kBN - 1) / kBN;
    const int64_t tilesM = (args.rows + kBM - 1) / kBM;
    const int die = blockIdx.x % 8;
    const int64_t local = blockIdx.x / 8;
    const int64_t tm = local / tilesN * 8 + die;
    const int tn = (int)(local % tilesN);
    if (tm >= tilesM) return;
    const int64_t m0 = tm * kBM;
    const int n0 = tn * kBN;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, col = lane & 15, quad = lane >> 4;
    const int wm = wave / kWN, wn = wave % kWN;

    i32x4 acc[kNB][kTN][kTM];
#pragma unroll
    for (int b = 0; b < kNB; b++)
#pragma unroll
        for (int j = 0; j < kTN; j++)
#pragma unroll
            for (int i = 0; i < kTM; i++) acc[b][j][i] = i32x4{ 0, 0, 0, 0 };

    // Rows past the operand's end lie past the descriptor's, pieces past a
    // row's width are sent there: both arrive as zeros.  (A piece with a byte
    // of a row in it is read whole: it lies in one page with that byte.)
    const int copyRow = threadIdx.x / kPieces;
    const auto copyPanel = [&](const int8_t* data, int64_t all, int64_t stride, int64_t row0, int rows, int k0, int at, bool weights) {
        const int8_t* base = data + row0 * stride;
        const int have = (int)(all - row0 < rows ? all - row0 : rows);
        const int c = (threadIdx.x % kPieces ^ (weights ? bReader<kRun>(copyRow) : copyRow & 7)) * 16;
        if constexpr (kDirect) {
            const i32x4 from = descriptor(base, have * (int)stride);
            const bool within = k0 + c < args.width;
#pragma unroll
            for (int i = 0; i < rows / kCopyRows; i++)
                copyToLds(from, within ? (copyRow + i * kCopyRows) * (int)stride + c : kOutside, k0,
                          ldsAddress(stages) + at + (i * kThreads + wave * 64) * 16);
        } else {
#pragma unroll
            for (int i = 0; i < rows / kCopyRows; i++) {
                const int row = copyRow + i * kCopyRows;
                const uint4 piece = loadBytes(base + row * stride + k0 + c, row < have ? args.width - k0 - c : 0);
                *reinterpret_cast<uint4*>(stages + at + (i * kThreads + threadIdx.x) * 16) = piece;
            }
        }
    };
    const auto copyStage = [&](int step, int at) {
        copyPanel(args.x, args.rows, args.xRow, m0, kBM, step * kRowBytes, at, false);
#pragma unroll
        for (int b = 0; b < kNB; b++)
            copyPanel(args.w[b], args.columns, args.wRow[b], n0, kBN, step * kRowBytes, at + (kBM + b * kBN) * kRowBytes, true);
    };
    const int aRow = (wm * kTM * 16 + col) * kRowBytes, piece0 = (quad ^ (col & 7)) * 16;
    const int bRow = (wn * kTN * 16 + (col >> 2) * kRun + (col & 3)) * kRowBytes;
    const int steps = (args.width + kRowBytes - 1) / kRowBytes;
    const auto multiply = [&](const char* lds, int step) {
        const bool cut = kDirect && step == steps - 1 && args.width % 16 != 0;
#pragma unroll
        for (int half = 0; half < 2; half++) {
            __builtin_amdgcn_sched_barrier(0);      // the fragments of one half at a time
            const char* aAt = lds + (aRow + (piece0 ^ half * 64));
            const char* bAt = lds + kBM * kRowBytes + (bRow + (piece0 ^ half * 64));
            uint4 a[kTM];
#pragma unroll
            for (int i = 0; i < kTM; i++) a[i] = *reinterpret_cast<const uint4*>(aAt + i * 16 * kRowBytes);
            if (cut) {
                const int have = args.width - step * kRowBytes - half * 64 - quad * 16;
#pragma unroll
                for (int i = 0; i < kTM; i++) a[i] = firstBytes(a[i], have);
            }
#pragma unroll
            for (int p = 0; p < kNB; p++)
#pragma unroll
                for (int j = 0; j < kTN; j++) {
                    const uint4 b = *reinterpret_cast<const uint4*>(bAt + (p * kBN + j * 4) * kRowBytes);
#pragma unroll
                    for (int i = 0; i < kTM; i++) acc[p][j][i] = mma(b, a[i], acc[p][j][i]);
                }
        }
    };

    copyStage(0, 0);
    waitCopies();
    __syncthreads();
    for (int step = 0; step < steps; step++) {
        if (step + 1 < steps) copyStage(step + 1, ((step + 1) & 1) * kStage);
        multiply(stages + (step & 1) * kStage, step);
        waitCopies();
        __syncthreads();
    }

    // a lane's columns: kRun neighbours from n on, of row `col` of each tile
    const int n = n0 + wn * kTN * 16 + quad * kRun;
    float scale[kNB][kRun], bias[kRun];
#pragma unroll
    for (int e = 0; e < kRun; e++) {
        const int at = n + e < args.columns ? n + e : args.columns - 1;
#pragma unroll
        for (int b = 0; b < kNB; b++) scale[b][e] = args.wScale[b][at];
        bias[e] = args.bias ? biasOf(args, at) : 0.0f;
    }
#pragma unroll
    for (int i = 0; i < kTM; i++) {
        const int64_t row = m0 + (wm * kTM + i) * 16 + col;
        if (row >= args.rows) continue;
        const float xScale = args.xScale[row];
        float y[kRun];
#pragma unroll
        for (int j = 0; j < kTN; j++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int at = j * 4 + e;
                const float both[2] = { scale[0][at], scale[kNB - 1][at] };
                y[at] = valueOf<kGated>(args, acc[0][j][i][e], acc[kNB - 1][j][i][e], xScale, both, bias[at]);
            }
        if (args.type == CARL_OP_F32) storeRun<float, kRun>(args, row, n, y);
        else if (args.type == CARL_OP_BF16) storeRun<bf16, kRun>(args, row, n, y);
        else storeRun<f16, kRun>(args, row, n, y);
    }
}

// ---- thin ----------------------------------------------------------------------

// A product of at most 64 rows a workgroup, which is a matter of latency: 16
// columns a workgroup, its eight waves taking the sum's blocks in turn,
// fragments straight from memory, whatever its alignment, to registers, one
// exchange at the end.
template <bool kGated, int kTM> __global__ __launch_bounds__(512) void int8ThinKernel(const Args args)
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
#pragma unroll 2
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
    float y[4];
#pragma unroll
    for (int e = 0; e < 4; e++) {
        const int at = n + e < args.columns ? n + e : args.columns - 1;
        const float scale[2] = { args.wScale[0][at], kGated ? args.wScale[1][at] : 0.0f };
        y[e] = valueOf<kGated>(args, sum[0][e], sum[kNB - 1][e], args.xScale[m], scale, args.bias ? biasOf(args, at) : 0.0f);
    }
    if (args.type == CARL_OP_F32) storeRun<float, 4>(args, m, n, y);
    else if (args.type == CARL_OP_BF16) storeRun<bf16, 4>(args, m, n, y);
    else storeRun<f16, 4>(args, m, n, y);
}

// ---- launches ------------------------------------------------------------------

constexpr int64_t kMostRows = (int64_t)1 << 28, kThinRows = 128;

template <bool kGated, bool kDirect, int kBM, int kBN, int kWM, int kWN> void launchTile(const Args& a, hipStream_t stream)
{
    const int64_t tilesM = (a.rows + kBM - 1) / kBM, tilesN = (a.columns + kBN - 1) / kBN;
    int8ProductKernel<kGated, kDirect, kBM, kBN, kWM, kWN><<<dim3((unsigned)((tilesM + 7) / 8 * 8 * tilesN)), kWM * kWN * 64, 0, stream>>>(a);
}

// Rows that a descriptor can take: whole 16-byte pieces, one row after another.
bool inPieces(const void* p, int64_t stride, int width)
{
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride % 16 == 0 && stride >= width && stride <= (int64_t)1 << 22;
}

template <bool kGated, bool kDirect> void launchProduct(const Args& a, hipStream_t stream)
{
    const auto tiles = [&](int rows, int columns) { return (a.rows + rows - 1) / rows * ((a.columns + columns - 1) / columns); };
    if (tiles(128, 128) >= 256) launchTile<kGated, kDirect, 128, 128, 2, 2>(a, stream);
    else launchTile<kGated, kDirect, 64, 64, 2, 2>(a, stream);
}

template <bool kGated> void launchAll(const Args& a, hipStream_t stream)
{
    if (a.rows <= kThinRows) {
        const unsigned columns = (unsigned)((a.columns + 15) / 16);
        if (a.rows <= 16) int8ThinKernel<kGated, 1><<<dim3(columns), 512, 0, stream>>>(a);
        else if (a.rows <= 32) int8ThinKernel<kGated, 2><<<dim3(columns), 512, 0, stream>>>(a);
        else int8ThinKernel<kGated, 4><<<dim3(columns, (unsigned)((a.rows + 63) / 64)), 512, 0, stream>>>(a);
        return;
    }
    const bool direct = inPieces(a.x, a.xRow, a.width) && inPieces(a.w[0], a.wRow[0], a.width)
                     && (!kGated || inPieces(a.w[1], a.wRow[1], a.width));
    if (direct) launchProduct<kGated, true>(a, stream);
    else launchProduct<kGated, false>(a, stream);
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
    if (p->rows < 0 || p->rows > kMostRows || tiles > (int64_t)1 << 22) return fail(CARL_ERR_VALUE, "rows are out of range");
    if (gated && p->bias) return fail(CARL_ERR_VALUE, "the gated product has no bias");
    if (p->rows == 0) return CARL_OK;
    if (!p->x || !p->x_scale || !p->w || !p->w_scale || (gated && !p->w_up_scale) || !p->y) return fail(CARL_ERR_VALUE, "null product tensor");
    const Args a{ p->x, { p->w, p->w_up }, p->x_row, { p->w_row, p->w_up_row }, p->rows, p->x_scale, { p->w_scale, p->w_up_scale },
                  p->bias, p->y, p->width, p->columns, p->type, p->activation };
    if (gated) launchAll<true>(a, (hipStream_t)stream);
    else launchAll<false>(a, (hipStream_t)stream);
    return launched("8-bit product");
}
