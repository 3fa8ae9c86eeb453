// ffn_kernel.h - the kernels of ffn.h, for one element type.
#pragma once

#include <algorithm>

#include "ffn.h"
#include "lds.h"
#include "status.h"

namespace carl {

typedef __attribute__((address_space(3))) i16x4 LdsI16x4;


// A lane's 16 bytes of either operand: row or column lane%16 of a 16x16 tile,
// 16/size neighbouring steps of the sum from 16/size times lane/16 on.
template <typename T> struct Mma;
template <> struct Mma<float> {
    static __device__ inline f32x4 run(uint4 a, uint4 b, f32x4 c)
    {
        const f32x4 x = __builtin_bit_cast(f32x4, a), y = __builtin_bit_cast(f32x4, b);
#pragma unroll
        for (int j = 0; j < 4; j++) c = __builtin_amdgcn_mfma_f32_16x16x4f32(x[j], y[j], c, 0, 0, 0);
        return c;
    }
};
template <> struct Mma<bf16> {
    static __device__ inline f32x4 run(uint4 a, uint4 b, f32x4 c)
    {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
};
template <> struct Mma<f16> {
    static __device__ inline f32x4 run(uint4 a, uint4 b, f32x4 c)
    {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    }
};

// act(g), and its slope where asked for.  The hardware's exponential and
// reciprocal are good to a unit in the last place each.
__device__ inline float activate(float g, int activation, float* slopeOut = nullptr)
{
    float z = g, slope = 1.0f;
    if (activation == CARL_GELU) {
        const float c = 1.5957691216057308f, g2 = g * g;       // 2 sqrt(2 / pi)
        z = c * (g + 0.044715f * g2 * g);
        slope = c * (1.0f + 0.134145f * fminf(g2, 1e30f));     // finite: it meets zeros in the tails
    }
    const float s = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(z * -1.44269504088896341f));
    const float act = g * s;
    if (slopeOut) *slopeOut = s + act * (1.0f - s) * slope;
    return act;
}

// ---- product -------------------------------------------------------------------

// Rows of a panel sit in LDS with their 16-byte pieces permuted, so that eight
// lanes reading one piece of eight rows meet all banks: by the lane's number
// mod 8 that reads the row, halved where a row has but four pieces.  That is
// the row mod 8 in a's panels, and in b's, whose rows the lanes read in runs
// of kRun (below), what bReader() says.
template <int kRun> __device__ inline int bReader(int row) { return (row & 3) | (row / kRun & 1) << 2; }

// kRowBytes: of a panel's row in a stage, 128 or 64.
template <typename T, int kKind, int kBM, int kBN, int kWM, int kWN, int kRowBytes> struct ProductShape {
    static constexpr int kNA = kKind == kProductGrad ? 2 : 1, kNB = kKind == kProductPlain ? 1 : kKind == kProductGate ? 2 : 3;
    static constexpr int kThreads = kWM * kWN * 64;
    static constexpr int kTM = kBM / kWM / 16, kTN = kBN / kWN / 16;
    static constexpr int kRun = 4 * kTN;
    static constexpr int kStage = (kNA * kBM + kNB * kBN) * kRowBytes;
    static constexpr int kPieces = kRowBytes / 16, kCopyRows = kThreads / kPieces;      // rows that the workgroup copies at once
    static_assert(kBM % kCopyRows == 0 && kBN % kCopyRows == 0, "whole copies");
    static_assert(kCopyRows % 8 == 0 && kCopyRows % (2 * kRun) == 0, "one permutation for a thread's pieces");
};

template <typename T, int kKind, int kBM, int kBN, int kWM, int kWN, int kRowBytes>
__global__ __launch_bounds__((ProductShape<T, kKind, kBM, kBN, kWM, kWN, kRowBytes>::kThreads)) void productKernel(const ProductArgs args)
{
    using S = ProductShape<T, kKind, kBM, kBN, kWM, kWN, kRowBytes>;
    constexpr int kE = 16 / sizeof(T), kStep = kRowBytes / sizeof(T);
    constexpr int kNA = S::kNA, kNB = S::kNB, kTM = S::kTM, kTN = S::kTN, kRun = S::kRun, kThreads = S::kThreads;

    __shared__ __align__(1024) char stages[2 * S::kStage];

    // The tiles of one row of tiles run next to each other on one of the 8
    // dies (blocks are dealt to them in turn), so that a's rows are read from
    // memory once and b stays in that die's cache.
    const int tilesN = (args.n + kBN - 1) / kBN;
    const int64_t tilesM = (args.m + kBM - 1) / kBM;
    const int die = blockIdx.x % 8;
    const int64_t local = blockIdx.x / 8;
    const int64_t tm = local / tilesN * 8 + die;
    const int tn = (int)(local % tilesN);
    if (tm >= tilesM) return;
    const int64_t m0 = tm * kBM;
    const int n0 = tn * kBN;

    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, col = lane & 15, quad = lane >> 4;
    const int wm = wave / kWN, wn = wave % kWN;

    f32x4 acc[kNB][kTN][kTM];
#pragma unroll
    for (int b = 0; b < kNB; b++)
#pragma unroll
        for (int j = 0; j < kTN; j++)
#pragma unroll
            for (int i = 0; i < kTM; i++) acc[b][j][i] = f32x4{ 0.f, 0.f, 0.f, 0.f };

    // Rows past the operand's end lie past the descriptor's, pieces past a
    // row's width are sent there: both arrive as zeros.
    const int copyRow = threadIdx.x / S::kPieces;
    const auto copyPanel = [&](const Panel& p, int64_t row0, int rows, int k0, uint32_t lds, bool weights) {
        const T* base = static_cast<const T*>(p.data) + row0 * p.stride;
        const int have = (int)(p.rows - row0 < rows ? p.rows - row0 : rows), strideBytes = (int)(p.stride * sizeof(T));
        const i32x4 from = descriptor(base, have * strideBytes);
        const int reader = weights ? bReader<kRun>(copyRow) : copyRow & 7;
        const int c = (threadIdx.x % S::kPieces ^ (kRowBytes == 128 ? reader : reader >> 1)) * 16;
        const bool within = c < (p.width - k0) * (int)sizeof(T);
        const int at = copyRow * strideBytes + c;
#pragma unroll
        for (int i = 0; i < rows / S::kCopyRows; i++)
            copyToLds(from, within ? at + i * S::kCopyRows * strideBytes : kOutside, k0 * (int)sizeof(T), lds + (i * kThreads + wave * 64) * 16);
    };
    const int steps0 = (args.a[0].width + kStep - 1) / kStep;
    const int steps = kKind == kProductPlain && args.terms == 2 ? steps0 + (args.a[1].width + kStep - 1) / kStep : steps0;
    const auto copyStage = [&](int step, uint32_t lds) {
        if constexpr (kKind == kProductPlain) {
            const int term = step >= steps0, k0 = (term ? step - steps0 : step) * kStep;
            copyPanel(args.a[term], m0, kBM, k0, lds, false);
            copyPanel(args.b[term], n0, kBN, k0, lds + kBM * kRowBytes, true);
        } else {
#pragma unroll
            for (int i = 0; i < kNA; i++) copyPanel(args.a[i], m0, kBM, step * kStep, lds + i * kBM * kRowBytes, false);
#pragma unroll
            for (int i = 0; i < kNB; i++) copyPanel(args.b[i], n0, kBN, step * kStep, lds + (kNA * kBM + i * kBN) * kRowBytes, true);
        }
    };
    // Tile i of a's: rows lane%16 of the tile.  Tile j of b's: row lane%16 is
    // column (lane%16)/4 kRun + 4 j + lane%4 of the wave's, so that a lane's
    // rows 4 quad + i of all tiles are kRun neighbouring columns of the result.
    const int aRow = (wm * kTM * 16 + col) * kRowBytes, piece0 = (quad ^ (kRowBytes == 128 ? col & 7 : (col & 7) >> 1)) * 16;
    const int bRow = (wn * kTN * 16 + (col >> 2) * kRun + (col & 3)) * kRowBytes;
    const auto multiply = [&](const char* lds) {
#pragma unroll
        for (int half = 0; half < kRowBytes / 64; half++) {
            __builtin_amdgcn_sched_barrier(0);      // the fragments of one half at a time
            const char* aAt = lds + (aRow + (piece0 ^ half * 64));
            const char* bAt = lds + kNA * kBM * kRowBytes + (bRow + (piece0 ^ half * 64));
            uint4 a[kNA][kTM];
#pragma unroll
            for (int p = 0; p < kNA; p++)
#pragma unroll
                for (int i = 0; i < kTM; i++) a[p][i] = *reinterpret_cast<const uint4*>(aAt + (p * kBM + i * 16) * kRowBytes);
#pragma unroll
            for (int p = 0; p < kNB; p++)
#pragma unroll
                for (int j = 0; j < kTN; j++) {
                    const uint4 b = *reinterpret_cast<const uint4*>(bAt + (p * kBN + j * 4) * kRowBytes);
#pragma unroll
                    for (int i = 0; i < kTM; i++) acc[p][j][i] = Mma<T>::run(b, a[kNA == 2 && p == 2 ? 1 : 0][i], acc[p][j][i]);
                }
        }
    };

    const uint32_t lds = ldsAddress(stages);
    copyStage(0, lds);
    waitCopies();
    __syncthreads();
    for (int step = 0; step < steps; step++) {
        if (step + 1 < steps) copyStage(step + 1, lds + ((step + 1) & 1) * S::kStage);
        multiply(stages + (step & 1) * S::kStage);
        waitCopies();
        __syncthreads();
    }

    const auto store = [&](void* out, int64_t row, const float (&x)[kRun]) {
        const int n = n0 + wn * kTN * 16 + quad * kRun;
        T* to = static_cast<T*>(out) + row * args.outStride + n;
        if (args.outWide && n + kRun <= args.outWidth) {
            constexpr int kPiece = kRun < kE ? kRun : kE;
#pragma unroll
            for (int e = 0; e < kRun; e += kPiece) {
                vec<T, kPiece> v;
#pragma unroll
                for (int i = 0; i < kPiece; i++) v[i] = (T)x[e + i];
                *reinterpret_cast<vec<T, kPiece>*>(to + e) = v;
            }
        } else {
#pragma unroll
            for (int e = 0; e < kRun; e++)
                if (n + e < args.outWidth) to[e] = (T)x[e];
        }
    };
    float scaleFirst = 1.0f, scaleRest = 1.0f;
    if constexpr (std::is_same_v<T, f16>) {
        scaleFirst = *args.scale[0];
        if constexpr (kKind == kProductGrad) scaleRest = *args.scale[1];
    }
#pragma unroll
    for (int i = 0; i < kTM; i++) {
        const int64_t row = m0 + (wm * kTM + i) * 16 + col;
        if (row >= args.m) continue;
        float first[kRun], second[kRun], third[kRun];
#pragma unroll
        for (int j = 0; j < kTN; j++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int at = j * 4 + e;
                if constexpr (kKind == kProductPlain) first[at] = acc[0][j][i][e];
                else {
                    const float up = acc[1][j][i][e];
                    float slope;
                    const float act = activate(acc[0][j][i][e], args.activation, &slope);
                    first[at] = act * up;
                    if constexpr (kKind == kProductGrad) {
                        const float dh = acc[kNB - 1][j][i][e];
                        second[at] = dh * up * slope;
                        third[at] = dh * act;
                    }
                }
            }
        if constexpr (std::is_same_v<T, f16>) {
#pragma unroll
            for (int e = 0; e < kRun; e++) {
                first[e] *= scaleFirst;
                if constexpr (kKind == kProductGrad) {
                    second[e] *= scaleRest;
                    third[e] *= scaleRest;
                }
            }
        }
        // the padding of rows is zero whatever a row holds (an infinity meets
        // the zeros past the weights' last row)
        if (kKind != kProductPlain && n0 + kBN > args.n) {
            const int n = n0 + wn * kTN * 16 + quad * kRun;
#pragma unroll
            for (int e = 0; e < kRun; e++) {
                if (n + e < args.n) continue;
                first[e] = 0.0f;
                if constexpr (kKind == kProductGrad) second[e] = third[e] = 0.0f;
            }
        }
        store(args.out[0], row, first);
        if constexpr (kKind == kProductGrad) {
            store(args.out[1], row, second);
            store(args.out[2], row, third);
        }
    }
}

// ---- thin ----------------------------------------------------------------------

// A product of at most 64 rows a workgroup (16 kTM), which is a matter of
// latency: 16 columns a workgroup, its eight waves taking the sum's blocks in
// turn, fragments straight from memory to registers, one exchange at the end.
// Addresses may be any (the hardware takes 16 bytes from each), so weights
// that the large products would lay out anew are read as they lie.  34 rows of
// 256 by 683: the block's two launches 14.0 us before, laid out and in tiles
// of 64 rows, now 9.5 us.  Up to 16 rows h goes from one launch to the other
// in float32 and meets w_down as two terms of bfloat16 (8.0 us for 16 rows
// either way; for 34 it would be 12.3 us); float16, whose range holds neither h
// nor such terms, runs that product in float32 whatever the rows.  h's rows are
// padded with zeros to multiples of 64.
constexpr float kMostBf16 = 0x1.fep127f;

template <typename T> __device__ inline uint4 loadAny(const T* p, int have)
{
    constexpr int kE = 16 / sizeof(T);
    vec<T, kE> r;
    if (have >= kE) __builtin_memcpy(&r, p, 16);
    else
#pragma unroll
        for (int j = 0; j < kE; j++) r[j] = j < have ? p[j] : T(0);
    return __builtin_bit_cast(uint4, r);
}

template <typename T, bool kGate, int kTM> __global__ __launch_bounds__(512) void thinKernel(const ThinArgs args)
{
    constexpr int kE = 16 / sizeof(T), kBlock = 4 * kE, kWaves = 8, kNB = kGate ? 2 : 1;
    __shared__ f32x4 parts[kWaves][kNB][kTM][64];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, col = lane & 15, quad = lane >> 4;
    const int n0 = blockIdx.x * 16, m0 = blockIdx.y * 16 * kTM;
    // rows past the end are the last one again; their results are not stored
    const int n = n0 + col < args.n ? n0 + col : args.n - 1;
    using H = std::conditional_t<kTM == 1 || std::is_same_v<T, f16>, float, T>;
    using A = std::conditional_t<kGate, T, H>;
    const T* b[kNB];
    b[0] = static_cast<const T*>(args.b0) + (int64_t)n * args.k;
    if constexpr (kGate) b[1] = static_cast<const T*>(args.b1) + (int64_t)n * args.k;
    const A* a[kTM];
#pragma unroll
    for (int i = 0; i < kTM; i++) {
        const int m = m0 + i * 16 + col;
        a[i] = static_cast<const A*>(args.a) + (int64_t)(m < args.m ? m : args.m - 1) * args.aStride;
    }
    f32x4 acc[kNB][kTM];
#pragma unroll
    for (int p = 0; p < kNB; p++)
#pragma unroll
        for (int i = 0; i < kTM; i++) acc[p][i] = f32x4{ 0.f, 0.f, 0.f, 0.f };
#pragma unroll 2
    for (int k = wave * kBlock + quad * kE; k - quad * kE < args.k; k += kWaves * kBlock) {
        const int have = args.k - k;
        uint4 w[kNB];
#pragma unroll
        for (int p = 0; p < kNB; p++) w[p] = loadAny(b[p] + k, have);
#pragma unroll
        for (int i = 0; i < kTM; i++) {
            if constexpr (kGate || std::is_same_v<H, T>) {
                const uint4 x = kGate ? loadAny(a[i] + k, have) : *reinterpret_cast<const uint4*>(a[i] + k);
#pragma unroll
                for (int p = 0; p < kNB; p++) acc[p][i] = Mma<T>::run(w[p], x, acc[p][i]);
            } else {
                const f32x4 lo = *reinterpret_cast<const f32x4*>(a[i] + k), hi = *reinterpret_cast<const f32x4*>(a[i] + k + 4);
                if constexpr (std::is_same_v<T, bf16>) {
                    const auto h = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
                    // a first term that is never infinite: the second takes what passes it
                    auto near = h;
#pragma unroll
                    for (int j = 0; j < 8; j++) near[j] = __builtin_amdgcn_fmed3f(h[j], -kMostBf16, kMostBf16);
                    const auto first = fromFloat<T, 8>(near), second = fromFloat<T, 8>(h - toFloat<T, 8>(first));
                    acc[0][i] = Mma<T>::run(w[0], __builtin_bit_cast(uint4, first), acc[0][i]);
                    acc[0][i] = Mma<T>::run(w[0], __builtin_bit_cast(uint4, second), acc[0][i]);
                } else {
                    const auto weights = toFloat<T, 8>(__builtin_bit_cast(vec<T, 8>, w[0]));
#pragma unroll
                    for (int j = 0; j < 4; j++) acc[0][i] = __builtin_amdgcn_mfma_f32_16x16x4f32(weights[j], lo[j], acc[0][i], 0, 0, 0);
#pragma unroll
                    for (int j = 0; j < 4; j++) acc[0][i] = __builtin_amdgcn_mfma_f32_16x16x4f32(weights[4 + j], hi[j], acc[0][i], 0, 0, 0);
                }
            }
        }
    }
#pragma unroll
    for (int p = 0; p < kNB; p++)
#pragma unroll
        for (int i = 0; i < kTM; i++) parts[wave][p][i][lane] = acc[p][i];
    __syncthreads();
    if (wave >= kTM) return;
    f32x4 sum[kNB];
#pragma unroll
    for (int p = 0; p < kNB; p++) {
        sum[p] = parts[0][p][wave][lane];
        for (int w = 1; w < kWaves; w++) sum[p] += parts[w][p][wave][lane];
    }
    const int m = m0 + wave * 16 + col;
    if (m >= args.m) return;
    using Out = std::conditional_t<kGate, H, T>;
    Out* out = static_cast<Out*>(args.out) + m * args.outStride + n0 + quad * 4;
    for (int e = 0; e < 4; e++) {
        const bool in = n0 + quad * 4 + e < args.n;
        if constexpr (kGate) out[e] = (Out)(in ? activate(sum[0][e], args.activation) * sum[1][e] : 0.0f);
        else if (in) out[e] = (T)sum[0][e];
    }
}

// ---- outer ---------------------------------------------------------------------

// A panel's stage is kStep rows of kB columns.  Its columns' 16-byte pieces are
// permuted by the row so that the rows that one read touches meet other banks.
template <typename T> __device__ inline int outerSwizzle(int row)
{
    if constexpr (sizeof(T) == 4) return (row >> 2 & 3) * 4;
    else return ((row & 3) | (row >> 3 & 1) << 2) * 2;
}

template <typename T, int kB, int kWM, int kWN>
__global__ __launch_bounds__(kWM* kWN * 64) void outerKernel(const OuterArgs args)
{
    constexpr int kThreads = kWM * kWN * 64, kE = 16 / sizeof(T), kStep = 128 / sizeof(T);
    constexpr int kTM = kB / kWM / 16, kTN = kB / kWN / 16;
    constexpr int kPieces = kB / kE, kPanel = kStep * kB * (int)sizeof(T);
    constexpr int kStage = 2 * kPanel;
    __shared__ __align__(1024) char stages[2 * kStage];

    const int job = blockIdx.y;
    // a tile's splits next to each other (with 8 of them, or a multiple, a
    // split's rows go through one die's cache; other counts spread them)
    const int split = (int)(blockIdx.x % args.splits), tile = (int)(blockIdx.x / args.splits);
    const int m = args.m[job], n = args.n[job], tilesN = (n + kB - 1) / kB;
    if (tile >= tilesN * ((m + kB - 1) / kB)) return;
    const int m0 = tile / tilesN * kB, n0 = tile % tilesN * kB;
    const int64_t k0 = split * args.splitRows, k1 = k0 + args.splitRows < args.k ? k0 + args.splitRows : args.k;

    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, col = lane & 15, quad = lane >> 4;
    const int wm = wave / kWN, wn = wave % kWN;
    f32x4 acc[kTN][kTM];
#pragma unroll
    for (int j = 0; j < kTN; j++)
#pragma unroll
        for (int i = 0; i < kTM; i++) acc[j][i] = f32x4{ 0.f, 0.f, 0.f, 0.f };

    constexpr int kCopyRows = kThreads / kPieces;       // rows that the workgroup copies at once
    const int copyRow = threadIdx.x / kPieces;
    const auto copyPanel = [&](const Panel& p, int64_t row0, int col0, uint32_t lds) {
        const T* base = static_cast<const T*>(p.data) + row0 * p.stride + col0;
        const int have = (int)(k1 - row0 < kStep ? k1 - row0 : kStep), strideBytes = (int)(p.stride * sizeof(T));
        // the last row ends with its width, not with its stride
        const int records = (have - 1) * strideBytes + (p.width - col0) * (int)sizeof(T);
        const i32x4 from = descriptor(base, records);
#pragma unroll
        for (int i = 0; i < kStep / kCopyRows; i++) {
            const int row = i * kCopyRows + copyRow;
            const int c = ((threadIdx.x % kPieces) ^ outerSwizzle<T>(row)) * 16;
            const int at = row < have && c < (p.width - col0) * (int)sizeof(T) ? row * strideBytes + c : kOutside;
            copyToLds(from, at, 0, lds + (i * kThreads + wave * 64) * 16);
        }
    };
    const auto copyStage = [&](int64_t k, uint32_t lds) {
        copyPanel(args.p[job], k, m0, lds);
        copyPanel(args.q[job], k, n0, lds + kPanel);
    };
    // columns 16 c .. 16 c + 15 of the stage's rows, a lane's share of step `half`
    const auto fragment = [&](const char* lds, int c, int half) {
        if constexpr (sizeof(T) == 4) {
            f32x4 x;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int row = half * 16 + quad * 4 + j, piece = c * 4 + (col >> 2);
                x[j] = *reinterpret_cast<const float*>(lds + (row * kPieces + (piece ^ outerSwizzle<T>(row))) * 16 + (col & 3) * 4);
            }
            return __builtin_bit_cast(uint4, x);
        } else {
            // each read transposes 4 rows x 16 columns held by 16 lanes
            i16x4 x[2];
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const int row = half * 32 + quad * 8 + j * 4 + (col >> 2), piece = c * 2 + (col >> 1 & 1);
                x[j] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                    (LdsI16x4*)(lds + (row * kPieces + (piece ^ outerSwizzle<T>(row))) * 16 + (col & 1) * 8));
            }
            return __builtin_bit_cast(uint4, __builtin_shufflevector(x[0], x[1], 0, 1, 2, 3, 4, 5, 6, 7));
        }
    };
    const auto multiply = [&](const char* lds) {
#pragma unroll
        for (int half = 0; half < 2; half++) {
            __builtin_amdgcn_sched_barrier(0);
            uint4 p[kTM];
#pragma unroll
            for (int i = 0; i < kTM; i++) p[i] = fragment(lds, wm * kTM + i, half);
#pragma unroll
            for (int j = 0; j < kTN; j++) {
                const uint4 q = fragment(lds + kPanel, wn * kTN + j, half);
#pragma unroll
                for (int i = 0; i < kTM; i++) acc[j][i] = Mma<T>::run(q, p[i], acc[j][i]);
            }
        }
    };

    const uint32_t lds = ldsAddress(stages);
    if (k0 < k1) copyStage(k0, lds);
    waitCopies();
    __syncthreads();
    int stage = 0;
    for (int64_t k = k0; k < k1; k += kStep) {
        if (k + kStep < k1) copyStage(k + kStep, lds + (stage ^ 1) * kStage);
        multiply(stages + stage * kStage);
        waitCopies();
        __syncthreads();
        stage ^= 1;
    }
    float* part = args.part[job] + (int64_t)split * m * n;
#pragma unroll
    for (int i = 0; i < kTM; i++) {
        const int f = m0 + (wm * kTM + i) * 16 + col;
        if (f >= m) continue;
#pragma unroll
        for (int j = 0; j < kTN; j++) {
            const int d = n0 + (wn * kTN + j) * 16 + quad * 4;
            float* to = part + (int64_t)f * n + d;
            if (n % 4 == 0 && d + 4 <= n) *reinterpret_cast<f32x4*>(to) = acc[j][i];
            else
                for (int e = 0; e < 4; e++)
                    if (d + e < n) to[e] = acc[j][i][e];
        }
    }
}

template <typename T> __global__ __launch_bounds__(256) void sumKernel(const SumArgs args)
{
    const SumJob& job = args.job[blockIdx.y];
    const float scale = std::is_same_v<T, f16> && job.scale ? *job.scale : 1.0f;
    for (int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x; e < job.count; e += (int64_t)gridDim.x * 256) {
        float x = 0.0f;
        for (int s = 0; s < args.splits; s++) x += job.part[s * job.count + e];
        static_cast<T*>(job.out)[e] = (T)(std::is_same_v<T, f16> ? x * scale : x);
    }
}

// Copies with rows padded by zeros, or transposes, tile by tile of 32 x 32.
template <typename T> __global__ __launch_bounds__(256) void packKernel(const PackArgs args)
{
    __shared__ T tile[32][33];
    const PackJob& job = args.job[blockIdx.y];
    const T* from = static_cast<const T*>(job.from);
    T* to = static_cast<T*>(job.to);
    const int x = threadIdx.x & 31, y = threadIdx.x >> 5;
    // of the destination
    const int64_t rows = job.transposed ? job.cols : job.rows, across = (job.toStride + 31) / 32;
    const int64_t tiles = (rows + 31) / 32 * across;
    for (int64_t t = blockIdx.x; t < tiles; t += gridDim.x) {
        const int64_t r0 = t / across * 32, c0 = t % across * 32;
        if (job.transposed) {
            for (int i = y; i < 32; i += 8) {
                const int64_t r = c0 + i, c = r0 + x;
                tile[i][x] = r < job.rows && c < job.cols ? from[r * job.fromStride + c] : T(0);
            }
            __syncthreads();
        }
        for (int i = y; i < 32; i += 8) {
            const int64_t r = r0 + i, c = c0 + x;
            if (r >= rows || c >= job.toStride) continue;
            to[r * job.toStride + c] = job.transposed ? tile[x][i] : c < job.cols ? from[r * job.fromStride + c] : T(0);
        }
        if (job.transposed) __syncthreads();
    }
}

// ---- launches ------------------------------------------------------------------

template <typename T, int kKind, int kBM, int kBN, int kWM, int kWN, int kRowBytes>
int launchProductShape(const ProductArgs& args, hipStream_t stream)
{
    const int64_t tilesM = (args.m + kBM - 1) / kBM, tilesN = (args.n + kBN - 1) / kBN;
    const int64_t blocks = (tilesM + 7) / 8 * 8 * tilesN;
    productKernel<T, kKind, kBM, kBN, kWM, kWN, kRowBytes><<<dim3((unsigned)blocks), kWM * kWN * 64, 0, stream>>>(args);
    return launched("feed-forward product");
}

// The largest tiles whose number still keeps the 256 compute units busy, by a
// sweep over 2,048 to 262,144 rows of 256 to 1,024 by 688 to 2,816 (us):
//   16 bits  gate   2,048 x 256 x 688   64 x 32 5.8   128 x 128 7.8      8,192 x 512 x 1,408   40.6 and 34.4
//                   8,192 x 1,024 x 2,816   128 x 128 113   256 x 128 97.7      262,144 x 512 x 1,408   908 and 1,005
//            grad   2,048 x 256 x 688   64 x 32 10.1   128 x 128 12.3     8,192 x 512 x 1,408   96.5 and 56.4
//            plain  2,048 x 1,408 to 512   64 x 64 12.0   128 x 128 18.6     8,192 x 2,816 to 1,024   86.2 and 49.7
//                   32,768 x 1,408 to 512   128 x 128 52.9   256 x 256 45.9  8,192 x 2,816 to 1,024   49.7 and 69.4
//   float32  gate   2,048 x 512 x 1,408   64 x 32 56.5   128 x 64 69.7    32,768 x 512 x 1,408   883 and 742
//            grad   2,048 x 512 x 1,408   64 x 64 84   128 x 64 107       32,768 x 512 x 1,408   1,153 and 1,102
//            plain  2,048 x 1,408 to 512   64 x 64 36.9   128 x 64 56.9     8,192 x 2,816 to 1,024   402 and 379
//                   62,000 x 684 to 256   128 x 128 188   256 x 256 194
// At 262,144 rows of 512 by 1,408 in bfloat16 gate runs at 860 TFLOP/s, grad at
// 590 and plain at 940 to 1,070 (the library's products of the same operands'
// layout: 1,320 to 1,580 for large ones, 875 and 1,260 for gate's and plain's
// sizes).  gate and grad are bound by their tiles' short sums (512), under which
// the copies' latency and the stores of h, dg and du (2.2 GB: 470 us of grad's
// 1,920) do not disappear; float32 by its matrix instructions (102 to 110
// TFLOP/s; the library's product 154).
template <typename T> int launchProduct(int kind, const ProductArgs& args, hipStream_t stream)
{
    constexpr bool wide = sizeof(T) == 4;
    const auto tiles = [&](int rows, int columns) { return (args.m + rows - 1) / rows * ((args.n + columns - 1) / columns); };
    if (kind == kProductGate) {
        if constexpr (wide) {
            if (tiles(128, 64) >= 1536) return launchProductShape<T, kProductGate, 128, 64, 2, 2, 64>(args, stream);
        } else {
            if (tiles(128, 128) >= 256 && args.a[0].width >= 1024) return launchProductShape<T, kProductGate, 256, 128, 2, 4, 128>(args, stream);
            if (tiles(128, 128) >= 128) return launchProductShape<T, kProductGate, 128, 128, 2, 4, 64>(args, stream);
        }
        return launchProductShape<T, kProductGate, 64, 32, 2, 2, 128>(args, stream);
    }
    if (kind == kProductGrad) {
        if constexpr (wide) {
            if (tiles(128, 64) >= 1536) return launchProductShape<T, kProductGrad, 128, 64, 2, 2, 64>(args, stream);
            if (tiles(64, 64) >= 512) return launchProductShape<T, kProductGrad, 64, 64, 2, 2, 64>(args, stream);
        } else if (tiles(128, 128) >= 128) return launchProductShape<T, kProductGrad, 128, 128, 2, 4, 128>(args, stream);
        return launchProductShape<T, kProductGrad, 64, 32, 2, 2, 128>(args, stream);
    }
    if constexpr (wide) {
        if (tiles(128, 128) >= 512) return launchProductShape<T, kProductPlain, 128, 128, 2, 2, 64>(args, stream);
        if (tiles(128, 64) >= 256) return launchProductShape<T, kProductPlain, 128, 64, 2, 2, 128>(args, stream);
    } else {
        if (tiles(256, 256) >= 256) return launchProductShape<T, kProductPlain, 256, 256, 2, 4, 128>(args, stream);
        if (tiles(128, 128) >= 256) return launchProductShape<T, kProductPlain, 128, 128, 2, 2, 128>(args, stream);
    }
    if (tiles(64, 64) >= 256) return launchProductShape<T, kProductPlain, 64, 64, 2, 2, 128>(args, stream);
    return launchProductShape<T, kProductPlain, 64, 32, 2, 2, 128>(args, stream);
}

template <typename T, bool kGate> void launchThinRows(const ThinArgs& args, hipStream_t stream)
{
    // h's padding is written too, as zeros
    const unsigned columns = (unsigned)(kGate ? args.outStride / 16 : (args.n + 15) / 16);
    if (args.m <= 16) thinKernel<T, kGate, 1><<<dim3(columns), 512, 0, stream>>>(args);
    else if (args.m <= 32) thinKernel<T, kGate, 2><<<dim3(columns), 512, 0, stream>>>(args);
    else thinKernel<T, kGate, 4><<<dim3(columns, (unsigned)((args.m + 63) / 64)), 512, 0, stream>>>(args);
}

template <typename T> int launchThin(bool gate, const ThinArgs& args, hipStream_t stream)
{
    if (gate) launchThinRows<T, true>(args, stream);
    else launchThinRows<T, false>(args, stream);
    return launched("feed-forward product of few rows");
}

template <typename T> int launchOuter(const OuterArgs& args, int tile, hipStream_t stream)
{
    int tiles = 0;
    for (int j = 0; j < args.jobs; j++)
        tiles = std::max(tiles, ((args.m[j] + tile - 1) / tile) * ((args.n[j] + tile - 1) / tile));
    const dim3 grid((unsigned)(tiles * args.splits), (unsigned)args.jobs);
    if (tile == 256) outerKernel<T, 256, 2, 4><<<grid, 512, 0, stream>>>(args);
    else outerKernel<T, 128, 2, 2><<<grid, 256, 0, stream>>>(args);
    return launched("weight gradient product");
}

template <typename T> int launchPack(const PackArgs& args, hipStream_t stream)
{
    int64_t tiles = 1;
    for (int j = 0; j < args.jobs; j++) {
        const PackJob& p = args.job[j];
        tiles = std::max(tiles, ((p.transposed ? p.cols : p.rows) + 31) / 32 * ((p.toStride + 31) / 32));
    }
    packKernel<T><<<dim3((unsigned)std::min<int64_t>(tiles, 16384), (unsigned)args.jobs), 256, 0, stream>>>(args);
    return launched("operand packing");
}

template <typename T> int launchSum(const SumArgs& args, hipStream_t stream)
{
    int64_t count = 1;
    for (int j = 0; j < args.jobs; j++) count = std::max(count, args.job[j].count);
    sumKernel<T><<<dim3((unsigned)std::min<int64_t>((count + 255) / 256, 8192), (unsigned)args.jobs), 256, 0, stream>>>(args);
    return launched("weight gradient sum");
}

}  // namespace carl
