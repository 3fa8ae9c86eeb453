// attention_kernel.h - the chunked kernel of attention.h, for one element type.
#pragma once

#include "attention.h"
#include "status.h"

namespace carl {

// One product of 16x16 tiles over one (x4: 16 steps of the sum) or two (x8: 32
// steps) fragments of each operand.
__device__ inline f32x4 mma(f32x4 a, f32x4 b, f32x4 c)
{
#pragma unroll
    for (int j = 0; j < 4; j++) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], b[j], c, 0, 0, 0);
    return c;
}
__device__ inline f32x4 mma(vec<float, 8> a, vec<float, 8> b, f32x4 c)
{
#pragma unroll
    for (int j = 0; j < 8; j++) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], b[j], c, 0, 0, 0);
    return c;
}
__device__ inline f32x4 mma(bf16x8 a, bf16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
__device__ inline f32x4 mma(f16x8 a, f16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }

template <typename V> __device__ inline auto both(V a, V b) { return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7); }

// From column `at` on: of rows 4 quad .. 4 quad + 3 of a 16-row block of LDS,
// the lane's column at + lane%16.
__device__ inline f32x4 columns(const float* rows, int stride, int at, int col, int quad)
{
    f32x4 x;
#pragma unroll
    for (int j = 0; j < 4; j++) x[j] = rows[(quad * 4 + j) * stride + at + col];
    return x;
}
typedef __attribute__((address_space(3))) i16x4 LdsI16x4;
template <typename T> __device__ inline vec<T, 4> columns(const T* rows, int stride, int at, int col, int quad)
{
    // transposes 4 rows x 16 columns held by 16 lanes
    return __builtin_bit_cast(vec<T, 4>, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (LdsI16x4*)(rows + (quad * 4 + (col >> 2)) * stride + at + (col & 3) * 4)));
}

// How products with float32 factors run (the memory read by a, what enters it
// from b): bfloat16 as terms of that type, two and three of them; float16
// rows, whose terms would leave its range, and float32 as float32.
template <typename T> struct Long {
    using type = float;
    static constexpr int kIn = 1, kOut = 1;
};
template <> struct Long<bf16> {
    using type = bf16;
    static constexpr int kIn = 2, kOut = 3;
};

// x as kTerms addends of type T, largest first.
template <typename T, int kTerms> __device__ inline void split(f32x4 x, vec<T, 4> (&out)[kTerms])
{
#pragma unroll
    for (int i = 0; i < kTerms; i++) {
        out[i] = fromFloat<T, 4>(x);
        if (i + 1 < kTerms) x -= toFloat<T, 4>(out[i]);
    }
}

// 16 bytes of a row from address p, element by element; zero past `have`.
template <typename T> __device__ inline uint4 loadPiece(const T* p, int have)
{
    constexpr int kE = 16 / sizeof(T);
    vec<T, kE> r;
#pragma unroll
    for (int j = 0; j < kE; j++) r[j] = j < have ? p[j] : T(0);
    return __builtin_bit_cast(uint4, r);
}

// The bits that tell a non-finite value, for the elements of one word: with the
// low one added to the exponent's field, all ones carry into the sign's place.
template <typename T> struct Exponent;
template <> struct Exponent<float> {
    static constexpr uint32_t kField = 0x7f800000u, kOne = 0x00800000u, kCarry = 0x80000000u;
};
template <> struct Exponent<bf16> {
    static constexpr uint32_t kField = 0x7f807f80u, kOne = 0x00800080u, kCarry = 0x80008000u;
};
template <> struct Exponent<f16> {
    static constexpr uint32_t kField = 0x7c007c00u, kOne = 0x04000400u, kCarry = 0x80008000u;
};

template <typename T> __device__ inline uint32_t nonFinite(uint4 x)
{
    using X = Exponent<T>;
    return ((x.x & X::kField) + X::kOne) | ((x.y & X::kField) + X::kOne) | ((x.z & X::kField) + X::kOne)
         | ((x.w & X::kField) + X::kOne);
}

template <typename T, int kA, int kC_, int kSteps> struct Shape {
    static constexpr int kWaves = kC_ / 16 < 4 ? kC_ / 16 : 4;
    static constexpr int kThreads = kWaves * 64;
    static constexpr int kPad = 16 / sizeof(T);
    static constexpr int kStrideA = kA + kPad, kStrideC = kC_ + kPad, kStrideP = kSteps + kPad;
    static constexpr int kPieceA = kA * (int)sizeof(T) / 16, kPieceC = kC_ * (int)sizeof(T) / 16;   // 16-byte pieces of a row
    static constexpr int kLoadsA = kSteps * kPieceA / kThreads, kLoadsC = kSteps * kPieceC / kThreads;
    // waves of a SIMD that the registers leave room for
    static constexpr int kResident = kA * kC_ <= 64 * 128 && sizeof(T) == 2 || kA * kC_ <= 64 * 64 ? 2 : 1;
    static_assert(kSteps * kPieceA % kThreads == 0 && kSteps * kPieceC % kThreads == 0, "whole loads");
};

template <typename T, int kA, int kCd, int kSteps, bool kStates>
__global__ __launch_bounds__((Shape<T, kA, kCd, kSteps>::kThreads), (Shape<T, kA, kCd, kSteps>::kResident))
void attentionKernel(const Pass pass, const int firstRole, const int roles)
{
    using S = Shape<T, kA, kCd, kSteps>;
    constexpr int kWaves = S::kWaves, kThreads = S::kThreads;
    constexpr int kBlocks = kSteps / 16;             // 16-step blocks of a chunk, an even number
    constexpr int kTilesA = kA / 16;                 // of the memory's rows, an even number
    constexpr int kOwn = kCd / 16 / kWaves;          // column tiles of a wave
    constexpr int kE = 16 / sizeof(T);
    using L = Long<T>;
    using LT = typename L::type;

    __shared__ __align__(16) T sA[kStates ? 1 : kSteps * S::kStrideA];
    __shared__ __align__(16) T sB[kSteps * S::kStrideA];
    __shared__ __align__(16) T sC[kSteps * S::kStrideC];
    __shared__ __align__(16) T sP[kStates ? 1 : kSteps * S::kStrideP];

    // Blocks are dealt to the 8 dies in turn.  The roles of one unit and the
    // heads of one sequence, which read the same rows or lines, run on one.
    const int die = blockIdx.x % 8, local = blockIdx.x / 8;
    const int64_t groups = pass.batch * pass.segments;
    int64_t group;
    int head;
    if (pass.dealGroups) {
        group = (int64_t)(local / roles / pass.heads) * 8 + die;
        head = local / roles % pass.heads;
    } else {
        const int64_t unit = (int64_t)(local / roles) * 8 + die;
        group = unit / pass.heads;
        head = (int)(unit % pass.heads);
    }
    if (group >= groups) return;
    const Role& r = pass.role[firstRole + local % roles];
    const int64_t batch = group % pass.batch, segment = group / pass.batch;
    const int lane = threadIdx.x & 63, col = lane & 15, quad = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const bool backwards = r.backwards != 0;

    const int64_t begin = segment * pass.segmentSteps;
    const int64_t end = begin + pass.segmentSteps < pass.steps ? begin + pass.segmentSteps : pass.steps;
    const int chunks = (int)((end - begin + kSteps - 1) / kSteps);
    const T* aRows = static_cast<const T*>(r.a.data) + batch * r.a.batch + head / r.aHeads * r.a.head;
    const T* bRows = static_cast<const T*>(r.b.data) + batch * r.b.batch + head / r.bHeads * r.b.head;
    const T* cRows = static_cast<const T*>(r.c.data) + batch * r.c.batch + head / r.cHeads * r.c.head;

    // -infinity times zero steps is no NaN
    const float decay2 = fmaxf(pass.logDecay[head] * 1.44269504088896341f, -1e30f);
    const auto power = [&](int steps) { return __builtin_amdgcn_exp2f(decay2 * (float)steps); };

    const int64_t size = (int64_t)r.dimA * r.dimC, unitState = batch * pass.heads + head;
    const int64_t partState = segment * pass.batch * pass.heads + unitState;
    // A lane's elements of the memory: rows 16 m + 4 quad + i, column 16 (wave's
    // tile) + col.  Through a descriptor, past whose end lies what the padding
    // would hold: read as zero, written nowhere.
    f32x4 memory[kOwn][kTilesA];
    const auto memoryAt = [&](bool swapped, int o, int m, int i) {
        const int x = m * 16 + quad * 4 + i, y = (wave * kOwn + o) * 16 + col;
        return x < r.dimA && y < r.dimC ? (swapped ? y * r.dimA + x : x * r.dimC + y) * 4 : (int)0x80000000u;
    };
    {
        const float* from = nullptr;
        bool swapped = false;
        if (!kStates) {
            if (pass.segments > 1) from = r.parts + partState * size;
            else if (r.first) {
                from = r.first + unitState * size;
                swapped = r.firstSwapped != 0;
            }
        }
        const auto d = __builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(from), 0, from ? (int)size * 4 : 0, 0x00027000);
#pragma unroll
        for (int o = 0; o < kOwn; o++)
#pragma unroll
            for (int m = 0; m < kTilesA; m++)
#pragma unroll
                for (int i = 0; i < 4; i++)
                    memory[o][m][i] = from ? __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(d, memoryAt(swapped, o, m, i), 0, 0)) : 0.0f;
    }

    // Chunks follow time in the pass's direction, and so do the rows of a chunk
    // in LDS: what comes first is in row 0.
    const auto chunkStart = [&](int n) { return begin + (int64_t)(backwards ? chunks - 1 - n : n) * kSteps; };

    // Rows on the way to LDS, in 16-byte pieces.  Past the chunk's last row that
    // row is read again, and cleared when it is put down.  Pieces need addresses
    // of 4 bytes, and are read word by word where a row ends within one; rows
    // of other addresses are copied element by element when they are due.
    uint4 nextA[kStates ? 1 : S::kLoadsA], nextB[S::kLoadsA], nextC[S::kLoadsC];
    const auto fetchRows = [&](auto& next, const T* rows, int64_t step, int64_t t0, int pieces, int dim) {
        const int have = (int)(end - t0 < kSteps ? end - t0 : kSteps);
        const int row = threadIdx.x / pieces, at = threadIdx.x % pieces * kE, rowsAtOnce = kThreads / pieces;
        const char* base = reinterpret_cast<const char*>(rows + t0 * step + (at < dim ? at : 0));
        const bool whole = dim % kE == 0;
        const int words = at < dim ? (dim - at) * (int)sizeof(T) / 4 : 0;
#pragma unroll
        for (int i = 0; i < (int)(sizeof(next) / sizeof(next[0])); i++) {
            const int mine = row + i * rowsAtOnce, within = mine < have ? mine : have - 1;
            const char* from = base + (backwards ? have - 1 - within : within) * (step * (int64_t)sizeof(T));
            if (whole) next[i] = *reinterpret_cast<const uint4*>(from);
            else {
                const uint32_t* w = reinterpret_cast<const uint32_t*>(from);
                next[i] = make_uint4(w[0], w[words > 1 ? 1 : 0], w[words > 2 ? 2 : 0], w[words > 3 ? 3 : 0]);
            }
        }
    };
    const auto fetch = [&](int n) {
        const int64_t t0 = chunkStart(n);
        if constexpr (!kStates)
            if (r.aGrain >= 4) fetchRows(nextA, aRows, r.a.step, t0, S::kPieceA, r.dimA);
        if (r.bGrain >= 4) fetchRows(nextB, bRows, r.b.step, t0, S::kPieceA, r.dimA);
        if (r.cGrain >= 4) fetchRows(nextC, cRows, r.c.step, t0, S::kPieceC, r.dimC);
    };
    uint32_t odd = 0;         // carry bits of non-finite values in this chunk's b and c
    const auto put = [&](auto& next, T* lds, int stride, int pieces, bool look, int grain, int dim, const T* rows, int64_t step,
                         int64_t t0, int have) {
        const int at = threadIdx.x % pieces * kE;
        T* to = lds + threadIdx.x / pieces * stride + at;
        if (grain < 4) {
            for (int row = threadIdx.x / pieces; row < kSteps; row += kThreads / pieces) {
                uint4 x = make_uint4(0, 0, 0, 0);
                if (row < have) x = loadPiece<T>(rows + (t0 + (backwards ? have - 1 - row : row)) * step + at, dim - at);
                *reinterpret_cast<uint4*>(lds + row * stride + at) = x;
                if (look) odd |= nonFinite<T>(x);
            }
            return;
        }
        const int words = at < dim ? (dim - at) * (int)sizeof(T) / 4 : 0;
        const bool whole = have == kSteps && pieces * kE == dim;
#pragma unroll
        for (int i = 0; i < (int)(sizeof(next) / sizeof(next[0])); i++) {
            uint4 x = next[i];
            if (!whole) {
                const int left = threadIdx.x / pieces + i * (kThreads / pieces) < have ? words : 0;
                x = make_uint4(left > 0 ? x.x : 0, left > 1 ? x.y : 0, left > 2 ? x.z : 0, left > 3 ? x.w : 0);
            }
            *reinterpret_cast<uint4*>(to + i * (kThreads / pieces) * stride) = x;
            if (look) odd |= nonFinite<T>(x);
        }
    };

    float factor = 1.0f;      // of the memory over the whole segment
    if (chunks > 0) fetch(0);
    for (int n = 0; n < chunks; n++) {
        const int64_t t0 = chunkStart(n);
        const int have = end - t0 < kSteps ? (int)(end - t0) : kSteps;
        __syncthreads();
        odd = 0;
        if constexpr (!kStates) put(nextA, sA, S::kStrideA, S::kPieceA, false, r.aGrain, r.dimA, aRows, r.a.step, t0, have);
        put(nextB, sB, S::kStrideA, S::kPieceA, true, r.bGrain, r.dimA, bRows, r.b.step, t0, have);
        put(nextC, sC, S::kStrideC, S::kPieceC, true, r.cGrain, r.dimC, cRows, r.c.step, t0, have);
        // Bit t of `cuts`: row t sees nothing of the rows before it.  Forwards
        // that is where an episode starts; backwards, where the step after
        // (row t - 1) does, and a start at the chunk's first step, its last
        // row, closes the way out instead (bit 0: the way in).
        uint64_t cuts = 0;
        bool shut = false;
        if (pass.starts) {
            const uint64_t starts = __ballot(
                lane < have && pass.starts[batch * pass.startsBatch + (t0 + (backwards ? have - 1 - lane : lane)) * pass.startsStep] != 0);
            cuts = backwards ? starts << 1 & (~0ull >> (64 - have)) : starts;
            shut = backwards && (starts >> (have - 1) & 1);
        }
        // A weight of zero takes a finite row out of a product, but not an
        // infinity or a NaN: a chunk whose b or c hold one is summed step by
        // step, leaving out the steps that are not seen.
        const bool careful = __syncthreads_or((odd & Exponent<T>::kCarry) != 0) != 0;
        if (n + 1 < chunks) fetch(n + 1);

        // Rows [low(t), t] are what row t sees of the chunk.
        const auto low = [&](int t) {
            const uint64_t before = cuts & (~0ull >> (63 - t));
            return before ? 63 - __builtin_clzll(before) : 0;
        };
        // Rows [leave, have) are what the memory after the chunk sees.
        const int leave = shut ? have : cuts ? 63 - __builtin_clzll(cuts) : 0;
        const bool closed = cuts != 0 || shut;

        f32x4 acc[kOwn][kBlocks];
        if constexpr (!kStates) {
            // P^T, tile by tile: rows s, column t
            for (int tb = wave; tb < kBlocks; tb += kWaves) {
                const int t = tb * 16 + col, from = low(t);
                vec<T, 4> a[kTilesA];
#pragma unroll
                for (int k = 0; k < kTilesA; k++) a[k] = *reinterpret_cast<const vec<T, 4>*>(sA + t * S::kStrideA + k * 16 + quad * 4);
                for (int sb = 0; sb <= tb; sb++) {
                    f32x4 p = { 0.f, 0.f, 0.f, 0.f };
                    const T* rows = sB + (sb * 16 + col) * S::kStrideA + quad * 4;
#pragma unroll
                    for (int k = 0; k < kTilesA; k += 2)
                        p = mma(both(*reinterpret_cast<const vec<T, 4>*>(rows + k * 16), *reinterpret_cast<const vec<T, 4>*>(rows + k * 16 + 16)),
                                both(a[k], a[k + 1]), p);
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const int s = sb * 16 + quad * 4 + i;
                        const float w = p[i] * (power(t - s) * r.scaleP);
                        p[i] = s >= from && s <= t ? w : 0.0f;
                    }
                    *reinterpret_cast<vec<T, 4>*>(sP + t * S::kStrideP + sb * 16 + quad * 4) = fromFloat<T, 4>(p);
                }
                // blocks of s are met in pairs below
                if (tb % 2 == 0)
                    *reinterpret_cast<vec<T, 4>*>(sP + t * S::kStrideP + (tb + 1) * 16 + quad * 4) = vec<T, 4>{ T(0), T(0), T(0), T(0) };
            }
            // what the carried memory gives
#pragma unroll
            for (int o = 0; o < kOwn; o++)
#pragma unroll
                for (int tb = 0; tb < kBlocks; tb++) acc[o][tb] = f32x4{ 0.f, 0.f, 0.f, 0.f };
#pragma unroll
            for (int m = 0; m < kTilesA; m += 2) {
                vec<LT, 4> lo[kOwn][L::kIn], hi[kOwn][L::kIn];
#pragma unroll
                for (int o = 0; o < kOwn; o++) {
                    split<LT, L::kIn>(memory[o][m], lo[o]);
                    split<LT, L::kIn>(memory[o][m + 1], hi[o]);
                }
#pragma unroll
                for (int tb = 0; tb < kBlocks; tb++) {
                    const T* rows = sA + (tb * 16 + col) * S::kStrideA + m * 16 + quad * 4;
                    const auto a = both(__builtin_convertvector(*reinterpret_cast<const vec<T, 4>*>(rows), vec<LT, 4>),
                                        __builtin_convertvector(*reinterpret_cast<const vec<T, 4>*>(rows + 16), vec<LT, 4>));
#pragma unroll
                    for (int o = 0; o < kOwn; o++)
#pragma unroll
                        for (int i = 0; i < L::kIn; i++) acc[o][tb] = mma(both(lo[o][i], hi[o][i]), a, acc[o][tb]);
                }
            }
#pragma unroll
            for (int tb = 0; tb < kBlocks; tb++) {
                const int t = tb * 16 + col;
                const bool open = (cuts & (~0ull >> (63 - t))) == 0;
                const float in = power(t + r.inShift) * r.scaleIn;
                // a closed row takes nothing from the memory, whatever that holds
#pragma unroll
                for (int o = 0; o < kOwn; o++) acc[o][tb] = open ? acc[o][tb] * in : f32x4{ 0.f, 0.f, 0.f, 0.f };
            }
            __syncthreads();
        }

        const float keep = closed ? 0.0f : power(have);
        factor *= keep;
        // what row s weighs in the memory after the chunk
        const auto weightOut = [&](int s) {
            return s >= leave && s < have ? power(have - 1 - s + 1 - r.inShift) * r.scaleOut : 0.0f;
        };
        if (!careful) {
            vec<T, 4> c[kOwn][kBlocks];
#pragma unroll
            for (int o = 0; o < kOwn; o++)
#pragma unroll
                for (int sb = 0; sb < kBlocks; sb++)
                    c[o][sb] = columns(sC + sb * 16 * S::kStrideC, S::kStrideC, (wave * kOwn + o) * 16, col, quad);
            if constexpr (!kStates) {
#pragma unroll
                for (int tb = 0; tb < kBlocks; tb++)
#pragma unroll
                    for (int sb = 0; sb <= tb; sb += 2) {
                        const T* row = sP + (tb * 16 + col) * S::kStrideP + sb * 16 + quad * 4;
                        const auto p = both(*reinterpret_cast<const vec<T, 4>*>(row), *reinterpret_cast<const vec<T, 4>*>(row + 16));
#pragma unroll
                        for (int o = 0; o < kOwn; o++) acc[o][tb] = mma(both(c[o][sb], c[o][sb + 1]), p, acc[o][tb]);
                    }
            }
#pragma unroll
            for (int o = 0; o < kOwn; o++)
#pragma unroll
                for (int m = 0; m < kTilesA; m++) memory[o][m] = closed ? f32x4{ 0.f, 0.f, 0.f, 0.f } : memory[o][m] * keep;
#pragma unroll
            for (int sb = 0; sb < kBlocks; sb += 2) {
                f32x4 w[2];
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    w[0][j] = weightOut(sb * 16 + quad * 4 + j);
                    w[1][j] = weightOut(sb * 16 + 16 + quad * 4 + j);
                }
                vec<LT, 4> lo[kOwn][L::kOut], hi[kOwn][L::kOut];
#pragma unroll
                for (int o = 0; o < kOwn; o++) {
                    split<LT, L::kOut>(toFloat<T, 4>(c[o][sb]) * w[0], lo[o]);
                    split<LT, L::kOut>(toFloat<T, 4>(c[o][sb + 1]) * w[1], hi[o]);
                }
                const T* rows = sB + sb * 16 * S::kStrideA;
#pragma unroll
                for (int m = 0; m < kTilesA; m++) {
                    const auto b = both(__builtin_convertvector(columns(rows, S::kStrideA, m * 16, col, quad), vec<LT, 4>),
                                        __builtin_convertvector(columns(rows + 16 * S::kStrideA, S::kStrideA, m * 16, col, quad), vec<LT, 4>));
#pragma unroll
                    for (int o = 0; o < kOwn; o++)
#pragma unroll
                        for (int i = 0; i < L::kOut; i++) memory[o][m] = mma(b, both(lo[o][i], hi[o][i]), memory[o][m]);
                }
            }
        } else {
#pragma unroll
            for (int o = 0; o < kOwn; o++) {
                const int tile = (wave * kOwn + o) * 16;
                if constexpr (!kStates) {
#pragma unroll
                    for (int tb = 0; tb < kBlocks; tb++) {
                        const int t = tb * 16 + col;
#pragma unroll 1
                        for (int s = low(t); s <= t && s < have; s++)
#pragma unroll
                            for (int i = 0; i < 4; i++)
                                acc[o][tb][i] += (float)sP[t * S::kStrideP + s] * (float)sC[s * S::kStrideC + tile + quad * 4 + i];
                    }
                }
#pragma unroll
                for (int m = 0; m < kTilesA; m++) memory[o][m] = closed ? f32x4{ 0.f, 0.f, 0.f, 0.f } : memory[o][m] * keep;
#pragma unroll 1
                for (int s = leave; s < have; s++) {
                    const float x = (float)sC[s * S::kStrideC + tile + col] * weightOut(s);
#pragma unroll
                    for (int m = 0; m < kTilesA; m++)
#pragma unroll
                        for (int i = 0; i < 4; i++) memory[o][m][i] += (float)sB[s * S::kStrideA + m * 16 + quad * 4 + i] * x;
                }
            }
        }

        if constexpr (!kStates) {
            const int64_t row0 = batch * r.out.batch + (t0 + (backwards ? have - 1 : 0)) * r.out.step + head * r.out.head;
            const int64_t ahead = backwards ? -r.out.step : r.out.step;
            const bool quick = r.outWide && !r.outFloat && r.dimC % 4 == 0;
#pragma unroll
            for (int tb = 0; tb < kBlocks; tb++) {
                const int t = tb * 16 + col;
                if (t >= have) continue;
                const int64_t row = row0 + t * ahead;
#pragma unroll
                for (int o = 0; o < kOwn; o++) {
                    const int y = (wave * kOwn + o) * 16 + quad * 4;
                    if (quick) {
                        if (y < r.dimC) *reinterpret_cast<vec<T, 4>*>(static_cast<T*>(r.out.data) + row + y) = fromFloat<T, 4>(acc[o][tb]);
                        continue;
                    }
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        if (y + i >= r.dimC) continue;
                        if (r.outFloat) static_cast<float*>(r.out.data)[row + y + i] = acc[o][tb][i];
                        else static_cast<T*>(r.out.data)[row + y + i] = (T)acc[o][tb][i];
                    }
                }
            }
        }
    }

    float* to = nullptr;
    bool swapped = false;
    if (kStates) {
        to = r.parts + partState * size;
        if (threadIdx.x == 0) r.factors[partState] = factor;
    } else if (pass.segments == 1 && r.last) {
        to = r.last + unitState * size;
        swapped = r.lastSwapped != 0;
    }
    if (!to) return;
    const auto d = __builtin_amdgcn_make_buffer_rsrc(to, 0, (int)size * 4, 0x00027000);
#pragma unroll
    for (int o = 0; o < kOwn; o++)
#pragma unroll
        for (int m = 0; m < kTilesA; m++)
#pragma unroll
            for (int i = 0; i < 4; i++)
                __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(memory[o][m][i]), d, memoryAt(swapped, o, m, i), 0, 0);
}

template <typename T, int kA, int kCd, bool kStates>
void launchAttentionShape(const Pass& pass, int firstRole, int roles, hipStream_t stream)
{
    // float32 rows of 128 leave room for chunks of 32 steps
    constexpr int kSteps = sizeof(T) == 4 && (kA > 64 || kCd > 64) ? 32 : 64;
    const int64_t groups = pass.batch * pass.segments;
    const int64_t blocks = (pass.dealGroups ? (groups + 7) / 8 * pass.heads : (groups * pass.heads + 7) / 8) * 8 * roles;
    attentionKernel<T, kA, kCd, kSteps, kStates>
        <<<dim3((unsigned)blocks), Shape<T, kA, kCd, kSteps>::kThreads, 0, stream>>>(pass, firstRole, roles);
}

template <typename T, int kA, bool kStates>
void launchAttentionRows(const Pass& pass, int firstRole, int roles, hipStream_t stream)
{
    const int dim = pass.role[firstRole].dimC;
    if (dim <= 32) launchAttentionShape<T, kA, 32, kStates>(pass, firstRole, roles, stream);
    else if (dim <= 64) launchAttentionShape<T, kA, 64, kStates>(pass, firstRole, roles, stream);
    else launchAttentionShape<T, kA, 128, kStates>(pass, firstRole, roles, stream);
}

template <typename T, bool kStates>
void launchAttentionDims(const Pass& pass, int firstRole, int roles, hipStream_t stream)
{
    const int dim = pass.role[firstRole].dimA;
    if (dim <= 32) launchAttentionRows<T, 32, kStates>(pass, firstRole, roles, stream);
    else if (dim <= 64) launchAttentionRows<T, 64, kStates>(pass, firstRole, roles, stream);
    else launchAttentionRows<T, 128, kStates>(pass, firstRole, roles, stream);
}

template <typename T> int launchAttentionOf(const Pass& pass, int firstRole, int roles, bool states, hipStream_t stream)
{
    if (states) launchAttentionDims<T, true>(pass, firstRole, roles, stream);
    else launchAttentionDims<T, false>(pass, firstRole, roles, stream);
    return launched("linear attention");
}

}  // namespace carl
