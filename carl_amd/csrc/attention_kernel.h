// attention_kernel.h - the chunked kernel of attention.h, for one element type.
#pragma once

#include "attention.h"
#include "status.h"

namespace carl {

template <typename T> struct Frag {
    using type = vec<T, 4>;
};

__device__ inline f32x4 mma(f32x4 a, f32x4 b, f32x4 c)
{
    for (int j = 0; j < 4; j++) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], b[j], c, 0, 0, 0);
    return c;
}

__device__ inline f32x4 mma(bf16x4 a, bf16x4 b, f32x4 c)
{
    return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(i16x4, a), __builtin_bit_cast(i16x4, b), c, 0, 0, 0);
}

__device__ inline f32x4 mma(f16x4 a, f16x4 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x16f16(a, b, c, 0, 0, 0); }

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

// kBytes of a row from address p, in pieces that its alignment allows; zero past `have` elements.
template <typename T> __device__ inline uint4 loadPiece(const T* p, int have, int grain)
{
    constexpr int kE = 16 / sizeof(T);
    if (have >= kE) {
        if (grain == 16) return *reinterpret_cast<const uint4*>(p);
        if (grain == 8) {
            const uint2 x = reinterpret_cast<const uint2*>(p)[0], y = reinterpret_cast<const uint2*>(p)[1];
            return make_uint4(x.x, x.y, y.x, y.y);
        }
        if (grain == 4) {
            const uint32_t* w = reinterpret_cast<const uint32_t*>(p);
            return make_uint4(w[0], w[1], w[2], w[3]);
        }
    }
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
    static_assert(kSteps * kPieceA % kThreads == 0 && kSteps * kPieceC % kThreads == 0, "whole loads");
};

template <typename T, int kA, int kCd, int kSteps, bool kStates>
__global__ __launch_bounds__((Shape<T, kA, kCd, kSteps>::kThreads)) void attentionKernel(const Pass pass, const int firstRole)
{
    using S = Shape<T, kA, kCd, kSteps>;
    constexpr int kWaves = S::kWaves, kThreads = S::kThreads;
    constexpr int kBlocks = kSteps / 16;             // 16-step blocks of a chunk
    constexpr int kTilesA = kA / 16;                 // of the memory's rows
    constexpr int kOwn = kCd / 16 / kWaves;          // column tiles of a wave
    constexpr int kE = 16 / sizeof(T);
    using L = Long<T>;

    __shared__ __align__(16) T sA[kStates ? 1 : kSteps * S::kStrideA];
    __shared__ __align__(16) T sB[kSteps * S::kStrideA];
    __shared__ __align__(16) T sC[kSteps * S::kStrideC];
    __shared__ __align__(16) T sP[kStates ? 1 : kSteps * S::kStrideP];

    const Role& r = pass.role[firstRole + blockIdx.y];
    const int64_t unit = blockIdx.x;
    const int head = (int)(unit % pass.heads);
    const int64_t batch = unit / pass.heads % pass.batch, segment = unit / pass.heads / pass.batch;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, col = lane & 15, quad = lane >> 4;

    const int64_t begin = segment * pass.segmentSteps;
    const int64_t end = begin + pass.segmentSteps < pass.steps ? begin + pass.segmentSteps : pass.steps;
    const int64_t chunks = (end - begin + kSteps - 1) / kSteps;
    const T* aRows = static_cast<const T*>(r.a.data) + batch * r.a.batch + head / r.aHeads * r.a.head;
    const T* bRows = static_cast<const T*>(r.b.data) + batch * r.b.batch + head / r.bHeads * r.b.head;
    const T* cRows = static_cast<const T*>(r.c.data) + batch * r.c.batch + head / r.cHeads * r.c.head;

    // -infinity times zero steps is no NaN
    const float decay2 = fmaxf(pass.logDecay[head] * 1.44269504088896341f, -1e30f);
    const auto power = [&](int steps) { return exp2f(decay2 * (float)steps); };

    f32x4 memory[kOwn][kTilesA];
    {
        const int64_t size = (int64_t)r.dimA * r.dimC, unitState = batch * pass.heads + head;
        const float* from = nullptr;
        bool swapped = false;
        if (!kStates) {
            if (pass.segments > 1) from = r.parts + (segment * pass.batch * pass.heads + unitState) * size;
            else if (r.first) {
                from = r.first + unitState * size;
                swapped = r.firstSwapped != 0;
            }
        }
#pragma unroll
        for (int o = 0; o < kOwn; o++)
#pragma unroll
            for (int m = 0; m < kTilesA; m++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int x = m * 16 + quad * 4 + i, y = (wave * kOwn + o) * 16 + col;
                    const bool in = from && x < r.dimA && y < r.dimC;
                    memory[o][m][i] = in ? from[swapped ? (int64_t)y * r.dimA + x : (int64_t)x * r.dimC + y] : 0.0f;
                }
    }

    uint4 nextA[kStates ? 1 : S::kLoadsA], nextB[S::kLoadsA], nextC[S::kLoadsC];
    const auto chunkStart = [&](int64_t n) { return begin + (r.backwards ? chunks - 1 - n : n) * kSteps; };
    const auto fetchRows = [&](auto& next, const T* rows, int64_t step, int64_t t0, int pieces, int dim, int grain) {
#pragma unroll
        for (int i = 0; i < (int)(sizeof(next) / sizeof(next[0])); i++) {
            const int piece = i * kThreads + threadIdx.x;
            const int row = piece / pieces, at = piece % pieces * kE;
            const int64_t t = t0 + row;
            next[i] = t < end && at < dim ? loadPiece<T>(rows + t * step + at, dim - at, grain) : make_uint4(0, 0, 0, 0);
        }
    };
    const auto fetch = [&](int64_t n) {
        const int64_t t0 = chunkStart(n);
        if constexpr (!kStates) fetchRows(nextA, aRows, r.a.step, t0, S::kPieceA, r.dimA, r.aGrain);
        fetchRows(nextB, bRows, r.b.step, t0, S::kPieceA, r.dimA, r.bGrain);
        fetchRows(nextC, cRows, r.c.step, t0, S::kPieceC, r.dimC, r.cGrain);
    };
    uint32_t odd = 0;         // carry bits of non-finite values in this chunk's b and c
    const auto put = [&](const auto& next, T* rows, int stride, int pieces) {
#pragma unroll
        for (int i = 0; i < (int)(sizeof(next) / sizeof(next[0])); i++) {
            const int piece = i * kThreads + threadIdx.x;
            *reinterpret_cast<uint4*>(rows + piece / pieces * stride + piece % pieces * kE) = next[i];
            odd |= nonFinite<T>(next[i]);
        }
    };
    // column `at` of rows 4 quad .. 4 quad + 3 of the 16-row block
    const auto columns = [&](const T* rows, int stride, int block, int at) {
        vec<T, 4> x;
#pragma unroll
        for (int j = 0; j < 4; j++) x[j] = rows[(block * 16 + quad * 4 + j) * stride + at];
        return x;
    };

    float factor = 1.0f;      // of the memory over the whole segment
    if (chunks > 0) fetch(0);
    for (int64_t n = 0; n < chunks; n++) {
        const int64_t t0 = chunkStart(n);
        const int have = end - t0 < kSteps ? (int)(end - t0) : kSteps;
        __syncthreads();
        if constexpr (!kStates) put(nextA, sA, S::kStrideA, S::kPieceA);
        odd = 0;
        put(nextB, sB, S::kStrideA, S::kPieceA);
        put(nextC, sC, S::kStrideC, S::kPieceC);
        // A weight of zero takes a finite row out of a product, but not an
        // infinity or a NaN: a chunk whose b or c hold one is summed step by
        // step, leaving out the steps that are not seen.
        const bool careful = __syncthreads_or((odd & Exponent<T>::kCarry) != 0) != 0;
        if (n + 1 < chunks) fetch(n + 1);

        // bit t: step t of the chunk starts an episode
        uint64_t starts = 0;
        if (pass.starts)
            starts = __ballot(lane < have && pass.starts[batch * pass.startsBatch + (t0 + lane) * pass.startsStep] != 0);
        const int all = __popcll(starts);
        const auto episode = [&](int t) { return __popcll(starts & (~0ull >> (63 - t))); };

        if constexpr (!kStates) {
            for (int tile = wave; tile < kBlocks * kBlocks; tile += kWaves) {
                const int tb = tile / kBlocks, sb = tile % kBlocks;
                const int t = tb * 16 + col, mine = episode(t);
                f32x4 p = { 0.f, 0.f, 0.f, 0.f };
                if (r.backwards ? sb >= tb : sb <= tb) {
#pragma unroll
                    for (int k = 0; k < kTilesA; k++) {
                        const auto b = *reinterpret_cast<const vec<T, 4>*>(sB + (sb * 16 + col) * S::kStrideA + k * 16 + quad * 4);
                        const auto a = *reinterpret_cast<const vec<T, 4>*>(sA + t * S::kStrideA + k * 16 + quad * 4);
                        p = mma(b, a, p);
                    }
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const int s = sb * 16 + quad * 4 + i, gap = r.backwards ? s - t : t - s;
                        p[i] = gap >= 0 && episode(s) == mine ? p[i] * (power(gap) * r.scaleP) : 0.0f;
                    }
                }
                *reinterpret_cast<vec<T, 4>*>(sP + t * S::kStrideP + sb * 16 + quad * 4) = fromFloat<T, 4>(p);
            }
            __syncthreads();
            for (int tb = 0; tb < kBlocks; tb++) {
                const int t = tb * 16 + col, mine = episode(t);
                const bool open = r.backwards ? mine == all : mine == 0;
                const float in = open ? power(r.backwards ? have - 1 - t : t + 1) * r.scaleIn : 0.0f;
#pragma unroll
                for (int o = 0; o < kOwn; o++) {
                    const int at = (wave * kOwn + o) * 16;
                    f32x4 within = { 0.f, 0.f, 0.f, 0.f }, carried = { 0.f, 0.f, 0.f, 0.f };
                    if (careful) {
                        for (int s = r.backwards ? t : 0; s < (r.backwards ? have : t + 1); s++)
                            if (episode(s) == mine)
                                for (int i = 0; i < 4; i++)
                                    within[i] += (float)sP[t * S::kStrideP + s] * (float)sC[s * S::kStrideC + at + quad * 4 + i];
                    } else {
#pragma unroll
                    for (int sb = 0; sb < kBlocks; sb++) {
                        if (r.backwards ? sb < tb : sb > tb) continue;
                        const auto p = *reinterpret_cast<const vec<T, 4>*>(sP + t * S::kStrideP + sb * 16 + quad * 4);
                        within = mma(columns(sC, S::kStrideC, sb, at + col), p, within);
                    }
                    }
#pragma unroll
                    for (int m = 0; m < kTilesA; m++) {
                        const auto a = *reinterpret_cast<const vec<T, 4>*>(sA + t * S::kStrideA + m * 16 + quad * 4);
                        vec<typename L::type, 4> terms[L::kIn];
                        split<typename L::type, L::kIn>(memory[o][m], terms);
#pragma unroll
                        for (int i = 0; i < L::kIn; i++) carried = mma(terms[i], __builtin_convertvector(a, vec<typename L::type, 4>), carried);
                    }
                    // a closed step takes nothing from the memory, whatever that holds
                    f32x4 out = within;
                    if (open) out += carried * in;
                    const int y = at + quad * 4;
                    if (t >= have || y >= r.dimC) continue;
                    const int64_t to = batch * r.out.batch + (t0 + t) * r.out.step + head * r.out.head + y;
                    if (r.outFloat) {
                        float* x = static_cast<float*>(r.out.data) + to;
                        if (r.outWide && y + 4 <= r.dimC) *reinterpret_cast<f32x4*>(x) = out;
                        else
                            for (int i = 0; i < 4; i++)
                                if (y + i < r.dimC) x[i] = out[i];
                    } else {
                        T* x = static_cast<T*>(r.out.data) + to;
                        if (r.outWide && y + 4 <= r.dimC) *reinterpret_cast<vec<T, 4>*>(x) = fromFloat<T, 4>(out);
                        else
                            for (int i = 0; i < 4; i++)
                                if (y + i < r.dimC) x[i] = (T)out[i];
                    }
                }
            }
        }

        // the memory: kept where no episode starts in the chunk, and what the chunk adds
        const float keep = all == 0 ? power(have) : 0.0f;
        factor *= keep;
#pragma unroll
        for (int o = 0; o < kOwn; o++) {
#pragma unroll
            for (int m = 0; m < kTilesA; m++)
                memory[o][m] = all == 0 ? memory[o][m] * keep : f32x4{ 0.f, 0.f, 0.f, 0.f };
            if (careful) {
                for (int s = 0; s < have; s++) {
                    if (episode(s) != (r.backwards ? 0 : all)) continue;
                    const float c = (float)sC[s * S::kStrideC + (wave * kOwn + o) * 16 + col]
                                  * (power(r.backwards ? s + 1 : have - 1 - s) * r.scaleOut);
#pragma unroll
                    for (int m = 0; m < kTilesA; m++)
#pragma unroll
                        for (int i = 0; i < 4; i++)
                            memory[o][m][i] += (float)sB[s * S::kStrideA + m * 16 + quad * 4 + i] * c;
                }
                continue;
            }
#pragma unroll
            for (int sb = 0; sb < kBlocks; sb++) {
                f32x4 c = toFloat<T, 4>(columns(sC, S::kStrideC, sb, (wave * kOwn + o) * 16 + col));
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const int s = sb * 16 + quad * 4 + j;
                    const bool leaves = s < have && episode(s) == (r.backwards ? 0 : all);
                    c[j] = leaves ? c[j] * (power(r.backwards ? s + 1 : have - 1 - s) * r.scaleOut) : 0.0f;
                }
                vec<typename L::type, 4> terms[L::kOut];
                split<typename L::type, L::kOut>(c, terms);
#pragma unroll
                for (int m = 0; m < kTilesA; m++) {
                    const auto b = __builtin_convertvector(columns(sB, S::kStrideA, sb, m * 16 + col), vec<typename L::type, 4>);
#pragma unroll
                    for (int i = 0; i < L::kOut; i++) memory[o][m] = mma(b, terms[i], memory[o][m]);
                }
            }
        }
    }

    const int64_t size = (int64_t)r.dimA * r.dimC, unitState = batch * pass.heads + head;
    float* to = nullptr;
    bool swapped = false;
    if (kStates) {
        to = r.parts + (segment * pass.batch * pass.heads + unitState) * size;
        if (threadIdx.x == 0) r.factors[segment * pass.batch * pass.heads + unitState] = factor;
    } else if (pass.segments == 1 && r.last) {
        to = r.last + unitState * size;
        swapped = r.lastSwapped != 0;
    }
    if (to) {
#pragma unroll
        for (int o = 0; o < kOwn; o++)
#pragma unroll
            for (int m = 0; m < kTilesA; m++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int x = m * 16 + quad * 4 + i, y = (wave * kOwn + o) * 16 + col;
                    if (x < r.dimA && y < r.dimC)
                        to[swapped ? (int64_t)y * r.dimA + x : (int64_t)x * r.dimC + y] = memory[o][m][i];
                }
    }
}

template <typename T, int kA, int kCd, bool kStates>
void launchAttentionShape(const Pass& pass, int firstRole, int roles, hipStream_t stream)
{
    // float32 rows of 128 leave room for chunks of 32 steps
    constexpr int kSteps = sizeof(T) == 4 && (kA > 64 || kCd > 64) ? 32 : 64;
    const int64_t units = pass.batch * pass.heads * pass.segments;
    attentionKernel<T, kA, kCd, kSteps, kStates>
        <<<dim3((unsigned)units, (unsigned)roles), Shape<T, kA, kCd, kSteps>::kThreads, 0, stream>>>(pass, firstRole);
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
