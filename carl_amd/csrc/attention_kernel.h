// attention_kernel.h - the chunked kernel of attention.h, for one element type.
#pragma once

#include "attention.h"
#include "lds.h"
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

// A tile of rows in LDS: rows of kPieces 16-byte pieces, each row's permuted by
// its number so that the reads below meet all banks.
template <typename T, int kWidth> struct Tile {
    static constexpr int kBytes = kWidth * (int)sizeof(T), kPieces = kBytes / 16, kE = 16 / (int)sizeof(T);

    static __device__ inline int permuted(int row, int piece)
    {
        if constexpr (sizeof(T) == 4) return piece ^ (((row & 3) | (row >> 2 & 3) << 2) & (kPieces - 1));
        else if constexpr (kPieces == 4) return piece ^ (row >> 2 & 1) << 1;
        else return piece ^ ((row & 3) << 1 | (row >> 2 & 1));
    }
    static __device__ inline int at(int row, int element)
    {
        return row * kBytes + permuted(row, element / kE) * 16 + element % kE * (int)sizeof(T);
    }
    static __device__ inline float element(const char* tile, int row, int i) { return (float)*reinterpret_cast<const T*>(tile + at(row, i)); }

    // Row lane%16 of a 16-row block, elements 16 k + 4 quad + j; `lane` is
    // at(lane%16, 4 quad), and the block's rows come before `tile`.
    static __device__ inline vec<T, 4> row(const char* tile, int lane, int k)
    {
        return *reinterpret_cast<const vec<T, 4>*>(tile + (lane ^ k * 16 * (int)sizeof(T)));
    }

    // Column 16 m + lane%16 of rows 4 quad + j of a 16-row block; `lane` from columnLane().
    static __device__ inline int columnLane(int col, int quad)
    {
        return sizeof(T) == 4 ? at(quad * 4, col) : at(quad * 4 + (col >> 2), (col & 3) * 4);
    }
    static __device__ inline vec<T, 4> column(const char* tile, int lane, int m)
    {
        if constexpr (sizeof(T) == 4) {
            f32x4 x;
#pragma unroll
            for (int j = 0; j < 4; j++)
                x[j] = *reinterpret_cast<const float*>(tile + ((lane ^ m * 64 ^ j * 16) + j * kBytes));
            return x;
        } else      // transposes 4 rows x 16 columns held by 16 lanes
            return __builtin_bit_cast(vec<T, 4>, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (__attribute__((address_space(3))) i16x4*)(tile + (lane ^ m * 32))));
    }
};

// How products with float32 factors run.  bfloat16: the memory as it is read
// by a rounded once, like the weights within a chunk, so that an output's two
// parts are each as exact as the other; what enters the memory from c as three
// terms where the memory is handed to the caller, else as two.  float16, whose
// range holds neither (a . b passes 65,504 where each is 100 in 64 dimensions,
// and of a small gradient little is left above 2^-24), and float32: as float32.
template <typename T> struct Long {
    using type = float;
    static constexpr int kIn = 1, kOut = 1;
};
template <> struct Long<bf16> {
    using type = bf16;
    static constexpr int kIn = 1, kOut = 3;
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
    // A wave for each column tile of the memory, two tiles each of 128 columns:
    // eight waves would leave room for one workgroup (or spill) where four
    // leave it for two (2,048 x 64 of 128 bf16, gradients: 1.94 and 1.27 ms).
    static constexpr int kWaves = kC_ / 16 < 4 ? kC_ / 16 : 4;
    static constexpr int kThreads = kWaves * 64;
    using P = typename Long<T>::type;                // of the weights within a chunk
    static constexpr int kStrideP = kSteps + 16 / (int)sizeof(P);
    static constexpr int kTileA = kSteps * Tile<T, kA>::kBytes, kTileC = kSteps * Tile<T, kC_>::kBytes;
    static constexpr int kLoadsA = (kTileA / 16 + kThreads - 1) / kThreads, kLoadsC = (kTileC / 16 + kThreads - 1) / kThreads;
    static_assert(kTileA % 1024 == 0 && kTileC % 1024 == 0, "whole copies of a wave");
    // workgroups that LDS holds at once, as waves of a SIMD that the registers leave room for
    static constexpr int kLds = 2 * kTileA + kTileC + kSteps * kStrideP * (int)sizeof(P);
    static constexpr int kFit = 160 * 1024 / kLds, kMost = kA * kC_ > 64 * 128 ? 2 : kA * kC_ > 64 * 64 ? 3 : 4;
    static constexpr int kResident = kFit < kMost ? kFit : kMost;
    static_assert(kFit >= 1, "one workgroup");
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
    using L = Long<T>;
    using LT = typename L::type;
    using TileA = Tile<T, kA>;
    using TileC = Tile<T, kCd>;

    __shared__ __align__(1024) char sA[kStates ? 16 : S::kTileA];
    __shared__ __align__(1024) char sB[S::kTileA];
    __shared__ __align__(1024) char sC[S::kTileC];
    __shared__ __align__(16) LT sP[kStates ? 1 : kSteps * S::kStrideP];

    // Blocks are dealt to the 8 dies in turn.  The roles of one unit and the
    // heads of one sequence, which read the same rows or lines, run on one:
    // the grid is (8 x heads x roles, groups / 8).  With few groups (sequences
    // and their segments) units of one head are dealt instead.
    const int die = blockIdx.x % 8, batches = (int)pass.batch, groups = batches * pass.segments;
    int group, head, role = 0;
    {
        int unit = blockIdx.x / 8;
        if (roles == 2) {
            role = unit & 1;
            unit >>= 1;
        } else if (roles == 3) {
            role = unit % 3;
            unit /= 3;
        }
        if (pass.dealGroups) {
            group = blockIdx.y * 8 + die;
            head = unit;
        } else {
            unit = unit * 8 + die;
            group = unit / pass.heads;
            head = unit - group * pass.heads;
        }
    }
    if (group >= groups) return;
    const int segmentOf = pass.segments == 1 ? 0 : group / batches;
    const Role& r = pass.role[firstRole + role];
    const int64_t segment = segmentOf, batch = group - segmentOf * batches;
    const int lane = threadIdx.x & 63, col = lane & 15, quad = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const bool backwards = r.backwards != 0;
    const int dimA = r.dimA, dimC = r.dimC, inShift = r.inShift;

    const int64_t begin = segment * pass.segmentSteps;
    const int64_t end = begin + pass.segmentSteps < pass.steps ? begin + pass.segmentSteps : pass.steps;
    const int chunks = (int)((end - begin + kSteps - 1) / kSteps);
    const T* aRows = static_cast<const T*>(r.a.data) + batch * r.a.batch + head / r.aHeads * r.a.head;
    const T* bRows = static_cast<const T*>(r.b.data) + batch * r.b.batch + head / r.bHeads * r.b.head;
    const T* cRows = static_cast<const T*>(r.c.data) + batch * r.c.batch + head / r.cHeads * r.c.head;
    const int64_t aStep = r.a.step, bStep = r.b.step, cStep = r.c.step;
    const int aGrain = r.aGrain, bGrain = r.bGrain, cGrain = r.cGrain;

    // Of a decay that is zero or not a number, no steps are still a weight of
    // one: this product with zero is zero, whatever the other factor.
    const float decay2 = pass.logDecay[head] * 1.44269504088896341f;
    const auto power = [&](float steps) {
        float x;
        asm("v_mul_legacy_f32 %0, %1, %2" : "=v"(x) : "v"(decay2), "v"(steps));
        return __builtin_amdgcn_exp2f(x);
    };

    // A lane's elements of the memory: rows 16 m + 4 quad + i, column 16 (wave's
    // tile) + col.  Through a descriptor, past whose end lies what the padding
    // would hold: read as zero, written nowhere.
    const int64_t unitState = batch * pass.heads + head, partState = segment * pass.batch * pass.heads + unitState;
    const int size = dimA * dimC;
    f32x4 memory[kOwn][kTilesA];
    // visits with a lane's offset and, of the whole wave, what is added to it
    const auto eachMemory = [&](bool swapped, auto one, auto four) {
        const bool full = dimA == kA && dimC == kCd;
#pragma unroll
        for (int o = 0; o < kOwn; o++) {
            const int y = (wave * kOwn + o) * 16 + col;
            const int base = swapped ? (y * dimA + quad * 4) * 4 : (quad * 4 * dimC + y) * 4;
            if (swapped && dimA % 4 == 0) {
#pragma unroll
                for (int m = 0; m < kTilesA; m++)
                    four(o, m, full ? base : y < dimC && m * 16 + quad * 4 < dimA ? base + m * 64 : kOutside, full ? m * 64 : 0);
                continue;
            }
            const int row = swapped ? 4 : dimC * 4;
#pragma unroll
            for (int m = 0; m < kTilesA; m++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    if (full) one(o, m, i, base, (m * 16 + i) * row);
                    else one(o, m, i, y < dimC && m * 16 + quad * 4 + i < dimA ? base + (m * 16 + i) * row : kOutside, 0);
                }
        }
    };
    {
        const float* from = nullptr;
        bool swapped = false;
        if (!kStates) {
            if (pass.segments > 1) {
                const int64_t part = segment * pass.finer + (backwards ? pass.finer - 1 : 0);
                from = r.parts + (part * pass.batch * pass.heads + unitState) * size;
                swapped = r.partsSwapped != 0;
            } else if (r.first) {
                from = r.first + unitState * size;
                swapped = r.firstSwapped != 0;
            }
        }
        if (from) {
            const auto d = __builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(from), 0, size * 4, 0x00027000);
            eachMemory(
                swapped,
                [&](int o, int m, int i, int at, int more) {
                    memory[o][m][i] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(d, at, more, 0));
                },
                [&](int o, int m, int at, int more) {
                    memory[o][m] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(d, at, more, 0));
                });
        } else {
#pragma unroll
            for (int o = 0; o < kOwn; o++)
#pragma unroll
                for (int m = 0; m < kTilesA; m++) memory[o][m] = f32x4{ 0.f, 0.f, 0.f, 0.f };
        }
    }

    // Chunks follow time in the pass's direction, and so do the rows of a chunk
    // in LDS: what comes first is in row 0.
    const auto chunkStart = [&](int n) { return begin + (int64_t)(backwards ? chunks - 1 - n : n) * kSteps; };

    // A chunk's rows to LDS, by copies that a descriptor ends at the chunk's
    // last row (rows and pieces past it arrive as zeros).  They need addresses
    // of 4 bytes within 32 bits of the chunk's first; others go element by
    // element.  waitRows() waits for this thread's pieces, clears what lies
    // past the row's end in the last one, and looks for non-finite values.
    const auto copyRows = [&](auto tile, int loads, int thread, char* lds, const T* rows, int64_t step, int64_t t0, int have, int dim, int grain) {
        using Rows = decltype(tile);
        constexpr int kPieces = Rows::kPieces;
        const T* base = rows + t0 * step;
        if (grain >= 4) {
            const uint32_t stepBytes = (uint32_t)step * (uint32_t)sizeof(T), rowBytes = (uint32_t)dim * (uint32_t)sizeof(T);
            const i32x4 from = descriptor(base, (int)((uint32_t)(have - 1) * stepBytes + rowBytes));
            const uint32_t to = ldsAddress(lds) + wave * 1024;
            // rows that a thread copies, 16 or a multiple apart, are permuted alike
            constexpr int kAtOnce = kThreads / kPieces;
            if (kAtOnce % 16 == 0 && have == kSteps) {
                const uint32_t row = thread / kPieces, at = Rows::permuted(row, thread % kPieces) * 16;
                const uint32_t first = (backwards ? kSteps - 1 - row : row) * stepBytes + at;
                const uint32_t ahead = (backwards ? 0u - kAtOnce : kAtOnce) * stepBytes;
                const bool within = at < rowBytes;
#pragma unroll
                for (int i = 0; i < loads; i++) {
                    if (i * kThreads + wave * 64 >= kSteps * kPieces) break;
                    copyToLds(from, within ? (int)(first + i * ahead) : kOutside, 0, to + i * kThreads * 16);
                }
                return;
            }
#pragma unroll
            for (int i = 0; i < loads; i++) {
                if (i * kThreads + wave * 64 >= kSteps * kPieces) break;
                const int piece = i * kThreads + thread, row = piece / kPieces, at = Rows::permuted(row, piece % kPieces) * 16;
                const uint32_t t = backwards ? have - 1 - row : row;
                copyToLds(from, row < have && at < (int)rowBytes ? (int)(t * stepBytes + at) : kOutside, 0, to + i * kThreads * 16);
            }
            return;
        }
#pragma unroll 1
        for (int i = 0; i < loads; i++) {
            if (i * kThreads + wave * 64 >= kSteps * kPieces) break;
            const int piece = i * kThreads + thread, row = piece / kPieces, at = Rows::permuted(row, piece % kPieces) * Rows::kE;
            uint4 x = make_uint4(0, 0, 0, 0);
            if (row < have) x = loadPiece<T>(base + (backwards ? have - 1 - row : row) * step + at, dim - at);
            *reinterpret_cast<uint4*>(lds + piece * 16) = x;
        }
    };
    const auto waitRows = [&](auto tile, int loads, int thread, char* lds, int dim, bool look) {
        using Rows = decltype(tile);
        uint32_t odd = 0;         // carry bits of non-finite values
        if (dim % Rows::kE) {
#pragma unroll 1
            for (int i = 0; i < loads; i++) {
                if (i * kThreads + wave * 64 >= kSteps * Rows::kPieces) break;
                const int piece = i * kThreads + thread;
                if (Rows::permuted(piece / Rows::kPieces, piece % Rows::kPieces) != dim / Rows::kE) continue;
                for (int e = dim % Rows::kE; e < Rows::kE; e++) reinterpret_cast<T*>(lds + piece * 16)[e] = T(0);
            }
        }
        if (look)
#pragma unroll
            for (int i = 0; i < loads; i++) {
                if (i * kThreads + wave * 64 >= kSteps * Rows::kPieces) break;
                odd |= nonFinite<T>(*reinterpret_cast<const uint4*>(lds + (i * kThreads + thread) * 16));
            }
        return odd;
    };

    // the memory after the last chunk goes to the caller (or to the sums that do)
    const bool handed = r.last && (kStates || pass.segments == 1);
    // of the memory over the whole segment; with its sign set where a start closes
    // it (a weight that is zero in float32 closes nothing: a NaN stays)
    float factor = 1.0f;
#pragma unroll 1
    for (int n = 0; n < chunks; n++) {
        const int64_t t0 = chunkStart(n);
        const int have = end - t0 < kSteps ? (int)(end - t0) : kSteps;
        // Opaque, so that the many addresses made of it are made again for each
        // chunk and not kept (spilled) from before the loop.
        int thread = threadIdx.x;
        asm volatile("" : "+v"(thread));
        const int lane = thread & 63, col = lane & 15, quad = lane >> 4;
        __syncthreads();
        if constexpr (!kStates) copyRows(TileA{}, S::kLoadsA, thread, sA, aRows, aStep, t0, have, dimA, aGrain);
        copyRows(TileA{}, S::kLoadsA, thread, sB, bRows, bStep, t0, have, dimA, bGrain);
        copyRows(TileC{}, S::kLoadsC, thread, sC, cRows, cStep, t0, have, dimC, cGrain);
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
        waitCopies();
        uint32_t odd = 0;
        if constexpr (!kStates) waitRows(TileA{}, S::kLoadsA, thread, sA, dimA, false);
        odd |= waitRows(TileA{}, S::kLoadsA, thread, sB, dimA, true);
        odd |= waitRows(TileC{}, S::kLoadsC, thread, sC, dimC, true);
        const bool careful = __syncthreads_or((odd & Exponent<T>::kCarry) != 0) != 0;

        // where a lane's fragments lie: a row's neighbouring elements, columns of
        // rows, and the results' rows of P
        const int rowLane = TileA::at(col, quad * 4);
        const int columnLaneA = TileA::columnLane(col, quad), columnLaneC = TileC::columnLane(col, quad);
        LT* const pLane = sP + col * S::kStrideP + quad * 4;
        const float quadSteps = (float)(quad * 4), colSteps = (float)col;

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
            // (several waves share a column where there are more of them than columns)
            constexpr int kShare = kWaves > kBlocks ? kWaves / kBlocks : 1;
            for (int tb = wave % kBlocks; tb < kBlocks; tb += kWaves) {
                const int t = tb * 16 + col, from = cuts ? low(t) : 0;
                vec<T, 4> a[kTilesA];
#pragma unroll
                for (int k = 0; k < kTilesA; k++) a[k] = TileA::row(sA + tb * 16 * TileA::kBytes, rowLane, k);
                const int share = kShare > 1 ? wave / kBlocks : 0;
                float gap = (float)((tb - share) * 16) + colSteps - quadSteps;      // to the tile's first row of the lane
#pragma unroll 1
                for (int sb = share; sb <= tb; sb += kShare, gap -= 16.0f * kShare) {
                    f32x4 p = { 0.f, 0.f, 0.f, 0.f };
                    const char* rows = sB + sb * 16 * TileA::kBytes;
#pragma unroll
                    for (int k = 0; k < kTilesA; k += 2)
                        p = mma(both(TileA::row(rows, rowLane, k), TileA::row(rows, rowLane, k + 1)), both(a[k], a[k + 1]), p);
                    const int s = sb * 16 + quad * 4;
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const float w = p[i] * (power(gap - (float)i) * r.scaleP);
                        p[i] = s + i >= from && s + i <= t ? w : 0.0f;
                    }
                    *reinterpret_cast<vec<LT, 4>*>(pLane + tb * 16 * S::kStrideP + sb * 16) = fromFloat<LT, 4>(p);
                }
                // blocks of s are met in pairs below
                if (tb % 2 == 0 && share == 0)
                    *reinterpret_cast<vec<LT, 4>*>(pLane + tb * 16 * S::kStrideP + (tb + 1) * 16) = vec<LT, 4>{ LT(0), LT(0), LT(0), LT(0) };
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
                    const char* rows = sA + tb * 16 * TileA::kBytes;
                    const auto a = both(__builtin_convertvector(TileA::row(rows, rowLane, m), vec<LT, 4>),
                                        __builtin_convertvector(TileA::row(rows, rowLane, m + 1), vec<LT, 4>));
#pragma unroll
                    for (int o = 0; o < kOwn; o++)
#pragma unroll
                        for (int i = 0; i < L::kIn; i++) acc[o][tb] = mma(both(lo[o][i], hi[o][i]), a, acc[o][tb]);
                }
            }
            const int firstCut = cuts ? __builtin_ctzll(cuts) : 64;
            const float past16 = power(16.0f);
            float in = power(colSteps + (float)inShift) * r.scaleIn;
#pragma unroll
            for (int tb = 0; tb < kBlocks; tb++, in *= past16) {
                const bool open = tb * 16 + col < firstCut;
                // a closed row takes nothing from the memory, whatever that holds
#pragma unroll
                for (int o = 0; o < kOwn; o++) acc[o][tb] = open ? acc[o][tb] * in : f32x4{ 0.f, 0.f, 0.f, 0.f };
            }
            __syncthreads();
        }

        const float keep = closed ? 0.0f : power((float)have);
        factor = closed ? -1.0f : factor * keep;
        if (!careful) {
            vec<T, 4> c[kOwn][kBlocks];
#pragma unroll
            for (int o = 0; o < kOwn; o++)
#pragma unroll
                for (int sb = 0; sb < kBlocks; sb++)
                    c[o][sb] = TileC::column(sC + sb * 16 * TileC::kBytes, columnLaneC, wave * kOwn + o);
            if constexpr (!kStates) {
#pragma unroll
                for (int tb = 0; tb < kBlocks; tb++)
#pragma unroll
                    for (int sb = 0; sb <= tb; sb += 2) {
                        const LT* row = pLane + tb * 16 * S::kStrideP + sb * 16;
                        const auto p = both(*reinterpret_cast<const vec<LT, 4>*>(row), *reinterpret_cast<const vec<LT, 4>*>(row + 16));
#pragma unroll
                        for (int o = 0; o < kOwn; o++)
                            acc[o][tb] = mma(both(__builtin_convertvector(c[o][sb], vec<LT, 4>), __builtin_convertvector(c[o][sb + 1], vec<LT, 4>)),
                                             p, acc[o][tb]);
                    }
            }
            if (closed) {
#pragma unroll
                for (int o = 0; o < kOwn; o++)
#pragma unroll
                    for (int m = 0; m < kTilesA; m++) memory[o][m] = f32x4{ 0.f, 0.f, 0.f, 0.f };
            } else {
#pragma unroll
                for (int o = 0; o < kOwn; o++)
#pragma unroll
                    for (int m = 0; m < kTilesA; m++) memory[o][m] *= keep;
            }
            // What a row weighs in the memory after the chunk: of a full chunk
            // without cuts one power of the last row's and the decay from row to
            // row and block to block; of others each row's, and zero for those
            // that it does not see.
            f32x4 w[kBlocks];
            const float rest = (float)(have - inShift) - quadSteps;
            if (!closed && have == kSteps) {
                const float once = power(1.0f), past16 = power(16.0f);
                w[kBlocks - 1][3] = power(rest - (float)(kSteps - 13)) * r.scaleOut;
#pragma unroll
                for (int j = 2; j >= 0; j--) w[kBlocks - 1][j] = w[kBlocks - 1][j + 1] * once;
#pragma unroll
                for (int sb = kBlocks - 2; sb >= 0; sb--) w[sb] = w[sb + 1] * past16;
            } else {
#pragma unroll
                for (int sb = 0; sb < kBlocks; sb++)
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const int s = sb * 16 + quad * 4 + j;
                        w[sb][j] = s >= leave && s < have ? power(rest - (float)(sb * 16 + j)) * r.scaleOut : 0.0f;
                    }
            }
#pragma unroll
            for (int sb = 0; sb < kBlocks; sb += 2) {
                vec<LT, 4> lo[kOwn][L::kOut], hi[kOwn][L::kOut];
#pragma unroll
                for (int o = 0; o < kOwn; o++) {
                    split<LT, L::kOut>(toFloat<T, 4>(c[o][sb]) * w[sb], lo[o]);
                    split<LT, L::kOut>(toFloat<T, 4>(c[o][sb + 1]) * w[sb + 1], hi[o]);
                }
                const char* rows = sB + sb * 16 * TileA::kBytes;
#pragma unroll
                for (int m = 0; m < kTilesA; m++) {
                    const auto b = both(__builtin_convertvector(TileA::column(rows, columnLaneA, m), vec<LT, 4>),
                                        __builtin_convertvector(TileA::column(rows + 16 * TileA::kBytes, columnLaneA, m), vec<LT, 4>));
#pragma unroll
                    for (int o = 0; o < kOwn; o++)
#pragma unroll
                        for (int i = 0; i < L::kOut; i++)
                            if (i < 2 || handed) memory[o][m] = mma(b, both(lo[o][i], hi[o][i]), memory[o][m]);
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
                                acc[o][tb][i] += (float)sP[t * S::kStrideP + s] * TileC::element(sC, s, tile + quad * 4 + i);
                    }
                }
#pragma unroll
                for (int m = 0; m < kTilesA; m++) memory[o][m] = closed ? f32x4{ 0.f, 0.f, 0.f, 0.f } : memory[o][m] * keep;
#pragma unroll 1
                for (int s = leave; s < have; s++) {
                    const float x = TileC::element(sC, s, tile + col) * (power((float)(have - inShift - s)) * r.scaleOut);
                    int past = dimA - quad * 4;         // rows from here stay zero: theirs would be no number with an infinite x
                    asm volatile("" : "+v"(past));
#pragma unroll
                    for (int m = 0; m < kTilesA; m++)
#pragma unroll
                        for (int i = 0; i < 4; i++)
                            memory[o][m][i] += TileA::element(sB, s, m * 16 + quad * 4 + i) * (m * 16 + i < past ? x : 0.0f);
                }
            }
        }

        if constexpr (!kStates) {
            const int64_t outStep = r.out.step;
            const int64_t row0 = batch * r.out.batch + (t0 + (backwards ? have - 1 : 0)) * outStep + head * r.out.head;
            if (r.outWide && !r.outFloat) {
                const int y = wave * kOwn * 16 + quad * 4;
                T* const lane0 = static_cast<T*>(r.out.data) + row0 + (backwards ? -(int64_t)col : (int64_t)col) * outStep + y;
                const int64_t ahead = (backwards ? -16 : 16) * outStep;
#pragma unroll
                for (int tb = 0; tb < kBlocks; tb++)
#pragma unroll
                    for (int o = 0; o < kOwn; o++)
                        if (tb * 16 + col < have && y + o * 16 < dimC)
                            *reinterpret_cast<vec<T, 4>*>(lane0 + tb * ahead + o * 16) = fromFloat<T, 4>(acc[o][tb]);
            } else {
#pragma unroll
                for (int tb = 0; tb < kBlocks; tb++) {
                    const int t = tb * 16 + col;
                    if (t >= have) continue;
                    const int64_t row = row0 + (backwards ? -t : t) * outStep;
#pragma unroll
                    for (int o = 0; o < kOwn; o++)
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            const int y = (wave * kOwn + o) * 16 + quad * 4 + i;
                            if (y >= dimC) continue;
                            if (r.outFloat) static_cast<float*>(r.out.data)[row + y] = acc[o][tb][i];
                            else static_cast<T*>(r.out.data)[row + y] = (T)acc[o][tb][i];
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
    const auto d = __builtin_amdgcn_make_buffer_rsrc(to, 0, size * 4, 0x00027000);
    eachMemory(
        swapped,
        [&](int o, int m, int i, int at, int more) {
            __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(memory[o][m][i]), d, at, more, 0);
        },
        [&](int o, int m, int at, int more) {
            __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(vec<uint32_t, 4>, memory[o][m]), d, at, more, 0);
        });
}

template <typename T, int kA, int kCd, int kSteps, bool kStates>
void launchAttentionSteps(const Pass& pass, int firstRole, int roles, hipStream_t stream)
{
    const unsigned groups = (unsigned)(pass.batch * pass.segments), heads = (unsigned)pass.heads;
    const dim3 grid = pass.dealGroups ? dim3(8 * heads * roles, (groups + 7) / 8) : dim3((groups * heads + 7) / 8 * 8 * roles);
    attentionKernel<T, kA, kCd, kSteps, kStates>
        <<<grid, Shape<T, kA, kCd, kSteps>::kThreads, 0, stream>>>(pass, firstRole, roles);
}

template <typename T, int kA, int kCd, bool kStates>
void launchAttentionShape(const Pass& pass, int firstRole, int roles, hipStream_t stream)
{
    // Chunks of 64 steps (16,384 x 64, 8 heads of 64 in bfloat16, gradients:
    // 4.4 ms, in chunks of 32 4.9 ms); of 32 where no sequence is longer, and
    // where products run in float32, whose matrix instructions the longer
    // chunks' products within keep busy (4,096 x 64 of float32 with gradients:
    // 2.68 ms, in chunks of 64 3.59 ms; 16,384 x 64 of float16 9.24 and 10.05).
    constexpr bool large = std::is_same_v<typename Long<T>::type, float>;
    if constexpr (!kStates && !large) {
        if (pass.segmentSteps > 32) launchAttentionSteps<T, kA, kCd, 64, kStates>(pass, firstRole, roles, stream);
        else launchAttentionSteps<T, kA, kCd, 32, kStates>(pass, firstRole, roles, stream);
    } else
        launchAttentionSteps<T, kA, kCd, large ? 32 : 64, kStates>(pass, firstRole, roles, stream);
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
