// actions.hip - log-probabilities, entropies and choices of actions from rows
// of logits, and the gradients by them.
//
// Formulas, and what is not there: include/carl_amd_ops.h.  With m a head's
// largest logit, Z = sum exp(x - m) and A = sum exp(x - m) (x - m):
//   log p_a = x_a - m - log Z          H = log Z - A / Z
//   dx_j = dlp ([j = a] - p_j) - dH p_j (log p_j + H)
// The backward pass computes m, Z and A again: it reads the logits anyway.
//
// What bounds it: memory, and for short heads the exponentials and the chain of
// one head's steps (the simulator's 7 heads of 18 logits in bf16, masked: 1,048,576
// log-probabilities 24 us, 3.9 TB/s, and gradients 30, 4.3 TB/s; 131,072 best
// actions with noise 9.6, 2.5 TB/s; 62,000 rows of 90 in f32 9.3 and 12.8).  Two
// forms:
//   own     heads of up to 32.  A lane takes a row, in pieces of 16 bytes (masked
//           logits as -infinity), and keeps it in LDS, where heads of any size
//           can be found by an index; up to four waves take the same rows and
//           share their heads.
//   shared  8 to 64 lanes, or a workgroup, take a head together, straight from
//           memory, eight logits a lane in registers; of longer heads the rest is
//           read again for each step.  A lane's loads are of one logit and one
//           byte of the mask, and bound it: 20 M bf16 logits with a mask in heads
//           of 33 to 2,000 36 to 41 us, 1.6 to 1.7 TB/s (62,000 rows of 90 in f32
//           2.4 TB/s, their gradients 3.4).
#include <cmath>

#include "../../include/carl_amd_ops.h"
#include "elem.h"
#include "reduce.h"
#include "status.h"

using namespace carl;

namespace {

constexpr int kMostHeads = CARL_ACTIONS_MAX_HEADS;

struct Args {
    int64_t rows;
    const void* logits;
    int64_t logitsRow;
    const uint8_t* mask;
    int64_t maskRow;
    const void* actions;
    int64_t actionsRow;
    float *logProb, *entropy;
    const float *dLogProb, *dEntropy;
    int64_t dLogProbStep, dEntropyStep;
    void* dLogits;
    const float* noise;
    int64_t noiseRow;
    int32_t* best;
    int32_t k, heads, wide;
    int32_t first[kMostHeads + 1];      // of each head's logits, and their number
};

enum { kLogProb = 0, kGradient = 1, kBest = 2 };

constexpr float kNone = -__builtin_inff();

// A row's actions; those of 64 bits that 32 do not hold are as good as the
// nearest that they do: below 0, or past every head.
struct RowActions {
    const void* at;
    bool wide;
    __device__ RowActions(const Args& a, int64_t row)
        : at(static_cast<const char*>(a.actions) + row * a.actionsRow * (a.wide ? 8 : 4)), wide(a.wide)
    {
    }
    __device__ int operator[](int head) const
    {
        if (!wide) return static_cast<const int32_t*>(at)[head];
        const int64_t v = static_cast<const int64_t*>(at)[head];
        return v < INT32_MIN ? INT32_MIN : v > INT32_MAX ? INT32_MAX : (int)v;
    }
};

// Keys as unsigned numbers in their order: 0 for what is not available, NaN
// above all, both zeros alike.
__device__ inline uint32_t keyOf(float key, float logit)
{
    if (logit == kNone) return 0;
    if (key != key) return 0xffffffffu;
    const uint32_t u = __float_as_uint(key + 0.0f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// The hardware's exponential, logarithm and reciprocal are good to a unit in
// the last place each; Z is at least 1 where anything is available.
__device__ inline float exponential(float x) { return __builtin_amdgcn_exp2f(x * 1.44269504088896341f); }

// The larger number; of a number and a (quiet) NaN the number.  fmaxf takes two
// instructions where it does not see what its argument is, the first to make
// signalling NaN quiet; here they stay NaN.
__device__ inline float larger(float a, float b)
{
    float r;
    asm("v_max_f32 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
    return r;
}

// The largest of a head's logits as the others are taken from: 0 where nothing
// is available (or all of it is NaN, which Z then tells).
__device__ inline float baseOf(float most) { return most == kNone ? 0.0f : most; }

// The shares in Z and A of a logit with d = x - base and e = exp(d): none of
// what is not available, NaN of a NaN.
__device__ inline void addTo(float& z, float& a, float d, float e)
{
    z += e;
    a = __builtin_fmaf(e, fmaxf(d, -1e30f), a);
}

// What follows from a head's m, Z and A.
struct Sums {
    float base, logZ, inverse, entropy;
    __device__ Sums(float base_, float z, float a) : base(base_)
    {
        const bool some = z != 0.0f;
        logZ = some ? __builtin_amdgcn_logf(z) * 0.693147180559945309f : 0.0f;
        inverse = __builtin_amdgcn_rcpf(z);
        entropy = some ? logZ - a * inverse : 0.0f;
    }
    __device__ float logProb(float x) const { return x == kNone ? kNone : x - base - logZ; }
    // of an action that may be none, or past the last
    __device__ float taken(int action, int size, float x) const
    {
        return action < 0 ? 0.0f : action >= size ? __builtin_nanf("") : logProb(x);
    }
};

// By a logit x with d = x - base and e = exp(d).
__device__ inline float gradient(const Sums& s, float x, float d, float e, bool taken, float dLogProb, float dEntropy)
{
    const float p = e * s.inverse;
    // (p is 0 where log p may be -infinity)
    const float g = dLogProb * ((taken ? 1.0f : 0.0f) - p) - dEntropy * (p * (fmaxf(d, -1e30f) - s.logZ + s.entropy));
    return x == kNone ? 0.0f : g;
}

// What an action leaves of its log-probability's gradient; nothing where there is none.
__device__ inline float shareOf(int action, int size, const float* given, float dLogProb)
{
    return !given || action < 0 ? 0.0f : action >= size ? __builtin_nanf("") : dLogProb;
}

// ---- own -------------------------------------------------------------------------

constexpr int kOwnHead = 32;

// Every kShare-th of a row's pieces of kE elements from the one numbered `part`
// on, 32 elements on their way at once: each(first element, piece).  A last piece
// that is not whole begins earlier, and its first elements come twice; rows
// shorter than a piece come one by one.
template <int kE, int kShare, typename Load, typename Each> __device__ inline void inPieces(int n, int part, Load&& load, Each&& each)
{
    if (n < kE) {
        for (int j = part; j < n; j += kShare) each(j, load(j, std::integral_constant<int, 1>()));
        return;
    }
    constexpr int kAtOnce = 32 / kE;
    for (int j0 = part * kE; j0 < n; j0 += kAtOnce * kShare * kE) {
        decltype(load(0, std::integral_constant<int, kE>())) piece[kAtOnce];
#pragma unroll
        for (int i = 0; i < kAtOnce; i++) {
            const int j = j0 + i * kShare * kE;
            if (j < n) piece[i] = load(j + kE <= n ? j : n - kE, std::integral_constant<int, kE>());
        }
#pragma unroll
        for (int i = 0; i < kAtOnce; i++) {
            const int j = j0 + i * kShare * kE;
            if (j < n) each(j + kE <= n ? j : n - kE, piece[i]);
        }
    }
}

template <typename X, int kN> __device__ inline vec<X, kN> loadVec(const X* p)
{
    vec<X, kN> r;
    __builtin_memcpy(&r, p, sizeof(X) * kN);
    return r;
}

template <typename T, int kE> struct Piece {
    vec<T, kE> x;
    uint32_t there[(kE + 3) / 4];       // bytes, four to a word until they are used
    vec<float, kE> noise;
};

constexpr int kAhead = 4;
struct Ahead {
    float x[kAhead];
    uint32_t key[kAhead];
    int action;
};

// kShare waves take the same 64 rows, each every kShare-th head of them.
template <typename T, int kWhat, bool kMasked, bool kNoisy, int kShare> __global__ __launch_bounds__(64 * kShare) void ownKernel(const Args a)
{
    constexpr int kE = 16 / sizeof(T);
    extern __shared__ float rows[];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int logits = a.first[a.heads], across = logits | 1;      // odd: the lanes' rows begin in different banks
    float* const own = rows + lane * across;
    uint32_t* const keys = reinterpret_cast<uint32_t*>(rows + 64 * across + kAhead + lane * across);
    float* const results = rows + 64 * across + kAhead + lane;      // of a head, log-probability and entropy, 64 apart
    const auto handOver = [&]() {
        if constexpr (kShare > 1) __syncthreads();
    };
    for (int64_t row0 = (int64_t)blockIdx.x * 64; row0 < a.rows; row0 += (int64_t)gridDim.x * 64) {
        // (rows past the last are the last one again; their results are not stored)
        const bool mine = row0 + lane < a.rows;
        const int64_t row = mine ? row0 + lane : a.rows - 1;
        const T* const from = static_cast<const T*>(a.logits) + row * a.logitsRow;
        const auto load = [&](int j, auto n) {
            Piece<T, n()> p;
            p.x = loadVec<T, n()>(from + j);
            if constexpr (kMasked) __builtin_memcpy(p.there, a.mask + row * a.maskRow + j, n());
            if constexpr (kNoisy) p.noise = loadVec<float, n()>(a.noise + row * a.noiseRow + j);
            return p;
        };
        inPieces<kE, kShare>(logits, wave, load, [&](int j, const auto& p) {
            constexpr int n = sizeof(p.x) / sizeof(T);
#pragma unroll
            for (int i = 0; i < n; i++) {
                float x = (float)p.x[i];
                if constexpr (kMasked) x = p.there[i / 4] >> i % 4 * 8 & 0xff ? x : kNone;
                own[j + i] = x;
                if constexpr (kNoisy) keys[j + i] = keyOf(x + p.noise[i], x);
                else if constexpr (kWhat == kBest) keys[j + i] = keyOf(x, x);
            }
        });
        float logProb = 0.0f, entropy = 0.0f, dLogProb = 0.0f, dEntropy = 0.0f;
        if constexpr (kWhat == kGradient) {
            if (a.dLogProb) dLogProb = a.dLogProb[row * a.dLogProbStep];
            if (a.dEntropy) dEntropy = a.dEntropy[row * a.dEntropyStep];
        }
        handOver();
        const RowActions actions(a, row);
        // a head's first logits (and keys) and its action are read while the head before it is computed
        Ahead ahead;
        const auto read = [&](int h) {
            // (a shorter head's come with what lies after it)
            const int j = a.first[h];
#pragma unroll
            for (int i = 0; i < kAhead; i++) {
                ahead.x[i] = own[j + i];
                if constexpr (kWhat == kBest) ahead.key[i] = keys[j + i];
            }
            if constexpr (kWhat != kBest) ahead.action = actions[h];
        };
        if (wave < a.heads) read(wave);
        for (int h = wave; h < a.heads; h += kShare) {
            const Ahead now = ahead;
            if (h + kShare < a.heads) read(h + kShare);
            float* const x = own + a.first[h];
            const int n = a.first[h + 1] - a.first[h];
            // short heads by their length, which is the same for all lanes (a condition for each logit: 26 and 32 us for 24 and 30)
            const auto compute = [&](auto few) {
                float most = kNone, z = 0.0f, sum = 0.0f, d[kAhead], e[kAhead];
#pragma unroll
                for (int i = 0; i < kAhead; i++)
                    if (i < few()) most = larger(most, now.x[i]);
                for (int j = kAhead; few() == kAhead && j < n; j++) most = larger(most, x[j]);
                const float base = baseOf(most);
#pragma unroll
                for (int i = 0; i < kAhead; i++)
                    if (i < few()) {
                        d[i] = now.x[i] - base;
                        e[i] = exponential(d[i]);
                        addTo(z, sum, d[i], e[i]);
                    }
                for (int j = kAhead; few() == kAhead && j < n; j++) addTo(z, sum, x[j] - base, exponential(x[j] - base));
                const Sums s(base, z, sum);
                if constexpr (kWhat == kBest) {
                    const uint32_t* const key = keys + a.first[h];
                    const int64_t at = (row * a.heads + h) * a.k;
                    uint32_t lastKey = 0xffffffffu;
                    int last = -1;
                    for (int i = 0; i < a.k; i++) {
                        uint32_t largest = 0;
                        int best = -1;
                        float picked = kNone;
                        const auto consider = [&](int j, uint32_t u, float v) {
                            if (u > largest && (u < lastKey || (u == lastKey && j > last))) {
                                largest = u;
                                best = j;
                                picked = v;
                            }
                        };
#pragma unroll
                        for (int j = 0; j < kAhead; j++)
                            if (j < n) consider(j, now.key[j], now.x[j]);
                        for (int j = kAhead; few() == kAhead && j < n; j++) consider(j, key[j], x[j]);
                        if (mine) {
                            a.best[at + i] = best;
                            a.logProb[at + i] = s.logProb(picked);
                        }
                        lastKey = largest;
                        last = best < 0 ? n : best;
                    }
                } else if constexpr (kWhat == kLogProb) {
                    const int action = now.action;
                    const float taken = s.taken(action, n, x[action >= 0 && action < n ? action : 0]);
                    if constexpr (kShare == 1) {
                        logProb += taken;
                        entropy += s.entropy;
                    } else {
                        results[h * 128] = taken;
                        results[h * 128 + 64] = s.entropy;
                    }
                } else {
                    const float share = shareOf(now.action, n, a.dLogProb, dLogProb);
#pragma unroll
                    for (int i = 0; i < kAhead; i++)
                        if (i < few()) x[i] = gradient(s, now.x[i], d[i], e[i], i == now.action, share, dEntropy);
                    for (int j = kAhead; few() == kAhead && j < n; j++)
                        x[j] = gradient(s, x[j], x[j] - base, exponential(x[j] - base), j == now.action, share, dEntropy);
                }
            };
            if (n == 1) compute(std::integral_constant<int, 1>());
            else if (n == 2) compute(std::integral_constant<int, 2>());
            else if (n == 3) compute(std::integral_constant<int, 3>());
            else compute(std::integral_constant<int, kAhead>());
        }
        handOver();
        if constexpr (kWhat == kLogProb) {
            if (wave == 0 && mine) {
                if constexpr (kShare > 1)
                    for (int h = 0; h < a.heads; h++) {
                        logProb += results[h * 128];
                        entropy += results[h * 128 + 64];
                    }
                a.logProb[row] = logProb;
                a.entropy[row] = entropy;
            }
        } else if constexpr (kWhat == kGradient) {
            T* const to = static_cast<T*>(a.dLogits) + row * logits;
            const auto read = [&](int j, auto n) {
                vec<T, n()> r;
#pragma unroll
                for (int i = 0; i < n(); i++) r[i] = (T)own[j + i];
                return r;
            };
            if (mine) inPieces<kE, kShare>(logits, wave, read, [&](int j, const auto& r) { __builtin_memcpy(to + j, &r, sizeof(r)); });
        }
        handOver();
    }
}

// ---- shared ----------------------------------------------------------------------

constexpr int kSharedThreads = 256, kHeld = 8;

// A group of lanes for each head of a row; a workgroup has whole rows, and adds
// up their heads' results in order.
template <typename T, int kWhat, bool kMasked, bool kNoisy, int kLanes>
__global__ __launch_bounds__(kSharedThreads) void sharedKernel(const Args a, int rowsOf, int longest)
{
    constexpr int kGroups = kSharedThreads / kLanes;
    __shared__ float results[2][kGroups > kMostHeads ? kGroups : kMostHeads], slots[kSharedThreads / 64];
    __shared__ uint32_t bits[kSharedThreads / 64];
    __shared__ int firsts[kMostHeads + 1];
    const int lane = threadIdx.x % kLanes, group = threadIdx.x / kLanes;
    if ((int)threadIdx.x <= a.heads) firsts[threadIdx.x] = a.first[threadIdx.x];
    __syncthreads();
    const float inHeads = 1.0f / (float)a.heads;
    for (int64_t row0 = (int64_t)blockIdx.x * rowsOf; row0 < a.rows; row0 += (int64_t)gridDim.x * rowsOf) {
        const int rows = a.rows - row0 < rowsOf ? (int)(a.rows - row0) : rowsOf;
        for (int unit = group; unit < rows * a.heads; unit += kGroups) {
            const int r = (int)(((float)unit + 0.5f) * inHeads), h = unit - r * a.heads;       // (units are fewer than 128)
            const int64_t row = row0 + r;
            const int first = firsts[h], n = firsts[h + 1] - first;
            const T* const from = static_cast<const T*>(a.logits) + row * a.logitsRow + first;
            const uint8_t* const mask = kMasked ? a.mask + row * a.maskRow + first : nullptr;
            const float* const noise = kNoisy ? a.noise + row * a.noiseRow + first : nullptr;
            // eight logits a lane in registers, all on their way at once
            T in[kHeld];
            uint8_t there[kHeld];
            float more[kHeld], held[kHeld];
#pragma unroll
            for (int i = 0; i < kHeld; i++) {
                const int j = i * kLanes + lane;
                if (i * kLanes < longest && j < n) {
                    in[i] = from[j];
                    if constexpr (kMasked) there[i] = mask[j];
                    if constexpr (kNoisy) more[i] = noise[j];
                }
            }
#pragma unroll
            for (int i = 0; i < kHeld; i++) {
                held[i] = i * kLanes + lane < n ? (float)in[i] : kNone;
                if constexpr (kMasked) held[i] = there[i] ? held[i] : kNone;
                if constexpr (kNoisy) more[i] += held[i];
            }
            const auto load = [&](int j) {
                const float x = (float)from[j];
                return !kMasked || mask[j] ? x : kNone;
            };
            // f(j, logit, key): the conditions on `longest` are the same for all lanes
            const auto each = [&](auto&& f) {
#pragma unroll
                for (int i = 0; i < kHeld; i++)
                    if (i * kLanes < longest) f(i * kLanes + lane, held[i], kNoisy ? more[i] : held[i]);
                for (int j = kHeld * kLanes + lane; j < n; j += kLanes) {
                    const float x = load(j);
                    f(j, x, kNoisy ? x + noise[j] : x);
                }
            };
            float most = kNone, z = 0.0f, sum = 0.0f;
            each([&](int, float x, float) { most = fmaxf(most, x); });
            const float base = baseOf(overRow<Most, kLanes>(most, slots));
            each([&](int, float x, float) { addTo(z, sum, x - base, exponential(x - base)); });
            const float zAll = overRow<Add, kLanes>(z, slots), sumAll = overRow<Add, kLanes>(sum, slots);
            const Sums s(base, zAll, sumAll);
            if constexpr (kWhat == kBest) {
                const int64_t at = (row * a.heads + h) * a.k;
                if (kLanes == kSharedThreads && a.k > 1) {
                    // a lane's keys lie in LDS and its best one in registers, and only the lane whose key was taken looks for its
                    // next one
                    extern __shared__ uint32_t keys[];
                    each([&](int j, float x, float key) {
                        if (j < n) keys[j] = keyOf(key, x);
                    });
                    uint32_t largest = 0;
                    int best = INT32_MAX;
                    const auto look = [&]() {
                        largest = 0;
                        best = INT32_MAX;
#pragma unroll 8
                        for (int j = lane; j < n; j += kLanes) {
                            const uint32_t u = keys[j];
                            best = u > largest ? j : best;
                            largest = u > largest ? u : largest;
                        }
                    };
                    look();
                    for (int i = 0; i < a.k; i++) {
                        const uint32_t most = overRow<Most, kLanes>(largest, bits);
                        const int taken = (int)overRow<Least, kLanes>((uint32_t)(largest == most ? best : INT32_MAX), bits);
                        // (of nothing that is left, the first lane)
                        if (taken == INT32_MAX ? lane == 0 : best == taken) {
                            a.best[at + i] = taken == INT32_MAX ? -1 : taken;
                            a.logProb[at + i] = s.logProb(taken == INT32_MAX ? kNone : load(taken));
                            if (taken != INT32_MAX) {
                                keys[taken] = 0;
                                look();
                            }
                        }
                    }
                } else {
                    uint32_t lastKey = 0xffffffffu;
                    int last = -1;
                    for (int i = 0; i < a.k; i++) {
                        uint32_t largest = 0;
                        int best = INT32_MAX;
                        float picked = kNone;
                        each([&](int j, float x, float key) {
                            const uint32_t u = keyOf(key, x);
                            if (u > largest && (u < lastKey || (u == lastKey && j > last))) {
                                largest = u;
                                best = j;
                                picked = x;
                            }
                        });
                        lastKey = overRow<Most, kLanes>(largest, bits);
                        last = (int)overRow<Least, kLanes>((uint32_t)(largest == lastKey ? best : INT32_MAX), bits);
                        // (of nothing that is left, the group's first lane)
                        if (last == INT32_MAX ? lane == 0 : best == last) {
                            a.best[at + i] = last == INT32_MAX ? -1 : best;
                            a.logProb[at + i] = s.logProb(picked);
                        }
                    }
                }
            } else {
                const int action = RowActions(a, row)[h];
                if constexpr (kWhat == kLogProb) {
                    const float own = s.taken(action, n, action >= 0 && action < n ? load(action) : 0.0f);
                    if (lane == 0 && a.heads == 1) {
                        a.logProb[row] = own;
                        a.entropy[row] = s.entropy;
                    } else if (lane == 0) {
                        results[0][unit] = own;
                        results[1][unit] = s.entropy;
                    }
                } else {
                    const float share = shareOf(action, n, a.dLogProb, a.dLogProb ? a.dLogProb[row * a.dLogProbStep] : 0.0f);
                    const float dEntropy = a.dEntropy ? a.dEntropy[row * a.dEntropyStep] : 0.0f;
                    T* const to = static_cast<T*>(a.dLogits) + row * a.first[a.heads] + first;
                    each([&](int j, float x, float) {
                        if (j < n) to[j] = (T)gradient(s, x, x - base, exponential(x - base), j == action, share, dEntropy);
                    });
                }
            }
        }
        if (kWhat == kLogProb && a.heads > 1) {
            __syncthreads();
            if ((int)threadIdx.x < rows) {
                float logProb = 0.0f, entropy = 0.0f;
                for (int h = 0; h < a.heads; h++) {
                    logProb += results[0][threadIdx.x * a.heads + h];
                    entropy += results[1][threadIdx.x * a.heads + h];
                }
                a.logProb[row0 + threadIdx.x] = logProb;
                a.entropy[row0 + threadIdx.x] = entropy;
            }
            __syncthreads();
        }
    }
}

constexpr int64_t kMostRows = (int64_t)1 << 40, kMostBlocks = 1 << 16;

template <typename T, int kWhat> void launch(const Args& a, hipStream_t stream)
{
    int longest = 0;
    for (int h = 0; h < a.heads; h++) longest = longest > a.first[h + 1] - a.first[h] ? longest : a.first[h + 1] - a.first[h];
    const int logits = a.first[a.heads];
    const auto blocks = [&](int rows) {
        const int64_t n = (a.rows + rows - 1) / rows;
        return dim3((unsigned)(n < kMostBlocks ? n : kMostBlocks));
    };
    using std::false_type, std::integral_constant, std::true_type;
    // A lane for each row of short heads where the rows fit LDS and are many, or short themselves (us, best actions and
    // log-probabilities, a lane for each row and lanes for each head: 5 heads of 16, 250,000 rows 61, 20 and 121, 82; 16,384 rows
    // 10.3, 6.4 and 9.8, 8.2; 34 rows 9.0, 5.2 and 3.9, 4.1).
    const int ownArray = 64 * (logits | 1) + kAhead;
    const int ownBytes = (ownArray + (kWhat == kBest ? ownArray : kWhat == kLogProb ? a.heads * 128 : 0)) * 4;
    const bool own = longest <= kOwnHead && ownBytes <= 65536 && (logits <= 32 || a.rows >= 16384);
    // Waves for its 64 rows (the simulator's heads, one, two and four waves: 34 rows 7.5, 5.3, 4.0 and 4.7, 3.9, 3.1; 131,072
    // 11.4, 10.0, 10.2 and 7.4, 6.5, 7.3; 1,048,576 59, 53, 53 and 22, 24, 28; 8 heads of 8, 262,144 rows 84, 53, 35 and 27, 21, 16).
    const int share = a.rows <= 65536 || logits > 32 ? 4 : a.heads > 1 && (kWhat == kBest || a.rows <= 200000) ? 2 : 1;
    // Lanes of a head by a sweep over 20 M logits (us, log-probabilities): heads of 33 8 lanes 40, 16 lanes 69; of 90 16 lanes 34;
    // of 200 32 lanes 34, 64 lanes 56; of 513 64 lanes 35, a workgroup 80; of 2,000 64 lanes 40, a workgroup 33 (34 rows: 9 and 5).
    // A workgroup's choice of several (its keys in LDS, 16,384 logits, 1 row, the best 64: 119 us, read again for each 1,099) is
    // quicker from 769 logits on, and from 513 for few heads (5 best, a workgroup and 64 lanes: 1,000 heads of 700 9.1 and 11.9,
    // 10,000 51 and 36; of 1,000 56 and 70).
    const bool together = kWhat == kBest && a.k > 1 && (longest > 768 || a.rows * a.heads <= 2048);
    const auto with = [&](auto masked, auto noisy) {
        const auto shared = [&](auto lanes) {
            const int groups = kSharedThreads / lanes(), rows = groups > a.heads ? groups / a.heads : 1;
            const int bytes = kWhat == kBest && lanes() == kSharedThreads && a.k > 1 ? longest * 4 : 0;
            sharedKernel<T, kWhat, masked(), noisy(), lanes()><<<blocks(rows), kSharedThreads, bytes, stream>>>(a, rows, longest);
        };
        if (own) {
            const auto with = [&](auto share) {
                ownKernel<T, kWhat, masked(), noisy(), share()><<<blocks(64), 64 * share(), ownBytes, stream>>>(a);
            };
            if (share == 4) with(integral_constant<int, 4>());
            else if (share == 2) with(integral_constant<int, 2>());
            else with(integral_constant<int, 1>());
        } else if (longest <= 64) shared(integral_constant<int, 8>());
        else if (longest <= 128) shared(integral_constant<int, 16>());
        else if (longest <= 256) shared(integral_constant<int, 32>());
        else if (longest <= (together ? 512 : 1024)) shared(integral_constant<int, 64>());
        else shared(integral_constant<int, kSharedThreads>());
    };
    if constexpr (kWhat == kBest) {
        if (a.noise) return a.mask ? with(true_type(), true_type()) : with(false_type(), true_type());
    }
    if (a.mask) with(true_type(), false_type());
    else with(false_type(), false_type());
}

template <int kWhat> int launch(int type, const Args& a, hipStream_t stream)
{
    if (type == CARL_OP_F32) launch<float, kWhat>(a, stream);
    else if (type == CARL_OP_BF16) launch<bf16, kWhat>(a, stream);
    else launch<f16, kWhat>(a, stream);
    return launched(kWhat == kBest ? "choice of actions" : "log-probabilities of actions");
}

int check(const carl_actions* p, Args& a)
{
    if (!p) return fail(CARL_ERR_VALUE, "null action argument");
    if (p->type != CARL_OP_F32 && p->type != CARL_OP_BF16 && p->type != CARL_OP_F16) return fail(CARL_ERR_TYPE, "unknown element type");
    if (p->rows < 0 || p->rows > kMostRows) return fail(CARL_ERR_VALUE, "rows are out of range");
    if (p->heads < 1 || p->heads > kMostHeads) return fail(CARL_ERR_VALUE, "heads must be in [1, 64]");
    if (!p->sizes) return fail(CARL_ERR_VALUE, "null head sizes");
    a = Args{ p->rows, p->logits, p->logits_row, p->mask, p->mask_row, p->actions, p->actions_row, p->log_prob, p->entropy,
              p->d_log_prob, p->d_entropy, p->d_log_prob_step, p->d_entropy_step, p->d_logits, p->noise, p->noise_row, p->best,
              p->k, p->heads, p->actions_wide, {} };
    for (int h = 0; h < p->heads; h++) {
        if (p->sizes[h] < 1 || p->sizes[h] > CARL_ACTIONS_MAX_LOGITS - a.first[h])
            return fail(CARL_ERR_VALUE, "head sizes must be at least 1, and 16,384 in all at most");
        a.first[h + 1] = a.first[h] + p->sizes[h];
    }
    return CARL_OK;
}

}  // namespace

extern "C" {

int carl_action_log_prob(const carl_actions* p, void* stream)
{
    Args a;
    if (int rc = check(p, a)) return rc;
    if (a.rows == 0) return CARL_OK;
    if (!a.logits || !a.actions || !a.logProb || !a.entropy) return fail(CARL_ERR_VALUE, "null action tensor");
    return launch<kLogProb>(p->type, a, (hipStream_t)stream);
}

int carl_action_log_prob_backward(const carl_actions* p, void* stream)
{
    Args a;
    if (int rc = check(p, a)) return rc;
    if (a.rows == 0) return CARL_OK;
    if (!a.logits || !a.actions || !a.dLogits) return fail(CARL_ERR_VALUE, "null action tensor");
    return launch<kGradient>(p->type, a, (hipStream_t)stream);
}

int carl_top_actions(const carl_actions* p, void* stream)
{
    Args a;
    if (int rc = check(p, a)) return rc;
    if (p->k < 1 || p->k > CARL_ACTIONS_MAX_K) return fail(CARL_ERR_VALUE, "k must be in [1, 64]");
    if (a.rows == 0) return CARL_OK;
    if (!a.logits || !a.best || !a.logProb) return fail(CARL_ERR_VALUE, "null action tensor");
    return launch<kBest>(p->type, a, (hipStream_t)stream);
}

}  // extern "C"
