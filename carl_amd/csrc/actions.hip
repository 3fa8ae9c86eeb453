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
// one head's steps.  Two forms:
//   staged  rows of 2 to 64 logits in heads of up to 32.  A wave takes 64 rows,
//           brings them into LDS (masked logits as -infinity) with reads that
//           run on through the rows, and each lane works on a row of its own;
//           gradients go back the same way.
//   shared  16 or 64 lanes take a row together, straight from memory, eight
//           logits of a head a lane in registers; of longer heads the rest is
//           read again for each step.
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
    int32_t k, heads, wide, inOne;      // inOne: 2^32 / logits, rounded up
    int32_t first[kMostHeads + 1];      // of each head's logits, and their number
};

enum { kLogProb = 0, kGradient = 1, kBest = 2 };

constexpr float kNone = -__builtin_inff();

__device__ inline int64_t actionOf(const Args& a, int64_t row, int head)
{
    const int64_t at = row * a.actionsRow + head;
    return a.wide ? static_cast<const int64_t*>(a.actions)[at] : (int64_t)static_cast<const int32_t*>(a.actions)[at];
}

// Keys as unsigned numbers in their order: 0 for what is not available, NaN
// above all, both zeros alike.
__device__ inline uint32_t keyOf(float key, float logit)
{
    if (logit == kNone) return 0;
    if (key != key) return 0xffffffffu;
    const uint32_t u = __float_as_uint(key + 0.0f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// A head's m, Z and A, from which the rest follows.
struct Sums {
    float most, logZ, inverse, entropy;
    __device__ Sums(float m, float z, float a)
        : most(m), logZ(z == 0.0f ? 0.0f : logf(z)), inverse(1.0f / z), entropy(z == 0.0f ? 0.0f : logZ - a / z)
    {
        // (z is at least 1 where anything is available, and 0 where nothing is)
    }
    __device__ float logProb(float x) const { return x == kNone ? kNone : x - most - logZ; }
    // of an action that may be none, or past the last
    __device__ float taken(int64_t action, int size, float x) const
    {
        return action < 0 ? 0.0f : action >= size ? __builtin_nanf("") : logProb(x);
    }
};

// x's shares of Z and A.
__device__ inline void addTo(float& z, float& a, float x, float most)
{
    if (x == kNone) return;
    const float d = x - most, e = expf(d);
    z += e;
    a += e > 0.0f ? e * d : 0.0f;
}

__device__ inline float gradient(const Sums& s, float x, bool taken, float dLogProb, float dEntropy)
{
    if (x == kNone) return 0.0f;
    const float d = x - s.most, p = expf(d) * s.inverse;
    return dLogProb * ((taken ? 1.0f : 0.0f) - p) - dEntropy * (p > 0.0f ? p * (d - s.logZ + s.entropy) : p);
}

// What an action leaves of its log-probability's gradient.
__device__ inline float shareOf(int64_t action, int size, float dLogProb)
{
    return action < 0 ? 0.0f : action >= size ? __builtin_nanf("") : dLogProb;
}

// ---- staged ----------------------------------------------------------------------

constexpr int kStagedLogits = 64, kStagedHead = 32;

template <typename T, int kWhat> __global__ __launch_bounds__(64) void stagedKernel(const Args a)
{
    extern __shared__ float staged[];
    const int lane = threadIdx.x, logits = a.first[a.heads], across = logits | 1;      // odd: a lane's row starts in a bank of its own
    uint32_t* const keys = reinterpret_cast<uint32_t*>(staged + 64 * across);
    for (int64_t row0 = (int64_t)blockIdx.x * 64; row0 < a.rows; row0 += (int64_t)gridDim.x * 64) {
        const int rows = a.rows - row0 < 64 ? (int)(a.rows - row0) : 64;
        const T* const from = static_cast<const T*>(a.logits) + row0 * a.logitsRow;
        for (int e = lane; e < rows * logits; e += 64) {
            const int row = (int)__umulhi((uint32_t)e, (uint32_t)a.inOne), j = e - row * logits;
            const bool there = !a.mask || a.mask[(row0 + row) * a.maskRow + j];
            const float x = there ? (float)from[row * a.logitsRow + j] : kNone;
            staged[row * across + j] = x;
            if constexpr (kWhat == kBest) keys[row * across + j] = keyOf(a.noise ? x + a.noise[(row0 + row) * a.noiseRow + j] : x, x);
        }
        __syncthreads();
        if (lane < rows) {
            const int64_t row = row0 + lane;
            float* const own = staged + lane * across;
            float logProb = 0.0f, entropy = 0.0f, dLogProb = 0.0f, dEntropy = 0.0f;
            if constexpr (kWhat == kGradient) {
                if (a.dLogProb) dLogProb = a.dLogProb[row * a.dLogProbStep];
                if (a.dEntropy) dEntropy = a.dEntropy[row * a.dEntropyStep];
            }
            for (int h = 0; h < a.heads; h++) {
                float* const x = own + a.first[h];
                const int n = a.first[h + 1] - a.first[h];
                float most = kNone, z = 0.0f, sum = 0.0f;
                for (int j = 0; j < n; j++) most = fmaxf(most, x[j]);
                for (int j = 0; j < n; j++) addTo(z, sum, x[j], most);
                const Sums s(most, z, sum);
                if constexpr (kWhat == kBest) {
                    const uint32_t* const key = keys + lane * across + a.first[h];
                    const int64_t at = (row * a.heads + h) * a.k;
                    uint32_t lastKey = 0xffffffffu;
                    int last = -1;
                    for (int i = 0; i < a.k; i++) {
                        uint32_t most = 0;
                        int best = -1;
                        for (int j = 0; j < n; j++) {
                            const uint32_t u = key[j];
                            if (u > most && (u < lastKey || (u == lastKey && j > last))) {
                                most = u;
                                best = j;
                            }
                        }
                        a.best[at + i] = best;
                        a.logProb[at + i] = best < 0 ? kNone : s.logProb(x[best]);
                        lastKey = most;
                        last = best < 0 ? n : best;
                    }
                } else {
                    const int64_t action = actionOf(a, row, h);
                    const bool within = action >= 0 && action < n;
                    if constexpr (kWhat == kLogProb) {
                        logProb += s.taken(action, n, within ? x[action] : 0.0f);
                        entropy += s.entropy;
                    } else {
                        const float share = shareOf(action, n, dLogProb);
                        for (int j = 0; j < n; j++) x[j] = gradient(s, x[j], j == action, share, dEntropy);
                    }
                }
            }
            if constexpr (kWhat == kLogProb) {
                a.logProb[row] = logProb;
                a.entropy[row] = entropy;
            }
        }
        __syncthreads();
        if constexpr (kWhat == kGradient) {
            T* const to = static_cast<T*>(a.dLogits) + row0 * logits;
            for (int e = lane; e < rows * logits; e += 64) {
                const int row = (int)__umulhi((uint32_t)e, (uint32_t)a.inOne), j = e - row * logits;
                to[e] = (T)staged[row * across + j];
            }
            __syncthreads();
        }
    }
}

// ---- shared ----------------------------------------------------------------------

template <typename T, int kWhat, int kLanes> __global__ __launch_bounds__(256) void sharedKernel(const Args a)
{
    constexpr int kHeld = 8, kGroups = 256 / kLanes;
    const int lane = threadIdx.x % kLanes;
    for (int64_t row = (int64_t)blockIdx.x * kGroups + threadIdx.x / kLanes; row < a.rows; row += (int64_t)gridDim.x * kGroups) {
        float logProb = 0.0f, entropy = 0.0f, dLogProb = 0.0f, dEntropy = 0.0f;
        if constexpr (kWhat == kGradient) {
            if (a.dLogProb) dLogProb = a.dLogProb[row * a.dLogProbStep];
            if (a.dEntropy) dEntropy = a.dEntropy[row * a.dEntropyStep];
        }
        for (int h = 0; h < a.heads; h++) {
            const int first = a.first[h], n = a.first[h + 1] - first;
            const T* const from = static_cast<const T*>(a.logits) + row * a.logitsRow + first;
            const uint8_t* const mask = a.mask ? a.mask + row * a.maskRow + first : nullptr;
            const auto load = [&](int j) { return j < n && (!mask || mask[j]) ? (float)from[j] : kNone; };
            float held[kHeld];
#pragma unroll
            for (int i = 0; i < kHeld; i++) held[i] = load(i * kLanes + lane);
            const auto each = [&](auto&& f) {
#pragma unroll
                for (int i = 0; i < kHeld; i++) f(i * kLanes + lane, held[i]);
                for (int j = kHeld * kLanes + lane; j < n; j += kLanes) f(j, load(j));
            };
            float most = kNone, z = 0.0f, sum = 0.0f;
            each([&](int, float x) { most = fmaxf(most, x); });
            most = overLanes<Most, kLanes>(most);
            each([&](int, float x) { addTo(z, sum, x, most); });
            const Sums s(most, overLanes<Add, kLanes>(z), overLanes<Add, kLanes>(sum));
            if constexpr (kWhat == kBest) {
                const float* const noise = a.noise ? a.noise + row * a.noiseRow + first : nullptr;
                const int64_t at = (row * a.heads + h) * a.k;
                uint64_t last = 0;
                for (int i = 0; i < a.k; i++) {
                    // key, then the lower index; 0 for none
                    uint64_t best = 0;
                    each([&](int j, float x) {
                        const uint64_t u = keyOf(noise && x != kNone ? x + noise[j] : x, x);
                        const uint64_t own = u << 32 | (uint32_t)~j;
                        if (u && (i == 0 || own < last) && own > best) best = own;
                    });
                    for (int d = 1; d < kLanes; d *= 2) best = Most::of(best, (uint64_t)__shfl_xor((unsigned long long)best, d));
                    if (lane == 0) {
                        const int j = (int)~(uint32_t)best;
                        a.best[at + i] = best ? j : -1;
                        a.logProb[at + i] = best ? s.logProb(load(j)) : kNone;
                    }
                    last = best;
                }
            } else {
                const int64_t action = actionOf(a, row, h);
                if constexpr (kWhat == kLogProb) {
                    logProb += s.taken(action, n, action >= 0 && action < n ? load((int)action) : 0.0f);
                    entropy += s.entropy;
                } else {
                    const float share = shareOf(action, n, dLogProb);
                    T* const to = static_cast<T*>(a.dLogits) + row * a.first[a.heads] + first;
                    each([&](int j, float x) {
                        if (j < n) to[j] = (T)gradient(s, x, j == action, share, dEntropy);
                    });
                }
            }
        }
        if (kWhat == kLogProb && lane == 0) {
            a.logProb[row] = logProb;
            a.entropy[row] = entropy;
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
    if (logits > 1 && logits <= kStagedLogits && longest <= kStagedHead) {
        const int bytes = 64 * (logits | 1) * 4 * (kWhat == kBest ? 2 : 1);
        stagedKernel<T, kWhat><<<blocks(64), 64, bytes, stream>>>(a);
    } else if (longest <= 128) sharedKernel<T, kWhat, 16><<<blocks(16), 256, 0, stream>>>(a);
    else sharedKernel<T, kWhat, 64><<<blocks(4), 256, 0, stream>>>(a);
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
              p->k, p->heads, p->actions_wide, 0, {} };
    for (int h = 0; h < p->heads; h++) {
        if (p->sizes[h] < 1 || p->sizes[h] > CARL_ACTIONS_MAX_LOGITS - a.first[h])
            return fail(CARL_ERR_VALUE, "head sizes must be at least 1, and 16,384 in all at most");
        a.first[h + 1] = a.first[h] + p->sizes[h];
    }
    a.inOne = (int32_t)(uint32_t)((((uint64_t)1 << 32) + a.first[p->heads] - 1) / a.first[p->heads]);
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
