// adamw.hip - one AdamW step over many tensors, moments in 32 or in 8 bits.
//
// Formulas, codes and orders of rounding: include/carl_amd_ops.h.  Every
// operation is one IEEE binary32 operation (no contraction, divisions and
// square roots correctly rounded), so that a plain restatement of the formulas
// gives the same bits, 8-bit codes included.
//
// What bounds it: memory.  An element's step reads parameter, gradient and two
// moments and writes all but the gradient, 28 bytes in float32 and 16 with
// 8-bit moments, against about 40 (110) operations.  A wave takes blocks of
// 256 elements, four neighbours a lane, so that every access of float32 is 16
// bytes a lane and a block's scale is one reduction over the wave; the loads
// of a wave's kRows blocks are all in flight before the first is used.
// Tensors are found by their first chunk in a table that travels in the
// launch's arguments (kMost tensors a launch, nothing is uploaded).  51 M
// elements with 32-bit moments: 271 us, 5.3 TB/s.
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>
#include <string>

#include "../../include/carl_amd_ops.h"
#include "elem.h"
#include "status.h"

using namespace carl;

namespace {

constexpr int kBlock = CARL_ADAMW_BLOCK;
constexpr int kThreads = 256, kWaves = 4;
constexpr int kMost = 60;                      // tensors a launch: its arguments stay under 4 KB
constexpr int64_t kMostElements = (int64_t)1 << 33, kMostChunks = 1 << 23;   // 2^31 threads a launch

struct Entry {
    void* p;
    const void* g;
    void* m;
    void* v;
    float* ms;
    float* vs;
    int64_t n;
    int32_t firstChunk;
    uint8_t pType, gType, wide, pad;
};

struct Table {
    Entry t[kMost];
    int32_t count;
};

struct Hyper {
    float b1, c1, b2, c2, keep, rate, root, eps;
    const float* gradScale;
};

template <typename T> __device__ inline f32x4 loadAs(const void* base, int64_t at, int have, bool wide)
{
    const T* x = static_cast<const T*>(base) + at;
    if (wide && have == 4) return toFloat<T, 4>(*reinterpret_cast<const vec<T, 4>*>(x));
    f32x4 r = { 0.f, 0.f, 0.f, 0.f };
    for (int j = 0; j < 4; j++)
        if (j < have) r[j] = (float)x[j];
    return r;
}

template <typename T> __device__ inline void storeAs(void* base, int64_t at, int have, bool wide, f32x4 r)
{
    T* x = static_cast<T*>(base) + at;
    if (wide && have == 4) {
        *reinterpret_cast<vec<T, 4>*>(x) = fromFloat<T, 4>(r);
        return;
    }
    for (int j = 0; j < 4; j++)
        if (j < have) x[j] = (T)r[j];
}

__device__ inline f32x4 load(const void* base, int type, int64_t at, int have, bool wide)
{
    if (type == CARL_OP_F32) return loadAs<float>(base, at, have, wide);
    if (type == CARL_OP_BF16) return loadAs<bf16>(base, at, have, wide);
    return loadAs<f16>(base, at, have, wide);
}

__device__ inline void store(void* base, int type, int64_t at, int have, bool wide, f32x4 r)
{
    if (type == CARL_OP_F32) storeAs<float>(base, at, have, wide, r);
    else if (type == CARL_OP_BF16) storeAs<bf16>(base, at, have, wide, r);
    else storeAs<f16>(base, at, have, wide, r);
}

// four codes of a lane in one word
__device__ inline uint32_t loadCodes(const void* base, int64_t at, int have, bool wide)
{
    const uint8_t* x = static_cast<const uint8_t*>(base) + at;
    if (wide && have == 4) return *reinterpret_cast<const uint32_t*>(x);
    uint32_t r = 0;
    for (int j = 0; j < 4; j++)
        if (j < have) r |= (uint32_t)x[j] << (8 * j);
    return r;
}

__device__ inline void storeCodes(void* base, int64_t at, int have, bool wide, uint32_t r)
{
    uint8_t* x = static_cast<uint8_t*>(base) + at;
    if (wide && have == 4) {
        *reinterpret_cast<uint32_t*>(x) = r;
        return;
    }
    for (int j = 0; j < 4; j++)
        if (j < have) x[j] = (uint8_t)(r >> (8 * j));
}

__device__ inline f32x4 decodeFirst(uint32_t codes, float scale)
{
    f32x4 r;
    for (int j = 0; j < 4; j++) {
        const float u = (float)(int8_t)(codes >> (8 * j)) * (1.0f / 127.0f);
        r[j] = u * fabsf(u) * scale;
    }
    return r;
}

__device__ inline f32x4 decodeSecond(uint32_t codes, float scale)
{
    f32x4 r;
    for (int j = 0; j < 4; j++) {
        float u = (float)(uint8_t)(codes >> (8 * j)) * (1.0f / 255.0f);
        u = u * u;
        r[j] = u * u * scale;
    }
    return r;
}

// The largest magnitude over the wave's block; NaN where any is not finite.
// Bit patterns of magnitudes order as unsigned numbers, infinity and NaN last.
template <int kPattern> __device__ inline uint32_t maxOver(uint32_t x)
{
    const uint32_t o = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, kPattern, 0xf, 0xf, false);
    return o > x ? o : x;
}

__device__ inline float blockScale(f32x4 x)
{
    uint32_t most = 0;
    for (int j = 0; j < 4; j++) {
        const uint32_t u = __float_as_uint(x[j]) & 0x7fffffffu;
        most = u > most ? u : most;
    }
    // within each row of 16 lanes, then over the four rows
    most = maxOver<0xb1>(most);      // quad_perm: 1 0 3 2
    most = maxOver<0x4e>(most);      // quad_perm: 2 3 0 1
    most = maxOver<0x141>(most);     // row_half_mirror
    most = maxOver<0x140>(most);     // row_mirror
    uint32_t all = 0;
    for (int r = 0; r < 64; r += 16) {
        const uint32_t row = (uint32_t)__builtin_amdgcn_readlane((int)most, r);
        all = row > all ? row : all;
    }
    return __uint_as_float(all >= 0x7f800000u ? 0x7fc00000u : all);
}

// Codes are defined by divisions and square roots that are correctly rounded,
// about 25 operations for a first and 40 for a second moment.  The quick ones
// here are good to a unit in the last place each: together they move 127 (255)
// times the root by less than 5e-5 (1e-4), so only a value that close to the
// border between two codes needs the others.  Scales far from 1, whose
// reciprocals would leave the normal numbers, always take them.
__device__ inline bool plainScale(float scale) { return scale > 0x1p-100f && scale < 0x1p100f; }

__device__ inline float byBorder(float y) { return fabsf(fabsf(y - rintf(y)) - 0.5f); }      // distance from half way

__device__ inline uint32_t encodeFirst(f32x4 x, float scale)
{
    uint32_t r = 0;
    const float inverse = __builtin_amdgcn_rcpf(scale);
    for (int j = 0; j < 4; j++) {
        float y = 127.0f * __builtin_amdgcn_sqrtf(fabsf(x[j]) * inverse);
        if (!plainScale(scale) || byBorder(y) < 2e-4f) y = 127.0f * sqrtf(fabsf(x[j]) / scale);
        const float c = rintf(y);
        const int code = scale > 0.0f ? (x[j] < 0.0f ? -(int)c : (int)c) : 0;
        r |= (uint32_t)(code & 0xff) << (8 * j);
    }
    return r;
}

__device__ inline uint32_t encodeSecond(f32x4 x, float scale)
{
    uint32_t r = 0;
    const float inverse = __builtin_amdgcn_rcpf(scale);
    for (int j = 0; j < 4; j++) {
        float y = 255.0f * __builtin_amdgcn_sqrtf(__builtin_amdgcn_sqrtf(x[j] * inverse));
        if (!plainScale(scale) || byBorder(y) < 4e-4f) y = 255.0f * sqrtf(sqrtf(x[j] / scale));
        const float c = fmaxf(rintf(y), 1.0f);
        const uint32_t code = x[j] > 0.0f && scale > 0.0f ? (uint32_t)c : 0u;
        r |= code << (8 * j);
    }
    return r;
}

// kRows blocks a wave: 4 where the step fills the GPU several times over, 1
// where a wave more is worth more than loads ahead.
template <int kBits, int kRows> __global__ __launch_bounds__(kThreads) void adamwKernel(const Table table, const Hyper h)
{
    int lo = 0, hi = table.count - 1;
    const int chunk = (int)blockIdx.x;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (table.t[mid].firstChunk <= chunk) lo = mid;
        else hi = mid - 1;
    }
    const Entry e = table.t[lo];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const bool wide = e.wide != 0;
    const int64_t first = ((int64_t)(chunk - e.firstChunk) * kRows * kWaves + wave) * kBlock;

    f32x4 p[kRows], g[kRows], m[kRows], v[kRows];
    uint32_t mc[kRows], vc[kRows];
    float ms[kRows], vs[kRows];
#pragma unroll
    for (int i = 0; i < kRows; i++) {
        const int64_t block = first + (int64_t)i * kWaves * kBlock, at = block + lane * 4;
        const int have = at >= e.n ? 0 : e.n - at < 4 ? (int)(e.n - at) : 4;
        p[i] = load(e.p, e.pType, at, have, wide);
        g[i] = load(e.g, e.gType, at, have, wide);
        if constexpr (kBits == 8) {
            mc[i] = loadCodes(e.m, at, have, wide);
            vc[i] = loadCodes(e.v, at, have, wide);
            ms[i] = block < e.n ? e.ms[block / kBlock] : 0.0f;
            vs[i] = block < e.n ? e.vs[block / kBlock] : 0.0f;
        } else {
            m[i] = load(e.m, CARL_OP_F32, at, have, wide);
            v[i] = load(e.v, CARL_OP_F32, at, have, wide);
        }
    }
    const float gs = h.gradScale ? *h.gradScale : 1.0f;
#pragma unroll
    for (int i = 0; i < kRows; i++) {
        const int64_t block = first + (int64_t)i * kWaves * kBlock, at = block + lane * 4;
        const int have = at >= e.n ? 0 : e.n - at < 4 ? (int)(e.n - at) : 4;
        if constexpr (kBits == 8) {
            m[i] = decodeFirst(mc[i], ms[i]);
            v[i] = decodeSecond(vc[i], vs[i]);
        }
        for (int j = 0; j < 4; j++) {
            const float x = h.gradScale ? g[i][j] * gs : g[i][j];
            m[i][j] = m[i][j] * h.b1 + x * h.c1;
            v[i][j] = v[i][j] * h.b2 + (x * x) * h.c2;
            const float root = sqrtf(v[i][j]) * h.root + h.eps;
            p[i][j] = p[i][j] * h.keep - (m[i][j] * h.rate) / root;
        }
        store(e.p, e.pType, at, have, wide, p[i]);
        if constexpr (kBits == 8) {
            // lanes past the tensor's end hold zeros (a NaN scale aside, which
            // is the block's own): they never raise a scale
            if (block >= e.n) continue;
            const float s = blockScale(m[i]), r = blockScale(v[i]);
            storeCodes(e.m, at, have, wide, encodeFirst(m[i], s));
            storeCodes(e.v, at, have, wide, encodeSecond(v[i], r));
            if (lane == 0) {
                e.ms[block / kBlock] = s;
                e.vs[block / kBlock] = r;
            }
        } else {
            store(e.m, CARL_OP_F32, at, have, wide, m[i]);
            store(e.v, CARL_OP_F32, at, have, wide, v[i]);
        }
    }
}

__global__ __launch_bounds__(kThreads) void decodeKernel(const int8_t* m, const float* ms, const uint8_t* v,
                                                         const float* vs, int64_t n, float* mOut, float* vOut, bool wide)
{
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int64_t block = (int64_t)blockIdx.x * kWaves + wave, at = block * kBlock + lane * 4;
    if (at >= n) return;
    const int have = n - at < 4 ? (int)(n - at) : 4;
    storeAs<float>(mOut, at, have, wide, decodeFirst(loadCodes(m, at, have, wide), ms[block]));
    storeAs<float>(vOut, at, have, wide, decodeSecond(loadCodes(v, at, have, wide), vs[block]));
}

__global__ __launch_bounds__(kThreads) void encodeKernel(const float* m, const float* v, int64_t n, int8_t* mOut,
                                                         float* ms, uint8_t* vOut, float* vs, bool wide)
{
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int64_t block = (int64_t)blockIdx.x * kWaves + wave, at = block * kBlock + lane * 4;
    if (block * kBlock >= n) return;
    const int have = at >= n ? 0 : n - at < 4 ? (int)(n - at) : 4;
    const f32x4 a = loadAs<float>(m, at, have, wide), b = loadAs<float>(v, at, have, wide);
    const float s = blockScale(a), r = blockScale(b);
    storeCodes(mOut, at, have, wide, encodeFirst(a, s));
    storeCodes(vOut, at, have, wide, encodeSecond(b, r));
    if (lane == 0) {
        ms[block] = s;
        vs[block] = r;
    }
}

bool aligned(const void* p, int bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

int bytesOf(int type) { return type == CARL_OP_F32 ? 4 : 2; }

int checkType(int type)
{
    if (type != CARL_OP_F32 && type != CARL_OP_BF16 && type != CARL_OP_F16) return fail(CARL_ERR_TYPE, "unknown element type");
    return CARL_OK;
}

template <int kBits> void launch(bool many, int64_t chunks, hipStream_t stream, const Table& table, const Hyper& h)
{
    if (many) adamwKernel<kBits, 4><<<dim3((unsigned)chunks), kThreads, 0, stream>>>(table, h);
    else adamwKernel<kBits, 1><<<dim3((unsigned)chunks), kThreads, 0, stream>>>(table, h);
}

}  // namespace

extern "C" {

int carl_adamw_step(const carl_adamw_tensor* tensors, int count, const carl_adamw* hyper, void* stream)
{
    if (!hyper || (count > 0 && !tensors)) return fail(CARL_ERR_VALUE, "null AdamW argument");
    if (count < 0) return fail(CARL_ERR_VALUE, "count must be non-negative");
    if (hyper->bits != 8 && hyper->bits != 32) return fail(CARL_ERR_VALUE, "moments must have 8 or 32 bits");
    if (hyper->step < 1) return fail(CARL_ERR_VALUE, "step must be at least 1");
    const auto part = [](double x) { return x >= 0.0 && x < 1.0; };
    if (!part(hyper->beta1) || !part(hyper->beta2)) return fail(CARL_ERR_VALUE, "betas must be in [0, 1)");
    const auto amount = [](double x) { return x >= 0.0 && std::isfinite(x); };
    if (!amount(hyper->lr)) return fail(CARL_ERR_VALUE, "lr must be finite and non-negative");
    if (!amount(hyper->eps)) return fail(CARL_ERR_VALUE, "eps must be finite and non-negative");
    if (!amount(hyper->weight_decay)) return fail(CARL_ERR_VALUE, "weight_decay must be finite and non-negative");
    const bool eight = hyper->bits == 8;
    int64_t total = 0;
    for (int i = 0; i < count; i++) {
        const carl_adamw_tensor& t = tensors[i];
        if (t.n < 0 || t.n > kMostElements) return fail(CARL_ERR_VALUE, "a tensor's size is out of range");
        if (int rc = checkType(t.param_type)) return rc;
        if (int rc = checkType(t.grad_type)) return rc;
        if (t.n == 0) continue;
        if (!t.param || !t.grad || !t.exp_avg || !t.exp_avg_sq) return fail(CARL_ERR_VALUE, "null AdamW tensor");
        if (eight && (!t.exp_avg_scale || !t.exp_avg_sq_scale)) return fail(CARL_ERR_VALUE, "8-bit moments need their scales");
        total += t.n;
    }

    Hyper h;
    h.b1 = (float)hyper->beta1;
    h.c1 = (float)(1.0 - hyper->beta1);
    h.b2 = (float)hyper->beta2;
    h.c2 = (float)(1.0 - hyper->beta2);
    h.keep = (float)(1.0 - hyper->lr * hyper->weight_decay);
    h.rate = (float)(hyper->lr / (1.0 - std::pow(hyper->beta1, (double)hyper->step)));
    h.root = (float)(1.0 / std::sqrt(1.0 - std::pow(hyper->beta2, (double)hyper->step)));
    h.eps = (float)hyper->eps;
    h.gradScale = hyper->grad_scale;

    const bool many = total > (int64_t)4 << 20;
    const int64_t perChunk = (int64_t)kBlock * kWaves * (many ? 4 : 1);
    Table table;
    table.count = 0;
    int64_t chunks = 0;
    const auto flush = [&]() {
        if (table.count == 0) return (int)CARL_OK;
        if (eight) launch<8>(many, chunks, (hipStream_t)stream, table, h);
        else launch<32>(many, chunks, (hipStream_t)stream, table, h);
        table.count = 0;
        chunks = 0;
        return launched("AdamW step");
    };
    for (int i = 0; i < count; i++) {
        const carl_adamw_tensor& t = tensors[i];
        if (t.n == 0) continue;
        const int64_t own = (t.n + perChunk - 1) / perChunk;
        if (table.count == kMost || chunks + own > kMostChunks)
            if (int rc = flush()) return rc;
        const bool wide = aligned(t.param, 4 * bytesOf(t.param_type)) && aligned(t.grad, 4 * bytesOf(t.grad_type))
                       && aligned(t.exp_avg, eight ? 4 : 16) && aligned(t.exp_avg_sq, eight ? 4 : 16);
        table.t[table.count++] = Entry{ t.param, t.grad, t.exp_avg, t.exp_avg_sq, t.exp_avg_scale, t.exp_avg_sq_scale, t.n,
                                        (int32_t)chunks, (uint8_t)t.param_type, (uint8_t)t.grad_type, (uint8_t)wide, 0 };
        chunks += own;
    }
    return flush();
}

int carl_adamw_decode(const int8_t* m, const float* ms, const uint8_t* v, const float* vs, int64_t n, float* mOut,
                      float* vOut, void* stream)
{
    if (n < 0 || n > kMostElements) return fail(CARL_ERR_VALUE, "a tensor's size is out of range");
    if (n == 0) return CARL_OK;
    if (!m || !ms || !v || !vs || !mOut || !vOut) return fail(CARL_ERR_VALUE, "null moment");
    const bool wide = aligned(m, 4) && aligned(v, 4) && aligned(mOut, 16) && aligned(vOut, 16);
    const int64_t blocks = (n + kBlock * kWaves - 1) / (kBlock * kWaves);
    decodeKernel<<<dim3((unsigned)blocks), kThreads, 0, (hipStream_t)stream>>>(m, ms, v, vs, n, mOut, vOut, wide);
    return launched("moment decoding");
}

int carl_adamw_encode(const float* m, const float* v, int64_t n, int8_t* mOut, float* ms, uint8_t* vOut, float* vs,
                      void* stream)
{
    if (n < 0 || n > kMostElements) return fail(CARL_ERR_VALUE, "a tensor's size is out of range");
    if (n == 0) return CARL_OK;
    if (!m || !v || !mOut || !ms || !vOut || !vs) return fail(CARL_ERR_VALUE, "null moment");
    const bool wide = aligned(m, 16) && aligned(v, 16) && aligned(mOut, 4) && aligned(vOut, 4);
    const int64_t blocks = (n + kBlock * kWaves - 1) / (kBlock * kWaves);
    encodeKernel<<<dim3((unsigned)blocks), kThreads, 0, (hipStream_t)stream>>>(m, v, n, mOut, ms, vOut, vs, wide);
    return launched("moment encoding");
}

}  // extern "C"
