// norm.hip - root-mean-square norm with the addition before it, its gradients,
// and rows in 8 bits.
//
//   s = x + residual          u = s / sqrt(mean(s^2) + eps)          y = u w
//   d = r (g - u mean(g u)) + dsum     with g = dy w, r = 1 / sqrt(mean(s^2) + eps)
//   dw = sum over rows of dy u
//   codes of t = s w: m = max |t|, code = rint(t (127 / m)), scale = (m / 127) r
// The factor r cancels in the codes, so they come from s and w alone, with one
// rounding a step: whatever the order of the sum of squares, the same codes.
//
// What bounds it: memory.  A row's elements stay in registers between the
// reduction and the output, so each is read and written once, in pieces of 16
// bytes.  48,828 bf16 rows of 2,048: 69 us (5.8 TB/s), with the addition 135
// (5.9), backward 163 (4.9), to codes 46 (6.6).  Of all shapes only the gradients
// of more than 8,192 float32 elements run out of registers, by three a lane (2,000
// rows of 16,384 95 us, 4.1 TB/s; 4,000 of 8,192 87, 4.5).
// The sum s is rounded to the elements' type once, as it is kept, and the norm
// is that of the rounded sum: the backward pass reads it and needs nothing else.
#include <algorithm>
#include <cmath>

#include "../../include/carl_amd_ops.h"
#include "elem.h"
#include "reduce.h"
#include "status.h"

using namespace carl;

namespace {

enum { kPlain = 0, kNormCodes = 1, kRowCodes = 2 };

struct NormArgs {
    const void *x, *residual, *weight;
    int64_t xRow, residualRow, rows;
    int32_t width;
    float eps;
    void *sum, *y;
    int8_t* codes;
    int64_t codesRow;
    float* scale;
};

struct NormGradArgs {
    const void *s, *dy, *dsum, *weight;
    int64_t sRow, dyRow, dsumRow, rows;
    int32_t width;
    float eps;
    void* dx;
    void* dw;          // written by a launch of one workgroup
    float* part;       // [workgroups, width], of a launch of more
};

// Squares of values this large add up to less than float32's largest; of rows
// whose do not, and of none else, the squares are those of 2^-80 times the values.
constexpr float kMostSquares = 0x1p120f, kSmaller = 0x1p-80f;
constexpr float kLeast = 0x1p-100f;       // a row's largest magnitude counts as this much at least

// A row's piece of 16 bytes at element `at`, from any address.  The last one
// begins earlier where it would not be whole, at the row's end minus a piece:
// its first elements are the piece's before it, too, which get the same values
// from both, and which dupOf() keeps out of the sums.  Rows shorter than a piece
// are filled up with zeros.
template <typename T> constexpr int kOf = 16 / sizeof(T);

template <typename T> __device__ inline int dupOf(int at, int width)
{
    const int have = width - at;
    return have > 0 && have < kOf<T> && width >= kOf<T> ? kOf<T> - have : 0;
}

template <typename T> __device__ inline vec<T, kOf<T>> loadPiece(const T* row, int at, int width)
{
    vec<T, kOf<T>> r = {};
    if (at >= width) return r;
    if (width >= kOf<T>) __builtin_memcpy(&r, row + (at + kOf<T> <= width ? at : width - kOf<T>), 16);
    else
#pragma unroll
        for (int j = 0; j < kOf<T>; j++) r[j] = j < width ? row[j] : T(0);
    return r;
}

template <typename X, int kN> __device__ inline void storePiece(X* row, int at, int width, vec<X, kN> r)
{
    if (at >= width) return;
    if (width >= kN) __builtin_memcpy(row + (at + kN <= width ? at : width - kN), &r, sizeof(X) * kN);
    else
#pragma unroll
        for (int j = 0; j < kN; j++)
            if (j < width) row[j] = r[j];
}

template <typename T, int kKind, int kLanes, int kPieces>
__global__ __launch_bounds__((kLanes < 128 ? 256 : kLanes)) void normKernel(const NormArgs a)
{
    constexpr int kE = 16 / sizeof(T), kThreads = kLanes < 128 ? 256 : kLanes, kGroups = kThreads / kLanes;
    __shared__ float slots[kThreads / 64];
    __shared__ uint32_t bits[kThreads / 64];
    const int lane = threadIdx.x % kLanes;
    const bool tail = a.width % kE != 0;
    vec<float, kE> w[kPieces];
    if constexpr (kKind != kRowCodes)
#pragma unroll
        for (int p = 0; p < kPieces; p++) {
            const int at = (p * kLanes + lane) * kE;
            w[p] = toFloat<T, kE>(loadPiece(static_cast<const T*>(a.weight), at, a.width));
        }
    for (int64_t row = (int64_t)blockIdx.x * kGroups + threadIdx.x / kLanes; row < a.rows; row += (int64_t)gridDim.x * kGroups) {
        vec<float, kE> s[kPieces];
        vec<T, kE> in[kPieces], more[kPieces];
#pragma unroll
        for (int p = 0; p < kPieces; p++) {
            const int at = (p * kLanes + lane) * kE;
            in[p] = loadPiece(static_cast<const T*>(a.x) + row * a.xRow, at, a.width);
            if (kKind != kRowCodes && a.residual) more[p] = loadPiece(static_cast<const T*>(a.residual) + row * a.residualRow, at, a.width);
        }
#pragma unroll
        for (int p = 0; p < kPieces; p++) {
            s[p] = toFloat<T, kE>(in[p]);
            if (kKind != kRowCodes && a.residual) {
                const int at = (p * kLanes + lane) * kE;
                const auto kept = fromFloat<T, kE>(s[p] + toFloat<T, kE>(more[p]));
                storePiece<T, kE>(static_cast<T*>(a.sum) + row * a.width, at, a.width, kept);
                s[p] = toFloat<T, kE>(kept);
            }
        }
        float r = 1.0f;
        if constexpr (kKind != kRowCodes) {
            float squares, factor = 1.0f;
            const auto sumUp = [&]() {
                squares = 0.0f;
#pragma unroll
                for (int p = 0; p < kPieces; p++) {
                    const int dup = tail ? dupOf<T>((p * kLanes + lane) * kE, a.width) : 0;
#pragma unroll
                    for (int j = 0; j < kE; j++) squares += j < dup ? 0.0f : s[p][j] * s[p][j];
                }
                squares = overRow<Add, kLanes>(squares, slots);
            };
            sumUp();
            if (!(squares < kMostSquares)) {
                factor = kSmaller;
#pragma unroll
                for (int p = 0; p < kPieces; p++) s[p] *= factor;
                sumUp();
            }
            r = 1.0f / sqrtf(squares / (float)a.width + a.eps * factor * factor);
        }
        if constexpr (kKind == kPlain) {
#pragma unroll
            for (int p = 0; p < kPieces; p++) {
                const int at = (p * kLanes + lane) * kE;
                storePiece<T, kE>(static_cast<T*>(a.y) + row * a.width, at, a.width, fromFloat<T, kE>(s[p] * r * w[p]));
            }
        } else {
            // bit patterns of magnitudes order as unsigned numbers, infinity and NaN last
            uint32_t most = 0;
#pragma unroll
            for (int p = 0; p < kPieces; p++) {
                if constexpr (kKind == kNormCodes) s[p] *= w[p];
#pragma unroll
                for (int j = 0; j < kE; j++) most = Most::of(most, __float_as_uint(s[p][j]) & 0x7fffffffu);
            }
            most = overRow<Most, kLanes>(most, bits);
            const bool finite = most < 0x7f800000u;
            const float m = fmaxf(__uint_as_float(most), kLeast), inverse = finite ? 127.0f / m : 0.0f;
            if (lane == 0) a.scale[row] = finite ? m / 127.0f * r : __uint_as_float(0x7fc00000u);
#pragma unroll
            for (int p = 0; p < kPieces; p++) {
                vec<int8_t, kE> code;
#pragma unroll
                for (int j = 0; j < kE; j++) code[j] = finite ? (int8_t)(int)rintf(s[p][j] * inverse) : (int8_t)0;
                storePiece<int8_t, kE>(a.codes + row * a.codesRow, (p * kLanes + lane) * kE, a.width, code);
            }
        }
    }
}

template <typename T, int kLanes, int kPieces>
__global__ __launch_bounds__((kLanes < 128 ? 256 : kLanes)) void normGradKernel(const NormGradArgs a)
{
    constexpr int kE = 16 / sizeof(T), kThreads = kLanes < 128 ? 256 : kLanes, kGroups = kThreads / kLanes;
    constexpr int kColumns = kLanes * kPieces * kE;
    __shared__ __align__(32) float sums[kGroups > 1 ? kGroups * kColumns : kThreads / 64];
    float* const slots = sums;            // a row of a whole workgroup has no columns to add up
    const int lane = threadIdx.x % kLanes;
    const bool tail = a.width % kE != 0;
    vec<float, kE> w[kPieces], dw[kPieces];
#pragma unroll
    for (int p = 0; p < kPieces; p++) {
        const int at = (p * kLanes + lane) * kE;
        w[p] = toFloat<T, kE>(loadPiece(static_cast<const T*>(a.weight), at, a.width));
        dw[p] = vec<float, kE>(0.0f);
    }
    for (int64_t row = (int64_t)blockIdx.x * kGroups + threadIdx.x / kLanes; row < a.rows; row += (int64_t)gridDim.x * kGroups) {
        vec<T, kE> in[kPieces], out[kPieces], on[kPieces];
#pragma unroll
        for (int p = 0; p < kPieces; p++) {
            const int at = (p * kLanes + lane) * kE;
            in[p] = loadPiece(static_cast<const T*>(a.s) + row * a.sRow, at, a.width);
            out[p] = loadPiece(static_cast<const T*>(a.dy) + row * a.dyRow, at, a.width);
            if (a.dsum) on[p] = loadPiece(static_cast<const T*>(a.dsum) + row * a.dsumRow, at, a.width);
        }
        // sums of s^2 and of g s in one pass, with s times a power of two where its squares need one
        float squares, inner, factor = 1.0f;
        const auto sumUp = [&]() {
            squares = inner = 0.0f;
#pragma unroll
            for (int p = 0; p < kPieces; p++) {
                const auto s = toFloat<T, kE>(in[p]) * factor, g = toFloat<T, kE>(out[p]) * w[p];
                const int dup = tail ? dupOf<T>((p * kLanes + lane) * kE, a.width) : 0;
#pragma unroll
                for (int j = 0; j < kE; j++) {
                    squares += j < dup ? 0.0f : s[j] * s[j];
                    inner += j < dup ? 0.0f : g[j] * s[j];
                }
            }
            squares = overRow<Add, kLanes>(squares, slots);
            inner = overRow<Add, kLanes>(inner, slots);
        };
        sumUp();
        if (!(squares < kMostSquares)) {
            factor = kSmaller;
            sumUp();
        }
        const float r = 1.0f / sqrtf(squares / (float)a.width + a.eps * factor * factor);
        const float mean = inner / (float)a.width * r, own = r * factor;
#pragma unroll
        for (int p = 0; p < kPieces; p++) {
            const int at = (p * kLanes + lane) * kE;
            const auto u = toFloat<T, kE>(in[p]) * factor * r, dy = toFloat<T, kE>(out[p]);
            dw[p] += dy * u;
            if (!a.dx) continue;
            auto d = (dy * w[p] - u * mean) * own;
            if (a.dsum) d += toFloat<T, kE>(on[p]);
            storePiece<T, kE>(static_cast<T*>(a.dx) + row * a.width, at, a.width, fromFloat<T, kE>(d));
        }
    }
    if (!a.part && !a.dw) return;
    const auto write = [&](int column, float x) {
        if (column >= a.width) return;
        if (a.part) a.part[(int64_t)blockIdx.x * a.width + column] = x;
        else static_cast<T*>(a.dw)[column] = (T)x;
    };
    if constexpr (kGroups > 1) {
        float* const mine = sums + threadIdx.x / kLanes * kColumns;
#pragma unroll
        for (int p = 0; p < kPieces; p++) {
            const int at = (p * kLanes + lane) * kE, dup = tail ? dupOf<T>(at, a.width) : 0;
            if (dup == 0) *reinterpret_cast<vec<float, kE>*>(mine + at) = dw[p];
            else
#pragma unroll
                for (int j = 0; j < kE; j++)
                    if (j >= dup) mine[at - dup + j] = dw[p][j];
        }
        __syncthreads();
        for (int c = threadIdx.x; c < kColumns; c += kThreads) {
            float x = 0.0f;
#pragma unroll
            for (int g = 0; g < kGroups; g++) x += sums[g * kColumns + c];
            write(c, x);
        }
    } else {
#pragma unroll
        for (int p = 0; p < kPieces; p++) {
            const int at = (p * kLanes + lane) * kE, dup = tail ? dupOf<T>(at, a.width) : 0;
#pragma unroll
            for (int j = 0; j < kE; j++)
                if (j >= dup) write(at - dup + j, dw[p][j]);
        }
    }
}

// Workgroups' parts of dw: 64 columns a workgroup, the parts dealt to its 16 waves.
template <typename T> __global__ __launch_bounds__(1024) void partsKernel(const float* part, int parts, int width, T* dw)
{
    __shared__ float sums[16][64];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, column = blockIdx.x * 64 + lane;
    float x = 0.0f;
    if (column < width) {
        // eight loads on their way at once
        int i = wave;
        for (; i + 7 * 16 < parts; i += 8 * 16) {
            float own[8];
#pragma unroll
            for (int j = 0; j < 8; j++) own[j] = part[(int64_t)(i + j * 16) * width + column];
#pragma unroll
            for (int j = 0; j < 8; j++) x += own[j];
        }
        for (; i < parts; i += 16) x += part[(int64_t)i * width + column];
    }
    sums[wave][lane] = x;
    __syncthreads();
    if (wave != 0 || column >= width) return;
    for (int i = 1; i < 16; i++) x += sums[i][lane];
    dw[column] = (T)x;
}

constexpr int64_t kMostRows = (int64_t)1 << 40;

// The lanes that share a row, and the pieces that each takes of it.  Up to 256
// pieces lanes of a wave do, so that it holds several rows: most of what a row
// costs beside its bytes are a reduction's steps, which a wave takes for all its
// rows at once, and lanes without a piece (262,144 bf16 rows of 257: 54 us with 16
// lanes of three pieces, 96 with 64 of one).  Beyond it a workgroup does, of as
// few waves as keep its registers low and its lanes filled (42,140 bf16 rows of
// 2,373, 297 pieces, backward: 193 us with 128 lanes of three, 257 with 256 of
// two; of 1,408 in f32, 352 pieces, 325 with 192 of two and 394 with 128 of three).
// `wide` calls read two or three rows at once for each that the others read, and
// take more lanes at two borders (195,312 bf16 rows of 512: codes 46 us with 32
// lanes of two and 55 with 64 of one, norm with an addition 131 and 127).
template <typename T, typename F> void withShape(int width, bool wide, F&& run)
{
    const int pieces = (int)((width * sizeof(T) + 15) / 16);
    const auto shape = [&](auto lanes, auto each) { run(lanes, each); };
    using std::integral_constant;
#define SHAPE(lanes, each) shape(integral_constant<int, lanes>(), integral_constant<int, each>())
    if (pieces <= 8) SHAPE(8, 1);
    else if (pieces <= 16) SHAPE(16, 1);
    else if (pieces <= 32) SHAPE(32, 1);
    else if (pieces <= 48) SHAPE(16, 3);
    else if (pieces <= 64 && !wide) SHAPE(32, 2);
    else if (pieces <= 64) SHAPE(64, 1);
    else if (pieces <= 96) SHAPE(32, 3);
    else if (pieces <= 128) SHAPE(64, 2);
    else if (pieces <= 192) SHAPE(64, 3);
    else if (pieces <= 256) SHAPE(64, 4);
    else if (pieces <= 384) SHAPE((sizeof(T) == 4 ? 192 : 128), (sizeof(T) == 4 ? 2 : 3));
    else if (pieces <= 512) SHAPE(256, 2);
    else if (pieces <= 768) SHAPE(256, 3);
    else if (pieces <= 1024) SHAPE(512, 2);
    else if (pieces <= 1536 && !wide) SHAPE(512, 3);
    else if (sizeof(T) == 2 || pieces <= 2048) SHAPE(1024, 2);
    else if constexpr (sizeof(T) == 4) SHAPE(1024, 4);
#undef SHAPE
}

constexpr int groupsOf(int lanes) { return lanes < 128 ? 256 / lanes : 1; }
constexpr int threadsOf(int lanes) { return lanes < 128 ? 256 : lanes; }

// Enough workgroups to fill the GPU; each goes on with rows further down.
int blocksOf(int64_t rows, int lanes, int most)
{
    const int64_t groups = groupsOf(lanes);
    return (int)std::min<int64_t>((rows + groups - 1) / groups, (int64_t)most * 256 / std::max(lanes, 256));
}

constexpr int kForwardBlocks = 65536, kGradBlocks = 1024;

template <typename T, int kKind> void launchNorm(const NormArgs& a, hipStream_t stream)
{
    withShape<T>(a.width, kKind != kRowCodes && a.residual, [&](auto lanes, auto pieces) {
        normKernel<T, kKind, lanes(), pieces()><<<dim3(blocksOf(a.rows, lanes(), kForwardBlocks)), threadsOf(lanes()), 0, stream>>>(a);
    });
}

template <int kKind> int norm(int type, const NormArgs& a, hipStream_t stream)
{
    if (type == CARL_OP_F32) launchNorm<float, kKind>(a, stream);
    else if (type == CARL_OP_BF16) launchNorm<bf16, kKind>(a, stream);
    else launchNorm<f16, kKind>(a, stream);
    return launched("norm");
}

template <typename T> int gradBlocks(const carl_norm& n)
{
    int blocks = 0;
    withShape<T>(n.width, true, [&](auto lanes, auto) { blocks = blocksOf(n.rows, lanes(), kGradBlocks); });
    return blocks;
}

int gradBlocks(const carl_norm& n) { return n.type == CARL_OP_F32 ? gradBlocks<float>(n) : gradBlocks<bf16>(n); }

template <typename T> int normBackward(const carl_norm& n, hipStream_t stream)
{
    const int blocks = gradBlocks<T>(n);
    NormGradArgs a{ n.sum, n.dy, n.d_sum, n.weight, n.sum_row, n.dy_row, n.d_sum_row, n.rows, n.width, n.eps, n.d_x, nullptr, nullptr };
    if (n.d_weight && blocks > 1) a.part = static_cast<float*>(n.workspace);
    else a.dw = n.d_weight;
    withShape<T>(n.width, true, [&](auto lanes, auto pieces) {
        normGradKernel<T, lanes(), pieces()><<<dim3(blocks), threadsOf(lanes()), 0, stream>>>(a);
    });
    if (int rc = launched("norm's gradients")) return rc;
    if (!a.part) return CARL_OK;
    partsKernel<T><<<dim3((n.width + 63) / 64), 1024, 0, stream>>>(a.part, blocks, n.width, static_cast<T*>(n.d_weight));
    return launched("norm's weight gradient");
}

int checkNorm(const carl_norm* n, bool normed)
{
    if (!n) return fail(CARL_ERR_VALUE, "null norm argument");
    if (n->type != CARL_OP_F32 && n->type != CARL_OP_BF16 && n->type != CARL_OP_F16) return fail(CARL_ERR_TYPE, "unknown element type");
    if (n->width < 1 || n->width > CARL_NORM_MAX_DIM) return fail(CARL_ERR_VALUE, "width must be in [1, 16384]");
    if (n->rows < 0 || n->rows > kMostRows) return fail(CARL_ERR_VALUE, "rows are out of range");
    if (!normed) return CARL_OK;
    if (!(n->eps >= CARL_NORM_MIN_EPS) || !std::isfinite(n->eps)) return fail(CARL_ERR_VALUE, "eps must be finite and at least 1e-30");
    if (!n->weight) return fail(CARL_ERR_VALUE, "null weight");
    return CARL_OK;
}

NormArgs argsOf(const carl_norm& n)
{
    return { n.x, n.residual, n.weight, n.x_row, n.residual_row, n.rows, n.width, n.eps, n.sum, n.y, n.codes, n.codes_row, n.scale };
}

}  // namespace

extern "C" {

int carl_rms_norm(const carl_norm* n, void* stream)
{
    if (int rc = checkNorm(n, true)) return rc;
    if (n->rows == 0) return CARL_OK;
    if (!n->x || !n->y || (n->residual && !n->sum)) return fail(CARL_ERR_VALUE, "null norm tensor");
    return norm<kPlain>(n->type, argsOf(*n), (hipStream_t)stream);
}

int carl_rms_norm_int8(const carl_norm* n, void* stream)
{
    if (int rc = checkNorm(n, true)) return rc;
    if (n->rows == 0) return CARL_OK;
    if (!n->x || !n->codes || !n->scale || (n->residual && !n->sum)) return fail(CARL_ERR_VALUE, "null norm tensor");
    if (n->codes_row < n->width) return fail(CARL_ERR_VALUE, "rows of codes overlap");
    return norm<kNormCodes>(n->type, argsOf(*n), (hipStream_t)stream);
}

int carl_quantize_int8(const carl_norm* n, void* stream)
{
    if (int rc = checkNorm(n, false)) return rc;
    if (n->rows == 0) return CARL_OK;
    if (!n->x || !n->codes || !n->scale) return fail(CARL_ERR_VALUE, "null tensor of rows");
    if (n->codes_row < n->width) return fail(CARL_ERR_VALUE, "rows of codes overlap");
    return norm<kRowCodes>(n->type, argsOf(*n), (hipStream_t)stream);
}

int carl_rms_norm_workspace(const carl_norm* n, int64_t* bytes)
{
    if (!bytes) return fail(CARL_ERR_VALUE, "null norm argument");
    if (int rc = checkNorm(n, false)) return rc;
    const int blocks = gradBlocks(*n);
    *bytes = blocks > 1 ? (int64_t)blocks * n->width * 4 : 0;
    return CARL_OK;
}

int carl_rms_norm_backward(const carl_norm* n, void* stream)
{
    if (int rc = checkNorm(n, true)) return rc;
    if (!n->d_x && !n->d_weight) return CARL_OK;
    if (n->rows > 0 && (!n->sum || !n->dy)) return fail(CARL_ERR_VALUE, "null norm tensor");
    const hipStream_t s = (hipStream_t)stream;
    if (n->rows == 0) {
        if (!n->d_weight) return CARL_OK;
        const dim3 grid((n->width + 63) / 64);
        if (n->type == CARL_OP_F32) partsKernel<float><<<grid, 1024, 0, s>>>(nullptr, 0, n->width, static_cast<float*>(n->d_weight));
        else if (n->type == CARL_OP_BF16) partsKernel<bf16><<<grid, 1024, 0, s>>>(nullptr, 0, n->width, static_cast<bf16*>(n->d_weight));
        else partsKernel<f16><<<grid, 1024, 0, s>>>(nullptr, 0, n->width, static_cast<f16*>(n->d_weight));
        return launched("norm's weight gradient");
    }
    if (n->d_weight && !n->workspace && gradBlocks(*n) > 1) return fail(CARL_ERR_VALUE, "null workspace");
    if (n->type == CARL_OP_F32) return normBackward<float>(*n, s);
    if (n->type == CARL_OP_BF16) return normBackward<bf16>(*n, s);
    return normBackward<f16>(*n, s);
}

}  // extern "C"
