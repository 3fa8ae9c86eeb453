// ffn_f16.hip - the gated feed-forward block's kernels for f16 elements, and
// the factors that its intermediate values are written with.
#include "ffn_kernel.h"

template int carl::launchProduct<carl::f16>(int, const carl::ProductArgs&, hipStream_t);
template int carl::launchThin<carl::f16>(bool, const carl::ThinArgs&, hipStream_t);
template int carl::launchOuter<carl::f16>(const carl::OuterArgs&, int, hipStream_t);
template int carl::launchPack<carl::f16>(const carl::PackArgs&, hipStream_t);
template int carl::launchSum<carl::f16>(const carl::SumArgs&, hipStream_t);

namespace carl {
namespace {

// The largest sum of squares of a panel's finite rows, a workgroup's part of
// it.  As many lanes a row as it has 16-byte pieces (a power of two, at most a
// wave), four rows of each on their way at once.  Bound by memory's bytes.
__global__ __launch_bounds__(256) void normKernel(const ScaleArgs args)
{
    constexpr int kAtOnce = 4;
    __shared__ float parts[4];
    const Panel& p = args.rows[blockIdx.y];
    const int pieces = (p.width + 7) / 8;
    int lanes = 1;
    while (lanes < pieces && lanes < 64) lanes *= 2;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, each = 64 / lanes, piece0 = lane % lanes;
    const f16* const data = static_cast<const f16*>(p.data);
    float most = 0.0f;
    // (every lane of a wave takes part in its sums)
    for (int64_t first = ((int64_t)blockIdx.x * 4 + wave) * each * kAtOnce; first < p.rows; first += (int64_t)gridDim.x * 4 * each * kAtOnce) {
        float sum[kAtOnce] = {};
        for (int piece = piece0; piece < pieces; piece += lanes) {
            vec<f16, 8> x[kAtOnce];
#pragma unroll
            for (int i = 0; i < kAtOnce; i++) {
                const int64_t row = first + i * each + lane / lanes;
                x[i] = vec<f16, 8>{};
                if (row < p.rows) x[i] = *reinterpret_cast<const vec<f16, 8>*>(data + row * p.stride + piece * 8);
            }
#pragma unroll
            for (int i = 0; i < kAtOnce; i++) {
                const auto y = toFloat<f16, 8>(x[i]);
#pragma unroll
                for (int j = 0; j < 8; j++) sum[i] += y[j] * y[j];
            }
        }
#pragma unroll
        for (int i = 0; i < kAtOnce; i++) {
            for (int d = 1; d < lanes; d *= 2) sum[i] += __shfl_xor(sum[i], d);
            if (sum[i] < 0x1p120f && sum[i] > most) most = sum[i];
        }
    }
    for (int d = 1; d < 64; d *= 2) most = fmaxf(most, __shfl_xor(most, d));
    if (lane == 0) parts[wave] = most;
    __syncthreads();
    if (threadIdx.x == 0) args.part[blockIdx.y * kScaleBlocks + blockIdx.x] = fmaxf(fmaxf(parts[0], parts[1]), fmaxf(parts[2], parts[3]));
}

constexpr int kScaleThreads = 512;

// A power of two that takes `bound` to [2^14, 2^15], and its inverse.
__device__ inline void factorOf(float bound, float& scale, float& unscale)
{
    int exponent = 15;
    if (bound > 0.0f) (void)frexpf(bound, &exponent);
    scale = ldexpf(1.0f, 15 - exponent);
    unscale = ldexpf(1.0f, exponent - 15);
}

__global__ __launch_bounds__(kScaleThreads) void scaleKernel(const ScaleArgs args)
{
    __shared__ float parts[5][kScaleThreads / 64];
    for (int j = 0; j < args.panels; j++) {
        float most = 0.0f;
#pragma unroll
        for (int i = 0; i < kScaleBlocks; i += kScaleThreads) most = fmaxf(most, args.part[j * kScaleBlocks + i + threadIdx.x]);
        for (int d = 1; d < 64; d *= 2) most = fmaxf(most, __shfl_xor(most, d));
        if ((threadIdx.x & 63) == 0) parts[j][threadIdx.x >> 6] = most;
    }
    __syncthreads();
    if (threadIdx.x != 0) return;
    float norm[5] = {};
    for (int j = 0; j < args.panels; j++) {
        for (int i = 0; i < kScaleThreads / 64; i++) norm[j] = fmaxf(norm[j], parts[j][i]);
        norm[j] = sqrtf(norm[j]);
    }
    const float x = norm[0], gate = norm[1], up = norm[2], dy = norm[3], down = norm[4];
    factorOf(x * gate * x * up, args.scale[kScaleH], args.scale[kUnscaleH]);
    factorOf(dy * down * x * fmaxf(gate, up), args.scale[kScaleD], args.scale[kUnscaleD]);
}

}  // namespace

int launchScale(const ScaleArgs& args, hipStream_t stream)
{
    normKernel<<<dim3(kScaleBlocks, (unsigned)args.panels), 256, 0, stream>>>(args);
    if (int rc = launched("norms of rows")) return rc;
    scaleKernel<<<dim3(1), kScaleThreads, 0, stream>>>(args);
    return launched("factors of float16 values");
}

}  // namespace carl
