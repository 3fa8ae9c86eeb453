// reduce.h - sums and maxima over the lanes that share a row: 8 to 64 lanes of a
// wave, or all waves of a workgroup.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace carl {

struct Add {
    template <typename X> static __device__ inline X of(X a, X b) { return a + b; }
};
struct Most {
    template <typename X> static __device__ inline X of(X a, X b) { return a > b ? a : b; }
};

struct Least {
    template <typename X> static __device__ inline X of(X a, X b) { return a < b ? a : b; }
};

template <int kPattern> __device__ inline uint32_t lanesMoved(uint32_t x)
{
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, kPattern, 0xf, 0xf, false);
}
template <int kPattern> __device__ inline float lanesMoved(float x) { return __uint_as_float(lanesMoved<kPattern>(__float_as_uint(x))); }

__device__ inline uint32_t laneOf(uint32_t x, int lane) { return (uint32_t)__builtin_amdgcn_readlane((int)x, lane); }
__device__ inline float laneOf(float x, int lane) { return __uint_as_float(laneOf(__float_as_uint(x), lane)); }

// Over aligned groups of kLanes lanes, all of which take part; the same bits
// in every lane of a group.
template <typename Op, int kLanes, typename X> __device__ inline X overLanes(X x)
{
    static_assert(kLanes == 8 || kLanes == 16 || kLanes == 32 || kLanes == 64, "halves of rows of 16 lanes, or whole rows");
    x = Op::of(x, lanesMoved<0xb1>(x));      // quad_perm: 1 0 3 2
    x = Op::of(x, lanesMoved<0x4e>(x));      // quad_perm: 2 3 0 1
    x = Op::of(x, lanesMoved<0x141>(x));     // row_half_mirror
    if constexpr (kLanes > 8) x = Op::of(x, lanesMoved<0x140>(x));      // row_mirror
    if constexpr (kLanes == 32) x = Op::of(x, __shfl_xor(x, 16));
    if constexpr (kLanes == 64) x = Op::of(Op::of(laneOf(x, 0), laneOf(x, 16)), Op::of(laneOf(x, 32), laneOf(x, 48)));
    return x;
}

// Over all kThreads of a workgroup, through `slots` (kThreads / 64 of them,
// used by nothing else); the same bits in every thread.
template <typename Op, int kThreads, typename X> __device__ inline X overWorkgroup(X x, X* slots)
{
    x = overLanes<Op, 64>(x);
    if constexpr (kThreads > 64) {
        __syncthreads();                     // the last call's readers are done
        if ((threadIdx.x & 63) == 0) slots[threadIdx.x >> 6] = x;
        __syncthreads();
        x = slots[0];
#pragma unroll
        for (int i = 1; i < kThreads / 64; i++) x = Op::of(x, slots[i]);
    }
    return x;
}

// Over the lanes of a row, whichever they are.
template <typename Op, int kLanes, typename X> __device__ inline X overRow(X x, X* slots)
{
    if constexpr (kLanes <= 64) return overLanes<Op, kLanes>(x);
    else return overWorkgroup<Op, kLanes>(x, slots);
}

}  // namespace carl
