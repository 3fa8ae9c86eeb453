// elem.h - element types of the learner's operators: loads, stores and the
// conversions between them, rounding to nearest even.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>

namespace carl {

using bf16 = __bf16;
using f16 = _Float16;

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef f16 f16x8 __attribute__((ext_vector_type(8)));
typedef short i16x4 __attribute__((ext_vector_type(4)));

template <typename T, int N> struct VecOf { typedef T type __attribute__((ext_vector_type(N))); };
template <typename T, int N> using vec = typename VecOf<T, N>::type;

template <typename T, int N> __device__ inline vec<float, N> toFloat(vec<T, N> x)
{
    return __builtin_convertvector(x, vec<float, N>);
}

template <typename T, int N> __device__ inline vec<T, N> fromFloat(vec<float, N> x)
{
    return __builtin_convertvector(x, vec<T, N>);
}

}  // namespace carl
