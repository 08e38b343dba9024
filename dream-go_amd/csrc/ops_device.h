// Device side that the operators share: element types, activations, loads that need no more alignment than an element's.
#pragma once

#include "ops.h"

namespace dgnn {
namespace ops {

typedef _Float16 f16;
typedef __bf16 bf16;
typedef float floatx4 __attribute__((ext_vector_type(4)));

template <typename T, int N> struct VectorOf { typedef T type __attribute__((ext_vector_type(N))); };
template <typename T> struct VectorOf<T, 1> { typedef T type; };
template <typename T, int N> using vec = typename VectorOf<T, N>::type;

// N elements from an address that is aligned to an element: one wide load all the same (gfx950 takes unaligned ones).
template <typename T, int N>
__device__ __forceinline__ vec<T, N> load_vec(const T* p)
{
    typedef vec<T, N> V;
    typedef V Unaligned __attribute__((aligned(alignof(T))));
    return *reinterpret_cast<const Unaligned*>(p);
}

template <typename T, int N>
__device__ __forceinline__ void store_vec(T* p, vec<T, N> v)
{
    typedef vec<T, N> V;
    typedef V Unaligned __attribute__((aligned(alignof(T))));
    *reinterpret_cast<Unaligned*>(p) = v;
}

// A [n] operand whose type is only known to the host as "T or fp32".
template <typename T>
__device__ __forceinline__ float load_either(const void* p, int64_t i, bool is_float)
{
    return is_float ? static_cast<const float*>(p)[i] : (float)static_cast<const T*>(p)[i];
}

__device__ __forceinline__ float activate(float v, int activation)
{
    switch (activation) {
    case DGNN_ACT_RELU: return v < 0.0f ? 0.0f : v;
    case DGNN_ACT_TANH: return tanhf(v);
    case DGNN_ACT_GELU: return 0.5f * v * (1.0f + erff(v * 0.70710678118654752f));
    case DGNN_ACT_SILU: return v / (1.0f + expf(-v));
    default: return v;
    }
}

__device__ __forceinline__ float wave_sum(float v)
{
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
    return v;
}

}  // namespace ops
}  // namespace dgnn
