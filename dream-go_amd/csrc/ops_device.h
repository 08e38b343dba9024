// Device side that the operators share: element types, activations, loads that need no more alignment than an element's.
#pragma once

#include "ops.h"

#include <type_traits>

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

__device__ __forceinline__ float rcp(float v) { return __builtin_amdgcn_rcpf(v); }                          // one step off at most
__device__ __forceinline__ float exponential(float v) { return __builtin_amdgcn_exp2f(v * 1.44269504088896341f); }

// The activations in fp32, without branches: a wave does eight of them per lane in a row.  Errors are a few steps of fp32 beside max(1, |v|).
//   tanh  an odd polynomial up to 0.7 (of degree 11, fitted like gelu's, 1.5e-8 relative), 1 - 2 / (exp(2 |x|) + 1) with the sign beyond: within 9e-8 on a
//         grid (twice that where the sign goes into the exponent, the quotient being near 2 below zero)
//   gelu  v * Phi(v); Phi(-x) exp(x^2 / 2) is a polynomial of t = 1 / (1 + 0.3 x), fitted to it over 0 <= x <= 14 by least squares weighted for the
//         smallest largest relative error, 1.5e-7.  The tail is the product itself, not 1 - erf: below zero it keeps its digits (the exponent's own
//         rounding, x^2 / 2 times a few steps, is what it loses), and results are within 1.2e-7 of max(1, |v|) as measured on a grid
//   silu  v / (1 + exp(-v)), the quotient corrected to the last bit where the result stays fp32 (1.2e-7 of max(1, |v|) on a grid; fixup: where an infinity is
//         divided or divides); the product with the reciprocal alone, 1.4e-7, where it is rounded to sixteen bits, whose half step is 4e3 times that
__device__ __forceinline__ float tanh_of(float v)
{
    const float q = v * v, x = __builtin_fabsf(v);
    const float odd = v * __builtin_fmaf(q, __builtin_fmaf(q, __builtin_fmaf(q, __builtin_fmaf(q, __builtin_fmaf(q, -0.00513866218f, 0.0200919695f), -0.05355886f), 0.13329111f),
                          -0.333331913f), 1.0f);
    const float direct = __builtin_copysignf(1.0f - 2.0f * rcp(exponential(2.0f * x) + 1.0f), v);
    return x < 0.7f ? odd : direct;
}
__device__ __forceinline__ float gelu_of(float v)
{
    const float x = __builtin_fabsf(v), t = rcp(__builtin_fmaf(0.3f, x, 1.0f));
    const float p = t * __builtin_fmaf(t, __builtin_fmaf(t, __builtin_fmaf(t, __builtin_fmaf(t, __builtin_fmaf(t, __builtin_fmaf(t, __builtin_fmaf(t,
                        3.56747769e-2f, -1.57203108e-1f), 2.06353530e-1f), -5.36836721e-2f), 1.28561646e-1f), 9.99134853e-2f), 1.20753959e-1f), 1.19629301e-1f);
    const float tail = p * __builtin_amdgcn_exp2f(x * x * -0.72134752044448170f);           // Phi(-|v|)
    return v * (v < 0.0f ? tail : 1.0f - tail);
}
template <typename O>
__device__ __forceinline__ float silu_of(float v)
{
    const float d = 1.0f + exponential(-v), r = rcp(d), q = v * r;
    if constexpr (!__is_same(O, float)) return q;
    else return __builtin_amdgcn_div_fixupf(__builtin_fmaf(__builtin_fmaf(-q, d, v), r, q), d, v);
}

// O: what the result is rounded to.
template <typename O>
__device__ __forceinline__ float activate(float v, int activation)
{
    switch (activation) {
    case DGNN_ACT_RELU: return v < 0.0f ? 0.0f : v;
    case DGNN_ACT_TANH: return tanh_of(v);
    case DGNN_ACT_GELU: return gelu_of(v);
    case DGNN_ACT_SILU: return silu_of<O>(v);
    default: return v;
    }
}

// Kinds of activation that a kernel may be made for: what it does not need would still have to be fetched with its instructions.
enum Kind { kPlain, kSilu, kAny };              // identity and ReLU; SiLU; every one

// One branch for several values.
template <typename O, int N>
__device__ __forceinline__ void activate(float (&v)[N], int activation)
{
    switch (activation) {
    case DGNN_ACT_IDENTITY: break;
    case DGNN_ACT_RELU:
#pragma unroll
        for (int r = 0; r < N; ++r) v[r] = activate<O>(v[r], DGNN_ACT_RELU);
        break;
    case DGNN_ACT_TANH:
#pragma unroll
        for (int r = 0; r < N; ++r) v[r] = activate<O>(v[r], DGNN_ACT_TANH);
        break;
    case DGNN_ACT_GELU:
#pragma unroll
        for (int r = 0; r < N; ++r) v[r] = activate<O>(v[r], DGNN_ACT_GELU);
        break;
    default:
#pragma unroll
        for (int r = 0; r < N; ++r) v[r] = activate<O>(v[r], DGNN_ACT_SILU);
    }
}

template <Kind K, typename O, int N>
__device__ __forceinline__ void activate_kind(float (&v)[N], int activation)
{
    if constexpr (K == kAny) activate<O>(v, activation);
    else {
#pragma unroll
        for (int r = 0; r < N; ++r) v[r] = K == kSilu ? silu_of<O>(v[r]) : activation == DGNN_ACT_RELU && v[r] < 0.0f ? 0.0f : v[r];
    }
}

template <int Control>
__device__ __forceinline__ float moved(float v)
{
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), Control, 0xf, 0xf, true));
}

// The sum over a row of sixteen lanes, the same in every one of them: data-parallel moves, which cost no trip through LDS.
__device__ __forceinline__ float row_sum(float v)
{
    v += moved<0xb1>(v);                // quad_perm [1, 0, 3, 2]
    v += moved<0x4e>(v);                // quad_perm [2, 3, 0, 1]
    v += moved<0x141>(v);               // row_half_mirror
    return v + moved<0x140>(v);         // row_mirror
}

// The sum over a wave, the same in every lane.
__device__ __forceinline__ float wave_sum(float v)
{
    v = row_sum(v);
    const auto row = [&](int lane) { return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane)); };
    return (row(0) + row(16)) + (row(32) + row(48));
}

// The sums over the lanes of a wave that are equal modulo `period` (a power of two up to 64, the same in the whole wave), in every
// one of them -- in an order of its own: take one lane's.
template <int N>
__device__ __forceinline__ void periodic_sums(float (&v)[N], int period)
{
    const auto each = [&](auto sum) {
#pragma unroll
        for (int e = 0; e < N; ++e) v[e] = sum(v[e]);
    };
    // both halves of a swap with itself: the lower partner's value in every lane, and the upper one's
    const auto joined = [](auto both) { return __builtin_bit_cast(float, (unsigned)both[0]) + __builtin_bit_cast(float, (unsigned)both[1]); };
    if (period <= 1) each([](float x) { return x + moved<0xb1>(x); });
    if (period <= 2) each([](float x) { return x + moved<0x4e>(x); });
    if (period <= 4) each([](float x) { return x + moved<0x124>(x); });          // row_ror 4: with the next one, the four lanes 4 apart
    if (period <= 8) each([](float x) { return x + moved<0x128>(x); });          // row_ror 8
    if (period <= 16) each([&](float x) { const unsigned b = __builtin_bit_cast(unsigned, x); return joined(__builtin_amdgcn_permlane16_swap(b, b, false, false)); });
    if (period <= 32) each([&](float x) { const unsigned b = __builtin_bit_cast(unsigned, x); return joined(__builtin_amdgcn_permlane32_swap(b, b, false, false)); });
}

}  // namespace ops
}  // namespace dgnn
