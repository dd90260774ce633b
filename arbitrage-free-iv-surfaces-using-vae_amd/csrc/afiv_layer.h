// Device helpers shared by the layer kernels (afiv_linear.hip, afiv_norm.hip, afiv_ckpt.hip):
// element types, unaligned vector access, activations and the 8-bit checkpoint format.
#pragma once

#include "afiv_internal.h"

#include <type_traits>

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

// N consecutive elements, moved as one unaligned access (global memory takes dword-wide accesses at
// any address on this target, so ragged row lengths keep wide loads)
template <class T, int N>
struct Pack { T v[N]; };

template <class T, int N>
__device__ __forceinline__ Pack<T, N> load_pack(const T *p)
{
    Pack<T, N> r;
    __builtin_memcpy(&r, p, sizeof r);
    return r;
}
template <class T, int N>
__device__ __forceinline__ void store_pack(T *p, const Pack<T, N> &r)
{
    __builtin_memcpy(p, &r, sizeof r);
}
// the first n of N elements, zeros behind them
template <class T, int N>
__device__ __forceinline__ Pack<T, N> load_some(const T *p, int n)
{
    if (n >= N) return load_pack<T, N>(p);
    Pack<T, N> r;
#pragma unroll
    for (int i = 0; i < N; ++i) r.v[i] = i < n ? p[i] : T(0);
    return r;
}
template <class T, int N>
__device__ __forceinline__ void store_some(T *p, const Pack<T, N> &r, int n)
{
    if (n >= N) { store_pack(p, r); return; }
#pragma unroll
    for (int i = 0; i < N; ++i)
        if (i < n) p[i] = r.v[i];
}

// ---- activations ---------------------------------------------------------------------------
constexpr float AFIV_SLOPE = 0.2f;      // leaky_relu: the slope of the reference's stacks (cvae_model.py:118)

__device__ __forceinline__ float act_value(float z, int act)
{
    switch (act) {
        case AFIV_ACT_RELU: return z > 0.0f ? z : (z == z ? 0.0f : z);
        case AFIV_ACT_LEAKY_RELU: return z > 0.0f ? z : AFIV_SLOPE * z;
        case AFIV_ACT_TANH: return tanhf(z);
        case AFIV_ACT_GELU: return 0.5f * z * erfcf(z * -0.70710678f);
        case AFIV_ACT_SILU: return z / (1.0f + expf(-z));
        default: return z;
    }
}

__device__ __forceinline__ float act_derivative(float z, int act)
{
    switch (act) {
        case AFIV_ACT_RELU: return z > 0.0f ? 1.0f : 0.0f;
        case AFIV_ACT_LEAKY_RELU: return z > 0.0f ? 1.0f : AFIV_SLOPE;
        case AFIV_ACT_TANH: {                              // 4 e / (1 + e)^2, e = exp(-2 |z|): no cancellation at the ends
            const float e = expf(-2.0f * fabsf(z)), s = 1.0f + e;
            return 4.0f * e / (s * s);
        }
        case AFIV_ACT_GELU:
            return 0.5f * erfcf(z * -0.70710678f) + z * expf(-0.5f * z * z) * 0.39894228f;
        case AFIV_ACT_SILU: {                              // p (1 + z (1 - p)), 1 - p = e / (1 + e) at z >= 0
            const float e = expf(-fabsf(z)), r = 1.0f / (1.0f + e);
            const float p = z >= 0.0f ? r : e * r, q = z >= 0.0f ? e * r : r;
            return p + z * (p * q);
        }
        default: return 1.0f;
    }
}

// ---- 8-bit derivative codes ------------------------------------------------------------------
// relu, leaky_relu: 1 where z > 0, else 0.  The others: the derivative lies in [-0.13, 1.13]; steps
// of 1/200 put it at codes 1..253 around 27 = 0, with 0 and 1 exact and an error of at most 1/400
// (a third of what e4m3 loses near 1).  255 = NaN.
__device__ __forceinline__ uint8_t derivative_code(float z, int act)
{
    if (act == AFIV_ACT_RELU || act == AFIV_ACT_LEAKY_RELU) return z > 0.0f ? 1 : 0;
    const float d = act_derivative(z, act);
    return d == d ? (uint8_t)(int)(rintf(d * 200.0f) + 27.0f) : (uint8_t)255;
}
__device__ __forceinline__ float derivative_of_code(uint8_t c, int act)
{
    if (act == AFIV_ACT_RELU) return (float)c;
    if (act == AFIV_ACT_LEAKY_RELU) return c ? 1.0f : AFIV_SLOPE;
    return c == 255 ? __builtin_nanf("") : ((float)c - 27.0f) / 200.0f;
}

// ---- 8-bit checkpoints -----------------------------------------------------------------------
// 32 consecutive elements of a row share one scale byte E = the biased exponent of their largest
// finite magnitude (at least 1); an element is the nearest q 2^(E - 133), |q| <= 127, ties to even.
// Steps are powers of two, so packing rounds once and restoring is exact in every type that held the
// input.  Magnitudes above 127.5 steps (the top 1/256 of the block's binade) become 127 steps: off by
// less than one step, the others by at most half.  Elements that are not finite have code -128 and
// come back as NaN.
__device__ __forceinline__ float finite_abs(float x)
{
    const float a = fabsf(x);
    return a < __builtin_inff() ? a : 0.0f;
}
__device__ __forceinline__ int scale_byte(float amax)
{
    const int e = (int)(__float_as_uint(amax) >> 23);
    return e > 1 ? e : 1;
}
__device__ __forceinline__ int8_t eight_code(float x, int e)
{
    if (!(fabsf(x) < __builtin_inff())) return -128;
    const float q = rintf(__builtin_ldexpf(x, 133 - e));
    return (int8_t)(int)fminf(fmaxf(q, -127.0f), 127.0f);
}
__device__ __forceinline__ float eight_value(int8_t q, int e)
{
    return q == -128 ? __builtin_nanf("") : __builtin_ldexpf((float)q, e - 133);
}
