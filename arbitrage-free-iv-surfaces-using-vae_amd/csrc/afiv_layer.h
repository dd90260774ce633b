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
    static_assert(sizeof(T) * N % 4 == 0, "whole words");
    // joined as words: a branch that yields elements would take them apart, and so wait for its load, before it ends
    uint32_t w[sizeof(T) * N / 4];
    if (n >= N) __builtin_memcpy(w, p, sizeof w);
    else {
        Pack<T, N> r;
#pragma unroll
        for (int i = 0; i < N; ++i) r.v[i] = i < n ? p[i] : T(0);
        __builtin_memcpy(w, &r, sizeof w);
    }
    Pack<T, N> r;
    __builtin_memcpy(&r, w, sizeof r);
    return r;
}
// The same by one load of the N elements that end with these n (0 < n <= N), moved into place: no branch, so several can
// be on their way.  ahead: N - n elements stand before p; otherwise element by element.
template <class T, int N>
__device__ __forceinline__ Pack<T, N> load_ending(const T *p, int n, bool ahead)
{
    constexpr int W = sizeof(T) * N / 4;
    if (!ahead) return load_some<T, N>(p, n);
    uint32_t w[W];
    __builtin_memcpy(w, p - (N - n), sizeof w);
    const uint32_t by = (N - n) * sizeof(T);
#pragma unroll
    for (int s = W / 2; s > 0; s /= 2)
#pragma unroll
        for (int i = 0; i < W; ++i) w[i] = by & (4 * s) ? (i + s < W ? w[i + s] : 0) : w[i];
    if constexpr (sizeof(T) < 4) {
#pragma unroll
        for (int i = 0; i < W; ++i) w[i] = __builtin_amdgcn_alignbyte(i + 1 < W ? w[i + 1] : 0, w[i], by & 3);
    }
    Pack<T, N> r;
    __builtin_memcpy(&r, w, sizeof r);
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

// f(z) and f'(z); whichever the caller drops costs nothing.  Built on the hardware's 2^x and reciprocal (1 ulp
// each) and, for erfc, a polynomial, at a third of the library functions' instructions, which an epilogue of 128
// outputs a lane feels.  Relative errors, in FP32 half steps (2^-24): gelu 16 + 1.5 z^2, silu 8 + 2 |z|, tanh' 12 + 4 |z|,
// gelu' and silu' as gelu and silu, of the sum of their terms' magnitudes.  The growing part comes from the exponent
// alone: its two or three roundings stand for a number that 2^x multiplies up, and it is only felt where f or f' is about
// to vanish; in absolute terms all are within a few half steps of max(1, |z|).
template <int ACT>
__device__ __forceinline__ void act_both(float z, float &f, float &d)
{
    if constexpr (ACT == AFIV_ACT_RELU) {
        f = z > 0.0f ? z : (z == z ? 0.0f : z);
        d = z > 0.0f ? 1.0f : 0.0f;
    } else if constexpr (ACT == AFIV_ACT_LEAKY_RELU) {
        f = z > 0.0f ? z : AFIV_SLOPE * z;
        d = z > 0.0f ? 1.0f : AFIV_SLOPE;
    } else if constexpr (ACT == AFIV_ACT_TANH) {
        // e = exp(-2 |z|): f = (1 - e) / (1 + e), f' = 4 e / (1 + e)^2, neither of which cancels far from zero;
        // near zero f is its Taylor polynomial (next term under 1e-8 of it at 1/4)
        const float a = fabsf(z);
        const float e = __builtin_amdgcn_exp2f(a * -2.88539008f), r = __builtin_amdgcn_rcpf(1.0f + e), q = a * a;
        const float near = a + a * q * (-0.333333333f + q * (0.133333333f + q * (-0.0539682540f + q * 0.0218694885f)));
        f = copysignf(a < 0.25f ? near : (1.0f - e) * r, z);
        if (z != z) f = z;
        d = 4.0f * e * r * r;
    } else if constexpr (ACT == AFIV_ACT_GELU) {
        // Phi(-|z|) = exp(-z^2/2) erfcx(|z|/sqrt 2) / 2, erfcx(x) = P(t), t = 1 / (1 + 0.45 x): least squares fit of
        // equal relative error, degree 8
        const float a = fabsf(z);
        const float t = __builtin_amdgcn_rcpf(1.0f + 0.318198052f * a);
        const float dens = __builtin_amdgcn_exp2f(z * z * -0.721347520f);          // exp(-z^2/2)
        float p = 0.0694841657f;
        p = p * t - 0.251303992f;
        p = p * t + 0.228051490f;
        p = p * t + 0.0224661360f;
        p = p * t + 0.198119277f;
        p = p * t + 0.225212867f;
        p = p * t + 0.254090404f;
        p = p * t + 0.253880022f;
        const float tail = 0.5f * p * t * dens, phi = z > 0.0f ? 1.0f - tail : tail;
        // z Phi and z exp(-z^2/2) vanish at -infinity
        f = z == -__builtin_inff() ? 0.0f : z * phi;
        d = phi + (a == __builtin_inff() ? 0.0f : z * dens * 0.39894228f);
    } else if constexpr (ACT == AFIV_ACT_SILU) {
        // p = 1 / (1 + exp(-z)): f = z p, f' = p + z p (1 - p), from e = exp(-|z|)
        const float e = __builtin_amdgcn_exp2f(fabsf(z) * -1.44269504f), r = __builtin_amdgcn_rcpf(1.0f + e);
        const float p = z >= 0.0f ? r : e * r, q = z >= 0.0f ? e * r : r;
        f = z == -__builtin_inff() ? 0.0f : z * p;
        d = p + (fabsf(z) == __builtin_inff() ? 0.0f : z * (p * q));
    } else {
        f = z;
        d = 1.0f;
    }
}

// calls f with the activation as a compile-time constant, so that loops stand inside the choice
template <class F>
__device__ __forceinline__ void with_act(int act, F &&f)
{
    switch (act) {
        case AFIV_ACT_RELU: f(std::integral_constant<int, AFIV_ACT_RELU>()); break;
        case AFIV_ACT_LEAKY_RELU: f(std::integral_constant<int, AFIV_ACT_LEAKY_RELU>()); break;
        case AFIV_ACT_TANH: f(std::integral_constant<int, AFIV_ACT_TANH>()); break;
        case AFIV_ACT_GELU: f(std::integral_constant<int, AFIV_ACT_GELU>()); break;
        case AFIV_ACT_SILU: f(std::integral_constant<int, AFIV_ACT_SILU>()); break;
        default: f(std::integral_constant<int, AFIV_ACT_NONE>()); break;
    }
}

// ---- 8-bit derivative codes ------------------------------------------------------------------
// relu, leaky_relu: 1 where z > 0, else 0.  The others: the derivative lies in [-0.13, 1.13]; steps
// of 1/200 put it at codes 1..253 around 27 = 0, with 0 and 1 exact and an error of at most 1/400
// (a third of what e4m3 loses near 1).  255 = NaN.
template <int ACT>
__device__ __forceinline__ uint8_t derivative_code(float z, float d)
{
    if constexpr (ACT == AFIV_ACT_RELU || ACT == AFIV_ACT_LEAKY_RELU) return z > 0.0f ? 1 : 0;
    return d == d ? (uint8_t)(int)(rintf(d * 200.0f) + 27.0f) : (uint8_t)255;
}
template <int ACT>
__device__ __forceinline__ float derivative_of_code(uint8_t c)
{
    if constexpr (ACT == AFIV_ACT_RELU) return (float)c;
    if constexpr (ACT == AFIV_ACT_LEAKY_RELU) return c ? 1.0f : AFIV_SLOPE;
    return c == 255 ? __builtin_nanf("") : ((float)c - 27.0f) * 0.005f;      // within one FP32 rounding of the quotient
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
