// What the dense products share (tfc_dense_act.hip, tfc_dense_narrow.hip): activations, the cut of fp32 into bf16 pieces, the matrix
// instructions.
#pragma once

#include <type_traits>

#include "tfc_types.h"

namespace {

typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef tfc_u32x4 uintx4;
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short shortx4 __attribute__((ext_vector_type(4)));

// FAST (16-bit results): exp as the power of 2 of x log2(e), 1/x as a single instruction.  exp is off by what its argument's rounding makes of
// it, |x| 2^-24 of the result, 2^-17 at most over the range in which it is not 0 or inf, and 1/x by 2^-23; half a step of the result is 2^-9 or 2^-12.
template <bool FAST>
__device__ __forceinline__ float exp_(float x) {
    return FAST ? __expf(x) : expf(x);
}
template <bool FAST>
__device__ __forceinline__ float inv_(float x) {
    return FAST ? __builtin_amdgcn_rcpf(x) : 1.f / x;
}
template <bool FAST>
__device__ __forceinline__ float sigmoid_(float x) {
    return inv_<FAST>(1.f + exp_<FAST>(-x));
}
// The normal distribution's tail beyond |x|, half of erfc(z) with z = |x| / sqrt 2; bell = exp(-x^2 / 2).  FAST: erfc(z) = t q(t) exp(-z^2),
// t = 1 / (1 + z / 2), with q a fit of degree 8 of erfc(z) exp(z^2) / t on 0 < t <= 1 that is off by at most 6e-7 (relative, in the
// tail too).
template <bool FAST>
__device__ __forceinline__ float tail_(float x, float bell) {
    const float z = 0.70710678118654752440f * fabsf(x);
    if (!FAST) return 0.5f * erfcf(z);
    const float t = __builtin_amdgcn_rcpf(1.f + 0.5f * z);
    float q = -0.021927181631326675f;
    q = q * t + 0.11047209799289703f;
    q = q * t - 0.18857893347740173f;
    q = q * t + 0.08813999593257904f;
    q = q * t + 0.013894896022975445f;
    q = q * t + 0.09286484122276306f;
    q = q * t + 0.12302764505147934f;
    q = q * t + 0.1410595327615738f;
    q = q * t + 0.14104732871055603f;
    return t * q * bell;
}
template <bool FAST>
__device__ __forceinline__ float bell_(float x) {
    return exp_<FAST>(-0.5f * x * x);
}

template <bool FAST>
__device__ __forceinline__ float act_eval(int act, float x) {
    switch (act) {
        // (the log of 1 .. 2 to 2^-23 absolute, which is what is left of it beside ln 2)
        case TFC_ACT_SSP: return fmaxf(x, 0.f) + __logf(1.f + exp_<FAST>(-fabsf(x))) - 0.69314718055994530942f;
        case TFC_ACT_SILU: return x * sigmoid_<FAST>(x);
        case TFC_ACT_TANH: return tanhf(x);
        case TFC_ACT_ABS: return fabsf(x);
        case TFC_ACT_SIGMOID: return sigmoid_<FAST>(x);
        case TFC_ACT_GELU: {
            const float h = tail_<FAST>(x, FAST ? bell_<FAST>(x) : 0.f);
            return x * (x > 0.f ? 1.f - h : h);  // (+inf stays +inf)
        }
        default: return x;
    }
}

// The same on an array: one branch for all of it, so that its elements' chains run side by side.
template <bool FAST, int N>
__device__ __forceinline__ void act_apply(int act, float (&v)[N]) {
#define TFC_ACT_CASE(A)                                              \
    case A: {                                                        \
        _Pragma("unroll") for (int j = 0; j < N; ++j) v[j] = act_eval<FAST>(A, v[j]); \
        break;                                                       \
    }
    switch (act) {
        TFC_ACT_CASE(TFC_ACT_SSP)
        TFC_ACT_CASE(TFC_ACT_SILU)
        TFC_ACT_CASE(TFC_ACT_TANH)
        TFC_ACT_CASE(TFC_ACT_ABS)
        TFC_ACT_CASE(TFC_ACT_SIGMOID)
        TFC_ACT_CASE(TFC_ACT_GELU)
        default: break;
    }
#undef TFC_ACT_CASE
}

template <bool FAST>
__device__ __forceinline__ float act_grad(int act, float x) {
    switch (act) {
        case TFC_ACT_SSP: return sigmoid_<FAST>(x);
        case TFC_ACT_SILU: {
            const float s = sigmoid_<FAST>(x);
            return s * (1.f + x * (1.f - s));
        }
        case TFC_ACT_TANH: {
            const float t = tanhf(x);
            return 1.f - t * t;
        }
        case TFC_ACT_ABS: return x > 0.f ? 1.f : (x < 0.f ? -1.f : 0.f);
        case TFC_ACT_SIGMOID: {
            const float s = sigmoid_<FAST>(x);
            return s * (1.f - s);
        }
        case TFC_ACT_GELU: {
            const float bell = bell_<FAST>(x), h = tail_<FAST>(x, bell);
            return (x > 0.f ? 1.f - h : h) + x * 0.39894228040143267794f * bell;
        }
        default: return 1.f;
    }
}

template <bool FAST, int N>
__device__ __forceinline__ void act_grad_apply(int act, float (&v)[N]) {
#define TFC_ACT_CASE(A)                                              \
    case A: {                                                        \
        _Pragma("unroll") for (int j = 0; j < N; ++j) v[j] = act_grad<FAST>(A, v[j]); \
        break;                                                       \
    }
    switch (act) {
        TFC_ACT_CASE(TFC_ACT_SSP)
        TFC_ACT_CASE(TFC_ACT_SILU)
        TFC_ACT_CASE(TFC_ACT_TANH)
        TFC_ACT_CASE(TFC_ACT_ABS)
        TFC_ACT_CASE(TFC_ACT_SIGMOID)
        TFC_ACT_CASE(TFC_ACT_GELU)
        default:
            _Pragma("unroll") for (int j = 0; j < N; ++j) v[j] = 1.f;
    }
#undef TFC_ACT_CASE
}

template <class T>
struct Pieces {
    static constexpr int N = std::is_same<T, float>::value ? 3 : 1;
    static constexpr int K = std::is_same<T, float>::value ? 32 : 64;  // contraction length of a step
};

// Eight consecutive k of one row, as fragments of the matrix instruction.
struct Unit3 {
    uintx4 h, m, l;
};
__device__ __forceinline__ Unit3 split8(const float (&x)[8]) {
    Unit3 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const unsigned u0 = __float_as_uint(x[2 * i]), u1 = __float_as_uint(x[2 * i + 1]);
        r.h[i] = __builtin_amdgcn_perm(u1, u0, 0x07060302u);  // upper halves: cut, not rounded, so that nothing overflows
        const float a0 = x[2 * i] - __uint_as_float(u0 & 0xffff0000u), a1 = x[2 * i + 1] - __uint_as_float(u1 & 0xffff0000u);
        const bf16x2 mm = {(__bf16)a0, (__bf16)a1};
        const unsigned mu = __builtin_bit_cast(unsigned, mm);
        r.m[i] = mu;
        const bf16x2 ll = {(__bf16)(a0 - __uint_as_float(mu << 16)), (__bf16)(a1 - __uint_as_float(mu & 0xffff0000u))};
        r.l[i] = __builtin_bit_cast(unsigned, ll);
    }
    return r;
}

// What is left of x behind its rounding to 16 bits.  fp16: times 2^11, so that it does not fall below the type's range (products with
// it are scaled back).
constexpr float TFC_LO_SCALE = 2048.f;
template <class T>
__device__ __forceinline__ float second_piece(T, float x) {
    const float hi = (float)(T)x, left = x - hi;
    return fabsf(hi) < __builtin_inff() ? (std::is_same<T, tfc_f16>::value ? left * TFC_LO_SCALE : left) : 0.f;
}

// Factor of dz = act'(z) dy in 16 bits, undone in the products' own: act' is up to 1.13, and dy up to the type's largest.  (act_cst goes into
// the products' factor for the same reason.)
constexpr float TFC_DZ_SCALE = 0.5f;

__device__ __forceinline__ floatx16 mma(tfc_bf16, uintx4 a, uintx4 b, floatx16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ floatx16 mma(tfc_f16, uintx4 a, uintx4 b, floatx16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

template <class T>
using Mma = std::conditional_t<std::is_same<T, float>::value, tfc_bf16, T>;  // what the matrix instruction takes

__device__ __forceinline__ void wave_step() {  // LDS written by the wave's lanes is read by its other lanes
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// Six of the nine piece products, smallest first: pieces of one operand and of the other.
constexpr int TFC_TERM_B[6] = {0, 2, 1, 0, 1, 0}, TFC_TERM_A[6] = {2, 0, 1, 1, 0, 0};

}  // namespace

// tfc_dense_narrow.hip: the backward pass of a layer of at most 64 x 64 in one kernel.
constexpr int TFC_NARROW = 64;
inline bool tfc_dense_is_narrow(int64_t n, int64_t k) { return n <= TFC_NARROW && k <= TFC_NARROW && n > 0 && k > 0; }
int64_t tfc_dense_narrow_partials(int64_t m);
int tfc_dense_narrow_bwd(const tfc_dense_bwd_desc* d, float* part, hipStream_t stream);
