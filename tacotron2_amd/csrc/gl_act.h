// Activations of the dense-layer and group-norm kernels, their derivatives, and the element types they run on.
#pragma once
#include <hip/hip_runtime.h>

typedef _Float16 gl_f16;
typedef __bf16 gl_bf16;

template <int N> struct gl_int { static constexpr int value = N; };

__device__ __forceinline__ float gl_to_f32(float v) { return v; }
__device__ __forceinline__ float gl_to_f32(gl_bf16 v) { return (float)v; }
__device__ __forceinline__ float gl_to_f32(gl_f16 v) { return (float)v; }

// R, here and below: the type of the results.  What is FINE is for float32; the rest is for 16-bit ones, next to whose half step
// (2^-12, 2^-9) it errs little.
template <typename R> constexpr bool gl_fine = __is_same(R, float);

// exp(z) = 2^(z log2 e).  The product's rounding moves the result by up to |z| 2^-24 of it.  FINE: 2^n 2^f with a whole n, where f
// takes along what the product and float32's log2 e lose; n stays within the range in which f alone makes infinity or zero.
template <bool FINE>
__device__ __forceinline__ float gl_exp(float z) {
    constexpr float k = 1.44269504088896341f;
    if constexpr (FINE) {
        constexpr float k_rest = (float)(1.44269504088896341 - (double)k);
        const float n = __builtin_amdgcn_fmed3f(__builtin_rintf(z * k), -200.0f, 200.0f);
        return __builtin_amdgcn_ldexpf(__builtin_amdgcn_exp2f(fmaf(z, k_rest, fmaf(z, k, -n))), (int)n);
    } else {
        const float t = z * k;
        const bool low = t < -120.0f;                        // subnormal results: 2^64 up, then down with one rounding
        return __builtin_amdgcn_exp2f(t + (low ? 64.0f : 0.0f)) * (low ? 0x1p-64f : 1.0f);
    }
}

template <bool FINE>
__device__ __forceinline__ float gl_sigmoid(float z) {
    if constexpr (FINE) return __builtin_amdgcn_rcpf(1.0f + gl_exp<true>(-z));
    else return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(z * -1.44269504088896341f));
}

// Phi(-a) / exp(-a^2 / 2) for a >= 0, in the form of Hastings' approximations: t P(t), t = 1 / (1 + c a).  c and P are fitted by
// weighted least squares (Lawson's weights) for the smallest relative error over a <= 14.6, where the result leaves float32's
// range: 2^-24.9 with nine terms; 2^-20.6 with seven, for bfloat16 (55 104 x 512 -> 2048: two terms are 4 us of 155).
template <int TERMS>
__device__ __forceinline__ float gl_phi_ratio(float a) {
    static_assert(TERMS == 9 || TERMS == 7);
    const float t = __builtin_amdgcn_rcpf(fmaf(a, TERMS == 9 ? 0.35f : 0.265f, 1.0f));
    float p;
    if constexpr (TERMS == 9) {
        p = fmaf(t, -2.915946483e-02f, 1.440387674e-01f);
        p = fmaf(p, t, -2.558555896e-01f);
        p = fmaf(p, t, 1.593390985e-01f);
        p = fmaf(p, t, -2.322604228e-02f);
        p = fmaf(p, t, 1.055584544e-01f);
        p = fmaf(p, t, 1.198197353e-01f);
        p = fmaf(p, t, 1.398637337e-01f);
        p = fmaf(p, t, 1.396212914e-01f);
    } else {
        p = fmaf(t, -6.778700520e-02f, 1.952730320e-01f);
        p = fmaf(p, t, -6.636279412e-02f);
        p = fmaf(p, t, 1.424932325e-01f);
        p = fmaf(p, t, 8.294662721e-02f);
        p = fmaf(p, t, 1.078367668e-01f);
        p = fmaf(p, t, 1.055998295e-01f);
    }
    return t * p;
}
// exp(-a^2 / 2).  FINE: with what a^2 and its product with log2(e) / 2 lose; a is cut off where the result has long been zero.
template <bool FINE>
__device__ __forceinline__ float gl_gauss(float a) {
    if constexpr (!FINE) return __builtin_amdgcn_exp2f(a * a * -0.72134752044448170f);
    else {
        constexpr float k = -0.72134752044448170f;           // -log2(e) / 2, and what float32 leaves of it
        constexpr float k_rest = (float)(-0.72134752044448170 - (double)k);
        a = __builtin_amdgcn_fmed3f(a, 0.0f, 16.0f);
        const float s = a * a, t = s * k;
        const float rest = fmaf(fmaf(a, a, -s), k, fmaf(s, k_rest, fmaf(s, k, -t)));
        const float e = __builtin_amdgcn_exp2f(t);
        return fmaf(e, rest * 0.69314718055994531f, e);
    }
}

// act(z).  Every branch on `act` is uniform: a kernel argument or a template constant.  For many values at once take
// gl_with_act around the loop: a branch a value scatters the code that runs over all activations of all values.
template <typename R>
__device__ __forceinline__ float gl_act(float z, int act) {
    constexpr bool FINE = gl_fine<R>;
    switch (act) {
        case GL_ACT_RELU: return z < 0.0f ? 0.0f : z;                  // NaN stays NaN
        case GL_ACT_SILU: return z * gl_sigmoid<FINE>(z);
        case GL_ACT_GELU: {                                            // z Phi(z), Phi(z) = 1 - Phi(-z): no tail is a difference
            const float h = gl_phi_ratio<__is_same(R, gl_bf16) ? 7 : 9>(fabsf(z)) * gl_gauss<FINE>(fabsf(z));
            return z * (z > 0.0f ? 1.0f - h : h);
        }
        case GL_ACT_TANH: {
            // (1 - e) / (1 + e) with e = exp(-2 |z|); near zero, where 1 - e cancels, z + z^3 P(z^2): P the series (left out is
            // 3.6e-7 of it at 0.25), FINE a fit by weighted least squares over |z| <= 0.6 (3e-9 of it)
            const float a = fabsf(z), e = FINE ? gl_exp<true>(-2.0f * a) : __builtin_amdgcn_exp2f(a * -2.88539008177792681f);
            const float far = copysignf((1.0f - e) * __builtin_amdgcn_rcpf(1.0f + e), z);
            const float q = z * z;
            float p;
            if constexpr (FINE) {
                p = fmaf(q, -5.895131993e-03f, 2.079595110e-02f);
                p = fmaf(q, p, -5.378382476e-02f);
                p = fmaf(q, p, 1.333192407e-01f);
                p = fmaf(q, p, -3.333329800e-01f);
            } else {
                p = fmaf(q, fmaf(q, -0.0539682540f, 0.133333333f), -0.333333333f);
            }
            return a < (FINE ? 0.6f : 0.25f) ? fmaf(z * q, p, z) : far;
        }
        case GL_ACT_EXP: return gl_exp<FINE>(z);
        default: return z;
    }
}

// act'(z).  R: the type of dy.  Phi has all its terms here: unrounded sums of gradients are made of it.
template <typename R>
__device__ __forceinline__ float gl_act_grad(float z, int act) {
    constexpr bool FINE = gl_fine<R>;
    switch (act) {
        case GL_ACT_RELU: return z > 0.0f ? 1.0f : (z != z ? z : 0.0f);
        case GL_ACT_SILU: {
            if constexpr (FINE) {                                      // s(z) and 1 - s(z) from exp(-|z|) <= 1, neither a difference
                const float e = gl_exp<true>(-fabsf(z)), r = __builtin_amdgcn_rcpf(1.0f + e), s = z < 0.0f ? e * r : r;
                return fmaf(z * s, z < 0.0f ? r : e * r, s);
            }
            const float s = gl_sigmoid<false>(z);
            return fmaf(z * s, 1.0f - s, s);
        }
        case GL_ACT_GELU: {                                            // Phi(z) + z phi(z)
            const float a = fabsf(z), e = gl_gauss<FINE>(a), h = gl_phi_ratio<9>(a) * e;
            return fmaf(z * e, 0.39894228040143268f, z < 0.0f ? h : 1.0f - h);
        }
        case GL_ACT_TANH: {                                            // 4 e / (1 + e)^2 with e = exp(-2 |z|)
            const float e = FINE ? gl_exp<true>(-2.0f * fabsf(z)) : __builtin_amdgcn_exp2f(fabsf(z) * -2.88539008177792681f);
            const float r = __builtin_amdgcn_rcpf(1.0f + e);
            return 4.0f * e * r * r;
        }
        case GL_ACT_EXP: return gl_exp<FINE>(z);
        default: return 1.0f;
    }
}

// f(gl_int<the activation>)
template <typename F>
__device__ __forceinline__ void gl_with_act(int act, F f) {
    switch (act) {
        case GL_ACT_RELU: f(gl_int<GL_ACT_RELU>()); break;
        case GL_ACT_SILU: f(gl_int<GL_ACT_SILU>()); break;
        case GL_ACT_GELU: f(gl_int<GL_ACT_GELU>()); break;
        case GL_ACT_TANH: f(gl_int<GL_ACT_TANH>()); break;
        case GL_ACT_EXP: f(gl_int<GL_ACT_EXP>()); break;
        default: f(gl_int<GL_ACT_NONE>());
    }
}
