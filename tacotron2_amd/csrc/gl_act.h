// Activations of the dense-layer and group-norm kernels, their derivatives, and the element types they run on.
#pragma once
#include <hip/hip_runtime.h>

typedef _Float16 gl_f16;
typedef __bf16 gl_bf16;

template <int N> struct gl_int { static constexpr int value = N; };

__device__ __forceinline__ float gl_to_f32(float v) { return v; }
__device__ __forceinline__ float gl_to_f32(gl_bf16 v) { return (float)v; }
__device__ __forceinline__ float gl_to_f32(gl_f16 v) { return (float)v; }

// act(z).  Every branch is uniform: `act` is a kernel argument or a template constant.
__device__ __forceinline__ float gl_act(float z, int act) {
    switch (act) {
        case GL_ACT_RELU: return z < 0.0f ? 0.0f : z;                  // NaN stays NaN
        case GL_ACT_SILU: return z / (1.0f + expf(-z));
        case GL_ACT_GELU: return 0.5f * z * (1.0f + erff(z * 0.70710678118654752f));
        case GL_ACT_TANH: return tanhf(z);
        case GL_ACT_EXP: return expf(z);
        default: return z;
    }
}

// act'(z)
__device__ __forceinline__ float gl_act_grad(float z, int act) {
    switch (act) {
        case GL_ACT_RELU: return z > 0.0f ? 1.0f : (z != z ? z : 0.0f);
        case GL_ACT_SILU: {
            const float s = 1.0f / (1.0f + expf(-z));
            return s * (1.0f + z * (1.0f - s));
        }
        case GL_ACT_GELU:
            return 0.5f * (1.0f + erff(z * 0.70710678118654752f)) + z * expf(-0.5f * z * z) * 0.39894228040143268f;
        case GL_ACT_TANH: {
            const float t = tanhf(z);
            return 1.0f - t * t;
        }
        case GL_ACT_EXP: return expf(z);
        default: return 1.0f;
    }
}
