// Group norm with an activation, channels last, and its gradients (include/gl_hip.h).
//
//   xh = (x - mean) rstd,  y = act(xh gamma + beta)          mean, rstd per (utterance, group) over its live frames
//   du = dy act'(xh gamma + beta);  v = du gamma;  p = mean(v), q = mean(v xh) per (utterance, group)
//   dx = rstd (v - p - xh q);  dgamma = sum du xh,  dbeta = sum du per channel over all live frames
#include "gl_internal.h"
#include "gl_act.h"

namespace {

__device__ __forceinline__ int live_frames(const int* frames, int b, int T) {
    return frames ? max(0, min(frames[b], T)) : T;
}

// Sum over the 256 threads of a workgroup, the same value in every thread; s: 4 floats of LDS.
__device__ __forceinline__ float block_sum(float v, float* s) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
    __syncthreads();
    return (s[0] + s[1]) + (s[2] + s[3]);
}

// grid (groups, B): mean first, then the squared distances from it (no cancellation whatever the level of x)
template <typename T>
__global__ void __launch_bounds__(256) k_norm_stats(const T* __restrict__ x, long long stride, const int* __restrict__ frames,
                                                    float* __restrict__ stats, int Tn, int n, float eps) {
    __shared__ float s[4];
    const int g = blockIdx.x, b = blockIdx.y;
    const int live = live_frames(frames, b, Tn);
    const long long count = (long long)live * n;
    const T* base = x + (long long)b * Tn * stride + g * n;
    float sum = 0.0f;
    for (long long e = threadIdx.x; e < count; e += 256) sum += gl_to_f32(base[e / n * stride + e % n]);
    const float mean = count ? block_sum(sum, s) / (float)count : 0.0f;
    float m2 = 0.0f;
    for (long long e = threadIdx.x; e < count; e += 256) {
        const float d = gl_to_f32(base[e / n * stride + e % n]) - mean;
        m2 += d * d;
    }
    m2 = block_sum(m2, s);
    if (threadIdx.x == 0) {
        float* o = stats + 2 * ((long long)b * gridDim.x + g);
        o[0] = mean;
        o[1] = count ? 1.0f / sqrtf(m2 / (float)count + eps) : 0.0f;
    }
}

template <typename T>
__global__ void __launch_bounds__(256) k_norm_apply(const T* __restrict__ x, long long x_stride, const T* __restrict__ gamma,
                                                    const T* __restrict__ beta, const int* __restrict__ frames,
                                                    const float* __restrict__ stats, T* __restrict__ y, long long y_stride,
                                                    int Tn, int C, int n, int act) {
    const int b = blockIdx.y;
    const int live = live_frames(frames, b, Tn);
    const int G = C / n;
    const long long count = (long long)Tn * C;
    for (long long e = (long long)blockIdx.x * 256 + threadIdx.x; e < count; e += (long long)gridDim.x * 256) {
        const int t = (int)(e / C), c = (int)(e % C);
        const long long row = (long long)b * Tn + t;
        float v = 0.0f;
        if (t < live) {
            const float* st = stats + 2 * ((long long)b * G + c / n);
            const float xh = (gl_to_f32(x[row * x_stride + c]) - st[0]) * st[1];
            v = gl_act(xh * (gamma ? gl_to_f32(gamma[c]) : 1.0f) + (beta ? gl_to_f32(beta[c]) : 0.0f), act);
        }
        y[row * y_stride + c] = (T)v;
    }
}

// grid (groups, B): per channel sums over the live frames (parts [B][2][C]: sum du xh, sum du) and the group's p, q
template <typename T>
__global__ void __launch_bounds__(256) k_norm_back_sums(const T* __restrict__ dy, long long dy_stride, const T* __restrict__ x,
                                                        long long x_stride, const float* __restrict__ stats,
                                                        const T* __restrict__ gamma, const T* __restrict__ beta,
                                                        const int* __restrict__ frames, float* __restrict__ parts,
                                                        float* __restrict__ pq, int Tn, int C, int n, int act) {
    __shared__ float s[4];
    const int g = blockIdx.x, b = blockIdx.y;
    const int live = live_frames(frames, b, Tn);
    const float mean = stats[2 * ((long long)b * gridDim.x + g)], rstd = stats[2 * ((long long)b * gridDim.x + g) + 1];
    float p = 0.0f, q = 0.0f;
    for (int c = g * n; c < (g + 1) * n; ++c) {
        const float ga = gamma ? gl_to_f32(gamma[c]) : 1.0f, be = beta ? gl_to_f32(beta[c]) : 0.0f;
        float a0 = 0.0f, a1 = 0.0f;
        for (int t = threadIdx.x; t < live; t += 256) {
            const long long row = (long long)b * Tn + t;
            const float xh = (gl_to_f32(x[row * x_stride + c]) - mean) * rstd;
            const float du = gl_to_f32(dy[row * dy_stride + c]) * gl_act_grad(xh * ga + be, act);
            a0 += du * xh;
            a1 += du;
        }
        a0 = block_sum(a0, s);
        a1 = block_sum(a1, s);
        if (threadIdx.x == 0) {
            parts[((long long)b * 2 + 0) * C + c] = a0;
            parts[((long long)b * 2 + 1) * C + c] = a1;
        }
        p += a1 * ga;
        q += a0 * ga;
    }
    if (threadIdx.x == 0) {
        const float count = (float)((long long)live * n);
        float* o = pq + 2 * ((long long)b * gridDim.x + g);
        o[0] = live ? p / count : 0.0f;
        o[1] = live ? q / count : 0.0f;
    }
}

template <typename T>
__global__ void __launch_bounds__(256) k_norm_back_apply(const T* __restrict__ dy, long long dy_stride,
                                                         const T* __restrict__ x, long long x_stride,
                                                         const float* __restrict__ stats, const float* __restrict__ pq,
                                                         const T* __restrict__ gamma, const T* __restrict__ beta,
                                                         const int* __restrict__ frames, T* __restrict__ dx,
                                                         long long dx_stride, int Tn, int C, int n, int act) {
    const int b = blockIdx.y;
    const int live = live_frames(frames, b, Tn);
    const int G = C / n;
    const long long count = (long long)Tn * C;
    for (long long e = (long long)blockIdx.x * 256 + threadIdx.x; e < count; e += (long long)gridDim.x * 256) {
        const int t = (int)(e / C), c = (int)(e % C);
        const long long row = (long long)b * Tn + t;
        float v = 0.0f;
        if (t < live) {
            const float* st = stats + 2 * ((long long)b * G + c / n);
            const float* o = pq + 2 * ((long long)b * G + c / n);
            const float ga = gamma ? gl_to_f32(gamma[c]) : 1.0f, be = beta ? gl_to_f32(beta[c]) : 0.0f;
            const float xh = (gl_to_f32(x[row * x_stride + c]) - st[0]) * st[1];
            const float du = gl_to_f32(dy[row * dy_stride + c]) * gl_act_grad(xh * ga + be, act);
            v = st[1] * (du * ga - o[0] - xh * o[1]);
        }
        dx[row * dx_stride + c] = (T)v;
    }
}

template <typename T>
__global__ void __launch_bounds__(256) k_norm_back_join(const float* __restrict__ parts, T* __restrict__ dgamma,
                                                        T* __restrict__ dbeta, int B, int C) {
    const int c = blockIdx.x * 256 + threadIdx.x;
    if (c >= C) return;
    float a0 = 0.0f, a1 = 0.0f;
    for (int b = 0; b < B; ++b) {
        a0 += parts[((long long)b * 2 + 0) * C + c];
        a1 += parts[((long long)b * 2 + 1) * C + c];
    }
    if (dgamma) dgamma[c] = (T)a0;
    if (dbeta) dbeta[c] = (T)a1;
}

inline long long ceil_div(long long a, long long b) { return (a + b - 1) / b; }
inline long long align16(long long b) { return (b + 15) / 16 * 16; }

int check_norm(int B, int T, int C, int groups, int dtype, int act, const char* who) {
    if (dtype < GL_F32 || dtype > GL_F16) return gl_set_error(GL_ERR_INVALID, "%s: dtype=%d", who, dtype);
    if (act < GL_ACT_NONE || act > GL_ACT_EXP) return gl_set_error(GL_ERR_INVALID, "%s: activation=%d", who, act);
    if (B < 0 || B > 65535) return gl_set_error(GL_ERR_INVALID, "%s: B=%d outside [0, 65535]", who, B);
    if (T < 0) return gl_set_error(GL_ERR_INVALID, "%s: T=%d", who, T);
    if (C < 1 || C > (1 << 20)) return gl_set_error(GL_ERR_INVALID, "%s: channels=%d outside [1, 2^20]", who, C);
    if (groups < 1 || groups > C || C % groups)
        return gl_set_error(GL_ERR_INVALID, "%s: %d channels do not divide into %d groups", who, C, groups);
    return 0;
}
int check_stride(long long stride, int cols, const char* what, const char* who) {
    if (stride < cols || stride > (1LL << 31))
        return gl_set_error(GL_ERR_INVALID, "%s: %s row stride %lld outside [%d, 2^31]", who, what, stride, cols);
    return 0;
}
int check_workspace(const void* ws, long long have, long long need, const char* who) {
    if (!ws || have < need)
        return gl_set_error(GL_ERR_INVALID, "%s: workspace of %lld bytes needed, %lld given", who, need, ws ? have : 0LL);
    if ((uintptr_t)ws % 16) return gl_set_error(GL_ERR_INVALID, "%s: workspace must be 16-byte aligned", who);
    return 0;
}
long long stats_bytes(int B, int groups) { return align16(8LL * B * groups); }

unsigned apply_blocks(int B, int T, int C) {
    long long per = ceil_div((long long)T * C, 256 * 8), most = 256 * 16 / B;
    if (most < 1) most = 1;
    return (unsigned)(per < 1 ? 1 : per < most ? per : most);
}

template <typename T>
int norm(const void* x, long long x_stride, const void* gamma, const void* beta, const int* frames, void* y,
         long long y_stride, float* stats, int B, int Tn, int C, int groups, int act, float eps, hipStream_t st) {
    const int n = C / groups;
    hipLaunchKernelGGL((k_norm_stats<T>), dim3(groups, B), dim3(256), 0, st, (const T*)x, x_stride, frames, stats, Tn, n, eps);
    GL_HIP_CHECK(hipGetLastError());
    hipLaunchKernelGGL((k_norm_apply<T>), dim3(apply_blocks(B, Tn, C), B), dim3(256), 0, st, (const T*)x, x_stride,
                       (const T*)gamma, (const T*)beta, frames, stats, (T*)y, y_stride, Tn, C, n, act);
    GL_HIP_CHECK(hipGetLastError());
    return 0;
}

template <typename T>
int norm_back(const void* dy, long long dy_stride, const void* x, long long x_stride, const float* stats, const void* gamma,
              const void* beta, const int* frames, void* dx, long long dx_stride, void* dgamma, void* dbeta, int B, int Tn,
              int C, int groups, int act, void* ws, hipStream_t st) {
    const int n = C / groups;
    float* pq = (float*)ws;
    float* parts = (float*)((char*)ws + stats_bytes(B, groups));
    if (B > 0 && Tn > 0) {
        hipLaunchKernelGGL((k_norm_back_sums<T>), dim3(groups, B), dim3(256), 0, st, (const T*)dy, dy_stride, (const T*)x,
                           x_stride, stats, (const T*)gamma, (const T*)beta, frames, parts, pq, Tn, C, n, act);
        GL_HIP_CHECK(hipGetLastError());
        if (dx) {
            hipLaunchKernelGGL((k_norm_back_apply<T>), dim3(apply_blocks(B, Tn, C), B), dim3(256), 0, st, (const T*)dy, dy_stride,
                               (const T*)x, x_stride, stats, pq, (const T*)gamma, (const T*)beta, frames, (T*)dx, dx_stride, Tn,
                               C, n, act);
            GL_HIP_CHECK(hipGetLastError());
        }
    }
    if (dgamma || dbeta) {
        hipLaunchKernelGGL((k_norm_back_join<T>), dim3((unsigned)ceil_div(C, 256)), dim3(256), 0, st, parts, (T*)dgamma,
                           (T*)dbeta, Tn > 0 ? B : 0, C);
        GL_HIP_CHECK(hipGetLastError());
    }
    return 0;
}

}  // namespace

extern "C" {

long long gl_group_norm_workspace(int B, int T, int channels, int groups, int dtype) {
    if (check_norm(B, T, channels, groups, dtype, 0, "gl_group_norm_workspace")) return GL_ERR_INVALID;
    return stats_bytes(B, groups);
}

int gl_group_norm(const void* x, long long x_stride, const void* gamma, const void* beta, const int* frames, void* y,
                  long long y_stride, float* stats, int B, int T, int channels, int groups, int dtype, int activation,
                  float eps, void* workspace, long long workspace_bytes, void* stream) {
    int rc = check_norm(B, T, channels, groups, dtype, activation, "gl_group_norm");
    if (!rc && !(eps >= 0.0f)) rc = gl_set_error(GL_ERR_INVALID, "gl_group_norm: eps=%g", (double)eps);
    if (rc || B == 0) return rc;
    if (T > 0 && (!x || !y)) return gl_set_error(GL_ERR_INVALID, "gl_group_norm: NULL buffer");
    rc = check_stride(x_stride, channels, "x", "gl_group_norm");
    if (!rc) rc = check_stride(y_stride, channels, "y", "gl_group_norm");
    if (!rc) rc = check_workspace(workspace, workspace_bytes, stats_bytes(B, groups), "gl_group_norm");
    if (rc) return rc;
    if (T == 0 && !stats) return 0;
    float* s = stats ? stats : (float*)workspace;
    const hipStream_t st = (hipStream_t)stream;
#define GL_NORM(T_)                                                                                                     \
    norm<T_>(x, x_stride, gamma, beta, frames, y, y_stride, s, B, T, channels, groups, activation, eps, st)
    return dtype == GL_F32 ? GL_NORM(float) : dtype == GL_BF16 ? GL_NORM(gl_bf16) : GL_NORM(gl_f16);
#undef GL_NORM
}

long long gl_group_norm_backward_workspace(int B, int T, int channels, int groups, int dtype) {
    if (check_norm(B, T, channels, groups, dtype, 0, "gl_group_norm_backward_workspace")) return GL_ERR_INVALID;
    return stats_bytes(B, groups) + align16(8LL * B * channels);
}

int gl_group_norm_backward(const void* dy, long long dy_stride, const void* x, long long x_stride, const float* stats,
                           const void* gamma, const void* beta, const int* frames, void* dx, long long dx_stride,
                           void* dgamma, void* dbeta, int B, int T, int channels, int groups, int dtype,
                           int activation, void* workspace, long long workspace_bytes, void* stream) {
    int rc = check_norm(B, T, channels, groups, dtype, activation, "gl_group_norm_backward");
    if (rc) return rc;
    if (B > 0 && T > 0) {
        if (!dy || !x || !stats) return gl_set_error(GL_ERR_INVALID, "gl_group_norm_backward: NULL buffer");
        rc = check_stride(dy_stride, channels, "dy", "gl_group_norm_backward");
        if (!rc) rc = check_stride(x_stride, channels, "x", "gl_group_norm_backward");
        if (!rc && dx) rc = check_stride(dx_stride, channels, "dx", "gl_group_norm_backward");
        if (!rc)
            rc = check_workspace(workspace, workspace_bytes,
                                 gl_group_norm_backward_workspace(B, T, channels, groups, dtype), "gl_group_norm_backward");
        if (rc) return rc;
    }
    const hipStream_t st = (hipStream_t)stream;
#define GL_NORM(T_)                                                                                                     \
    norm_back<T_>(dy, dy_stride, x, x_stride, stats, gamma, beta, frames, dx, dx_stride, dgamma, dbeta, B, T, channels, \
                  groups, activation, workspace, st)
    return dtype == GL_F32 ? GL_NORM(float) : dtype == GL_BF16 ? GL_NORM(gl_bf16) : GL_NORM(gl_f16);
#undef GL_NORM
}

}  // extern "C"
