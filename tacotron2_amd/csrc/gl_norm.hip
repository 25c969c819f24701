// Group norm with an activation, channels last, and its gradients (include/gl_hip.h).
//
//   xh = (x - mean) rstd,  y = act(xh gamma + beta)          mean, rstd per (utterance, group) over its live frames
//   du = dy act'(xh gamma + beta);  v = du gamma;  p = mean(v), q = mean(v xh) per (utterance, group)
//   dx = rstd (v - p - xh q);  dgamma = sum du xh,  dbeta = sum du per channel over all live frames
//
// Bound by memory: x (and dy) in once, the result out once.  A workgroup that can hold its frames of some whole groups in
// registers (16 bytes x 8 a thread) does everything in one pass: "slab" kernels.  Longer utterances are cut into chunks of
// frames: statistics (sums) of the chunks, their join, and a second pass that applies them, the input then coming from the
// 256 MB cache behind the L2s where it fits.  Variances are sums of squared distances from a mean already known (of the slab
// or the chunk, joined with the distances between the means), never a difference of large sums.  All sums run in a
// fixed order.
#include <initializer_list>

#include "gl_internal.h"
#include "gl_act.h"

namespace {

constexpr int kHeld = 8;                 // vectors of V channels a thread holds
constexpr int kMaxThreads = 1024;
// Bytes of a slab's rows where whole groups and the chip allow.  64 ragged utterances of 861 x 512 bf16 with 32: 28.9 us, 64: 28.3,
// 128: 32; their gradients 58, 62, 70.
constexpr int kRowBytes = 64, kBackRowBytes = 32;
// threads of a gradient slab: it holds x and du in registers (16-bit: 96 of them, 1024 threads would spill)
template <typename T> constexpr int kBackThreads = sizeof(T) == 2 ? 512 : 1024;

__device__ __forceinline__ int live_frames(const int* frames, int b, int T) {
    return frames ? max(0, min(frames[b], T)) : T;
}

template <typename T, int V> struct vec_of { typedef T type __attribute__((ext_vector_type(V))); };
template <typename T> struct vec_of<T, 1> { typedef T type; };
template <typename T, int V>
__device__ __forceinline__ float get(const typename vec_of<T, V>::type& v, int k) {
    if constexpr (V == 1) return gl_to_f32(v);
    else return gl_to_f32(v[k]);
}
template <typename T, int V>
__device__ __forceinline__ void set(typename vec_of<T, V>::type& v, int k, float f) {
    if constexpr (V == 1) v = (T)f;
    else v[k] = (T)f;
}

// f(gl_int<the activation>): the kernel's own where it has one, else the argument's, chosen once around f's loop
template <int ACT, typename F>
__device__ __forceinline__ void act_for(int act, const F& f) {
    if constexpr (ACT < 0) gl_with_act(act, f);
    else f(gl_int<ACT>());
}

// Where a workgroup works: CB channels from c0 (whole groups), threads as rows x TP vectors.
struct Place {
    int CB, TP, RP, r, col;              // channels, threads per row, rows at a time, this thread's row and first channel
    bool on;
};
template <int V>
__device__ __forceinline__ Place place(int CB) {
    Place p;
    p.CB = CB;
    p.TP = CB / V;
    p.RP = blockDim.x / p.TP;
    p.r = threadIdx.x / p.TP;
    p.col = (threadIdx.x - p.r * p.TP) * V;
    p.on = p.r < p.RP;
    return p;
}

// Sums of v (V channels a thread) over the workgroup's rows, per channel, to tot[CB]; red: blockDim.x * V floats.
template <int V>
__device__ __forceinline__ void channel_sums(const float (&v)[V], const Place& p, float* red, float* tot) {
    __syncthreads();
    if (p.on)
#pragma unroll
        for (int k = 0; k < V; ++k) red[p.r * p.CB + p.col + k] = v[k];
    __syncthreads();
    // rows in `segs` interleaved segments first where there are threads for it, then the segments
    const int nt = blockDim.x;
    const int segs = min(p.RP, nt / p.CB);
    if (segs > 1) {
        const int c = threadIdx.x % p.CB, s = threadIdx.x / p.CB;
        float a = 0.0f;
        if (s < segs)
            for (int r = s; r < p.RP; r += segs) a += red[r * p.CB + c];
        __syncthreads();
        if (s < segs) red[s * p.CB + c] = a;
        __syncthreads();
    }
    const int rows = segs > 1 ? segs : p.RP;
    for (int c = threadIdx.x; c < p.CB; c += nt) {
        float a = 0.0f;
        for (int r = 0; r < rows; ++r) a += red[r * p.CB + c];
        tot[c] = a;
    }
    __syncthreads();
}
// f(c) summed over the channels of each of the block's groups to out[group], a wave per group
template <typename F>
__device__ __forceinline__ void group_sums(const Place& p, int n, float* out, F f) {
    const int lane = threadIdx.x & 63, waves = blockDim.x / 64;
    for (int g = threadIdx.x / 64; g < p.CB / n; g += waves) {
        float a = 0.0f;
        for (int c = lane; c < n; c += 64) a += f(g * n + c);
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) a += __shfl_xor(a, o);
        if (lane == 0) out[g] = a;
    }
    __syncthreads();
}

// V values of gamma or beta from channel c on
template <typename T, int V>
__device__ __forceinline__ void load_vector(const T* p, int c, float none, float (&v)[V]) {
    typedef typename vec_of<T, V>::type vT;
    if (!p) {
#pragma unroll
        for (int k = 0; k < V; ++k) v[k] = none;
    } else if ((uintptr_t)p % sizeof(vT) == 0) {             // c is a multiple of V
        const vT t = *(const vT*)(p + c);
#pragma unroll
        for (int k = 0; k < V; ++k) v[k] = get<T, V>(t, k);
    } else {
#pragma unroll
        for (int k = 0; k < V; ++k) v[k] = gl_to_f32(p[c + k]);
    }
}
template <typename T, int V>
__device__ __forceinline__ void load_affine(const T* gamma, const T* beta, int c, float (&ga)[V], float (&be)[V]) {
    load_vector<T, V>(gamma, c, 1.0f, ga);
    load_vector<T, V>(beta, c, 0.0f, be);
}
// pairs [group][2] of the groups of channels c .. c + V - 1
template <int V>
__device__ __forceinline__ void load_pairs(const float* pairs, int c, int n, float (&first)[V], float (&second)[V]) {
    if (n % V == 0) {                                        // one group
        const float f = pairs[2 * (c / n)], g = pairs[2 * (c / n) + 1];
#pragma unroll
        for (int k = 0; k < V; ++k) {
            first[k] = f;
            second[k] = g;
        }
    } else {
#pragma unroll
        for (int k = 0; k < V; ++k) {
            first[k] = pairs[2 * ((c + k) / n)];
            second[k] = pairs[2 * ((c + k) / n) + 1];
        }
    }
}

// Vectors inside one group, rows and groups on whole powers of two of lanes: sums run through shuffles.
struct Lanes {
    bool even;
    int gl;                              // lanes of a row that share a group
};
template <int V>
__device__ __forceinline__ Lanes lanes_of(const Place& p, int n) {
    Lanes l;
    l.gl = n / V;
    l.even = n % V == 0 && (p.TP & (p.TP - 1)) == 0 && (l.gl & (l.gl - 1)) == 0 && l.gl <= 64;
    return l;
}
// The sum over rows and channels of this thread's group, in every thread.  red: floats, waves x lanes of a row's groups.
// Alternate two buffers between calls: only one barrier is inside.
__device__ __forceinline__ float group_total(float s, const Place& p, const Lanes& l, float* red) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
    for (int o = 1; o < l.gl; o <<= 1) s += __shfl_xor(s, o);
    for (int o = p.TP; o < 64; o <<= 1) s += __shfl_xor(s, o);
    const int per = min(p.TP, 64);                           // lanes of a row in a wave; TP / per waves make a row
    const int slot = (lane & (per - 1)) / l.gl, slots = per / l.gl;
    if (lane < per && (lane & (l.gl - 1)) == 0) red[wave * slots + slot] = s;
    __syncthreads();
    const int seg = p.TP / per;
    s = 0.0f;
    for (int w = wave % seg; w < waves; w += seg) s += red[w * slots + slot];
    return s;
}
template <int V>
__device__ __forceinline__ float total(const float (&v)[V]) {
    float s = v[0];
#pragma unroll
    for (int k = 1; k < V; ++k) s += v[k];
    return s;
}
// Sums over rows per channel, where rows are whole powers of two of lanes: tot[CB] written, a barrier behind it.  red: waves x CB
template <int V>
__device__ __forceinline__ void channel_totals(float (&v)[V], const Place& p, float* red, float* tot) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
    for (int o = p.TP; o < 64; o <<= 1)
#pragma unroll
        for (int k = 0; k < V; ++k) v[k] += __shfl_xor(v[k], o);
    const int seg = max(1, p.TP / 64), width = p.CB / seg;   // channels of a wave
    if (lane < p.TP)
#pragma unroll
        for (int k = 0; k < V; ++k) red[wave * width + (lane & 63) * V + k] = v[k];
    __syncthreads();
    for (int c = threadIdx.x; c < p.CB; c += blockDim.x) {
        float a = 0.0f;
        for (int w = c / width; w < waves; w += seg) a += red[w * width + c % width];
        tot[c] = a;
    }
    __syncthreads();
}

// One pass: statistics and result of CB channels of utterance b.  grid (blocks of channels x B), see block_of().  Bound by
// memory and the activation's arithmetic in turn (a workgroup loads, sums, then writes; a CU holds few of them): 64 ragged
// utterances of 861 x 512 bf16 silu 25 us (94 MB, 3.7 TB/s); one utterance of 641 x 512 7.7 us.
// Neighbouring blocks share cache lines where CB channels are less than 128 bytes: they go to one XCD (ids 8 apart).
struct Blocks {
    int per_b, total;                    // blocks of channels per utterance, and in all
    int CB, C;                           // channels of a block (the last may have fewer), of a row
};
__device__ __forceinline__ bool block_of(const Blocks& k, int& b, int& c0, int& CB) {
    const int per = (k.total + 7) / 8;
    const int id = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
    if ((int)(blockIdx.x >> 3) >= per || id >= k.total) return false;
    b = id / k.per_b;
    c0 = (id - b * k.per_b) * k.CB;
    CB = min(k.CB, k.C - c0);
    return true;
}

// EVEN: see Lanes; one group a vector then, so its mean and deviation are single registers.
template <typename T, int V, int ACT, bool EVEN>
__global__ void __launch_bounds__(kMaxThreads) k_norm_slab(const T* x, long long x_stride, const T* __restrict__ gamma,
                                                           const T* __restrict__ beta, const int* __restrict__ frames,
                                                           T* y, long long y_stride, float* __restrict__ stats, int Tn, int n,
                                                           int act, float eps, Blocks blocks) {
    typedef typename vec_of<T, V>::type vT;
    extern __shared__ float lds[];
    int b, c0, CB;
    if (!block_of(blocks, b, c0, CB)) return;
    const Place p = place<V>(CB);
    float* red = lds;                                        // [threads * V]
    float* tot = red + blockDim.x * (V > 1 ? V : 2);                       // [CB]
    float* mean_g = tot + CB;                                // [CB / n] each
    float* rstd_g = mean_g + CB / n;
    const int live = live_frames(frames, b, Tn);
    const int c = c0 + p.col;
    const T* xb = x + (long long)b * Tn * x_stride + c;
    vT held[kHeld];
    float v[V];
#pragma unroll
    for (int k = 0; k < V; ++k) v[k] = 0.0f;
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
        const int t = p.r + i * p.RP;
        if (p.on && t < live) held[i] = *(const vT*)(xb + (long long)t * x_stride);
    }
#pragma unroll
    for (int i = 0; i < kHeld; ++i)
        if (p.on && p.r + i * p.RP < live)
#pragma unroll
            for (int k = 0; k < V; ++k) v[k] += get<T, V>(held[i], k);
    const float count = (float)((long long)live * n);
    const float inv = live ? 1.0f / count : 0.0f;
    const Lanes l = lanes_of<V>(p, n);
    float mean[V], ga[V], be[V];
    if (p.on) load_affine<T, V>(gamma, beta, c, ga, be);     // arrives under the sums
    const auto squares = [&] {
#pragma unroll
        for (int k = 0; k < V; ++k) v[k] = 0.0f;
#pragma unroll
        for (int i = 0; i < kHeld; ++i)
            if (p.on && p.r + i * p.RP < live)
#pragma unroll
                for (int k = 0; k < V; ++k) {
                    const float d = get<T, V>(held[i], k) - mean[k];
                    v[k] = fmaf(d, d, v[k]);
                }
    };
    if constexpr (EVEN) {
        const float m = group_total(total<V>(v), p, l, red) * inv;
#pragma unroll
        for (int k = 0; k < V; ++k) mean[k] = m;
        squares();
        const float m2 = group_total(total<V>(v), p, l, red + blockDim.x);
        const float rstd = live ? 1.0f / sqrtf(m2 * inv + eps) : 0.0f;
        if (stats && p.r == 0 && p.col % n == 0) {
            float* o = stats + 2 * ((long long)b * (blocks.C / n) + c / n);
            o[0] = m;
            o[1] = rstd;
        }
#pragma unroll
        for (int k = 0; k < V; ++k) ga[k] *= rstd;
    } else {
        channel_sums<V>(v, p, red, tot);
        group_sums(p, n, mean_g, [&](int k) { return tot[k]; });
#pragma unroll
        for (int k = 0; k < V; ++k) mean[k] = p.on ? mean_g[(p.col + k) / n] * inv : 0.0f;
        squares();
        channel_sums<V>(v, p, red, tot);
        group_sums(p, n, rstd_g, [&](int k) { return tot[k]; });
        for (int g = threadIdx.x; g < CB / n; g += blockDim.x) {
            const float rstd = live ? 1.0f / sqrtf(rstd_g[g] * inv + eps) : 0.0f;
            rstd_g[g] = rstd;
            if (stats) {
                float* o = stats + 2 * ((long long)b * (blocks.C / n) + c0 / n + g);
                o[0] = mean_g[g] * inv;
                o[1] = rstd;
            }
        }
        __syncthreads();
        if (p.on)
#pragma unroll
            for (int k = 0; k < V; ++k) ga[k] *= rstd_g[(p.col + k) / n];
    }
    if (!p.on) return;
    T* yb = y + (long long)b * Tn * y_stride + c;
    act_for<ACT>(act, [&](auto a) {
#pragma unroll
        for (int i = 0; i < kHeld; ++i) {
            const int t = p.r + i * p.RP;
            if (t >= Tn) continue;
            vT o = vT{};
            if (t < live)
#pragma unroll
                for (int k = 0; k < V; ++k) set<T, V>(o, k, gl_act<T>(fmaf(get<T, V>(held[i], k) - mean[k], ga[k], be[k]), decltype(a)::value));
            *(vT*)(yb + (long long)t * y_stride) = o;
        }
    });
}

// Chunks of RP * kHeld frames, all channels: mean and sum of squared distances per group.  grid (chunks, B);
// parts [B][groups][chunks][2].  51 680 x 256 float32: 12.5 us (4.2 TB/s), the join below 3.8, k_norm_apply 18 (5.9 TB/s, its
// input from the cache).
template <typename T, int V>
__global__ void __launch_bounds__(kMaxThreads) k_norm_chunk(const T* __restrict__ x, long long x_stride, const int* __restrict__ frames,
                                                    float* __restrict__ parts, int Tn, int C, int n) {
    typedef typename vec_of<T, V>::type vT;
    extern __shared__ float lds[];
    const Place p = place<V>(C);
    float* red = lds;
    float* tot = red + blockDim.x * (V > 1 ? V : 2);
    float* mean_g = tot + C;
    float* m2_g = mean_g + C / n;
    const int b = blockIdx.y, rows = p.RP * kHeld;
    const int live = live_frames(frames, b, Tn);
    const int t0 = blockIdx.x * rows, here = max(0, min(rows, live - t0));
    const T* xb = x + ((long long)b * Tn + t0) * x_stride + p.col;
    vT held[kHeld];
    float v[V], mean[V];
#pragma unroll
    for (int k = 0; k < V; ++k) v[k] = 0.0f;
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
        const int t = p.r + i * p.RP;
        if (p.on && t < here) held[i] = *(const vT*)(xb + (long long)t * x_stride);
    }
#pragma unroll
    for (int i = 0; i < kHeld; ++i)
        if (p.on && p.r + i * p.RP < here)
#pragma unroll
            for (int k = 0; k < V; ++k) v[k] += get<T, V>(held[i], k);
    const float inv = here ? 1.0f / (float)(here * n) : 0.0f;
    const Lanes l = lanes_of<V>(p, n);
    const auto squares = [&] {
#pragma unroll
        for (int k = 0; k < V; ++k) v[k] = 0.0f;
#pragma unroll
        for (int i = 0; i < kHeld; ++i)
            if (p.on && p.r + i * p.RP < here)
#pragma unroll
                for (int k = 0; k < V; ++k) {
                    const float d = get<T, V>(held[i], k) - mean[k];
                    v[k] = fmaf(d, d, v[k]);
                }
    };
    if (l.even) {
        const float m = group_total(total<V>(v), p, l, red) * inv;
#pragma unroll
        for (int k = 0; k < V; ++k) mean[k] = m;
        squares();
        const float m2 = group_total(total<V>(v), p, l, red + blockDim.x);
        if (p.r == 0 && p.col % n == 0) {
            float* o = parts + 2 * (((long long)b * (C / n) + p.col / n) * gridDim.x + blockIdx.x);
            o[0] = m;
            o[1] = m2;
        }
        return;
    }
    channel_sums<V>(v, p, red, tot);
    group_sums(p, n, mean_g, [&](int k) { return tot[k]; });
#pragma unroll
    for (int k = 0; k < V; ++k) mean[k] = p.on ? mean_g[(p.col + k) / n] * inv : 0.0f;
    squares();
    channel_sums<V>(v, p, red, tot);
    group_sums(p, n, m2_g, [&](int k) { return tot[k]; });
    for (int g = threadIdx.x; g < C / n; g += blockDim.x) {
        float* o = parts + 2 * (((long long)b * (C / n) + g) * gridDim.x + blockIdx.x);
        o[0] = mean_g[g] * inv;
        o[1] = m2_g[g];
    }
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

// grid (groups, B): joins the chunks' means and distances.  rows: frames of a chunk
__global__ void __launch_bounds__(256) k_norm_join(const float* __restrict__ parts, const int* __restrict__ frames,
                                                   float* __restrict__ stats, int Tn, int n, int chunks, int rows, float eps) {
    __shared__ float s[4];
    const int g = blockIdx.x, b = blockIdx.y;
    const int live = live_frames(frames, b, Tn);
    const float* in = parts + 2 * ((long long)b * gridDim.x + g) * chunks;
    auto frames_of = [&](int k) { return (float)max(0, min(rows, live - k * rows)); };
    float m = 0.0f;
    for (int k = threadIdx.x; k < chunks; k += 256) m += frames_of(k) * in[2 * k];
    m = live ? block_sum(m, s) / (float)live : 0.0f;
    float m2 = 0.0f;
    for (int k = threadIdx.x; k < chunks; k += 256) {
        const float d = in[2 * k] - m;
        m2 += in[2 * k + 1] + frames_of(k) * (float)n * d * d;
    }
    m2 = block_sum(m2, s);
    if (threadIdx.x == 0) {
        float* o = stats + 2 * ((long long)b * gridDim.x + g);
        o[0] = m;
        o[1] = live ? 1.0f / sqrtf(m2 / ((float)live * (float)n) + eps) : 0.0f;
    }
}

// grid (row blocks, B): y from x and the statistics
template <typename T, int V, int ACT>
__global__ void __launch_bounds__(kMaxThreads) k_norm_apply(const T* x, long long x_stride, const T* __restrict__ gamma,
                                                    const T* __restrict__ beta, const int* __restrict__ frames,
                                                    const float* __restrict__ stats, T* y, long long y_stride, int Tn, int C,
                                                    int n, int act) {
    typedef typename vec_of<T, V>::type vT;
    const Place p = place<V>(C);
    if (!p.on) return;
    const int b = blockIdx.y;
    const int live = live_frames(frames, b, Tn);
    float ga[V], be[V], mean[V];
    load_affine<T, V>(gamma, beta, p.col, ga, be);
    {
        float rstd[V];
        load_pairs<V>(stats + 2 * (long long)b * (C / n), p.col, n, mean, rstd);
#pragma unroll
        for (int k = 0; k < V; ++k) ga[k] *= rstd[k];
    }
    const T* xb = x + (long long)b * Tn * x_stride + p.col;
    T* yb = y + (long long)b * Tn * y_stride + p.col;
    const int step = gridDim.x * p.RP;
    act_for<ACT>(act, [&](auto a) {
#pragma unroll 4
        for (int t = blockIdx.x * p.RP + p.r; t < Tn; t += step) {
            vT o = vT{};
            if (t < live) {
                const vT in = *(const vT*)(xb + (long long)t * x_stride);
#pragma unroll
                for (int k = 0; k < V; ++k) set<T, V>(o, k, gl_act<T>(fmaf(get<T, V>(in, k) - mean[k], ga[k], be[k]), decltype(a)::value));
            }
            *(vT*)(yb + (long long)t * y_stride) = o;
        }
    });
}

// ---- gradients ----

// Of one element: d = x - mean and du; slope = rstd gamma.  Sums of du xh are those of du d, times rstd.
template <typename T, int V, int ACT>
__device__ __forceinline__ void du_d(const typename vec_of<T, V>::type& x, const typename vec_of<T, V>::type& dy, int k, float mean,
                                     float slope, float be, float& du, float& d) {
    d = get<T, V>(x, k) - mean;
    du = get<T, V>(dy, k) * gl_act_grad<T>(fmaf(d, slope, be), ACT);
}
// dx = rstd (du gamma - p - xh q) = du slope + d cq + cp
struct Back {
    float cp, cq;
};
__device__ __forceinline__ Back back_of(float rstd, float p, float q) { return {-rstd * p, -rstd * (rstd * q)}; }

// One pass, as k_norm_slab.  sums [B][2][C]: sum du xh, sum du per channel of the utterance.  64 ragged utterances of 861 x 512
// bf16 silu 43 us (131 MB, 3.0 TB/s): 157 registers leave three workgroups a CU, whose loads, sums and stores overlap little.  Four
// vectors a thread instead of eight, with more waves: 51 us; 64-byte rows in workgroups of 512: 47.
template <typename T, int V, int ACT, bool EVEN>
__global__ void __launch_bounds__(kBackThreads<T>) k_norm_back_slab(const T* dy, long long dy_stride, const T* __restrict__ x,
                                                                long long x_stride, const float* __restrict__ stats,
                                                                const T* __restrict__ gamma, const T* __restrict__ beta,
                                                                const int* __restrict__ frames, T* dx, long long dx_stride,
                                                                float* __restrict__ sums, int Tn, int n, int act, Blocks blocks) {
    typedef typename vec_of<T, V>::type vT;
    extern __shared__ float lds[];
    int b, c0, CB;
    if (!block_of(blocks, b, c0, CB)) return;
    const Place p = place<V>(CB);
    float* red = lds;
    float* tot = red + blockDim.x * (V > 1 ? V : 2);                       // [2][CB]
    float* pq = tot + 2 * CB;                                // [2][CB / n]
    const int live = live_frames(frames, b, Tn), C = blocks.C;
    const int c = c0 + p.col;
    const T* xb = x + (long long)b * Tn * x_stride + c;
    const T* db = dy + (long long)b * Tn * dy_stride + c;
    vT hx[kHeld], hd[kHeld];
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
        const int t = p.r + i * p.RP;
        if (p.on && t < live) {
            hx[i] = *(const vT*)(xb + (long long)t * x_stride);
            hd[i] = *(const vT*)(db + (long long)t * dy_stride);
        }
    }
    float du[kHeld][V];                                      // in place of dy from here on: the activation's slope is
                                                             // worked out once
    float ga[V], be[V], mean[V], rstd[V], slope[V], a0[V], a1[V];
#pragma unroll
    for (int k = 0; k < V; ++k) a0[k] = a1[k] = 0.0f;
    if (p.on) {
        load_affine<T, V>(gamma, beta, c, ga, be);
        if constexpr (EVEN) {
            const float* st = stats + 2 * ((long long)b * (C / n) + c / n);
            const float m = st[0], r = st[1];
#pragma unroll
            for (int k = 0; k < V; ++k) {
                mean[k] = m;
                rstd[k] = r;
            }
        } else {
            load_pairs<V>(stats + 2 * (long long)b * (C / n), c, n, mean, rstd);
        }
#pragma unroll
        for (int k = 0; k < V; ++k) slope[k] = rstd[k] * ga[k];
    }
#pragma unroll
    for (int i = 0; i < kHeld; ++i)
        if (p.on && p.r + i * p.RP < live)
            act_for<ACT>(act, [&](auto a) {
#pragma unroll
                for (int k = 0; k < V; ++k) {
                    float d;
                    du_d<T, V, decltype(a)::value>(hx[i], hd[i], k, mean[k], slope[k], be[k], du[i][k], d);
                    a0[k] = fmaf(du[i][k], d, a0[k]);
                    a1[k] += du[i][k];
                }
            });
    if (p.on)
#pragma unroll
        for (int k = 0; k < V; ++k) a0[k] *= rstd[k];
    const Lanes l = lanes_of<V>(p, n);
    const float scale = live ? 1.0f / (float)((long long)live * n) : 0.0f;
    Back end[V];
    if constexpr (EVEN) {
        float vp = 0.0f, vq = 0.0f;
#pragma unroll
        for (int k = 0; k < V; ++k) {
            vp = fmaf(a1[k], ga[k], vp);
            vq = fmaf(a0[k], ga[k], vq);
        }
        channel_totals<V>(a0, p, red, tot);
        channel_totals<V>(a1, p, red, tot + CB);
        for (int k = threadIdx.x; k < CB; k += blockDim.x) {
            sums[((long long)b * 2 + 0) * C + c0 + k] = tot[k];
            sums[((long long)b * 2 + 1) * C + c0 + k] = tot[CB + k];
        }
        if (!dx) return;
        vp = group_total(vp, p, l, red) * scale;
        vq = group_total(vq, p, l, red + blockDim.x) * scale;
#pragma unroll
        for (int k = 0; k < V; ++k) end[k] = back_of(rstd[k], vp, vq);
    } else {
        channel_sums<V>(a0, p, red, tot);
        channel_sums<V>(a1, p, red, tot + CB);
        for (int k = threadIdx.x; k < CB; k += blockDim.x) {
            sums[((long long)b * 2 + 0) * C + c0 + k] = tot[k];
            sums[((long long)b * 2 + 1) * C + c0 + k] = tot[CB + k];
            const float g = gamma ? gl_to_f32(gamma[c0 + k]) : 1.0f;
            tot[k] *= g;
            tot[CB + k] *= g;
        }
        if (!dx) return;
        __syncthreads();
        group_sums(p, n, pq, [&](int k) { return tot[CB + k]; });
        group_sums(p, n, pq + CB / n, [&](int k) { return tot[k]; });
        if (!p.on) return;
#pragma unroll
        for (int k = 0; k < V; ++k) end[k] = back_of(rstd[k], pq[(p.col + k) / n] * scale, pq[CB / n + (p.col + k) / n] * scale);
    }
    T* ob = dx + (long long)b * Tn * dx_stride + c;
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
        const int t = p.r + i * p.RP;
        if (t >= Tn) continue;
        vT o = vT{};
        if (t < live)
#pragma unroll
            for (int k = 0; k < V; ++k)
                set<T, V>(o, k, fmaf(du[i][k], slope[k], fmaf(get<T, V>(hx[i], k) - mean[k], end[k].cq, end[k].cp)));
        *(vT*)(ob + (long long)t * dx_stride) = o;
    }
}

// grid (chunks, B): per channel sums of a run of `rows` frames to parts [B][chunks][2][C].  51 680 x 256 f16 silu 15 us (53 MB,
// 3.5 TB/s), its join 3.9, k_norm_back_apply 18 (79 MB, 4.5 TB/s).
template <typename T, int V, int ACT>
__global__ void __launch_bounds__(kMaxThreads) k_norm_back_chunk(const T* __restrict__ dy, long long dy_stride, const T* __restrict__ x,
                                                         long long x_stride, const float* __restrict__ stats,
                                                         const T* __restrict__ gamma, const T* __restrict__ beta,
                                                         const int* __restrict__ frames, float* __restrict__ parts, int Tn, int C,
                                                         int n, int rows, int act) {
    typedef typename vec_of<T, V>::type vT;
    extern __shared__ float lds[];
    const Place p = place<V>(C);
    float* red = lds;
    float* tot = red + blockDim.x * (V > 1 ? V : 2);
    const int b = blockIdx.y;
    const int live = live_frames(frames, b, Tn);
    const int t0 = blockIdx.x * rows, t1 = min(t0 + rows, live);
    float slope[V], be[V], mean[V], rstd[V], a0[V], a1[V];
#pragma unroll
    for (int k = 0; k < V; ++k) a0[k] = a1[k] = 0.0f;
    if (p.on) {
        load_affine<T, V>(gamma, beta, p.col, slope, be);
        load_pairs<V>(stats + 2 * (long long)b * (C / n), p.col, n, mean, rstd);
#pragma unroll
        for (int k = 0; k < V; ++k) slope[k] *= rstd[k];
        const T* xb = x + (long long)b * Tn * x_stride + p.col;
        const T* db = dy + (long long)b * Tn * dy_stride + p.col;
        act_for<ACT>(act, [&](auto a) {
#pragma unroll 4
            for (int t = t0 + p.r; t < t1; t += p.RP) {
                const vT vx = *(const vT*)(xb + (long long)t * x_stride);
                const vT vd = *(const vT*)(db + (long long)t * dy_stride);
#pragma unroll
                for (int k = 0; k < V; ++k) {
                    float du, d;
                    du_d<T, V, decltype(a)::value>(vx, vd, k, mean[k], slope[k], be[k], du, d);
                    a0[k] = fmaf(du, d, a0[k]);
                    a1[k] += du;
                }
            }
        });
#pragma unroll
        for (int k = 0; k < V; ++k) a0[k] *= rstd[k];
    }
    float* o = parts + ((long long)b * gridDim.x + blockIdx.x) * 2 * C;
    const bool even = (p.TP & (p.TP - 1)) == 0;
    if (even) channel_totals<V>(a0, p, red, tot);
    else channel_sums<V>(a0, p, red, tot);
    for (int c = threadIdx.x; c < C; c += blockDim.x) o[c] = tot[c];
    __syncthreads();
    if (even) channel_totals<V>(a1, p, red, tot);
    else channel_sums<V>(a1, p, red, tot);
    for (int c = threadIdx.x; c < C; c += blockDim.x) o[C + c] = tot[c];
}

// grid (blocks of 16 of the 2 C columns, utterances): sums [2][C] over the parts [parts][2][C]; thread (column, one of 64
// lanes over the parts).  Few workgroups on little data: what counts is how many loads run at once (1024 parts of 2 x 256: 3.9 us,
// with 16 lanes 7.4).  affine: these are dgamma and dbeta.
template <typename T>
__global__ void __launch_bounds__(1024) k_norm_back_join(const float* __restrict__ parts, float* __restrict__ sums,
                                                         T* __restrict__ dgamma, T* __restrict__ dbeta, int C, int n_parts,
                                                         bool affine) {
    __shared__ float s[16][16];
    const int k = threadIdx.x & 15, l = threadIdx.x >> 4, c = blockIdx.x * 16 + k, b = blockIdx.y;
    float a = 0.0f;
    if (c < 2 * C) {
        const float* in = parts + (long long)b * n_parts * 2 * C + c;
#pragma unroll 8
        for (int j = l; j < n_parts; j += 64) a += in[(long long)j * 2 * C];
    }
    a += __shfl_xor(a, 16);
    a += __shfl_xor(a, 32);
    if ((l & 3) == 0) s[l >> 2][k] = a;
    __syncthreads();
    if (l || c >= 2 * C) return;
    a = s[0][k];
#pragma unroll
    for (int j = 1; j < 16; ++j) a += s[j][k];
    if (sums) sums[(long long)b * 2 * C + c] = a;
    if (!affine) return;
    if (c < C && dgamma) dgamma[c] = (T)a;
    if (c >= C && dbeta) dbeta[c - C] = (T)a;
}

template <typename T, int V, int ACT>
__global__ void __launch_bounds__(kMaxThreads) k_norm_back_apply(const T* dy, long long dy_stride, const T* __restrict__ x,
                                                         long long x_stride, const float* __restrict__ stats,
                                                         const float* __restrict__ sums, const T* __restrict__ gamma,
                                                         const T* __restrict__ beta, const int* __restrict__ frames, T* dx,
                                                         long long dx_stride, int Tn, int C, int n, int act) {
    typedef typename vec_of<T, V>::type vT;
    extern __shared__ float lds[];                           // [2][C] weighted sums, [groups][2] p, q
    const Place p = place<V>(C);
    const int b = blockIdx.y;
    const int live = live_frames(frames, b, Tn);
    float slope[V], be[V], mean[V], rstd[V];
    if (p.on) {
        load_affine<T, V>(gamma, beta, p.col, slope, be);
        load_pairs<V>(stats + 2 * (long long)b * (C / n), p.col, n, mean, rstd);
    }
    float* pairs = lds + 2 * C;
    for (int c = threadIdx.x; c < C; c += blockDim.x) {
        const float g = gamma ? gl_to_f32(gamma[c]) : 1.0f;
        lds[c] = sums[((long long)b * 2 + 0) * C + c] * g;
        lds[C + c] = sums[((long long)b * 2 + 1) * C + c] * g;
    }
    __syncthreads();
    const float scale = live ? 1.0f / (float)((long long)live * n) : 0.0f;
    for (int g = threadIdx.x >> 6; g < C / n; g += blockDim.x >> 6) {
        float sp = 0.0f, sq = 0.0f;
        for (int c = threadIdx.x & 63; c < n; c += 64) {
            sp += lds[C + g * n + c];
            sq += lds[g * n + c];
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) {
            sp += __shfl_xor(sp, o);
            sq += __shfl_xor(sq, o);
        }
        if ((threadIdx.x & 63) == 0) {
            pairs[2 * g] = sp * scale;
            pairs[2 * g + 1] = sq * scale;
        }
    }
    __syncthreads();
    if (!p.on) return;
    Back end[V];
    {
        float gp[V], gq[V];
        load_pairs<V>(pairs, p.col, n, gp, gq);
#pragma unroll
        for (int k = 0; k < V; ++k) {
            slope[k] *= rstd[k];
            end[k] = back_of(rstd[k], gp[k], gq[k]);
        }
    }
    const T* xb = x + (long long)b * Tn * x_stride + p.col;
    const T* db = dy + (long long)b * Tn * dy_stride + p.col;
    T* ob = dx + (long long)b * Tn * dx_stride + p.col;
    const int step = gridDim.x * p.RP;
    act_for<ACT>(act, [&](auto a) {
#pragma unroll 2
        for (int t = blockIdx.x * p.RP + p.r; t < Tn; t += step) {
            vT o = vT{};
            if (t < live) {
                const vT vx = *(const vT*)(xb + (long long)t * x_stride);
                const vT vd = *(const vT*)(db + (long long)t * dy_stride);
#pragma unroll
                for (int k = 0; k < V; ++k) {
                    float du, d;
                    du_d<T, V, decltype(a)::value>(vx, vd, k, mean[k], slope[k], be[k], du, d);
                    set<T, V>(o, k, fmaf(du, slope[k], fmaf(d, end[k].cq, end[k].cp)));
                }
            }
            *(vT*)(ob + (long long)t * dx_stride) = o;
        }
    });
}

// ---- rows that no workgroup spans (more than 1024 vectors, or channels of 64 KiB of sums), element by element: 8 x 861 x 2050
// float32 in 2 groups 89 us (44 for the chunks, 41 to apply; 113 MB), its gradients 78 ----

// grid (groups, B, chunks of `rows` frames): as k_norm_chunk
template <typename T>
__global__ void __launch_bounds__(256) k_norm_plain_chunk(const T* __restrict__ x, long long stride, const int* __restrict__ frames,
                                                    float* __restrict__ parts, int Tn, int n, int rows) {
    __shared__ float s[4];
    const int g = blockIdx.x, b = blockIdx.y, k = blockIdx.z;
    const int t0 = k * rows, here = max(0, min(rows, live_frames(frames, b, Tn) - t0));
    const T* base = x + ((long long)b * Tn + t0) * stride + (long long)g * n;
    // 256 threads on `across` channels of 256 / across frames at a time
    const int across = min(n, 256), c0 = threadIdx.x % across, r0 = threadIdx.x / across, step = 256 / across;
    const float inv = here ? 1.0f / ((float)here * (float)n) : 0.0f;
    float sum = 0.0f;
    if (r0 < step)
        for (int t = r0; t < here; t += step)
            for (int c = c0; c < n; c += across) sum += gl_to_f32(base[t * stride + c]);
    const float mean = block_sum(sum, s) * inv;
    float m2 = 0.0f;
    if (r0 < step)
        for (int t = r0; t < here; t += step)
            for (int c = c0; c < n; c += across) {
                const float d = gl_to_f32(base[t * stride + c]) - mean;
                m2 = fmaf(d, d, m2);
            }
    m2 = block_sum(m2, s);
    if (threadIdx.x == 0) {
        float* o = parts + 2 * (((long long)b * gridDim.x + g) * gridDim.z + k);
        o[0] = mean;
        o[1] = m2;
    }
}

template <typename T>
__global__ void __launch_bounds__(256) k_norm_plain_apply(const T* x, long long x_stride, const T* __restrict__ gamma,
                                                    const T* __restrict__ beta, const int* __restrict__ frames,
                                                    const float* __restrict__ stats, T* y, long long y_stride,
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
            v = gl_act<T>(xh * (gamma ? gl_to_f32(gamma[c]) : 1.0f) + (beta ? gl_to_f32(beta[c]) : 0.0f), act);
        }
        y[row * y_stride + c] = (T)v;
    }
}

// grid (blocks of 256 channels, B, chunks): as k_norm_back_chunk, a thread a channel
template <typename T>
__global__ void __launch_bounds__(256) k_norm_plain_back_chunk(const T* __restrict__ dy, long long dy_stride, const T* __restrict__ x,
                                                        long long x_stride, const float* __restrict__ stats,
                                                        const T* __restrict__ gamma, const T* __restrict__ beta,
                                                        const int* __restrict__ frames, float* __restrict__ parts, int Tn, int C,
                                                        int n, int rows, int act) {
    const int c = blockIdx.x * 256 + threadIdx.x, b = blockIdx.y, k = blockIdx.z;
    if (c >= C) return;
    const int t0 = k * rows, here = max(0, min(rows, live_frames(frames, b, Tn) - t0));
    const float* st = stats + 2 * ((long long)b * (C / n) + c / n);
    const float mean = st[0], rstd = st[1];
    const float slope = rstd * (gamma ? gl_to_f32(gamma[c]) : 1.0f), be = beta ? gl_to_f32(beta[c]) : 0.0f;
    const T* xb = x + ((long long)b * Tn + t0) * x_stride + c;
    const T* db = dy + ((long long)b * Tn + t0) * dy_stride + c;
    float a0 = 0.0f, a1 = 0.0f;
#pragma unroll 4
    for (int t = 0; t < here; ++t) {
        const float d = gl_to_f32(xb[t * x_stride]) - mean;
        const float du = gl_to_f32(db[t * dy_stride]) * gl_act_grad<T>(fmaf(d, slope, be), act);
        a0 = fmaf(du, d, a0);
        a1 += du;
    }
    float* o = parts + ((long long)b * gridDim.z + k) * 2 * C;
    o[c] = a0 * rstd;
    o[C + c] = a1;
}

// grid (groups, B): p and q of a group from the sums [B][2][C]
template <typename T>
__global__ void __launch_bounds__(256) k_norm_plain_back_pq(const float* __restrict__ sums, const T* __restrict__ gamma,
                                                      const int* __restrict__ frames, float* __restrict__ pq, int Tn, int C, int n) {
    __shared__ float s[4];
    const int g = blockIdx.x, b = blockIdx.y, live = live_frames(frames, b, Tn);
    float p = 0.0f, q = 0.0f;
    for (int c = g * n + threadIdx.x; c < (g + 1) * n; c += 256) {
        const float ga = gamma ? gl_to_f32(gamma[c]) : 1.0f;
        q = fmaf(sums[((long long)b * 2 + 0) * C + c], ga, q);
        p = fmaf(sums[((long long)b * 2 + 1) * C + c], ga, p);
    }
    p = block_sum(p, s);
    q = block_sum(q, s);
    if (threadIdx.x == 0) {
        const float inv = live ? 1.0f / ((float)live * (float)n) : 0.0f;
        float* o = pq + 2 * ((long long)b * gridDim.x + g);
        o[0] = p * inv;
        o[1] = q * inv;
    }
}

template <typename T>
__global__ void __launch_bounds__(256) k_norm_plain_back_apply(const T* dy, long long dy_stride,
                                                         const T* __restrict__ x, long long x_stride,
                                                         const float* __restrict__ stats, const float* __restrict__ pq,
                                                         const T* __restrict__ gamma, const T* __restrict__ beta,
                                                         const int* __restrict__ frames, T* dx,
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
            const float du = gl_to_f32(dy[row * dy_stride + c]) * gl_act_grad<T>(xh * ga + be, act);
            v = st[1] * (du * ga - o[0] - xh * o[1]);
        }
        dx[row * dx_stride + c] = (T)v;
    }
}

// ---- host ----

inline long long ceil_div(long long a, long long b) { return (a + b - 1) / b; }
inline long long align16(long long b) { return (b + 15) / 16 * 16; }

int check_norm(int B, int T, int C, int groups, int dtype, int act, const char* who) {
    if (dtype < GL_F32 || dtype > GL_F16) return gl_set_error(GL_ERR_INVALID, "%s: dtype=%d", who, dtype);
    if (act < GL_ACT_NONE || act > GL_ACT_EXP) return gl_set_error(GL_ERR_INVALID, "%s: activation=%d", who, act);
    if (B < 0 || B > 65535) return gl_set_error(GL_ERR_INVALID, "%s: B=%d outside [0, 65535]", who, B);
    if (T < 0 || T > (1 << 30)) return gl_set_error(GL_ERR_INVALID, "%s: T=%d outside [0, 2^30]", who, T);
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
// Elements start on whole multiples of their own size.
int check_elements(std::initializer_list<const void*> arrays, int size, const char* who) {
    for (const void* p : arrays)
        if ((uintptr_t)p % size) return gl_set_error(GL_ERR_INVALID, "%s: %p is not on its elements' size", who, p);
    return 0;
}
int check_workspace(const void* ws, long long have, long long need, const char* who) {
    if (need == 0) return 0;
    if (!ws || have < need)
        return gl_set_error(GL_ERR_INVALID, "%s: workspace of %lld bytes needed, %lld given", who, need, ws ? have : 0LL);
    if ((uintptr_t)ws % 16) return gl_set_error(GL_ERR_INVALID, "%s: workspace must be 16-byte aligned", who);
    return 0;
}

long long stats_bytes(int B, int groups) { return align16(8LL * B * groups); }

size_t lds_bytes(int threads, int V, int CB, int n, int totals) {
    return sizeof(float) * ((size_t)threads * (V > 1 ? V : 2) + (size_t)totals * CB + 2 * (size_t)(CB / n));
}
constexpr size_t kMaxLds = 65536;

// How a call is cut.  kind 0: slabs, 1: chunks, 2: element by element (rows that no workgroup spans)
struct Cut {
    int kind, threads;
    Blocks blocks;                       // slabs
    int rows, chunks;                    // chunks: frames of one, and how many
};
// Chunks of the gradients' sums, two workgroups a CU: 51 680 x 256 bf16 in 256 chunks 36.6 us, 512: 36.4, 1024: 43.7, 2048: 46.8
constexpr int kWorkgroups = 512;
int threads_for(int tp, long long rows, int most) {          // the fewest threads whose rows hold `rows` frames, or 0
    for (int t = 256; t <= most; t *= 2)
        if (t >= tp && (long long)(t / tp) * kHeld >= rows) return t;
    return 0;
}
Cut cut_for(int B, int T, int C, int groups, int size, int V, int most, int row_bytes) {
    Cut c = {};
    const int n = C / groups;
    int k = 1;
    while (k < groups && (n * k) % V) ++k;                   // whole groups on whole vectors
    if (n * k % V == 0 && threads_for(n * k / V, T, most) && lds_bytes(kMaxThreads, V, n * k, n, 2) <= kMaxLds) {
        // more groups to a block, to row_bytes a row, while the slab fits and the blocks fill the chip
        for (int m = 2 * k; m <= groups && (long long)n * k * size < row_bytes; m += k)
            if (groups % m == 0 && threads_for(n * m / V, T, most) && (long long)B * (groups / m) >= 256) k = m;
        c.kind = 0;
        c.threads = threads_for(n * k / V, T, most);
        c.blocks = {(int)ceil_div(groups, k), 0, n * k, C};
        const long long total = (long long)B * c.blocks.per_b;
        if (total * c.threads < 0xff000000LL) {              // what one launch can have
            c.blocks.total = (int)total;
            return c;
        }
        c = {};
    }
    if (C / V > kMaxThreads || lds_bytes(kMaxThreads, V, C, n, 1) > kMaxLds) {
        c.kind = 2;
        const long long chunks = 1024 / ((long long)B * groups);
        c.rows = (int)ceil_div(T, chunks < 1 ? 1 : chunks);
        if (c.rows < 1) c.rows = 1;
        c.chunks = (int)ceil_div(T, c.rows);
        return c;
    }
    c.kind = 1;
    c.threads = C / V > 512 ? 1024 : 512;
    c.rows = c.threads / (C / V) * kHeld;
    c.chunks = (int)ceil_div(T, c.rows);
    return c;
}
// frames of a chunk of the gradients' sums: enough chunks to fill the chip, 32 frames at least
int back_rows(int B, int T) {
    const long long chunks = B >= kWorkgroups ? 1 : kWorkgroups / B;
    const long long r = ceil_div(T, chunks);
    return (int)(r < 32 ? 32 : r);
}
unsigned apply_blocks(int B, int T, int rows_at_a_time) {
    const long long per = ceil_div(T, 8LL * rows_at_a_time), most = 4096 / B;
    return (unsigned)(per < 1 ? 1 : per < most ? per : most < 1 ? 1 : most);
}
unsigned plain_blocks(int B, int T, int C) {
    long long per = ceil_div((long long)T * C, 256 * 8), most = 256 * 16 / B;
    if (most < 1) most = 1;
    return (unsigned)(per < 1 ? 1 : per < most ? per : most);
}
// Lanes::even of every block of a cut (the last block of an utterance may have fewer groups: powers of two divide them too)
bool even_blocks(const Cut& c, int C, int n, int V) {
    auto pow2 = [](int v) { return v > 0 && (v & (v - 1)) == 0; };
    const int last = C - (c.blocks.per_b - 1) * c.blocks.CB;
    return n % V == 0 && pow2(n / V) && n / V <= 64 && pow2(c.blocks.CB / V) && pow2(last / V);
}

// f(gl_int<the activation>) where loads are of 16 bytes, f(gl_int<-1>) elsewhere: those kernels choose by themselves
template <bool FIXED, typename F>
int with_act(int act, F f) {
    if constexpr (!FIXED) return f(gl_int<-1>());
    else
        switch (act) {
            case GL_ACT_RELU: return f(gl_int<GL_ACT_RELU>());
            case GL_ACT_SILU: return f(gl_int<GL_ACT_SILU>());
            case GL_ACT_GELU: return f(gl_int<GL_ACT_GELU>());
            case GL_ACT_TANH: return f(gl_int<GL_ACT_TANH>());
            case GL_ACT_EXP: return f(gl_int<GL_ACT_EXP>());
            default: return f(gl_int<GL_ACT_NONE>());
        }
}
// How many channels are moved at once: 16 bytes, or as much of that as divides the channels and the arrays' alignment.
struct Array {
    const void* p;
    long long stride;
};
int channels_at_once(int C, int size, std::initializer_list<Array> arrays) {
    int V = 16 / size;
    for (const Array& a : arrays)
        while (a.p && V > 1 && ((uintptr_t)a.p % (V * size) || a.stride % V)) V /= 2;
    while (C % V) V /= 2;
    return V;
}

// workspace: [statistics where the caller wants none] [parts of the chunks]
long long parts_bytes(int B, int T, int C, int groups, int dtype) {
    const int size = dtype == GL_F32 ? 4 : 2;
    long long most = 0;
    for (int V = 16 / size; V; V /= 2) {                     // alignment is not known to the query
        if (C % V) continue;
        const Cut c = cut_for(B, T, C, groups, size, V, kMaxThreads, kRowBytes);
        if (c.kind && 8LL * B * groups * c.chunks > most) most = 8LL * B * groups * c.chunks;
    }
    return align16(most);
}
long long norm_bytes(int B, int T, int C, int groups, int dtype) {
    const int size = dtype == GL_F32 ? 4 : 2;
    bool slabs = B && T;
    for (int V = 16 / size; V; V /= 2)
        if (slabs && C % V == 0) slabs = cut_for(B, T, C, groups, size, V, kMaxThreads, kRowBytes).kind == 0;
    return slabs ? 0 : stats_bytes(B, groups) + (B && T ? parts_bytes(B, T, C, groups, dtype) : 0);
}
long long back_parts_bytes(int B, int T, int C) {
    return B && T ? align16(8LL * B * ceil_div(T, back_rows(B, T)) * C) : 0;
}
// workspace of the gradients: [p, q] [sums B x 2 x C] [parts of the chunks]
long long back_bytes(int B, int T, int C, int groups) {
    return stats_bytes(B, groups) + align16(8LL * B * C) + back_parts_bytes(B, T, C);
}

struct Norm {
    const void* x;
    long long x_stride;
    const void *gamma, *beta;
    const int* frames;
    int B, T, C, groups, act;
    hipStream_t st;
};

template <typename T, int V>
int norm_fwd(const Norm& a, void* y, long long y_stride, float* stats, float* given, float* parts, float eps) {
    const int n = a.C / a.groups;
    const T *x = (const T*)a.x, *ga = (const T*)a.gamma, *be = (const T*)a.beta;
    Cut c = a.T ? cut_for(a.B, a.T, a.C, a.groups, sizeof(T), V, kMaxThreads, kRowBytes) : Cut{2};
    if (c.kind == 0)
        return with_act<V * sizeof(T) == 16>(a.act, [&](auto act) -> int {
            const bool even = even_blocks(c, a.C, n, V);
            auto kernel = even ? k_norm_slab<T, V, decltype(act)::value, true> : k_norm_slab<T, V, decltype(act)::value, false>;
            hipLaunchKernelGGL(kernel, dim3((unsigned)((c.blocks.total + 7) / 8 * 8)), dim3(c.threads), lds_bytes(c.threads, V, c.blocks.CB, n, 1), a.st, x, a.x_stride, ga, be, a.frames,
                               (T*)y, y_stride, given, a.T, n, a.act, eps, c.blocks);
            GL_HIP_CHECK(hipGetLastError());
            return 0;
        });
    if (c.kind == 1) {
        hipLaunchKernelGGL((k_norm_chunk<T, V>), dim3(c.chunks, a.B), dim3(c.threads), lds_bytes(c.threads, V, a.C, n, 1), a.st, x,
                           a.x_stride, a.frames, parts, a.T, a.C, n);
        GL_HIP_CHECK(hipGetLastError());
        hipLaunchKernelGGL(k_norm_join, dim3(a.groups, a.B), dim3(256), 0, a.st, parts, a.frames, stats, a.T, n, c.chunks, c.rows, eps);
        GL_HIP_CHECK(hipGetLastError());
        return with_act<V * sizeof(T) == 16>(a.act, [&](auto act) -> int {
            hipLaunchKernelGGL((k_norm_apply<T, V, decltype(act)::value>),
                               dim3(apply_blocks(a.B, a.T, c.threads / (a.C / V)), a.B), dim3(c.threads), 0, a.st, x, a.x_stride,
                               ga, be, a.frames, stats, (T*)y, y_stride, a.T, a.C, n, a.act);
            GL_HIP_CHECK(hipGetLastError());
            return 0;
        });
    }
    if (c.chunks) {
        hipLaunchKernelGGL((k_norm_plain_chunk<T>), dim3(a.groups, a.B, c.chunks), dim3(256), 0, a.st, x, a.x_stride, a.frames, parts, a.T,
                           n, c.rows);
        GL_HIP_CHECK(hipGetLastError());
    }
    hipLaunchKernelGGL(k_norm_join, dim3(a.groups, a.B), dim3(256), 0, a.st, parts, a.frames, stats, a.T, n, c.chunks, c.rows, eps);
    GL_HIP_CHECK(hipGetLastError());
    if (!a.T) return 0;
    hipLaunchKernelGGL((k_norm_plain_apply<T>), dim3(plain_blocks(a.B, a.T, a.C), a.B), dim3(256), 0, a.st, x, a.x_stride, ga, be,
                       a.frames, stats, (T*)y, y_stride, a.T, a.C, n, a.act);
    GL_HIP_CHECK(hipGetLastError());
    return 0;
}

template <typename T, int V>
int norm_back(const Norm& a, const void* dy_, long long dy_stride, const float* stats, void* dx_, long long dx_stride, float* pq,
              float* sums, float* parts, void* dgamma, void* dbeta, bool* done) {
    const int n = a.C / a.groups;
    const T *x = (const T*)a.x, *ga = (const T*)a.gamma, *be = (const T*)a.beta, *dy = (const T*)dy_;
    T* dx = (T*)dx_;
    const Cut c = cut_for(a.B, a.T, a.C, a.groups, sizeof(T), V, kBackThreads<T>, kBackRowBytes);
    if (c.kind == 0)
        return with_act<V * sizeof(T) == 16>(a.act, [&](auto act) -> int {
            const bool even = even_blocks(c, a.C, n, V);
            auto kernel = even ? k_norm_back_slab<T, V, decltype(act)::value, true> : k_norm_back_slab<T, V, decltype(act)::value, false>;
            hipLaunchKernelGGL(kernel, dim3((unsigned)((c.blocks.total + 7) / 8 * 8)), dim3(c.threads), lds_bytes(c.threads, V, c.blocks.CB, n, 2), a.st, dy, dy_stride, x, a.x_stride,
                               stats, ga, be, a.frames, dx, dx_stride, sums, a.T, n, a.act, c.blocks);
            GL_HIP_CHECK(hipGetLastError());
            return 0;
        });
    if (c.kind == 1) {
        const int rows = back_rows(a.B, a.T), chunks = (int)ceil_div(a.T, rows);
        *done = a.B == 1;                                    // the join writes dgamma and dbeta
        return with_act<V * sizeof(T) == 16>(a.act, [&](auto act) -> int {
            constexpr int ACT = decltype(act)::value;
            hipLaunchKernelGGL((k_norm_back_chunk<T, V, ACT>), dim3(chunks, a.B), dim3(c.threads),
                               lds_bytes(c.threads, V, a.C, n, 1), a.st, dy, dy_stride, x, a.x_stride, stats, ga, be, a.frames, parts,
                               a.T, a.C, n, rows, a.act);
            GL_HIP_CHECK(hipGetLastError());
            hipLaunchKernelGGL((k_norm_back_join<T>), dim3((unsigned)ceil_div(2 * a.C, 16), a.B), dim3(1024), 0, a.st, parts, sums,
                               (T*)dgamma, (T*)dbeta, a.C, chunks, *done);
            GL_HIP_CHECK(hipGetLastError());
            if (!dx) return 0;
            hipLaunchKernelGGL((k_norm_back_apply<T, V, ACT>), dim3(apply_blocks(a.B, a.T, c.threads / (a.C / V)), a.B),
                               dim3(c.threads), sizeof(float) * (2 * a.C + 2 * (a.C / n)), a.st, dy, dy_stride, x, a.x_stride, stats,
                               sums, ga, be, a.frames, dx, dx_stride, a.T, a.C, n, a.act);
            GL_HIP_CHECK(hipGetLastError());
            return 0;
        });
    }
    const int rows = back_rows(a.B, a.T), chunks = (int)ceil_div(a.T, rows);
    *done = a.B == 1;
    hipLaunchKernelGGL((k_norm_plain_back_chunk<T>), dim3((unsigned)ceil_div(a.C, 256), a.B, chunks), dim3(256), 0, a.st, dy, dy_stride, x,
                       a.x_stride, stats, ga, be, a.frames, parts, a.T, a.C, n, rows, a.act);
    GL_HIP_CHECK(hipGetLastError());
    hipLaunchKernelGGL((k_norm_back_join<T>), dim3((unsigned)ceil_div(2 * a.C, 16), a.B), dim3(1024), 0, a.st, parts, sums,
                       (T*)dgamma, (T*)dbeta, a.C, chunks, *done);
    GL_HIP_CHECK(hipGetLastError());
    if (!dx) return 0;
    hipLaunchKernelGGL((k_norm_plain_back_pq<T>), dim3(a.groups, a.B), dim3(256), 0, a.st, sums, ga, a.frames, pq, a.T, a.C, n);
    GL_HIP_CHECK(hipGetLastError());
    hipLaunchKernelGGL((k_norm_plain_back_apply<T>), dim3(plain_blocks(a.B, a.T, a.C), a.B), dim3(256), 0, a.st, dy, dy_stride, x,
                       a.x_stride, stats, pq, ga, be, a.frames, dx, dx_stride, a.T, a.C, n, a.act);
    GL_HIP_CHECK(hipGetLastError());
    return 0;
}

}  // namespace

extern "C" {

long long gl_group_norm_workspace(int B, int T, int channels, int groups, int dtype) {
    if (check_norm(B, T, channels, groups, dtype, 0, "gl_group_norm_workspace")) return GL_ERR_INVALID;
    return norm_bytes(B, T, channels, groups, dtype);
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
    if (!rc) rc = check_elements({x, gamma, beta, y}, dtype == GL_F32 ? 4 : 2, "gl_group_norm");
    if (!rc) rc = check_elements({frames, stats}, 4, "gl_group_norm");
    if (!rc) rc = check_workspace(workspace, workspace_bytes, norm_bytes(B, T, channels, groups, dtype), "gl_group_norm");
    if (rc) return rc;
    if (T == 0 && !stats) return 0;
    float* s = stats ? stats : (float*)workspace;
    float* parts = (float*)((char*)workspace + stats_bytes(B, groups));
    const Norm a = {x, x_stride, gamma, beta, frames, B, T, channels, groups, activation, (hipStream_t)stream};
    const int V = channels_at_once(channels, dtype == GL_F32 ? 4 : 2, {{x, x_stride}, {y, y_stride}});
#define GL_NORM(T_, V_) \
    case V_: return norm_fwd<T_, V_>(a, y, y_stride, s, stats, parts, eps);
#define GL_NORM16(T_) \
    switch (V) { GL_NORM(T_, 8) GL_NORM(T_, 4) GL_NORM(T_, 2) GL_NORM(T_, 1) }
    if (dtype == GL_BF16) GL_NORM16(gl_bf16)
    else if (dtype == GL_F16) GL_NORM16(gl_f16)
    else switch (V) { GL_NORM(float, 4) GL_NORM(float, 2) GL_NORM(float, 1) }
    return 0;                                                // not reached
#undef GL_NORM16
#undef GL_NORM
}

long long gl_group_norm_backward_workspace(int B, int T, int channels, int groups, int dtype) {
    if (check_norm(B, T, channels, groups, dtype, 0, "gl_group_norm_backward_workspace")) return GL_ERR_INVALID;
    return back_bytes(B, T, channels, groups);
}

int gl_group_norm_backward(const void* dy, long long dy_stride, const void* x, long long x_stride, const float* stats,
                           const void* gamma, const void* beta, const int* frames, void* dx, long long dx_stride,
                           void* dgamma, void* dbeta, int B, int T, int channels, int groups, int dtype,
                           int activation, void* workspace, long long workspace_bytes, void* stream) {
    int rc = check_norm(B, T, channels, groups, dtype, activation, "gl_group_norm_backward");
    if (!rc) rc = check_elements({dy, x, gamma, beta, dx, dgamma, dbeta}, dtype == GL_F32 ? 4 : 2, "gl_group_norm_backward");
    if (!rc) rc = check_elements({frames, stats}, 4, "gl_group_norm_backward");
    if (rc) return rc;
    const hipStream_t st = (hipStream_t)stream;
    float* pq = (float*)workspace;
    float* sums = (float*)((char*)workspace + stats_bytes(B, groups));
    bool done = false;
    if (B > 0 && T > 0) {
        if (!dy || !x || !stats) return gl_set_error(GL_ERR_INVALID, "gl_group_norm_backward: NULL buffer");
        rc = check_stride(dy_stride, channels, "dy", "gl_group_norm_backward");
        if (!rc) rc = check_stride(x_stride, channels, "x", "gl_group_norm_backward");
        if (!rc && dx) rc = check_stride(dx_stride, channels, "dx", "gl_group_norm_backward");
        if (!rc)
            rc = check_workspace(workspace, workspace_bytes, back_bytes(B, T, channels, groups), "gl_group_norm_backward");
        if (rc) return rc;
        float* parts = (float*)((char*)sums + align16(8LL * B * channels));
        const Norm a = {x, x_stride, gamma, beta, frames, B, T, channels, groups, activation, st};
        const int V = channels_at_once(channels, dtype == GL_F32 ? 4 : 2, {{x, x_stride}, {dy, dy_stride}, {dx, dx_stride}});
#define GL_NORM(T_, V_)                                                                                                        \
    case V_: rc = norm_back<T_, V_>(a, dy, dy_stride, stats, dx, dx_stride, pq, sums, parts, dgamma, dbeta, &done); break;
#define GL_NORM16(T_) \
    switch (V) { GL_NORM(T_, 8) GL_NORM(T_, 4) GL_NORM(T_, 2) GL_NORM(T_, 1) }
        if (dtype == GL_BF16) GL_NORM16(gl_bf16)
        else if (dtype == GL_F16) GL_NORM16(gl_f16)
        else switch (V) { GL_NORM(float, 4) GL_NORM(float, 2) GL_NORM(float, 1) }
#undef GL_NORM16
#undef GL_NORM
        if (rc) return rc;
    }
    if ((dgamma || dbeta) && !done) {
        const dim3 grid((unsigned)ceil_div(2 * channels, 16));   // over the utterances
        const int n = T > 0 ? B : 0;
#define GL_AFFINE(T_)                                                                                                          \
    hipLaunchKernelGGL((k_norm_back_join<T_>), grid, dim3(1024), 0, st, sums, (float*)nullptr, (T_*)dgamma, (T_*)dbeta, channels, n, true)
        if (dtype == GL_F32) GL_AFFINE(float);
        else if (dtype == GL_BF16) GL_AFFINE(gl_bf16);
        else GL_AFFINE(gl_f16);
#undef GL_AFFINE
        GL_HIP_CHECK(hipGetLastError());
    }
    return 0;
}

}  // extern "C"
