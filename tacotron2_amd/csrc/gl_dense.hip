// Dense layers of the learned mel inversion: y = act(x W^T + b) + r and its gradients (include/gl_hip.h).
//
// All three products are C[i][j] = sum_q P(i, q) Q(j, q):
//   forward   P = x  [rows][inputs],   Q = W  [outputs][inputs]      both contiguous in q
//   dx        P = dz [rows][outputs],  Q(j, q) = W[q][j]             Q contiguous in j
//   dweight   P(i, q) = dz[q][i],      Q(j, q) = x[q][j]             both contiguous in i / j, q = frames
// Which kernel, by sizes alone (the workspace query and the call must agree):
//   up to 8 rows (forward): k_dense_few, one wave (or part of one) a column: W is read once, nothing else counts;
//   small gradients: k_dense_back_small, one launch and a join: launches are what counts;
//   16-bit types: the tiles of gl_mm16.h, on copies padded to whole chunks where a width is not a multiple of 8;
//   float32 with enough work: the same tiles on planes of 16 bits;
//   the rest, and operands whose rows start off 16 bytes against their widths: k_dense_any, element by element, on
//   v_mfma_f32_32x32x16 or, for float32, v_mfma_f32_32x32x2_f32.
// Sums are float32 everywhere.  Q is the matrix instruction's A operand: the accumulator's registers then run along j, the
// contiguous direction of C.
#include <initializer_list>
#include <type_traits>

#include "gl_dense.h"

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
template <typename T, int N> struct vecn { typedef T type __attribute__((ext_vector_type(N))); };
typedef gl_operand Operand;
typedef gl_epilogue Epilogue;

constexpr int kTile = 64;        // rows and columns of C per workgroup (4 waves, 32 x 32 each)
constexpr int kBQ = 32;          // contraction indexes staged per step
constexpr long long kMostBlocks = 1 << 23;   // of 256 threads: a launch has less than 2^32
constexpr int kCUs = 256;        // compute units of an MI355X: the work split must not depend on the moment

// A product of k_dense_any.  With DZ, P is dy and Z the preactivation: the first factor is dz = dy act'(z), rounded to T or split
// into two planes, and `sums` ([parts][I]) or, without parts, `db` gets the unrounded dz's sums over q, from the tiles at j = 0.
struct AnyArgs {
    Operand P, Q, Z;             // base null: zeros
    Epilogue e;
    long long I, nq, q_per_part;
    int J, tiles_j, n_tiles, act;
    bool p_along, q_along;       // staged along q (P and Z alike), or eight rows of one q
    float* sums;
    void* db;
};

// Any size, stride and alignment.  A thread stages eight consecutive elements of each side, two steps ahead of the
// products.  V: 1, or 16 bytes of T: loads are 16 bytes wide (the sides' pointers, strides and sizes allow it).
// T: what is multiplied, TY: what is written, TD: what dy and z are.  TWO: the first factor is in two planes (gl_split).
// Bound by latency where it is small, by the LDS traffic of 4-byte elements where it is not: 641 x 80 -> 512 float32 8.3 us,
// 2000 x 500 -> 700 float32 32 us (43 TF).
template <typename T, typename TY, typename TD, int V, bool DZ, bool TWO>
__device__ __forceinline__ void any_tiles(const AnyArgs& a, long long first, long long step, int part, const int* __restrict__ flags) {
    constexpr bool k16 = sizeof(T) == 2;
    constexpr int kPitch = k16 ? kBQ + 8 : kBQ + 1;
    __shared__ __attribute__((aligned(16))) T Ps[kTile * kPitch];
    __shared__ __attribute__((aligned(16))) T Qs[kTile * kPitch];
    __shared__ __attribute__((aligned(16))) T Ls[TWO ? kTile * kPitch : 8];      // P's lower plane
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, li = lane & 31, lk = lane >> 5;
    const long long q_begin = (long long)part * a.q_per_part;
    const long long q_end = q_begin + a.q_per_part < a.nq ? q_begin + a.q_per_part : a.nq;
    const int wi = (wave >> 1) * 32, wj = (wave & 1) * 32;
    // this thread's eight elements: of row r along q, or of contraction index q across rows
    auto spot = [&](bool along, int& r, int& q) {
        r = along ? threadIdx.x >> 2 : (threadIdx.x & 7) * 8;
        q = along ? (threadIdx.x & 3) * 8 : threadIdx.x >> 3;
    };
    // Loads them and says how many exist.  No branch around a load: one would have to wait for it.
    auto fetch = [&](auto (&v)[8], const Operand& o, bool along, long long r0, long long rn, long long q0) -> int {
        typedef typename std::remove_reference<decltype(v[0])>::type U;
        constexpr int VU = V > 1 ? 16 / sizeof(U) : 1;
        typedef typename vecn<U, VU>::type vU;
        int r, q;
        spot(along, r, q);
        const U* at = (const U*)o.base + (r0 + r) * o.is + (q0 + q) * o.qs;
        const long long left = along ? (r0 + r < rn ? q_end - (q0 + q) : 0) : (q0 + q < q_end ? rn - (r0 + r) : 0);
        const int have = (int)min(max(left, 0LL), 8LL);
#pragma unroll
        for (int k = 0; k < 8; k += VU) {
            const vU t = *(const vU*)(k < have ? at + k : (const U*)o.base);
#pragma unroll
            for (int u = 0; u < VU; ++u) {
                if constexpr (VU == 1) v[k] = t[0];
                else v[k + u] = t[u];
            }
        }
        return have;
    };
    auto deposit = [&](T* dst, bool along, const T (&v)[8]) {
        int r, q;
        spot(along, r, q);
        if (k16 && along) {                                  // uniform; a row's eight lie on 16 bytes
            typedef typename vecn<T, 8>::type v8;
            v8 t;
#pragma unroll
            for (int k = 0; k < 8; ++k) t[k] = v[k];
            *(v8*)(dst + r * kPitch + q) = t;
            return;
        }
        const int across = along ? 1 : kPitch;
#pragma unroll
        for (int k = 0; k < 8; ++k) dst[r * kPitch + q + k * across] = v[k];
    };
    for (long long tile = first; tile < a.n_tiles; tile += step) {
        if (flags && !flags[tile]) continue;                 // uniform over the workgroup
        const long long i0 = tile / a.tiles_j * kTile;
        const int j0 = (int)(tile % a.tiles_j) * kTile;
        f32x16 acc, low;
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[r] = low[r] = 0.0f;
        float bias[16];                                      // arrives under the products
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const int j = j0 + wj + (r & 3) + 8 * (r >> 2) + 4 * lk;
            bias[r] = !DZ && a.e.bias && !a.e.partial && j < a.J ? gl_to_f32(((const T*)a.e.bias)[j]) : 0.0f;
        }
        struct Staged {
            TD p[8], z[8];
            T q[8];
            int p_have, q_have;
        };
        Operand below = a.P;                                 // the lower plane, where there is one in memory
        if (TWO && !DZ) below.base = (const T*)a.P.base + a.P.plane;
        float sum[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) sum[k] = 0.0f;
        auto load = [&](Staged& t, long long q0) {
            if (q0 >= q_end) return;                         // uniform, as all conditions outside of fetch
            t.p_have = fetch(t.p, a.P, a.p_along, i0, a.I, q0);
            if (DZ && a.act != GL_ACT_NONE) fetch(t.z, a.Z, a.p_along, i0, a.I, q0);
            if (TWO && !DZ) fetch(t.z, below, a.p_along, i0, a.I, q0);
            t.q_have = a.Q.base ? fetch(t.q, a.Q, a.q_along, j0, a.J, q0) : 0;
        };
        auto multiply = [&](Staged& t, long long q0) {
            if (q0 >= q_end) return;
            T pt[8], pl[8];
            if constexpr (DZ) {
                float d[8];
                gl_with_act(a.act, [&](auto act) {
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        d[k] = gl_to_f32(t.p[k]);
                        if constexpr (decltype(act)::value != GL_ACT_NONE) d[k] *= gl_act_grad<TD>(gl_to_f32(t.z[k]), decltype(act)::value);
                    }
                });
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    d[k] = k < t.p_have ? d[k] : 0.0f;
                    sum[k] += d[k];
                    if constexpr (TWO) gl_split(d[k], pt[k], pl[k]);
                    else pt[k] = (T)d[k];
                }
            } else {
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    pt[k] = k < t.p_have ? t.p[k] : (T)0.0f;
                    if constexpr (TWO) pl[k] = k < t.p_have ? t.z[k] : (T)0.0f;
                }
            }
#pragma unroll
            for (int k = 0; k < 8; ++k) t.q[k] = k < t.q_have ? t.q[k] : (T)0.0f;
            __syncthreads();
            deposit(Ps, a.p_along, pt);
            if constexpr (TWO) deposit(Ls, a.p_along, pl);
            deposit(Qs, a.q_along, t.q);
            __syncthreads();
            load(t, q0 + 2 * kBQ);
            if constexpr (k16) {
                typedef typename vecn<T, 8>::type v8;
#pragma unroll
                for (int s = 0; s < kBQ; s += 16) {
                    const v8 x = *(const v8*)(Qs + (wj + li) * kPitch + s + 8 * lk);
                    auto product = [&](const T* side, f32x16 c) -> f32x16 {
                        const v8 y = *(const v8*)(side + (wi + li) * kPitch + s + 8 * lk);
                        if constexpr (__is_same(T, gl_bf16)) return __builtin_amdgcn_mfma_f32_32x32x16_bf16(x, y, c, 0, 0, 0);
                        else return __builtin_amdgcn_mfma_f32_32x32x16_f16(x, y, c, 0, 0, 0);
                    };
                    acc = product(Ps, acc);
                    if constexpr (TWO) low = product(Ls, low);
                }
            } else {
#pragma unroll
                for (int s = 0; s < kBQ; s += 2)
                    acc = __builtin_amdgcn_mfma_f32_32x32x2f32(Qs[(wj + li) * kPitch + s + lk], Ps[(wi + li) * kPitch + s + lk],
                                                               acc, 0, 0, 0);
            }
        };
        Staged even, odd;
        load(even, q_begin);
        load(odd, q_begin + kBQ);
        for (long long q0 = q_begin; q0 < q_end; q0 += 2 * kBQ) {
            multiply(even, q0);
            multiply(odd, q0 + kBQ);
        }
        if constexpr (TWO)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[r] = fmaf(low[r], kSplitStep<T>, acc[r]);
        if constexpr (DZ) {
            if ((a.sums || a.db) && j0 == 0) {               // not p_along: thread = (8 rows, one of 32 indexes)
                __shared__ float red[4][kTile];
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    sum[k] += __shfl_xor(sum[k], 8);
                    sum[k] += __shfl_xor(sum[k], 16);
                    sum[k] += __shfl_xor(sum[k], 32);
                }
                __syncthreads();
                if (lane < 8)
#pragma unroll
                    for (int k = 0; k < 8; ++k) red[wave][lane * 8 + k] = sum[k];
                __syncthreads();
                const int c = threadIdx.x;
                if (c < kTile && i0 + c < a.I) {
                    const float s = (red[0][c] + red[1][c]) + (red[2][c] + red[3][c]);
                    if (a.sums) a.sums[part * a.I + i0 + c] = s;
                    else ((T*)a.db)[i0 + c] = (T)s;
                }
            }
        }
        const long long i = i0 + wi + li;
        if (i >= a.I || !(a.e.partial || a.e.y)) continue;
        const Epilogue& e = a.e;
        typedef typename vecn<TY, 4>::type v4;
        // four columns next to each other: f(first column, how many exist, the sums)
        auto quads = [&](auto f) {
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int j = j0 + wj + 8 * g + 4 * lk;
                if (j < a.J) f(j, min(a.J - j, 4), 4 * g);
            }
        };
        auto put = [&](TY* o, int n, int r) {
            v4 t;
#pragma unroll
            for (int k = 0; k < 4; ++k) t[k] = (TY)acc[r + k];
            if (e.quads) *(v4*)o = t;
            else
                for (int k = 0; k < n; ++k) o[k] = t[k];
        };
        if (e.partial) {
            quads([&](int j, int n, int r) {
                float* o = e.partial + ((long long)part * a.I + i) * a.J + j;
                if (a.J % 4 == 0) *(f32x4*)o = f32x4{acc[r], acc[r + 1], acc[r + 2], acc[r + 3]};
                else
                    for (int k = 0; k < n; ++k) o[k] = acc[r + k];
            });
            continue;
        }
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[r] += bias[r];
        if (e.z) quads([&](int j, int n, int r) { put((TY*)e.z + i * e.z_stride + j, n, r); });
        gl_with_act(e.act, [&](auto act) {
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[r] = gl_act<TY>(acc[r], decltype(act)::value);
        });
        if (e.residual)
            quads([&](int j, int n, int r) {
                const TY* from = (const TY*)e.residual + i * e.r_stride + j;
                v4 t = v4{};
                if (e.quads) t = *(const v4*)from;
                else
                    for (int k = 0; k < n; ++k) t[k] = from[k];
#pragma unroll
                for (int k = 0; k < 4; ++k) acc[r + k] += gl_to_f32(t[k]);
            });
        quads([&](int j, int n, int r) { put((TY*)e.y + i * e.y_stride + j, n, r); });
    }
}

// grid (workgroups, parts); workgroups walk over the tiles.  flags: only the tiles whose flag is set.
template <typename T, typename TO, int V, bool TWO>
__global__ void __launch_bounds__(256) k_dense_any(AnyArgs a, const int* __restrict__ flags) {
    if (flags) {                                             // all of this workgroup's at once: there is hardly ever one
        int set = 0;
        for (long long tile = blockIdx.x + (long long)threadIdx.x * gridDim.x; tile < a.n_tiles; tile += 256LL * gridDim.x)
            set |= flags[tile];
        if (!__syncthreads_or(set)) return;
    }
    any_tiles<T, TO, T, V, false, TWO>(a, blockIdx.x, gridDim.x, blockIdx.y, flags);
}

// The gradients of a small layer in one launch: tiles (times parts) of dx, then of dweight, whose first ones sum dz for dbias.
// dz is worked out from dy and z by every tile that reads it.  641 x 80 -> 512 float32: 11.6 us and 5.8 for the join, where a pass
// for dz, its sums, two products and their joins took 35 us.
template <typename T, typename TO, int V, bool TWO>
__global__ void __launch_bounds__(256) k_dense_back_small(AnyArgs x, AnyArgs w, int x_blocks) {
    const bool second = (int)blockIdx.x >= x_blocks;
    const AnyArgs a = second ? w : x;
    const int block = blockIdx.x - (second ? x_blocks : 0), part = block / a.n_tiles;
    any_tiles<T, T, TO, V, true, TWO>(a, block - part * a.n_tiles, a.n_tiles, part, nullptr);
}

// Its join: elements of dx, then of dweight (where there are parts of them), then of dbias.  V divides `inputs`.
struct BackJoin {
    const float *x, *w, *d;              // parts
    int x_parts, w_parts;
    long long x_n, w_n;                  // elements of a part; 0: written already
    void *dx, *dw, *db;
    long long dx_stride, dw_stride;
    int inputs, outputs;                 // outputs: of dbias to sum
};
template <typename T, int V>
__global__ void __launch_bounds__(256) k_dense_back_join(BackJoin k) {
    typedef typename vecn<float, V>::type vf;
    const long long n = k.x_n + k.w_n + k.outputs;
    for (long long at = ((long long)blockIdx.x * 256 + threadIdx.x) * V; at < n; at += (long long)gridDim.x * 256 * V) {
        if (at >= k.x_n + k.w_n) {
            const int c0 = (int)(at - k.x_n - k.w_n);
            for (int c = c0; c < c0 + V && c < k.outputs; ++c) {
                float s = 0.0f;
#pragma unroll 8
                for (int p = 0; p < k.w_parts; ++p) s += k.d[(long long)p * k.outputs + c];
                ((T*)k.db)[c] = (T)s;
            }
            continue;
        }
        const bool second = at >= k.x_n;
        const long long e = second ? at - k.x_n : at, part = second ? k.w_n : k.x_n;
        const float* in = (second ? k.w : k.x) + e;
        const int parts = second ? k.w_parts : k.x_parts;
        vf s = *(const vf*)in;
#pragma unroll 8
        for (int p = 1; p < parts; ++p) s += *(const vf*)(in + p * part);
        const long long i = e / k.inputs;
        T* o = (T*)(second ? k.dw : k.dx) + i * (second ? k.dw_stride : k.dx_stride) + (e - i * k.inputs);
#pragma unroll
        for (int v = 0; v < V; ++v) o[v] = (T)s[v];
    }
}

// Sums the parts of a split contraction in their order and finishes the elements, V at a time.  Bound by memory: 2048 x 512 in
// 16 parts 13 us (5.2 TB/s).
template <typename T, typename TO, int V>
__global__ void __launch_bounds__(256) k_dense_join(Epilogue e, long long I, int J, int parts) {
    typedef typename vecn<float, V>::type vf;
    const long long n = I * J;
    for (long long at = ((long long)blockIdx.x * 256 + threadIdx.x) * V; at < n; at += (long long)gridDim.x * 256 * V) {
        vf s = *(const vf*)(e.partial + at);
#pragma unroll 4
        for (int p = 1; p < parts; ++p) s += *(const vf*)(e.partial + p * n + at);
        const long long i = at / J;
        const int j = (int)(at - i * J);
#pragma unroll
        for (int v = 0; v < V; ++v) {
            gl_finish<T, TO>(e, i, j + v, s[v]);
        }
    }
}

// The same for float32 through planes: a workgroup 16 rows of a 64 x 64 block, which are left as they were and flagged (a byte of
// the block's flag) where the planes do not give one of their sums.  V divides J.  Bound by memory and, with few blocks, by how many
// loads run at once: 264 x 512 in 42 parts 8 us (a workgroup a whole block: 15), 512 x 512 in 24 parts 6.
constexpr int kJoinRows = 16;
template <int V>
__device__ __forceinline__ void join_rows(const Epilogue& e, long long i0, int j0, long long I, int J, int parts, unsigned char* flag) {
    typedef typename vecn<float, V>::type vf;
    constexpr int kAcross = kTile / V, kRows = 256 / kAcross, kEach = kJoinRows / kRows, kAtOnce = 12 / kEach;
    const int j = j0 + (threadIdx.x % kAcross) * V;
    const long long i1 = i0 + threadIdx.x / kAcross, n = I * J;
    auto real = [&](int k) { return j < J && i1 + k * kRows < I; };
    vf s[kEach];
    const float* from[kEach];
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
        s[k] = vf{};
        from[k] = e.partial + (real(k) ? (i1 + k * kRows) * J + j : 0);
    }
    for (int p = 0; p < parts; p += kAtOnce) {               // no branch around a load: one would have to wait for it
        vf t[kAtOnce][kEach];
#pragma unroll
        for (int o = 0; o < kAtOnce; ++o)
#pragma unroll
            for (int k = 0; k < kEach; ++k) t[o][k] = *(const vf*)(from[k] + min(p + o, parts - 1) * n);
#pragma unroll
        for (int o = 0; o < kAtOnce; ++o)
#pragma unroll
            for (int k = 0; k < kEach; ++k) s[k] += p + o < parts ? t[o][k] : vf{};
    }
    if (flag) {
        bool bad = false;
#pragma unroll
        for (int k = 0; k < kEach; ++k) {
            if (!real(k)) continue;
            const long long i = i1 + k * kRows;
#pragma unroll
            for (int v = 0; v < V; ++v) {
                bad |= !(fabsf(s[k][v]) < INFINITY);
                if (e.scale_p) {
                    const gl_scale p = {e.scale_p[i]}, q = {e.scale_q[j + v]};
                    bad |= !gl_halves_give(ldexpf(s[k][v], p.e() + q.e()), p, q, (float)e.exact_nq);
                }
            }
        }
        bad = __syncthreads_or(bad);
        if (threadIdx.x == 0) *flag = bad;
        if (bad) return;
    }
#pragma unroll
    for (int k = 0; k < kEach; ++k)
        if (real(k))
#pragma unroll
            for (int v = 0; v < V; ++v) gl_finish<float, float>(e, i1 + k * kRows, j + v, s[k][v]);
}
// grid (blocks, their runs of 16 rows)
template <int V>
__global__ void __launch_bounds__(256) k_dense_join_rows(Epilogue e, long long I, int J, int parts, int tiles_j) {
    const int tile = blockIdx.x, run = blockIdx.y;
    if (run == 0 && threadIdx.x == 0) e.flags[gridDim.x + tile] = 0;         // the count of k_dense_repair
    join_rows<V>(e, (long long)(tile / tiles_j) * kTile + run * kJoinRows, tile % tiles_j * kTile, I, J, parts,
                 (unsigned char*)(e.flags + tile) + run);
}

// And the flagged rows from the operands themselves, a block in as many parts, each a workgroup's: the one that ends last joins
// them, in their order.  grid (workgroups, parts).  Nobody waits.  4.6 us where no flag is set; dweight of 40 000 x 512 -> 264 with
// one infinite gradient 0.23 ms (a loop over the frames in one thread for every sum: 50 ms).
template <int V>
__global__ void __launch_bounds__(256) k_dense_repair(AnyArgs a, Epilogue e, int parts) {
    __shared__ int last;
    int set = 0;                                             // all of this workgroup's at once: there is hardly ever one
    for (long long tile = blockIdx.x + (long long)threadIdx.x * gridDim.x; tile < a.n_tiles; tile += 256LL * gridDim.x) set |= e.flags[tile];
    if (!__syncthreads_or(set)) return;
    for (long long tile = blockIdx.x; tile < a.n_tiles; tile += gridDim.x) {
        const unsigned flags = e.flags[tile];
        if (!flags) continue;                                // uniform over the workgroup
        any_tiles<float, float, float, 1, false, false>(a, tile, a.n_tiles, blockIdx.y, nullptr);
        __threadfence();
        __syncthreads();
        if (threadIdx.x == 0) last = atomicAdd(e.flags + a.n_tiles + tile, 1) == parts - 1;
        __syncthreads();
        const bool mine = last;
        __syncthreads();
        if (!mine) continue;
        __threadfence();
        for (int run = 0; run < kTile / kJoinRows; ++run)
            if (flags >> (8 * run) & 0xff)
                join_rows<V>(e, tile / a.tiles_j * kTile + run * kJoinRows, (int)(tile % a.tiles_j) * kTile, a.I, a.J, parts, nullptr);
    }
}

// Up to ROWS frames: L lanes a column (as many as 16-byte pieces of its weights, to 64), 64 / L columns a wave.  W streams
// through once and bounds it: 1 x 2048 -> 8192 bf16 5.4 us (6.2 TB/s, W in the cache behind the L2s); 8 rows, whose x no longer
// stays in the L1, 19 us.  1 x 512 -> 1025 3.3 us, a launch.
template <typename T, typename TO, int ROWS, int V>
__global__ void __launch_bounds__(256) k_dense_few(const T* __restrict__ x, long long x_stride, const T* __restrict__ w,
                                                   long long w_stride, Epilogue e, int rows, int K, int N, int L) {
    typedef typename vecn<T, V>::type vT;
    constexpr int kAtOnce = V * sizeof(T) >= 8 ? 2 : 4;      // pieces a lane has on the way
    const int lane = threadIdx.x & 63, l = lane & (L - 1);
    const int n = (blockIdx.x * 4 + (threadIdx.x >> 6)) * (64 / L) + lane / L;
    float acc[ROWS];
#pragma unroll
    for (int m = 0; m < ROWS; ++m) acc[m] = 0.0f;
    if (n < N) {
        const T* wn = w + n * w_stride;
#pragma unroll kAtOnce
        for (int k = l * V; k < K; k += L * V) {
            const vT wv = *(const vT*)(wn + k);
#pragma unroll
            for (int m = 0; m < ROWS; ++m) {
                const vT xv = *(const vT*)(x + min(m, rows - 1) * x_stride + k);     // rows past the last: once more, unused
#pragma unroll
                for (int v = 0; v < V; ++v) acc[m] = fmaf(gl_to_f32(xv[v]), gl_to_f32(wv[v]), acc[m]);
            }
        }
    }
    // over the L lanes: first each half takes half of the rows over, until a lane has one, then that row's sum alone
    int m = 0, o = L / 2;
#pragma unroll
    for (int half = ROWS / 2; half > 0; half /= 2, o >>= 1) {
        const bool up = l & o;
#pragma unroll
        for (int k = 0; k < half; ++k) {
            const float got = __shfl_xor(up ? acc[k] : acc[k + half], o);
            acc[k] = (up ? acc[k + half] : acc[k]) + got;
        }
        if (up) m += half;
    }
    const int same = max(2 * o, 1) - 1;                      // lanes that differ in these bits have the same row
    for (; o > 0; o >>= 1) acc[0] += __shfl_xor(acc[0], o);
    if (n < N && m < rows && (l & same) == 0) gl_finish<T, TO>(e, m, n, acc[0]);
}

// Copies two matrices of as many columns, one after the other, into rows of whole chunks: zeros up to `padded` columns.
// PLANES 3: float32 into three bfloat16 planes.  Rows may start anywhere, so elements are read one by one: 55 104 x 513 bf16 30 us
// (3.8 TB/s).
struct Packed {
    const void* in;
    long long in_stride, rows;
    void* out;
};
template <typename T, int PLANES>
__global__ void __launch_bounds__(256) k_dense_pack(Packed first, Packed second, int cols, int padded) {
    const int per_row = padded / 8;
    const long long n = (first.rows + second.rows) * per_row;
    for (long long at = (long long)blockIdx.x * 256 + threadIdx.x; at < n; at += (long long)gridDim.x * 256) {
        const long long row = at / per_row;
        const int c = (int)(at - row * per_row) * 8;
        const bool other = row >= first.rows;
        const long long r = other ? row - first.rows : row, plane = (other ? second.rows : first.rows) * padded;
        const T* src = (const T*)(other ? second.in : first.in) + r * (other ? second.in_stride : first.in_stride) + c;
        void* out = other ? second.out : first.out;
        T v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = c + k < cols ? src[k] : (T)0.0f;
        if constexpr (PLANES == 1) {
            typename vecn<T, 8>::type o;
#pragma unroll
            for (int k = 0; k < 8; ++k) o[k] = v[k];
            *(typename vecn<T, 8>::type*)((T*)out + r * padded + c) = o;
        } else {
            typedef typename vecn<gl_bf16, 8>::type v8;
            v8 h, m, l;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                h[k] = (gl_bf16)v[k];
                const float d = v[k] - (float)h[k];          // exact
                m[k] = (gl_bf16)d;
                l[k] = (gl_bf16)(d - (float)m[k]);
            }
            gl_bf16* o = (gl_bf16*)out + r * padded + c;
            *(v8*)o = h;
            *(v8*)(o + plane) = m;
            *(v8*)(o + 2 * plane) = l;
        }
    }
}

// Rows of two float32 matrices, one after the other, into two planes of f16 each and their gl_scale; zeros up to `padded`
// columns.  A wave a row, which it reads twice: for its largest value, and, from the L1 or L2, to convert it.  Bound by memory:
// 7912 rows of 1024 12.7 us (5.1 TB/s).
struct Halves {
    const float* in;
    long long in_stride, rows;
    gl_f16* out;
    int* scale;
};
template <bool VEC>
__global__ void __launch_bounds__(256) k_dense_halves(Halves a, Halves b, int cols, int padded) {
    const int lane = threadIdx.x & 63;
    for (long long at = (long long)blockIdx.x * 4 + (threadIdx.x >> 6); at < a.rows + b.rows; at += (long long)gridDim.x * 4) {
        const bool second = at >= a.rows;
        const Halves h = second ? b : a;
        const long long r = second ? at - a.rows : at;
        const float* src = h.in + r * h.in_stride;
        auto load = [&](int c, float (&v)[8]) {
            if constexpr (VEC) {
                const f32x4 lo = *(const f32x4*)(src + min(c, cols - 4)), hi = *(const f32x4*)(src + min(c + 4, cols - 4));
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    v[k] = c < cols ? lo[k] : 0.0f;
                    v[4 + k] = c + 4 < cols ? hi[k] : 0.0f;
                }
            } else {
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const float t = src[min(c + k, cols - 1)];
                    v[k] = c + k < cols ? t : 0.0f;
                }
            }
        };
        unsigned most = 0;                                   // of |x|, as bits: NaN above infinity above the rest
#pragma unroll 2
        for (int c = lane * 8; c < padded; c += 512) {
            float v[8];
            load(c, v);
#pragma unroll
            for (int k = 0; k < 8; ++k) most = max(most, __builtin_bit_cast(unsigned, v[k]) & 0x7fffffffu);
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) most = max(most, (unsigned)__shfl_xor((int)most, o));
        const bool wild = most >= 0x7f800000u;
        const int e = wild || most == 0 ? 0 : 15 - __builtin_amdgcn_frexp_expf(__builtin_bit_cast(float, most));
        bool small = false;
#pragma unroll 2
        for (int c = lane * 8; c < padded; c += 512) {
            typedef typename vecn<gl_f16, 8>::type v8;
            float v[8];
            v8 hi, lo;
            load(c, v);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const float s = wild ? 0.0f : ldexpf(v[k], e);
                small |= v[k] != 0.0f && fabsf(s) < 0x1p-13f;
                hi[k] = (gl_f16)s;
                lo[k] = (gl_f16)((s - (float)hi[k]) * 4096.0f);
            }
            gl_f16* o = h.out + r * padded + c;
            *(v8*)o = hi;
            *(v8*)(o + h.rows * padded) = lo;
        }
        small = __any(small);
        if (lane == 0) h.scale[r] = gl_scale::of(e, small, wild).bits;
    }
}

// dz = dy act'(z), as the products read it (splits_dz() says which): rounded to T, in two planes of T, or, float32, in three of
// bfloat16 beside `exact`; zeros up to dz_stride columns, and column sums of the unrounded dz over this workgroup's frames.
// grid (blocks of 64 V columns, parts of the frames); thread = (V columns, one of 4 frame lanes).  dz is a pass of its own, since
// both products read it and one of them transposed; it is bound by memory: 55 104 x 2048 gelu bf16 129 us (677 MB, 5.2 TB/s), two
// planes from float32 254 us (1.35 GB, 5.3 TB/s), from f16 164.
template <typename T, typename TO, int V, int PLANES>
__global__ void __launch_bounds__(256) k_dense_dz(const TO* __restrict__ dy, long long dy_stride, const TO* __restrict__ z,
                                                  long long z_stride, void* __restrict__ dz_, long long dz_stride, long long plane,
                                                  float* __restrict__ exact, float* __restrict__ parts, long long rows, int N, int rows_per_part, int act) {
    typedef typename vecn<TO, V>::type vI;
    __shared__ float s[4][64 * V];
    const int c = threadIdx.x & 63, r = threadIdx.x >> 6;
    const int n = (blockIdx.x * 64 + c) * V;                 // V divides N: a thread's columns exist or are padding, all of them
    const long long r0 = (long long)blockIdx.y * rows_per_part;
    const long long r1 = r0 + rows_per_part < rows ? r0 + rows_per_part : rows;
    const bool real = n < N;
    float sum[V];
#pragma unroll
    for (int v = 0; v < V; ++v) sum[v] = 0.0f;
    auto frames = [&](auto act) {
        constexpr int ACT = decltype(act)::value;
#pragma unroll 2
        for (long long i = r0 + r; i < r1; i += 4) {
            float d[V];
#pragma unroll
            for (int v = 0; v < V; ++v) d[v] = 0.0f;
            if (real) {
                const vI g = *(const vI*)(dy + i * dy_stride + n);
                vI zz = vI{};
                if constexpr (ACT != GL_ACT_NONE) zz = *(const vI*)(z + i * z_stride + n);
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    d[v] = gl_to_f32(g[v]);
                    if constexpr (ACT != GL_ACT_NONE) d[v] *= gl_act_grad<TO>(gl_to_f32(zz[v]), ACT);
                    sum[v] += d[v];
                }
            }
            if (!dz_) continue;
            if constexpr (PLANES == 1) {
                typename vecn<T, V>::type o;
#pragma unroll
                for (int v = 0; v < V; ++v) o[v] = (T)d[v];
                *(typename vecn<T, V>::type*)((T*)dz_ + i * dz_stride + n) = o;
            } else if constexpr (PLANES == 2) {
                typename vecn<T, V>::type h, l;
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    T high, below;
                    gl_split(d[v], high, below);
                    h[v] = high;
                    l[v] = below;
                }
                T* o = (T*)dz_ + i * dz_stride + n;
                *(typename vecn<T, V>::type*)o = h;
                *(typename vecn<T, V>::type*)(o + plane) = l;
            } else {
                typename vecn<gl_bf16, V>::type h, m, l;
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    h[v] = (gl_bf16)d[v];
                    const float e = d[v] - (float)h[v];
                    m[v] = (gl_bf16)e;
                    l[v] = (gl_bf16)(e - (float)m[v]);
                }
                gl_bf16* o = (gl_bf16*)dz_ + i * dz_stride + n;
                *(typename vecn<gl_bf16, V>::type*)o = h;
                *(typename vecn<gl_bf16, V>::type*)(o + plane) = m;
                *(typename vecn<gl_bf16, V>::type*)(o + 2 * plane) = l;
                if (exact) {
                    typename vecn<float, V>::type f;
#pragma unroll
                    for (int v = 0; v < V; ++v) f[v] = d[v];
                    *(typename vecn<float, V>::type*)(exact + i * dz_stride + n) = f;
                }
            }
        }
    };
    if (real || (dz_ && n < dz_stride)) gl_with_act(act, frames);
    if (!parts) return;
#pragma unroll
    for (int v = 0; v < V; ++v) s[r][c * V + v] = sum[v];
    __syncthreads();
    for (int k = threadIdx.x; k < 64 * V; k += 256) {
        const int col = blockIdx.x * 64 * V + k;
        if (col < N) parts[(long long)blockIdx.y * N + col] = (s[0][k] + s[1][k]) + (s[2][k] + s[3][k]);
    }
}

// Column sums over the parts: grid (blocks of 16 columns), thread (column, one of 64 lanes over the parts).  Latency: 511 parts
// of 2048 5.3 us.
template <typename T>
__global__ void __launch_bounds__(1024) k_dense_db(const float* __restrict__ parts, int n_parts, T* __restrict__ db, int N) {
    __shared__ float s[16][16];
    const int c = threadIdx.x & 15, l = threadIdx.x >> 4, n = blockIdx.x * 16 + c;
    float a = 0.0f;
    if (n < N)
#pragma unroll 8
        for (int p = l; p < n_parts; p += 64) a += parts[(long long)p * N + n];
    a += __shfl_xor(a, 16);
    a += __shfl_xor(a, 32);
    if ((l & 3) == 0) s[l >> 2][c] = a;
    __syncthreads();
    if (l || n >= N) return;
    a = s[0][c];
#pragma unroll
    for (int k = 1; k < 16; ++k) a += s[k][c];
    db[n] = (T)a;
}

template <typename T>
__global__ void __launch_bounds__(256) k_dense_zero(T* p, long long stride, int rows, int cols) {
    for (long long at = (long long)blockIdx.x * 256 + threadIdx.x; at < (long long)rows * cols; at += (long long)gridDim.x * 256)
        p[at / cols * stride + at % cols] = (T)0.0f;
}

// Parts of the contraction for k_dense_any: enough workgroups to fill half the chip, at least 4 steps each.
int n_splits(long long I, int J, long long nq) {
    const long long tiles = gl_ceil_div(I, kTile) * gl_ceil_div(J, kTile);
    long long s = kCUs / tiles;
    const long long most = gl_ceil_div(nq, 4 * kBQ);
    if (s > most) s = most;
    return s < 1 ? 1 : (int)s;
}
long long any_bytes(long long I, int J, long long nq) {
    const int s = n_splits(I, J, nq);
    return s > 1 ? gl_align16((long long)s * I * J * 4) : 0;
}

// 16-byte loads: pointer, rows and their length on 16 bytes.  length: of the contiguous direction
bool wide_loads(const Operand& o, long long length, int size) {
    const long long stride = o.qs == 1 ? o.is : o.qs;
    return !o.base || ((uintptr_t)o.base % 16 == 0 && stride * size % 16 == 0 && length * size % 16 == 0);
}

// Whether four columns of every array of results can be moved at once.
template <typename TO>
bool quads(const Epilogue& e, int J) {
    auto whole = [](const void* p, long long stride) { return !p || ((uintptr_t)p % (4 * sizeof(TO)) == 0 && stride % 4 == 0); };
    return J % 4 == 0 && whole(e.y, e.y_stride) && whole(e.z, e.z_stride) && whole(e.residual, e.r_stride);
}

template <typename T, typename TO, bool TWO>
int any_product(const Operand& P, const Operand& Q, Epilogue e, long long I, int J, long long nq, float* partial, hipStream_t st) {
    const int splits = n_splits(I, J, nq);
    const long long per = gl_ceil_div(gl_ceil_div(nq, splits), kBQ) * kBQ;
    const long long used = gl_ceil_div(nq, per);             // rounding up to whole steps may leave fewer parts
    const long long tiles = gl_ceil_div(I, kTile) * gl_ceil_div(J, kTile);
    if (tiles > 0x7fffffffLL) return gl_set_error(GL_ERR_INVALID, "gl_dense: %lld tiles are too many for one launch", tiles);
    e.partial = used > 1 ? partial : nullptr;
    e.exact_p = nullptr;
    e.quads = quads<TO>(e, J);
    const bool wide = wide_loads(P, P.qs == 1 ? nq : I, sizeof(T)) && wide_loads(Q, Q.qs == 1 ? nq : J, sizeof(T));
    auto kernel = wide ? k_dense_any<T, TO, 16 / sizeof(T), TWO> : k_dense_any<T, TO, 1, TWO>;
    const AnyArgs a = {P, Q, {}, e, I, nq, per, J, (int)gl_ceil_div(J, kTile), (int)tiles, GL_ACT_NONE, P.qs == 1,
                       Q.qs == 1, nullptr, nullptr};
    hipLaunchKernelGGL(kernel, dim3((unsigned)(tiles < kMostBlocks ? tiles : kMostBlocks), (unsigned)used), dim3(256), 0, st, a,
                       (const int*)nullptr);
    GL_HIP_CHECK(hipGetLastError());
    return used > 1 ? gl_dense_join<T, TO>(e, I, J, (int)used, st) : 0;
}

// Layers of fewer multiplications than this go as they are to k_dense_any (forward, where the tiles would need copies) and
// k_dense_back_small.  `odd`: widths off the 16 bytes that those load at once.  Microseconds a call there / on the tiles:
//   float32   forward   2000 x 512 -> 512 23 / 29, 2000 x 500 -> 700 34 / 34, 861 x 1024 -> 1024 41 / 36
//             odd       641 x 257 -> 513 18 / 24, 6888 x 81 -> 512 25 / 23, 2000 x 501 -> 701 54 / 37
//             backward  861 x 1024 -> 1024 73 / 90, 2000 x 1024 -> 1024 137 / 132, 6888 x 1024 -> 512 229 / 165
//             odd       641 x 257 -> 513 33 / 66, 6888 x 81 -> 512 101 / 75, 641 x 512 -> 1025 82 / 72
//   16 bits   odd       4000 x 17 -> 33 6.5 / 7.8, 641 x 81 -> 100 8.1 / 8.1, 61 x 948 -> 144 13.4 / 11.5, 641 x 257 -> 513 17 / 10
//             backward  861 x 512 -> 512 22 / 28, 6888 x 80 -> 512 40 / 35, 2000 x 512 -> 512 39 / 34
//             odd       641 x 129 -> 300 18 / 22, 2000 x 129 -> 300 25 / 25, 300 x 1001 -> 300 26 / 21
double small_layer(int dtype, int inputs, int outputs, bool back) {
    const int whole = dtype == GL_F32 ? 4 : 8;
    const bool odd = inputs % whole || (back && outputs % whole);
    if (dtype == GL_F32) return back ? (odd ? 3 << 26 : 3LL << 29) : odd ? 1 << 28 : 3 << 28;
    return back ? (odd ? 3 << 24 : 1 << 28) : 1 << 22;
}
bool is_small(long long rows, int inputs, int outputs, int dtype, bool back) {
    return (double)rows * inputs * outputs < small_layer(dtype, inputs, outputs, back);
}
int pad_to(int n) { return (n + kPadded - 1) / kPadded * kPadded; }
bool copies(int dtype, int width) { return dtype == GL_F32 || width % 8 != 0; }
long long copy_bytes(int dtype, long long rows, int cols) {
    return gl_align16(rows * pad_to(cols) * (dtype == GL_F32 ? 6LL : 2LL));
}
long long halves_bytes(long long rows, int cols) { return gl_align16(rows * pad_to(cols) * 4LL); }
// a flag and a count for every 64 x 64 block
long long flag_bytes(int dtype, long long I, int J) { return dtype == GL_F32 ? gl_align16(gl_ceil_div(I, 64) * gl_ceil_div(J, 64) * 8) : 0; }
// flags and parts of a product, whichever kernel takes it
long long partial_bytes(int dtype, long long I, int J, long long nq, bool any_q, bool fast) {
    const long long any = any_bytes(I, J, nq);
    const long long mm = dtype == GL_F32 && !fast ? 0 : gl_mm_partial_bytes(I, J, nq, any_q);
    return (any > mm ? any : mm) + (fast ? flag_bytes(dtype, I, J) : 0);
}

// Copies of `cols` columns of a and, where it has rows, b.
template <typename T>
int pack(const Packed& a, const Packed& b, int cols, hipStream_t st) {
    const int padded = pad_to(cols);
    const long long blocks = gl_ceil_div((a.rows + b.rows) * (padded / 8), 256);
    hipLaunchKernelGGL((k_dense_pack<T, sizeof(T) == 4 ? 3 : 1>), dim3((unsigned)(blocks < 8192 ? blocks : 8192)), dim3(256), 0, st, a, b, cols, padded);
    GL_HIP_CHECK(hipGetLastError());
    return 0;
}
// The operand that a copy is: of `rows` rows of `cols` columns, which lie across or along the contraction
Operand copied(const Packed& a, int cols, bool across) {
    const int padded = pad_to(cols);
    return across ? Operand{a.out, 1, padded, a.rows * padded, true} : Operand{a.out, padded, 1, a.rows * padded, true};
}

// The product on prepared operands (16-bit as they lie or copied, float32 in planes), else on the originals (P0, Q0).
template <typename T, typename TO, int SEG>
int product(const Operand& P, const Operand& Q, const Operand& P0, const Operand& Q0, Epilogue e, long long I, int J, long long nq,
            float* partial, bool fast, hipStream_t st) {
    if constexpr (sizeof(T) == 2) {
        if (gl_mm16_takes(P, Q, e, I, J, nq, sizeof(TO))) return gl_mm16<T, TO, T, SEG>(P, Q, e, I, J, nq, partial, st);
    } else if constexpr (SEG > 1) {
        if (fast && gl_mm16_takes(P, Q, e, I, J, nq, sizeof(TO))) {
            e.exact_p = (const float*)P0.base;
            e.exact_q = (const float*)Q0.base;
            e.exact_p_is = P0.is;
            e.exact_p_qs = P0.qs;
            e.exact_q_is = Q0.is;
            e.exact_q_qs = Q0.qs;
            e.exact_nq = nq;
            e.flags = (int*)partial;
            typedef typename std::conditional<SEG == 3, gl_f16, gl_bf16>::type Plane;
            return gl_mm16<Plane, float, float, SEG>(P, Q, e, I, J, nq, partial + flag_bytes(GL_F32, I, J) / 4, st);
        }
    }
    e.scale_p = nullptr;
    return any_product<T, TO, SEG == 2>(P0, Q0, e, I, J, nq, partial, st);
}

int check_types(int dtype, int out_dtype, int act, const char* who) {
    if (dtype < GL_F32 || dtype > GL_F16) return gl_set_error(GL_ERR_INVALID, "%s: dtype=%d", who, dtype);
    if (out_dtype != dtype && out_dtype != GL_F32)
        return gl_set_error(GL_ERR_INVALID, "%s: out_dtype=%d must be the dtype (%d) or GL_F32", who, out_dtype, dtype);
    if (act < GL_ACT_NONE || act > GL_ACT_EXP) return gl_set_error(GL_ERR_INVALID, "%s: activation=%d", who, act);
    return 0;
}
constexpr int kMaxWidth = 1 << 20;
int check_sizes(long long rows, int inputs, int outputs, const char* who) {
    if (rows < 0 || rows > 0x7fffffffLL) return gl_set_error(GL_ERR_INVALID, "%s: rows=%lld", who, rows);
    if (inputs < 1 || inputs > kMaxWidth || outputs < 1 || outputs > kMaxWidth)
        return gl_set_error(GL_ERR_INVALID, "%s: inputs=%d, outputs=%d outside [1, %d]", who, inputs, outputs, kMaxWidth);
    return 0;
}
int check_stride(long long stride, int cols, const char* what, const char* who) {
    if (stride < cols || stride > (1LL << 31))
        return gl_set_error(GL_ERR_INVALID, "%s: %s row stride %lld outside [%d, 2^31]", who, what, stride, cols);
    return 0;
}
// Elements start on whole multiples of their own size.
int check_elements(std::initializer_list<const void*> arrays, int dtype, const char* who) {
    for (const void* p : arrays)
        if ((uintptr_t)p % (dtype == GL_F32 ? 4 : 2)) return gl_set_error(GL_ERR_INVALID, "%s: %p is not on its elements' size", who, p);
    return 0;
}
int check_workspace(const void* ws, long long have, long long need, const char* who) {
    if (need == 0) return 0;
    if (!ws || have < need)
        return gl_set_error(GL_ERR_INVALID, "%s: workspace of %lld bytes needed, %lld given", who, need, ws ? have : 0LL);
    if ((uintptr_t)ws % 16) return gl_set_error(GL_ERR_INVALID, "%s: workspace must be 16-byte aligned", who);
    return 0;
}

// ---- forward ----
constexpr int kFewRows = 8;

// workspace: [copy of x] [copy of weight] [their scales, where the copies are halves of float32] [flags and parts]
struct FrontLayout {
    bool fast, copy;
    long long x_bytes, w_bytes, scale_bytes, partial;
    long long total() const { return x_bytes + w_bytes + scale_bytes + partial; }
};
FrontLayout front_layout(long long rows, int inputs, int outputs, int dtype) {
    FrontLayout l = {};
    if (rows <= kFewRows) return l;
    l.fast = !is_small(rows, inputs, outputs, dtype, false);
    l.copy = l.fast && copies(dtype, inputs);
    if (l.copy && dtype == GL_F32) {
        l.x_bytes = halves_bytes(rows, inputs);
        l.w_bytes = halves_bytes(outputs, inputs);
        l.scale_bytes = gl_align16((rows + outputs) * 4);
    } else if (l.copy) {
        l.x_bytes = copy_bytes(dtype, rows, inputs);
        l.w_bytes = copy_bytes(dtype, outputs, inputs);
    }
    l.partial = partial_bytes(dtype, rows, outputs, l.copy ? pad_to(inputs) : inputs, false, l.fast);
    return l;
}

template <typename T, typename TO, int ROWS>
int few(const void* x, long long x_stride, const void* w, long long w_stride, const Epilogue& e, int rows, int K, int N, hipStream_t st) {
    int V = 16 / sizeof(T);              // elements at once: what the widths and the arrays' alignment allow
    auto fits = [&](const void* p, long long stride) { return K % V == 0 && stride % V == 0 && (uintptr_t)p % (V * sizeof(T)) == 0; };
    while (V > 1 && (!fits(x, x_stride) || !fits(w, w_stride))) V /= 2;
    const int pieces = K / V;
    int L = kFewRows;                    // a lane for every row's result at least
    while (L < 64 && L < pieces) L *= 2;
    const unsigned grid = (unsigned)gl_ceil_div(N, 4 * (64 / L));
    auto kernel = V == 1 ? k_dense_few<T, TO, ROWS, 1> : V == 2 ? k_dense_few<T, TO, ROWS, 2>
                : V == 4 ? k_dense_few<T, TO, ROWS, 4> : k_dense_few<T, TO, ROWS, 16 / sizeof(T)>;
    hipLaunchKernelGGL(kernel, dim3(grid), dim3(256), 0, st, (const T*)x, x_stride, (const T*)w, w_stride, e, rows, K, N, L);
    GL_HIP_CHECK(hipGetLastError());
    return 0;
}

template <typename T, typename TO>
int forward(const void* x, long long x_stride, const void* w, long long w_stride, const Epilogue& e, long long rows,
            int inputs, int outputs, const FrontLayout& l, void* ws, hipStream_t st) {
    if (rows == 1) return few<T, TO, 1>(x, x_stride, w, w_stride, e, 1, inputs, outputs, st);
    if (rows == 2) return few<T, TO, 2>(x, x_stride, w, w_stride, e, 2, inputs, outputs, st);
    if (rows <= 4) return few<T, TO, 4>(x, x_stride, w, w_stride, e, (int)rows, inputs, outputs, st);
    if (rows <= kFewRows) return few<T, TO, kFewRows>(x, x_stride, w, w_stride, e, (int)rows, inputs, outputs, st);
    const Operand P0 = {x, x_stride, 1}, Q0 = {w, w_stride, 1};
    Operand P = P0, Q = Q0;
    char *at = (char*)ws, *w_copy = at + l.x_bytes, *scale = w_copy + l.w_bytes;
    float* partial = (float*)(scale + l.scale_bytes);
    if (!l.copy) return product<T, TO, 1>(P, Q, P0, Q0, e, rows, outputs, inputs, partial, l.fast, st);
    if constexpr (sizeof(T) == 2) {
        const Packed a = {x, x_stride, rows, at}, b = {w, w_stride, outputs, w_copy};
        const int rc = pack<T>(a, b, inputs, st);
        P = copied(a, inputs, false);
        Q = copied(b, inputs, false);
        return rc ? rc : product<T, TO, 1>(P, Q, P0, Q0, e, rows, outputs, inputs, partial, true, st);
    } else {
        const int padded = pad_to(inputs);
        Epilogue f = e;
        f.scale_p = (const int*)scale;
        f.scale_q = f.scale_p + rows;
        const Halves a = {(const float*)x, x_stride, rows, (gl_f16*)at, (int*)scale};
        const Halves b = {(const float*)w, w_stride, outputs, (gl_f16*)w_copy, (int*)scale + rows};
        const long long blocks = gl_ceil_div(rows + outputs, 4);
        const dim3 grid((unsigned)(blocks < 4096 ? blocks : 4096));
        if (wide_loads(P0, inputs, 4) && wide_loads(Q0, inputs, 4))
            hipLaunchKernelGGL((k_dense_halves<true>), grid, dim3(256), 0, st, a, b, inputs, padded);
        else
            hipLaunchKernelGGL((k_dense_halves<false>), grid, dim3(256), 0, st, a, b, inputs, padded);
        GL_HIP_CHECK(hipGetLastError());
        P = {at, padded, 1, rows * padded, true};
        Q = {w_copy, padded, 1, (long long)outputs * padded, true};
        return product<T, TO, 3>(P, Q, P0, Q0, f, rows, outputs, inputs, partial, true, st);
    }
}

// ---- backward ----
// Frames of a part of the column sums: about 2048 workgroups of k_dense_dz in all (its loads in flight then reach what the
// memory needs: 55 104 x 2048 bf16 gelu 190 us with 512 of them), 16 frames at least.
int rows_per_part(long long rows, int outputs) {
    const long long r = gl_ceil_div(rows, 2048 / gl_ceil_div(outputs, 512) + 1);
    return (int)(r < 16 ? 16 : r);
}

// One product of k_dense_back_small: parts for one workgroup a CU, of two steps at least, or for two, of eight; and no more
// than balance a part's steps with the join, where eight parts cost what a step does (24 125 x 64 -> 64 bf16: dweight in 256
// parts 44 us, in 78 32 us).
struct SmallSplit {
    long long tiles, per;
    int parts;
};
SmallSplit small_split(long long I, int J, long long nq) {
    SmallSplit s;
    s.tiles = gl_ceil_div(I, kTile) * gl_ceil_div(J, kTile);
    auto parts = [&](long long workgroups, int steps) {
        const long long fill = workgroups / s.tiles, most = nq / (steps * kBQ);
        return fill < most ? fill : most;
    };
    const long long one = parts(kCUs, 2), two = parts(2 * kCUs, 8);
    long long most = one > two ? one : two;
    while (most > 1 && 4 * most * most > nq) --most;
    s.per = gl_ceil_div(gl_ceil_div(nq, most > 1 ? most : 1), kBQ) * kBQ;
    s.parts = (int)gl_ceil_div(nq, s.per);
    return s;
}

// Whether 16-bit products take dz in two planes.  bfloat16 with a dy of its own type: once rounded (half a step a term, what dy
// itself has lost already: the gradients' error against 64 bits is 0.0023 of them where their own rounding makes 0.0017, and
// 55 104 x 512 -> 2048 gelu takes 374 us where two planes take 614).  A caller who keeps dy and z in float32 keeps dz to 2^-17
// of it (676 us, rounded once 463).  float16: dz falls below the type's range where dy does not (a mean over a batch's magnitudes
// has gradients of 2e-8, and act' makes them smaller), and sums over frames bring it back: two planes reach 2^-44 (633 us, rounded
// once 380).  Without an activation and with relu dz is dy or zero: it serves as it is where dy is of the products' type.
bool splits_dz(int dtype, int out_dtype, int act) {
    return dtype != GL_F32 && (out_dtype == GL_F32 || (dtype == GL_F16 && act > GL_ACT_RELU));
}

// workspace of a small layer: [parts of dx] [parts of dweight] [parts of dbias]; else
// [dz (unless dy serves), or its planes] [with planes: dz itself, for sums that are not finite] [copy of x]
// [copy of weight] [column-sum parts] [flags and parts of dx and dweight, one after the other on the stream: the larger]
struct BackLayout {
    bool small, own_dz, copy, planes, two;
    SmallSplit x, w;
    long long dz_stride, dz_bytes, dz32_bytes, x_bytes, w_bytes, parts_bytes, partial;
    long long total() const { return dz_bytes + dz32_bytes + x_bytes + w_bytes + parts_bytes + partial; }
};
BackLayout back_layout(long long rows, int inputs, int outputs, int dtype, int out_dtype, int act) {
    BackLayout l = {};
    l.two = splits_dz(dtype, out_dtype, act);
    l.small = is_small(rows, inputs, outputs, dtype, true);
    if (l.small) {
        l.x = small_split(rows, inputs, outputs);
        l.w = small_split(outputs, inputs, rows);
        if (l.x.parts > 1) l.x_bytes = gl_align16(4LL * l.x.parts * rows * inputs);
        if (l.w.parts > 1) l.w_bytes = gl_align16(4LL * l.w.parts * outputs * inputs);
        if (l.w.parts > 1) l.parts_bytes = gl_align16(4LL * l.w.parts * outputs);
        return l;
    }
    l.planes = dtype == GL_F32;
    // dy itself serves where nothing is to be multiplied, converted or padded
    l.own_dz = act != GL_ACT_NONE || dtype != out_dtype || (dtype != GL_F32 && outputs % 32) || l.planes;
    l.dz_stride = pad_to(outputs);
    if (l.own_dz) l.dz_bytes = gl_align16(rows * l.dz_stride * (l.planes ? 6 : l.two ? 4 : 2));
    if (l.planes && act != GL_ACT_NONE) l.dz32_bytes = gl_align16(rows * l.dz_stride * 4);
    l.copy = copies(dtype, inputs);
    if (l.copy) {
        l.x_bytes = copy_bytes(dtype, rows, inputs);
        l.w_bytes = copy_bytes(dtype, outputs, inputs);
    }
    l.parts_bytes = gl_align16(gl_ceil_div(rows, rows_per_part(rows, outputs)) * outputs * 4);
    const long long a = partial_bytes(dtype, rows, inputs, l.own_dz ? l.dz_stride : outputs, false, true);
    const long long b = partial_bytes(dtype, outputs, inputs, rows, true, true);
    l.partial = a > b ? a : b;
    return l;
}

template <typename T, typename TO, int V, int PLANES>
int dz_launch(const void* dy, long long dy_stride, const void* z, long long z_stride, void* dz, long long dz_stride, float* exact, float* parts,
              long long rows, int outputs, int act, hipStream_t st) {
    const int rpp = rows_per_part(rows, outputs);
    hipLaunchKernelGGL((k_dense_dz<T, TO, V, PLANES>), dim3((unsigned)gl_ceil_div(dz ? dz_stride : outputs, 64 * V),
                       (unsigned)gl_ceil_div(rows, rpp)), dim3(256), 0, st, (const TO*)dy, dy_stride, (const TO*)z, z_stride, dz,
                       dz_stride, rows * dz_stride, exact, parts, rows, outputs, rpp, act);
    GL_HIP_CHECK(hipGetLastError());
    return 0;
}
template <typename T, typename TO, int PLANES>
int dz_pass(const void* dy, long long dy_stride, const void* z, long long z_stride, void* dz, long long dz_stride, float* exact, float* parts,
            long long rows, int outputs, int act, hipStream_t st) {
    constexpr int V = 16 / sizeof(TO);   // 16 bytes at a time where rows and columns allow
    auto wide = [&](const void* p, long long stride) { return (uintptr_t)p % 16 == 0 && stride % V == 0; };
    if (outputs % V == 0 && wide(dy, dy_stride) && (act == GL_ACT_NONE || wide(z, z_stride)))
        return dz_launch<T, TO, V, PLANES>(dy, dy_stride, z, z_stride, dz, dz_stride, exact, parts, rows, outputs, act, st);
    return dz_launch<T, TO, 1, PLANES>(dy, dy_stride, z, z_stride, dz, dz_stride, exact, parts, rows, outputs, act, st);
}

template <typename T, typename TO, bool TWO>
int backward_small(const void* dy, long long dy_stride, const void* x, long long x_stride, const void* w, long long w_stride,
                   const void* z, long long z_stride, void* dx, long long dx_stride, void* dw, long long dw_stride, void* db,
                   long long rows, int inputs, int outputs, int act, const BackLayout& l, void* ws, hipStream_t st) {
    char* at = (char*)ws;
    AnyArgs a = {{dy, dy_stride, 1}, {w, 1, w_stride}, {z, z_stride, 1}, {}, rows, outputs, l.x.per, inputs,
                 (int)gl_ceil_div(inputs, kTile), (int)l.x.tiles, act, true, false, nullptr, nullptr};
    AnyArgs b = {{dy, 1, dy_stride}, {x, 1, x_stride}, {z, 1, z_stride}, {}, outputs, rows, l.w.per, inputs,
                 (int)gl_ceil_div(inputs, kTile), (int)l.w.tiles, act, false, false, nullptr, nullptr};
    a.e.y = dx;
    a.e.y_stride = dx_stride;
    b.e.y = dw;
    b.e.y_stride = dw_stride;
    if (!dw) {                           // sums of dz alone: one column of tiles
        b.Q.base = nullptr;
        b.tiles_j = 1;
        b.n_tiles = (int)gl_ceil_div(outputs, kTile);
    }
    a.e.quads = quads<T>(a.e, inputs);
    b.e.quads = quads<T>(b.e, inputs);
    if (dx && l.x.parts > 1) a.e.partial = (float*)at;
    if (dw && l.w.parts > 1) b.e.partial = (float*)(at + l.x_bytes);
    if (db && l.w.parts > 1) b.sums = (float*)(at + l.x_bytes + l.w_bytes);
    else b.db = db;
    const long long x_blocks = dx ? l.x.tiles * l.x.parts : 0, w_blocks = dw || db ? (long long)b.n_tiles * l.w.parts : 0;
    const bool v = wide_loads(a.P, outputs, sizeof(TO)) && (act == GL_ACT_NONE || wide_loads(a.Z, outputs, sizeof(TO))) &&
                   (!dx || wide_loads(a.Q, inputs, sizeof(T))) && (!dw || wide_loads(b.Q, inputs, sizeof(T)));
    auto kernel = v ? k_dense_back_small<T, TO, 16 / sizeof(T), TWO> : k_dense_back_small<T, TO, 1, TWO>;
    hipLaunchKernelGGL(kernel, dim3((unsigned)(x_blocks + w_blocks)), dim3(256), 0, st, a, b, (int)x_blocks);
    GL_HIP_CHECK(hipGetLastError());
    BackJoin j = {a.e.partial, b.e.partial, b.sums, l.x.parts, l.w.parts, a.e.partial ? rows * inputs : 0,
                  b.e.partial ? (long long)outputs * inputs : 0, dx, dw, db, dx_stride, dw_stride, inputs, b.sums ? outputs : 0};
    const long long n = j.x_n + j.w_n + j.outputs;
    if (n == 0) return 0;
    const int V = inputs % 4 == 0 ? 4 : 1;
    const long long blocks = gl_ceil_div(n, 256 * V);
    const dim3 grid((unsigned)(blocks < 4096 ? blocks : 4096));
    if (V == 4) hipLaunchKernelGGL((k_dense_back_join<T, 4>), grid, dim3(256), 0, st, j);
    else hipLaunchKernelGGL((k_dense_back_join<T, 1>), grid, dim3(256), 0, st, j);
    GL_HIP_CHECK(hipGetLastError());
    return 0;
}

template <typename T, typename TO, bool TWO>
int backward(const void* dy, long long dy_stride, const void* x, long long x_stride, const void* w, long long w_stride,
             const void* z, long long z_stride, void* dx, long long dx_stride, void* dw, long long dw_stride, void* db,
             long long rows, int inputs, int outputs, int act, const BackLayout& l, void* ws, hipStream_t st) {
    char* at = (char*)ws;
    const bool products = dx || dw;
    void* dz = l.own_dz && products ? at : nullptr;
    float* dz32 = l.dz32_bytes && products ? (float*)(at + l.dz_bytes) : nullptr;
    char* x_copy = at + l.dz_bytes + l.dz32_bytes;
    char* w_copy = x_copy + l.x_bytes;
    float* parts = (float*)(w_copy + l.w_bytes);
    float* partial = (float*)((char*)parts + l.parts_bytes);
    int rc = 0;
    if (dz || db) {
        float* sums = db ? parts : nullptr;
        rc = dz_pass<T, TO, sizeof(T) == 4 ? 3 : TWO ? 2 : 1>(dy, dy_stride, z, z_stride, dz, l.dz_stride, dz32, sums, rows, outputs, act, st);
        if (rc) return rc;
    }
    if (db) {
        hipLaunchKernelGGL((k_dense_db<T>), dim3((unsigned)gl_ceil_div(outputs, 16)), dim3(1024), 0, st, parts,
                           (int)gl_ceil_div(rows, rows_per_part(rows, outputs)), (T*)db, outputs);
        GL_HIP_CHECK(hipGetLastError());
    }
    // dz as the products read it, and as it is
    const void* d = dz ? (const void*)dz : dy;
    const long long d_stride = dz ? l.dz_stride : dy_stride, plane = rows * l.dz_stride;
    const bool padded = dz != nullptr;
    const void* d0 = !l.planes ? d : dz32 ? (const void*)dz32 : dy;
    const long long d0_stride = !l.planes ? d_stride : dz32 ? l.dz_stride : dy_stride;
    const Packed wp = {w, w_stride, dx ? outputs : 0, w_copy}, xp = {x, x_stride, dw ? rows : 0, x_copy};
    if (l.copy && products) rc = pack<T>(wp, xp, inputs, st);
    if (rc) return rc;
    constexpr int SEG = sizeof(T) == 4 ? 6 : TWO ? 2 : 1;
    Epilogue e = {};
    if (dx) {
        const Operand Q0 = {w, 1, w_stride}, Q = l.copy ? copied(wp, inputs, true) : Q0;
        e.y = dx;
        e.y_stride = dx_stride;
        rc = product<T, T, SEG>({d, d_stride, 1, plane, padded}, Q, {d0, d0_stride, 1, plane}, Q0, e, rows, inputs, outputs, partial, true, st);
        if (rc) return rc;
    }
    if (dw) {
        const Operand Q0 = {x, 1, x_stride}, Q = l.copy ? copied(xp, inputs, true) : Q0;
        e.y = dw;
        e.y_stride = dw_stride;
        rc = product<T, T, SEG>({d, 1, d_stride, plane, padded}, Q, {d0, 1, d0_stride, plane}, Q0, e, outputs, inputs, rows, partial, true, st);
    }
    return rc;
}

}  // namespace

template <typename T, typename TO>
int gl_dense_join(const gl_epilogue& e, long long I, int J, int parts, hipStream_t st) {
    const int V = J % 4 == 0 ? 4 : 1;
    const long long blocks = gl_ceil_div(I * J, 256 * V);
    const dim3 grid((unsigned)(blocks < 4096 ? blocks : 4096));
    if (V == 4) hipLaunchKernelGGL((k_dense_join<T, TO, 4>), grid, dim3(256), 0, st, e, I, J, parts);
    else hipLaunchKernelGGL((k_dense_join<T, TO, 1>), grid, dim3(256), 0, st, e, I, J, parts);
    GL_HIP_CHECK(hipGetLastError());
    return 0;
}
template int gl_dense_join<float, float>(const gl_epilogue&, long long, int, int, hipStream_t);
template int gl_dense_join<gl_bf16, gl_bf16>(const gl_epilogue&, long long, int, int, hipStream_t);
template int gl_dense_join<gl_bf16, float>(const gl_epilogue&, long long, int, int, hipStream_t);
template int gl_dense_join<gl_f16, gl_f16>(const gl_epilogue&, long long, int, int, hipStream_t);
template int gl_dense_join<gl_f16, float>(const gl_epilogue&, long long, int, int, hipStream_t);

int gl_dense_join_planes(const gl_epilogue& e, long long I, int J, long long nq, const gl_mm_plan& p, hipStream_t st) {
    const long long tiles = gl_ceil_div(I, kTile) * gl_ceil_div(J, kTile);
    const int tiles_j = (int)gl_ceil_div(J, kTile);
    const bool wide = J % 4 == 0;
    hipLaunchKernelGGL((wide ? k_dense_join_rows<4> : k_dense_join_rows<1>), dim3((unsigned)tiles, kTile / kJoinRows), dim3(256), 0, st, e, I, J,
                       p.parts, tiles_j);
    GL_HIP_CHECK(hipGetLastError());
    gl_epilogue f = {};
    f.partial = e.partial;
    const AnyArgs a = {{e.exact_p, e.exact_p_is, e.exact_p_qs}, {e.exact_q, e.exact_q_is, e.exact_q_qs}, {}, f, I, nq, p.per, J, tiles_j,
                       (int)tiles, GL_ACT_NONE, e.exact_p_qs == 1, e.exact_q_qs == 1, nullptr, nullptr};
    hipLaunchKernelGGL((wide ? k_dense_repair<4> : k_dense_repair<1>), dim3((unsigned)(tiles < 512 ? tiles : 512), p.parts), dim3(256), 0, st, a, e,
                       p.parts);
    GL_HIP_CHECK(hipGetLastError());
    return 0;
}

int gl_dense_flagged(const gl_epilogue& e, long long I, int J, long long nq, hipStream_t st) {
    const long long tiles = gl_ceil_div(I, kTile) * gl_ceil_div(J, kTile);
    gl_epilogue f = e;
    f.partial = nullptr;
    f.quads = quads<float>(e, J);
    const AnyArgs a = {{e.exact_p, e.exact_p_is, e.exact_p_qs}, {e.exact_q, e.exact_q_is, e.exact_q_qs}, {}, f, I, nq, nq, J,
                       (int)gl_ceil_div(J, kTile), (int)tiles, GL_ACT_NONE, e.exact_p_qs == 1, e.exact_q_qs == 1, nullptr, nullptr};
    hipLaunchKernelGGL((k_dense_any<float, float, 1, false>), dim3((unsigned)(tiles < 512 ? tiles : 512)), dim3(256), 0, st, a, e.flags);
    GL_HIP_CHECK(hipGetLastError());
    return 0;
}

// 256 x 256 tiles where they fill half the chip (parts included), else 128 x 128, else 64 x 64.  A part of the contraction has
// at least 2048 indexes with large tiles, 512 with medium and 256 with small ones: shorter ones cost more in the join than
// they fill (6888 x 1024 x 1024 float32 in two parts of large tiles 120 us, in one of medium ones 92).
gl_mm_plan gl_mm_plan_for(long long I, int J, long long nq, bool any_q) {
    auto split = [&](int b, long long least) -> gl_mm_plan {
        const long long tiles = gl_ceil_div(I, b) * gl_ceil_div(J, b);
        const long long fill = b == 256 ? kCUs : 2 * kCUs;
        long long parts = tiles * 2 > fill ? 1 : fill / tiles;
        if (parts > nq / least) parts = nq / least;
        if (parts > 64) parts = 64;
        if (parts < 1) parts = 1;
        const long long per = gl_ceil_div(gl_ceil_div(nq, parts), 64) * 64;
        return {0, (int)gl_ceil_div(nq, per), per};
    };
    if (J % 256 == 0 && I >= 256 && (any_q || nq % 32 == 0)) {
        gl_mm_plan p = split(256, 2048);
        if (gl_ceil_div(I, 256) * (J / 256) * p.parts >= 128) {
            p.kind = 2;
            return p;
        }
    }
    gl_mm_plan p = split(128, 512);
    if (I >= 96 && J >= 96 && gl_ceil_div(I, 128) * gl_ceil_div(J, 128) * p.parts >= 256) {
        p.kind = 1;
        return p;
    }
    return split(64, 256);
}

int gl_mm_first_columns(long long I, int J, long long nq, bool any_q, int out_size) {
    // columns that end inside a tile, and rows that start off 4 bytes, go to smaller tiles: the large ones have no registers
    // for a second way to store
    const int whole = J / 256 * 256;
    if (J % 2 && out_size == 2) return J;
    return whole > 0 && whole < J && gl_mm_plan_for(I, whole, nq, any_q).kind == 2 ? whole : J;
}

long long gl_mm_partial_bytes(long long I, int J, long long nq, bool any_q) {
    auto bytes = [&](int cols) {
        const gl_mm_plan p = gl_mm_plan_for(I, cols, nq, any_q);
        return p.parts > 1 ? (long long)p.parts * I * cols * 4 : 0;
    };
    const int first = gl_mm_first_columns(I, J, nq, any_q, 4);
    long long most = bytes(J);                               // in one launch, or in two: that goes by the result's type
    if (bytes(first) > most) most = bytes(first);
    if (first < J && bytes(J - first) > most) most = bytes(J - first);
    return gl_align16(most);
}

bool gl_mm16_takes(const gl_operand& P, const gl_operand& Q, const gl_epilogue& e, long long I, int J, long long nq, int out_size) {
    auto side = [&](const gl_operand& o, long long rows) {
        const long long stride = o.across() ? o.qs : o.is;
        return (uintptr_t)o.base % 16 == 0 && stride % 8 == 0 && stride <= (1 << 21) && (o.padded || (o.across() ? rows : nq) % 8 == 0);
    };
    auto out = [&](const void* p, long long stride) {        // stores of four bytes and more; single elements where J is odd
        return !p || (stride <= (1 << 20) && (J % 2 || ((uintptr_t)p % 4 == 0 && stride * out_size % 4 == 0)));
    };
    if (P.across() && !Q.across()) return false;
    return side(P, I) && side(Q, J) && out(e.y, e.y_stride) && out(e.z, e.z_stride) && out(e.residual, e.r_stride) && nq < (1LL << 31) - 64 &&
           gl_ceil_div(I, 64) * gl_ceil_div(J, 64) < (1LL << 24) - 8;   // workgroups of 256 threads in a launch
}

extern "C" {

long long gl_dense_workspace(long long rows, int inputs, int outputs, int dtype, int out_dtype) {
    if (check_types(dtype, out_dtype, 0, "gl_dense_workspace") || check_sizes(rows, inputs, outputs, "gl_dense_workspace"))
        return GL_ERR_INVALID;
    return rows ? front_layout(rows, inputs, outputs, dtype).total() : 0;
}

int gl_dense(const void* x, long long x_stride, const void* weight, long long w_stride, const void* bias,
             const void* residual, long long r_stride, void* y, long long y_stride, void* preactivation,
             long long z_stride, long long rows, int inputs, int outputs, int dtype, int out_dtype, int activation,
             void* workspace, long long workspace_bytes, void* stream) {
    int rc = check_types(dtype, out_dtype, activation, "gl_dense");
    if (!rc) rc = check_sizes(rows, inputs, outputs, "gl_dense");
    if (rc || rows == 0) return rc;
    if (!x || !weight || !y) return gl_set_error(GL_ERR_INVALID, "gl_dense: NULL buffer");
    rc = check_stride(x_stride, inputs, "x", "gl_dense");
    if (!rc) rc = check_stride(w_stride, inputs, "weight", "gl_dense");
    if (!rc) rc = check_stride(y_stride, outputs, "y", "gl_dense");
    if (!rc && residual) rc = check_stride(r_stride, outputs, "residual", "gl_dense");
    if (!rc && preactivation) rc = check_stride(z_stride, outputs, "preactivation", "gl_dense");
    if (!rc) rc = check_elements({x, weight, bias}, dtype, "gl_dense");
    if (!rc) rc = check_elements({residual, y, preactivation}, out_dtype, "gl_dense");
    const FrontLayout l = front_layout(rows, inputs, outputs, dtype);
    if (!rc) rc = check_workspace(workspace, workspace_bytes, l.total(), "gl_dense");
    if (rc) return rc;
    Epilogue e = {};
    e.bias = bias;
    e.residual = residual;
    e.r_stride = r_stride;
    e.y = y;
    e.y_stride = y_stride;
    e.z = preactivation;
    e.z_stride = z_stride;
    e.act = activation;
    const hipStream_t st = (hipStream_t)stream;
#define GL_FRONT(T, TO) forward<T, TO>(x, x_stride, weight, w_stride, e, rows, inputs, outputs, l, workspace, st)
    if (dtype == GL_F32) return GL_FRONT(float, float);
    if (dtype == GL_BF16) return out_dtype == GL_F32 ? GL_FRONT(gl_bf16, float) : GL_FRONT(gl_bf16, gl_bf16);
    return out_dtype == GL_F32 ? GL_FRONT(gl_f16, float) : GL_FRONT(gl_f16, gl_f16);
#undef GL_FRONT
}

long long gl_dense_backward_workspace(long long rows, int inputs, int outputs, int dtype, int out_dtype, int activation) {
    if (check_types(dtype, out_dtype, activation, "gl_dense_backward_workspace") ||
        check_sizes(rows, inputs, outputs, "gl_dense_backward_workspace"))
        return GL_ERR_INVALID;
    return rows ? back_layout(rows, inputs, outputs, dtype, out_dtype, activation).total() : 0;
}

int gl_dense_backward(const void* dy, long long dy_stride, const void* x, long long x_stride, const void* weight,
                      long long w_stride, const void* preactivation, long long z_stride, void* dx, long long dx_stride,
                      void* dweight, long long dw_stride, void* dbias, long long rows, int inputs, int outputs,
                      int dtype, int out_dtype, int activation, void* workspace, long long workspace_bytes,
                      void* stream) {
    int rc = check_types(dtype, out_dtype, activation, "gl_dense_backward");
    if (!rc) rc = check_sizes(rows, inputs, outputs, "gl_dense_backward");
    if (!rc && dweight) rc = check_stride(dw_stride, inputs, "dweight", "gl_dense_backward");
    if (!rc) rc = check_elements({x, weight, dx, dweight, dbias}, dtype, "gl_dense_backward");
    if (!rc) rc = check_elements({dy, preactivation}, out_dtype, "gl_dense_backward");
    if (rc) return rc;
    const hipStream_t st = (hipStream_t)stream;
    if (rows == 0) {                                         // empty sums
        auto zero = [&](void* p, long long stride, int r, int c) -> int {
            const long long blocks = gl_ceil_div((long long)r * c, 256);
            const dim3 grid((unsigned)(blocks < 4096 ? blocks : 4096));
            if (dtype == GL_F32) hipLaunchKernelGGL((k_dense_zero<float>), grid, dim3(256), 0, st, (float*)p, stride, r, c);
            else hipLaunchKernelGGL((k_dense_zero<gl_f16>), grid, dim3(256), 0, st, (gl_f16*)p, stride, r, c);
            GL_HIP_CHECK(hipGetLastError());
            return 0;
        };
        if (dweight) rc = zero(dweight, dw_stride, outputs, inputs);
        if (!rc && dbias) rc = zero(dbias, outputs, 1, outputs);
        return rc;
    }
    if (!dx && !dweight && !dbias) return 0;
    if (!dy || (dx && !weight) || (dweight && !x) || (activation != GL_ACT_NONE && !preactivation))
        return gl_set_error(GL_ERR_INVALID, "gl_dense_backward: NULL buffer");
    rc = check_stride(dy_stride, outputs, "dy", "gl_dense_backward");
    if (!rc && dweight) rc = check_stride(x_stride, inputs, "x", "gl_dense_backward");
    if (!rc && dx) rc = check_stride(w_stride, inputs, "weight", "gl_dense_backward");
    if (!rc && dx) rc = check_stride(dx_stride, inputs, "dx", "gl_dense_backward");
    if (!rc && activation != GL_ACT_NONE) rc = check_stride(z_stride, outputs, "preactivation", "gl_dense_backward");
    const BackLayout l = back_layout(rows, inputs, outputs, dtype, out_dtype, activation);
    if (!rc) rc = check_workspace(workspace, workspace_bytes, l.total(), "gl_dense_backward");
    if (rc) return rc;
#define GL_BACK(T, TO, TWO)                                                                                               \
    (l.small ? backward_small<T, TO, TWO> : backward<T, TO, TWO>)(dy, dy_stride, x, x_stride, weight, w_stride, preactivation,      \
        z_stride, dx, dx_stride, dweight, dw_stride, dbias, rows, inputs, outputs, activation, l, workspace, st)
    if (dtype == GL_F32) return GL_BACK(float, float, false);
    if (dtype == GL_BF16) return l.two ? GL_BACK(gl_bf16, float, true) : GL_BACK(gl_bf16, gl_bf16, false);
    if (out_dtype == GL_F32) return GL_BACK(gl_f16, float, true);
    return l.two ? GL_BACK(gl_f16, gl_f16, true) : GL_BACK(gl_f16, gl_f16, false);
#undef GL_BACK
}

}  // extern "C"
