// Dense layers of the learned mel inversion: y = act(x W^T + b) + r and its gradients (include/gl_hip.h).
//
// All three products are C[i][j] = sum_q P(i, q) Q(j, q):
//   forward   P = x  [rows][inputs],   Q = W  [outputs][inputs]      both contiguous in q
//   dx        P = dz [rows][outputs],  Q(j, q) = W[q][j]             Q contiguous in j
//   dweight   P(i, q) = dz[q][i],      Q(j, q) = x[q][j]             both contiguous in i / j, q = frames
// 16-bit types: v_mfma_f32_32x32x16 (8 consecutive q per lane), 32-bit: v_mfma_f32_32x32x2_f32; sums are fp32.  Q is the
// matrix instruction's A operand: the accumulator's registers then run along j, the contiguous direction of C.
#include "gl_dense.h"

namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
template <typename T> struct vec8 { typedef T type __attribute__((ext_vector_type(8))); };

constexpr int kTile = 64;        // rows and columns of C per workgroup (4 waves, 32 x 32 each)
constexpr int kBQ = 32;          // contraction indexes staged per step

typedef gl_operand Operand;
typedef gl_epilogue Epilogue;

// Any size, stride and alignment: elements are staged one by one.  grid (tiles, splits).
template <typename T, typename TO>
__global__ void __launch_bounds__(256) k_dense_any(Operand P, Operand Q, Epilogue e, long long I, int J, long long nq,
                                                   long long q_per_split, int tiles_j) {
    constexpr bool k16 = sizeof(T) == 2;
    constexpr int kPitch = k16 ? kBQ + 8 : kBQ + 1;
    __shared__ __attribute__((aligned(16))) T Ps[kTile * kPitch];
    __shared__ __attribute__((aligned(16))) T Qs[kTile * kPitch];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, li = lane & 31, lk = lane >> 5;
    const long long i0 = (long long)(blockIdx.x / tiles_j) * kTile;
    const int j0 = (int)(blockIdx.x % tiles_j) * kTile;
    const long long q_begin = (long long)blockIdx.y * q_per_split;
    const long long q_end = q_begin + q_per_split < nq ? q_begin + q_per_split : nq;
    const int wi = (wave >> 1) * 32, wj = (wave & 1) * 32;

    f32x16 acc;
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[r] = 0.0f;

    auto stage = [&](T* dst, const Operand& o, long long r0, long long rn, long long q0) {
        for (int e8 = threadIdx.x; e8 < kTile * kBQ; e8 += 256) {
            // consecutive threads along the contiguous direction
            const int r = o.qs == 1 ? e8 / kBQ : e8 % kTile;
            const int q = o.qs == 1 ? e8 % kBQ : e8 / kTile;
            T v = (T)0.0f;
            if (r0 + r < rn && q0 + q < q_end) v = ((const T*)o.base)[(r0 + r) * o.is + (q0 + q) * o.qs];
            dst[r * kPitch + q] = v;
        }
    };
    for (long long q0 = q_begin; q0 < q_end; q0 += kBQ) {
        __syncthreads();
        stage(Ps, P, i0, I, q0);
        stage(Qs, Q, j0, J, q0);
        __syncthreads();
        if constexpr (k16) {
            typedef typename vec8<T>::type v8;
#pragma unroll
            for (int s = 0; s < kBQ; s += 16) {
                const v8 a = *(const v8*)(Qs + (wj + li) * kPitch + s + 8 * lk);
                const v8 b = *(const v8*)(Ps + (wi + li) * kPitch + s + 8 * lk);
                if constexpr (__is_same(T, gl_bf16))
                    acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, acc, 0, 0, 0);
                else
                    acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, acc, 0, 0, 0);
            }
        } else {
#pragma unroll
            for (int s = 0; s < kBQ; s += 2)
                acc = __builtin_amdgcn_mfma_f32_32x32x2f32(Qs[(wj + li) * kPitch + s + lk], Ps[(wi + li) * kPitch + s + lk],
                                                           acc, 0, 0, 0);
        }
    }
    const long long i = i0 + wi + li;
    if (i >= I) return;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        const int j = j0 + wj + (r & 3) + 8 * (r >> 2) + 4 * lk;
        if (j >= J) continue;
        if (e.partial) e.partial[((long long)blockIdx.y * I + i) * J + j] = acc[r];
        else gl_finish<T, TO>(e, i, j, acc[r]);
    }
}

// Sums the parts of a split contraction in their order and finishes the element.
template <typename T, typename TO>
__global__ void __launch_bounds__(256) k_dense_join(Epilogue e, long long I, int J, int splits) {
    const long long n = I * J;
    for (long long at = (long long)blockIdx.x * 256 + threadIdx.x; at < n; at += (long long)gridDim.x * 256) {
        float s = 0.0f;
        for (int p = 0; p < splits; ++p) s += e.partial[p * n + at];
        const long long i = at / J;
        gl_finish<T, TO>(e, i, (int)(at - i * J), s);
    }
}

// dz = dy act'(z), rounded to T for the products that read it, and column sums over this workgroup's frames.
// grid (column blocks of 64, parts); thread = (column, one of 4 frame lanes).
template <typename T, typename TO>
__global__ void __launch_bounds__(256) k_dense_dz(const TO* __restrict__ dy, long long dy_stride, const TO* __restrict__ z,
                                                  long long z_stride, T* __restrict__ dz, long long dz_stride,
                                                  float* __restrict__ parts, long long rows, int N, int rows_per_part,
                                                  int act) {
    __shared__ float s[4][64];
    const int c = threadIdx.x & 63, r = threadIdx.x >> 6;
    const int n = blockIdx.x * 64 + c;
    const long long r0 = (long long)blockIdx.y * rows_per_part;
    const long long r1 = r0 + rows_per_part < rows ? r0 + rows_per_part : rows;
    float sum = 0.0f;
    if (n >= N && n < dz_stride && dz)                        // zeros up to the padded width
        for (long long i = r0 + r; i < r1; i += 4) dz[i * dz_stride + n] = (T)0.0f;
    if (n < N)
        for (long long i = r0 + r; i < r1; i += 4) {
            float d = gl_to_f32(dy[i * dy_stride + n]);
            if (act != GL_ACT_NONE) d *= gl_act_grad(gl_to_f32(z[i * z_stride + n]), act);
            if (dz) dz[i * dz_stride + n] = (T)d;
            sum += d;
        }
    s[r][c] = sum;
    __syncthreads();
    if (parts && r == 0 && n < N) parts[(long long)blockIdx.y * N + n] = (s[0][c] + s[1][c]) + (s[2][c] + s[3][c]);
}

template <typename T>
__global__ void __launch_bounds__(256) k_dense_db(const float* __restrict__ parts, int n_parts, T* __restrict__ db, int N) {
    const int n = blockIdx.x * 256 + threadIdx.x;
    if (n >= N) return;
    float s = 0.0f;
    for (int p = 0; p < n_parts; ++p) s += parts[(long long)p * N + n];
    db[n] = (T)s;
}

template <typename T>
__global__ void __launch_bounds__(256) k_dense_zero(T* p, long long stride, int rows, int cols) {
    for (long long at = (long long)blockIdx.x * 256 + threadIdx.x; at < (long long)rows * cols; at += (long long)gridDim.x * 256)
        p[at / cols * stride + at % cols] = (T)0.0f;
}

constexpr int kCUs = 256;        // compute units of an MI355X: the work split must not depend on the moment

// Parts of the contraction: enough workgroups to fill the chip twice, at least 8 steps each.
int n_splits(long long I, int J, long long nq) {
    const long long tiles = gl_ceil_div(I, kTile) * gl_ceil_div(J, kTile);
    long long s = 2 * kCUs / tiles;
    const long long most = gl_ceil_div(nq, 8 * kBQ);
    if (s > most) s = most;
    return s < 1 ? 1 : (int)s;
}
// workspace of a product's parts: whichever kernel takes it (that goes by alignment too, which the query does not know)
long long partial_bytes(long long I, int J, long long nq, int dtype, bool any_q = false, bool padded = false) {
    const int s = n_splits(I, J, nq);
    const long long any = s > 1 ? gl_align16((long long)s * I * J * 4) : 0;
    const long long mm = dtype == GL_F32 ? 0 : gl_mm_partial_bytes(I, J, padded ? gl_ceil_div(nq, 32) * 32 : nq, any_q);
    return any > mm ? any : mm;
}

template <typename T, typename TO>
int product(const Operand& P, const Operand& Q, Epilogue e, long long I, int J, long long nq, float* partial,
            hipStream_t st) {
    if constexpr (sizeof(T) == 2) {
        if (gl_mm16_takes(P, Q, e, I, J, nq, sizeof(TO))) return gl_mm16<T, TO>(P, Q, e, I, J, nq, partial, st);
    }
    const int splits = n_splits(I, J, nq);
    const long long per = gl_ceil_div(gl_ceil_div(nq, splits), kBQ) * kBQ;
    const long long used = gl_ceil_div(nq, per);                 // rounding up to whole steps may leave fewer parts
    const long long tiles = gl_ceil_div(I, kTile) * gl_ceil_div(J, kTile);
    if (tiles > 0x7fffffffLL) return gl_set_error(GL_ERR_INVALID, "gl_dense: %lld tiles are too many for one launch", tiles);
    e.partial = used > 1 ? partial : nullptr;
    hipLaunchKernelGGL((k_dense_any<T, TO>), dim3((unsigned)tiles, (unsigned)used), dim3(256), 0, st, P, Q, e, I, J, nq, per,
                       (int)gl_ceil_div(J, kTile));
    GL_HIP_CHECK(hipGetLastError());
    return used > 1 ? gl_dense_join<T, TO>(e, I, J, (int)used, st) : 0;
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
int check_workspace(const void* ws, long long have, long long need, const char* who) {
    if (need == 0) return 0;
    if (!ws || have < need)
        return gl_set_error(GL_ERR_INVALID, "%s: workspace of %lld bytes needed, %lld given", who, need, ws ? have : 0LL);
    if ((uintptr_t)ws % 16) return gl_set_error(GL_ERR_INVALID, "%s: workspace must be 16-byte aligned", who);
    return 0;
}

template <typename T, typename TO>
int forward(const void* x, long long x_stride, const void* w, long long w_stride, const Epilogue& e, long long rows,
            int inputs, int outputs, void* ws, hipStream_t st) {
    return product<T, TO>({x, x_stride, 1}, {w, w_stride, 1}, e, rows, outputs, inputs, (float*)ws, st);
}

constexpr int kMaxParts = 128;
int rows_per_part(long long rows) {
    const long long r = gl_ceil_div(rows, kMaxParts);
    return (int)(r < 64 ? 64 : r);
}

// workspace of the backward pass: [dz (unless dy serves)] [column-sum parts] [partials of dx and dweight, one after the
// other on the stream: the larger of the two]
struct BackLayout {
    bool own_dz;
    long long dz_stride, dz_bytes, parts_bytes, partial_bytes_;
    long long total() const { return dz_bytes + parts_bytes + partial_bytes_; }
};
int elem_size(int dtype) { return dtype == GL_F32 ? 4 : 2; }
BackLayout back_layout(long long rows, int inputs, int outputs, int dtype, int out_dtype, int act) {
    BackLayout l;
    // dy itself serves where nothing is to be multiplied, converted or padded
    l.dz_stride = gl_ceil_div(outputs, 32) * 32;
    l.own_dz = act != GL_ACT_NONE || dtype != out_dtype || (dtype != GL_F32 && outputs % 32);
    l.dz_bytes = l.own_dz ? gl_align16(rows * l.dz_stride * elem_size(dtype)) : 0;
    l.parts_bytes = gl_align16(gl_ceil_div(rows, rows_per_part(rows)) * outputs * 4);
    const long long a = partial_bytes(rows, inputs, outputs, dtype, false, l.own_dz), b = partial_bytes(outputs, inputs, rows, dtype, true);
    l.partial_bytes_ = a > b ? a : b;
    return l;
}

template <typename T, typename TO>
int backward(const void* dy, long long dy_stride, const void* x, long long x_stride, const void* w, long long w_stride,
             const void* z, long long z_stride, void* dx, long long dx_stride, void* dw, long long dw_stride, void* db,
             long long rows, int inputs, int outputs, int act, const BackLayout& l, void* ws, hipStream_t st) {
    char* at = (char*)ws;
    T* dz = l.own_dz ? (T*)at : nullptr;
    float* parts = (float*)(at + l.dz_bytes);
    float* partial = (float*)(at + l.dz_bytes + l.parts_bytes);
    if (dz || db) {
        const int rpp = rows_per_part(rows);
        const int n_parts = (int)gl_ceil_div(rows, rpp);
        hipLaunchKernelGGL((k_dense_dz<T, TO>), dim3((unsigned)gl_ceil_div(outputs, 64), (unsigned)n_parts), dim3(256), 0, st,
                           (const TO*)dy, dy_stride, (const TO*)z, z_stride, dz, l.dz_stride, db ? parts : nullptr,
                           rows, outputs, rpp, act);
        GL_HIP_CHECK(hipGetLastError());
        if (db) {
            hipLaunchKernelGGL((k_dense_db<T>), dim3((unsigned)gl_ceil_div(outputs, 256)), dim3(256), 0, st, parts, n_parts,
                               (T*)db, outputs);
            GL_HIP_CHECK(hipGetLastError());
        }
    }
    const void* d = dz ? (const void*)dz : dy;
    const long long d_stride = dz ? l.dz_stride : dy_stride;
    Epilogue e = {};
    if (dx) {
        e.y = dx;
        e.y_stride = dx_stride;
        int rc = product<T, T>({d, d_stride, 1, dz != nullptr}, {w, 1, w_stride}, e, rows, inputs, outputs, partial, st);
        if (rc) return rc;
    }
    if (dw) {
        e.y = dw;
        e.y_stride = dw_stride;
        return product<T, T>({d, 1, d_stride, dz != nullptr}, {x, 1, x_stride}, e, outputs, inputs, rows, partial, st);
    }
    return 0;
}

}  // namespace

template <typename T, typename TO>
int gl_dense_join(const gl_epilogue& e, long long I, int J, int parts, hipStream_t st) {
    const long long blocks = gl_ceil_div(I * J, 256);
    hipLaunchKernelGGL((k_dense_join<T, TO>), dim3((unsigned)(blocks < 4096 ? blocks : 4096)), dim3(256), 0, st, e, I, J, parts);
    GL_HIP_CHECK(hipGetLastError());
    return 0;
}
template int gl_dense_join<float, float>(const gl_epilogue&, long long, int, int, hipStream_t);
template int gl_dense_join<gl_bf16, gl_bf16>(const gl_epilogue&, long long, int, int, hipStream_t);
template int gl_dense_join<gl_bf16, float>(const gl_epilogue&, long long, int, int, hipStream_t);
template int gl_dense_join<gl_f16, gl_f16>(const gl_epilogue&, long long, int, int, hipStream_t);
template int gl_dense_join<gl_f16, float>(const gl_epilogue&, long long, int, int, hipStream_t);

// 256 x 256 tiles where they fill the chip (parts included), else 128 x 128, else 64 x 64.  A part has at least 512
// contraction indexes with large tiles and 256 with small ones: shorter ones cost more in the join than they fill.
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
        gl_mm_plan p = split(256, 512);
        if (gl_ceil_div(I, 256) * (J / 256) * p.parts >= 128) {
            p.kind = 2;
            return p;
        }
    }
    gl_mm_plan p = split(128, 256);
    if (I >= 96 && J >= 96 && gl_ceil_div(I, 128) * gl_ceil_div(J, 128) * p.parts >= 256) {
        p.kind = 1;
        return p;
    }
    return split(64, 256);
}

int gl_mm_first_columns(long long I, int J, long long nq, bool any_q) {
    const int whole = J / 256 * 256;
    return whole > 0 && whole < J && gl_mm_plan_for(I, whole, nq, any_q).kind == 2 ? whole : J;
}

long long gl_mm_partial_bytes(long long I, int J, long long nq, bool any_q) {
    const int first = gl_mm_first_columns(I, J, nq, any_q);
    const gl_mm_plan a = gl_mm_plan_for(I, first, nq, any_q);
    long long bytes = a.parts > 1 ? (long long)a.parts * I * first * 4 : 0;
    if (first < J) {
        const gl_mm_plan b = gl_mm_plan_for(I, J - first, nq, any_q);
        const long long more = b.parts > 1 ? (long long)b.parts * I * (J - first) * 4 : 0;
        if (more > bytes) bytes = more;
    }
    return gl_align16(bytes);
}

bool gl_mm16_takes(const gl_operand& P, const gl_operand& Q, const gl_epilogue& e, long long I, int J, long long nq, int out_size) {
    auto side = [&](const gl_operand& o, long long rows) {
        const long long stride = o.across() ? o.qs : o.is;
        return (uintptr_t)o.base % 16 == 0 && stride % 8 == 0 && stride <= (1 << 21) && (o.padded || (o.across() ? rows : nq) % 8 == 0);
    };
    auto out = [&](const void* p, long long stride) {        // stores of four bytes and more
        return !p || ((uintptr_t)p % 4 == 0 && stride * out_size % 4 == 0 && stride <= (1 << 20));
    };
    if (P.across() && !Q.across()) return false;
    return side(P, I) && side(Q, J) && out(e.y, e.y_stride) && out(e.z, e.z_stride) && out(e.residual, e.r_stride) && nq < (1LL << 31) &&
           gl_ceil_div(I, 64) * gl_ceil_div(J, 64) < (1LL << 31) - 8;
}

extern "C" {

long long gl_dense_workspace(long long rows, int inputs, int outputs, int dtype, int out_dtype) {
    if (check_types(dtype, out_dtype, 0, "gl_dense_workspace") || check_sizes(rows, inputs, outputs, "gl_dense_workspace"))
        return GL_ERR_INVALID;
    return rows ? partial_bytes(rows, outputs, inputs, dtype) : 0;
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
    if (!rc) rc = check_workspace(workspace, workspace_bytes, partial_bytes(rows, outputs, inputs, dtype), "gl_dense");
    if (rc) return rc;
    const Epilogue e = {bias, residual, r_stride, y, y_stride, preactivation, z_stride, activation, nullptr};
    const hipStream_t st = (hipStream_t)stream;
    if (dtype == GL_F32) return forward<float, float>(x, x_stride, weight, w_stride, e, rows, inputs, outputs, workspace, st);
    if (dtype == GL_BF16)
        return out_dtype == GL_F32 ? forward<gl_bf16, float>(x, x_stride, weight, w_stride, e, rows, inputs, outputs, workspace, st)
                                   : forward<gl_bf16, gl_bf16>(x, x_stride, weight, w_stride, e, rows, inputs, outputs, workspace, st);
    return out_dtype == GL_F32 ? forward<gl_f16, float>(x, x_stride, weight, w_stride, e, rows, inputs, outputs, workspace, st)
                               : forward<gl_f16, gl_f16>(x, x_stride, weight, w_stride, e, rows, inputs, outputs, workspace, st);
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
#define GL_BACK(T, TO)                                                                                                    \
    backward<T, TO>(dy, dy_stride, x, x_stride, weight, w_stride, preactivation, z_stride, dx, dx_stride, dweight,        \
                    dw_stride, dbias, rows, inputs, outputs, activation, l, workspace, st)
    if (dtype == GL_F32) return GL_BACK(float, float);
    if (dtype == GL_BF16) return out_dtype == GL_F32 ? GL_BACK(gl_bf16, float) : GL_BACK(gl_bf16, gl_bf16);
    return out_dtype == GL_F32 ? GL_BACK(gl_f16, float) : GL_BACK(gl_f16, gl_f16);
#undef GL_BACK
}

}  // extern "C"
