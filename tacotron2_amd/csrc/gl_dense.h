// Shared by the translation units of the dense layers: the products' operands and their dispatch.
#pragma once
#include "gl_internal.h"
#include "gl_act.h"

constexpr int kPadded = 64;      // contraction indexes that the products read at once from copies

struct gl_operand {              // element (i, q) at base[i * is + q * qs], one of is, qs is 1
    const void* base;
    long long is, qs;
    long long plane = 0;         // elements between the planes of an operand that has several
    bool padded = false;         // this library's own copy: zeros up to whole multiples of kPadded in the contiguous direction
    bool across() const { return is == 1 && qs != 1; }       // contiguous across the contraction
};

struct gl_epilogue {
    const void* bias;            // [J] of T or null
    const void* residual;        // of TO or null
    long long r_stride;
    void* y;
    long long y_stride;
    void* z;                     // of TO or null
    long long z_stride;
    int act;
    bool quads;                  // k_dense_any: four columns of y, z and residual lie on whole vectors
    float* partial;              // [parts][I][J]: sums of one part of the contraction, finished by k_dense_join
    // float32 through planes: the operands themselves, for the sums the planes do not give, and the flags of their blocks
    const float *exact_p, *exact_q;
    long long exact_p_is, exact_p_qs, exact_q_is, exact_q_qs, exact_nq;
    int* flags;
    const int *scale_p, *scale_q;    // float32 through halves: gl_scale of P's and Q's rows, else null
};

// A row of a float32 matrix in two planes of f16: x 2^e = h + l 2^-12 with h = f16(x 2^e), l = f16((x 2^e - h) 2^12) and the row's
// largest |x| 2^e in [2^14, 2^15).  Values of at least 2^-13 have 23 bits in it (float32's last one may be lost: 2^-23 of the
// value), smaller ones are off by 2^-37 at most: `small` says that there are such.  `wild`: the row holds an infinity or a NaN,
// and its planes zeros.
struct gl_scale {
    int bits;                    // e, small, wild
    static __host__ __device__ gl_scale of(int e, bool small, bool wild) { return {e * 4 + (small ? 1 : 0) + (wild ? 2 : 0)}; }
    __device__ int e() const { return bits >> 2; }
    __device__ bool small() const { return bits & 1; }
    __device__ bool wild() const { return bits & 2; }
};
// Whether the planes give a sum of nq products, `sum` = C 2^(e of P's row + e of Q's).  Small values move it by at most
// 3 nq 2^-37 2^15 in all; where that is more than 2^-23 of it, it is for the operands themselves.
__device__ __forceinline__ bool gl_halves_give(float sum, gl_scale p, gl_scale q, float nq) {
    const gl_scale both = {p.bits | q.bits};
    return !both.wild() && !(both.small() && fabsf(sum) < 6.0f * nq);
}

// A float32 value in two planes of a 16-bit type: v = high + low kSplitStep.  bfloat16 has the range for low to be what high leaves:
// off by 2^-17 |v| at most.  float16: what high leaves, 2^20 up, so that values below high's range stay: off by 2^-23 |v| from
// 2^-14, where high has all its bits, to 128; below, by min(2^-37, 2^-11 |v|), and 2^-45 where low runs out of bits too; above, where
// 2^20 times the rest may not fit, by half a step of float16.  Infinities, NaN and what rounds to infinity stay in high alone.
template <typename T> constexpr float kSplitStep = __is_same(T, gl_f16) ? 0x1p-20f : 1.0f;
template <typename T>
__device__ __forceinline__ void gl_split(float v, T& high, T& low) {
    high = (T)v;
    float rest = v - (float)high;                            // exact where it is finite
    if constexpr (__is_same(T, gl_f16)) rest = __builtin_amdgcn_fmed3f(rest * 0x1p20f, -65504.0f, 65504.0f);
    low = (T)(fabsf((float)high) < INFINITY ? rest : 0.0f);
}

static inline long long gl_ceil_div(long long a, long long b) { return (a + b - 1) / b; }
static inline long long gl_align16(long long b) { return (b + 15) / 16 * 16; }

// How a product of 16-bit operands on 16 bytes is split (gl_mm16_launch.h).  A pure function of the sizes: the workspace
// query and the call must agree, and results must not depend on the moment.
struct gl_mm_plan {
    int kind;                    // 0: 64 x 64 tiles, 1: 128 x 128, 2: 256 x 256 walked by one workgroup a CU
    int parts;                   // of the contraction
    long long per;               // contraction indexes in a part
};
// any_q: both sides are contiguous across the contraction, which may then have any length.  out_size: bytes of a result.
gl_mm_plan gl_mm_plan_for(long long I, int J, long long nq, bool any_q);
// columns the first of the product's two launches takes (the rest has its own plan): all, or a multiple of 256
int gl_mm_first_columns(long long I, int J, long long nq, bool any_q, int out_size);
long long gl_mm_partial_bytes(long long I, int J, long long nq, bool any_q);

// Whether the fast kernels take the operands as they lie, else the strided kernel does.
bool gl_mm16_takes(const gl_operand& P, const gl_operand& Q, const gl_epilogue& e, long long I, int J, long long nq, int out_size);
// T: gl_bf16 / gl_f16; TO: T or float; TB: type of the bias; SEG: products of planes that make C (gl_mm16.h), 6 or 3 for float32
// operands, 2 where P has two planes (gl_split), else 1
template <typename T, typename TO, typename TB, int SEG>
int gl_mm16(const gl_operand& P, const gl_operand& Q, gl_epilogue e, long long I, int J, long long nq, float* partial, hipStream_t st);

// sums the parts in their order and finishes the elements
template <typename T, typename TO>
int gl_dense_join(const gl_epilogue& e, long long I, int J, int parts, hipStream_t st);

// the same for float32 through planes; what those do not give is computed from the operands
int gl_dense_join_planes(const gl_epilogue& e, long long I, int J, long long nq, const gl_mm_plan& p, hipStream_t st);

// computes the 64 x 64 blocks that are flagged, on the float32 operands
int gl_dense_flagged(const gl_epilogue& e, long long I, int J, long long nq, hipStream_t st);

// sum -> (preactivation, y) of element (i, j)
template <typename T, typename TO>
__device__ __forceinline__ void gl_finish(const gl_epilogue& e, long long i, int j, float sum) {
    float z = sum;
    if (e.bias) z += gl_to_f32(((const T*)e.bias)[j]);
    if (e.z) ((TO*)e.z)[i * e.z_stride + j] = (TO)z;
    float y = gl_act<TO>(z, e.act);
    if (e.residual) y += gl_to_f32(((const TO*)e.residual)[i * e.r_stride + j]);
    ((TO*)e.y)[i * e.y_stride + j] = (TO)y;
}
