// C = P Q^T on the 16-bit matrix instructions, for operands whose rows start on 16 bytes and whose contiguous direction is
// a multiple of 8 elements (gl_dense.hip uses the strided kernel for the rest).
//
// A workgroup of (BM / WM) (BN / WN) waves owns a BM x BN tile; a wave owns WM x WN of it in registers.  Steps of BK run
// through a ring of ST stages in LDS, filled by buffer loads that write LDS directly (no registers, out-of-range chunks
// become zeros through the buffer's bounds check), one barrier a step:
//     wait for the own loads of stage k, barrier (all have landed, all waves are done with stage k - 1),
//     start the loads of stage k + ST - 1 into the slot of k - 1, read stage k, multiply.
//
// Stage layouts.  An operand contiguous in the contraction is [rows][BK] with 16-byte chunk c of row r at c ^ swizzle(r):
// the 16 rows a matrix instruction reads at one chunk then spread over all banks.  An operand contiguous across the
// contraction is [BK][columns], read by ds_read_b64_tr_b16 (4 contraction rows x 16 columns per 16 lanes, transposed on the
// way); its 32-byte pieces are XORed with the row so that the 8 rows of half a wave spread over all banks.  The swizzle is
// applied to the global address, since direct loads place consecutive lanes' chunks consecutively.
//
// Operands of more bits come in planes, and C is a sum of SEG products of planes.
//   2: P in two planes of Q's own type (gl_split): low x Q first, times kSplitStep, then high x Q.
// float32 operands: a block with a sum that the planes do not give is not written but flagged, and the float32 kernel computes it.
//   3: two planes of f16 per row (gl_scale), where a row of either side is one of the contraction: h l, l h, then, with the
//      sums times 2^-12, h h.  Left out is l l 2^-24 <= 2^-22 |x| |y| (h rounds at 2^-11 of a value), and either side is off by up
//      to 2^-23 of itself: 2^-21 |x| |y| in all at most, for a product whose both factors are the worst there are.
//   6: three planes of bfloat16, x = h + m + l with h = bf16(x), m = bf16(x - h), l = bf16(x - h - m), which need no scale (an
//      operand across the contraction has one per column): hh, hm, mh, mm, hl, lh; what is left out (ml, lm, ll) is below 2^-24
//      of |x| |y|.  Sums that are not finite are flagged: an infinity times a zero plane would be NaN.
//
// v_mfma_f32_16x16x32: A = Q rows (columns j of C), B = P rows (rows i of C): a lane's four accumulator registers are four
// consecutive j of one i.
#pragma once
#include "gl_dense.h"

namespace gl_mm {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
template <typename T, int N> struct vec { typedef T type __attribute__((ext_vector_type(N))); };

struct Side {                    // rows (or columns) of C x contraction
    const void* base;
    long long stride;            // elements between rows of the contiguous direction
    long long rows;              // rows that may be loaded: I (J), or more where zeros pad them
    long long plane;             // elements between the planes of a float32 operand
    int missing;                 // contraction indexes at the end that this side does not have (the other has zeros there)
};

template <typename T>
__device__ __forceinline__ f32x4 mfma16(s16x8 a, s16x8 b, f32x4 c) {
    typedef typename vec<T, 8>::type v8;
    if constexpr (__is_same(T, gl_bf16))
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0, 0, 0);
}

__device__ __forceinline__ void wait_loads(int n) {          // at most n vector memory operations outstanding
    switch (n) {
#define GL_WAIT(k) case k: asm volatile("s_waitcnt vmcnt(" #k ")" ::: "memory"); break;
        GL_WAIT(8) GL_WAIT(12) GL_WAIT(24) GL_WAIT(40)
#undef GL_WAIT
        default: asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    }
}

// A workgroup barrier behind which this wave's own LDS reads are done too: their slot may be overwritten
__device__ __forceinline__ void barrier() {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// The planes of the products, two bits each
template <int SEG> constexpr int kPlanesP = SEG == 2 ? 1 | 0 << 2 : SEG == 3 ? 0 | 1 << 2 | 0 << 4 : 0 | 0 << 2 | 1 << 4 | 1 << 6 | 0 << 8 | 2 << 10;
template <int SEG> constexpr int kPlanesQ = SEG == 2 ? 0 : SEG == 3 ? 1 | 0 << 2 | 0 << 4 : 0 | 1 << 2 | 0 << 4 | 1 << 6 | 2 << 8 | 0 << 10;
__device__ __forceinline__ int plane_of(int planes, int seg) { return planes >> (2 * seg) & 3; }

constexpr int kFlags = 0x00027000;                           // raw 32-bit buffer: bounds-checked, no format conversion
constexpr int kStream = 2;                                   // cache policy: non-temporal
constexpr int kOutside = 0x7fffff00;                         // an offset beyond every buffer: loads zeros

// One operand of a tile: LDS layout, loads and fragments.
//   R rows of C's side, TR: contiguous across the contraction
template <int R, int BK, bool TR, int WAVES, bool TEXT>
struct Stage {
    static constexpr int kLoads = (R * BK * 2 + 1024 * WAVES - 1) / (1024 * WAVES);   // 16-byte loads per lane and stage
    static constexpr int kBytes = kLoads * 1024 * WAVES;     // with whole loads of all waves: rows past R are zeros
    static_assert(!TR || (R % 32 == 0 && (R & (R - 1)) == 0), "pieces of 32 bytes are exchanged within a row");
    static constexpr int kRowChunks = TR ? R / 8 : BK / 8;   // chunks per LDS row
    const char* base;            // first element of the tile at the current step
    const char* start;           // and at the first one
    int stride2, n_rows;         // bytes per row of the contiguous direction; rows of C's side that exist
    int voff[kLoads];

    __device__ __forceinline__ static int swizzle(int row) {
        return BK == 32 ? (row >> 1) & 3 : row & 7;
    }
    __device__ __forceinline__ static int tr_swizzle(int q) { return (((q & 3) | ((q >> 3) & 1) << 2) << 1) & (R / 8 - 1); }

    __device__ __forceinline__ static int chunk_of(int i, int wave, int lane, int& row) {
        const int slot = (i * WAVES + wave) * 64 + lane;
        row = slot / kRowChunks;
        return (slot % kRowChunks) ^ (TR ? tr_swizzle(row) : swizzle(row));
    }
    // r0: first row of the tile, q0: first contraction index
    __device__ __forceinline__ void init(const Side& s, long long r0, long long q0, int wave, int lane) {
        n_rows = s.rows - r0 < R ? (int)(s.rows - r0) : R;
        stride2 = (int)s.stride * 2;
        base = (const char*)s.base + (TR ? q0 * s.stride + r0 : r0 * s.stride + q0) * 2;
        start = base;
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            int row;
            const int ch = chunk_of(i, wave, lane, row);
            voff[i] = (TR ? ch * 8 < n_rows : row < n_rows) ? row * stride2 + ch * 16 : kOutside;
        }
    }
    // krem: contraction indexes left at this step (<= 0: zeros).  Bytes to the end of the last row that exists; rows and
    // chunks beyond it load as zeros.
    __device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer(int krem) const {
        const int records = krem <= 0 ? 0 : TR ? (min(krem, BK) - 1) * stride2 + n_rows * 2 : (n_rows - 1) * stride2 + krem * 2;
        return __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, records, kFlags);
    }
    // One 16-byte load per lane straight into LDS.  TEXT (where a side is read transposed): with the builtin the compiler
    // waits for every load in flight before a transposing read, which may alias (dx of 55 104 x 2048 x 512: 210 us, so 127);
    // as text, wait_loads() and barrier() alone order them.  It has no register result.
    __device__ __forceinline__ void load_one(__amdgpu_buffer_rsrc_t rs, char* lds, int i, int v, int wave) const {
        auto at = (__attribute__((address_space(3))) char*)(lds + (i * WAVES + wave) * 1024);
        if constexpr (TEXT)
            asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
                         : : "s"(__builtin_amdgcn_readfirstlane((unsigned)(unsigned long long)at)), "v"(v), "s"(rs)
                         : "memory", "m0");
        else
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (__attribute__((address_space(3))) void*)at, 16, v, 0, 0, 0);
    }
    __device__ __forceinline__ void advance() { base += TR ? (long long)BK * stride2 : BK * 2; }
    __device__ __forceinline__ void load(char* lds, int krem, int wave, int lane) {
        const __amdgpu_buffer_rsrc_t rs = buffer(krem);
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            int v = voff[i];
            if (!TR && krem < BK) {                          // the last step: chunks past the row's end are another row's
                int row;
                if (chunk_of(i, wave, lane, row) * 8 >= krem) v = kOutside;
            }
            load_one(rs, lds, i, v, wave);
        }
        advance();
    }
    // 16 rows from r0 (a multiple of 16), contraction 32 ks .. +32: the lane's row is lane & 15, its 8 indexes 8 (lane >> 4)
    __device__ __forceinline__ static s16x8 frag(const char* lds, int r0, int ks, int lane) {
        if constexpr (TR) {
            const int p = lane & 15, g = lane >> 4;
            const int q = 32 * ks + 8 * g + (p >> 2);
            const int ch = (r0 / 8 + ((p & 3) >> 1)) ^ tr_swizzle(q);
            const char* at = lds + q * (R * 2) + ch * 16 + (p & 1) * 8;
            typedef __attribute__((address_space(3))) s16x4* lp;
            const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(at));
            const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(at + 4 * R * 2));
            return (s16x8){a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
        } else {
            const int row = r0 + (lane & 15);
            const int ch = ((lane >> 4) + 4 * ks) ^ swizzle(row);
            return *(const s16x8*)(lds + row * (BK * 2) + ch * 16);
        }
    }
};

struct Out {
    const void* bias;            // [J] of TB or null
    const void* residual;        // of TO or null
    long long r_stride;
    void* y;
    long long y_stride;
    void* z;                     // of TO or null
    long long z_stride;
    int act;                     // where the kernel does not fix it
    int* flags;                  // float32 operands: per 64 x 64 block of C, whether it is left to the float32 kernel; or null
    long long part_stride;       // elements of y between the results of two parts of the contraction (bias, residual and z
                                 // are null then)
    int odd;                     // rows start off 4 bytes: elements are stored one by one (TAIL kernels)
    const int *scale_p, *scale_q;    // SEG 3
};

template <typename T> struct bits;                          // what a buffer load or store of an element moves
template <> struct bits<float> { typedef unsigned type; };
template <> struct bits<gl_bf16> { typedef unsigned short type; };
template <> struct bits<gl_f16> { typedef unsigned short type; };
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

template <typename T>
__device__ __forceinline__ T load_at(__amdgpu_buffer_rsrc_t rs, int off) {
    if constexpr (sizeof(T) == 4) return __builtin_bit_cast(T, __builtin_amdgcn_raw_buffer_load_b32(rs, off, 0, 0));
    else return __builtin_bit_cast(T, __builtin_amdgcn_raw_buffer_load_b16(rs, off, 0, 0));
}
template <typename T>
__device__ __forceinline__ void store_at(T v, __amdgpu_buffer_rsrc_t rs, int off) {
    if constexpr (sizeof(T) == 4) __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(unsigned, v), rs, off, 0, 0);
    else __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(unsigned short, v), rs, off, 0, 0);
}

// A wave's bias: NI times four consecutive columns, kept packed until the sums start at it; zero past the last column.
template <typename TB, int NI>
__device__ __forceinline__ void load_bias(const Out& o, typename vec<TB, 4>::type (&bias)[NI], int j0, int J, int lane) {
    const int n_cols = o.bias && j0 < J ? min(J - j0, 16 * NI) : 0;
    const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc((void*)((const TB*)o.bias + (n_cols ? j0 : 0)), 0,
                                                                        n_cols * (int)sizeof(TB), kFlags);
#pragma unroll
    for (int n = 0; n < NI; ++n)
#pragma unroll
        for (int r = 0; r < 4; ++r) bias[n][r] = load_at<TB>(rs, (16 * n + 4 * (lane >> 4) + r) * (int)sizeof(TB));
}
template <typename TB, int MI, int NI>
__device__ __forceinline__ void start_sums(f32x4 (&acc)[MI][NI], const typename vec<TB, 4>::type (&bias)[NI]) {
#pragma unroll
    for (int n = 0; n < NI; ++n) {
        f32x4 b;
#pragma unroll
        for (int r = 0; r < 4; ++r) b[r] = gl_to_f32(bias[n][r]);
#pragma unroll
        for (int m = 0; m < MI; ++m) acc[m][n] = b;
    }
}

// A wave's block of an array with rows on 4 bytes: the buffer ends with the block's last row, so rows past it are dropped.
template <typename TO, int MI, int NI>
__device__ __forceinline__ __amdgpu_buffer_rsrc_t block_of(const void* p, long long stride, long long i0, int j0, long long I, int J) {
    const int rows = I - i0 < 16 * MI ? (int)(I - i0) : 16 * MI, cols = J - j0 < 16 * NI ? J - j0 : 16 * NI;
    return __builtin_amdgcn_make_buffer_rsrc((void*)((const TO*)p + i0 * stride + j0), 0,
                                             rows > 0 && cols > 0 ? ((rows - 1) * (int)stride + cols) * (int)sizeof(TO) : 0, kFlags);
}

// Stores a wave's block, rounded to TO; returns how many store instructions that were at least (the caller may leave that
// many outstanding).  TAIL: columns may end inside the block (a branch that costs registers).  LINES: rows on 128 bytes; the
// result then streams past the L2s, which keep Q and the rows of P (55 104 x 2048 x 512 bf16: 149 us, so 128; rows off 128 bytes
// would lose that way what the L2s merge: 55 104 x 1025 float32 105 us, so 132).
template <typename TO, bool TAIL, bool LINES, int MI, int NI>
__device__ __forceinline__ int put_block(TO* dst, long long stride, const f32x4 (&v)[MI][NI], long long i0, int j0, long long I,
                                         int J, int lane, bool odd) {
    typedef typename vec<TO, 4>::type to4;
    const int il = lane & 15, g4 = lane >> 4;
    constexpr bool kPair = sizeof(TO) == 2 && NI % 2 == 0;
    const __amdgpu_buffer_rsrc_t rs = block_of<TO, MI, NI>(dst, stride, i0, j0, I, J);
    const int stride_b = (int)stride * (int)sizeof(TO);
    auto round4 = [](const f32x4& f) {
        to4 t;
#pragma unroll
        for (int r = 0; r < 4; ++r) t[r] = (TO)f[r];
        return t;
    };
    if (!TAIL || (j0 + 16 * NI <= J && !odd)) {              // wave-uniform: whole column blocks
        // A lane's 16 bytes of two column groups: neighbouring lanes (rows 2 k and 2 k + 1) swap one, so that a store writes
        // 128 contiguous bytes of eight rows instead of 64 of sixteen: whole cache lines.
        const bool hi = lane & 1;
        constexpr int kCols = kPair ? 32 : 16;               // columns from one group to the other
        const int c0 = kPair ? 16 * (g4 & 1) + 8 * (g4 >> 1) : 4 * g4;
        int off_a = (il & ~1) * stride_b + (c0 + (hi ? kCols : 0)) * (int)sizeof(TO), off_b = off_a + stride_b;
        auto store2 = [&](const u32x4& x, const u32x4& y, int at) {
            u32x4 a, b;
#pragma unroll
            for (int d = 0; d < 4; ++d) {
                const unsigned got = __builtin_amdgcn_mov_dpp(hi ? x[d] : y[d], 0xB1, 0xF, 0xF, true);   // the lane beside
                a[d] = hi ? got : x[d];
                b[d] = hi ? y[d] : got;
            }
            __builtin_amdgcn_raw_buffer_store_b128(a, rs, off_a + at, 0, LINES ? kStream : 0);
            __builtin_amdgcn_raw_buffer_store_b128(b, rs, off_b + at, 0, LINES ? kStream : 0);
        };
#pragma unroll
        for (int m = 0; m < MI; ++m) {
            if constexpr (kPair) {
                // two 16-column blocks: quarter-waves swapped so that a lane holds 8 consecutive columns
                auto eight = [&](int n) -> u32x4 {
                    const u32x2 lo = __builtin_bit_cast(u32x2, round4(v[m][n])), up = __builtin_bit_cast(u32x2, round4(v[m][n + 1]));
                    const auto s0 = __builtin_amdgcn_permlane16_swap(lo[0], up[0], false, false);
                    const auto s1 = __builtin_amdgcn_permlane16_swap(lo[1], up[1], false, false);
                    return (u32x4){s0[0], s1[0], s0[1], s1[1]};
                };
                if constexpr (NI % 4 == 0) {
#pragma unroll
                    for (int n = 0; n < NI; n += 4) store2(eight(n), eight(n + 2), 32 * n);
                } else {
#pragma unroll
                    for (int n = 0; n < NI; n += 2)
                        __builtin_amdgcn_raw_buffer_store_b128(eight(n), rs, (16 * m + il) * stride_b + (c0 + 16 * n) * 2, 0, 0);
                }
            } else {
                static_assert(sizeof(TO) == 4 && NI % 2 == 0, "columns in pairs of blocks");
#pragma unroll
                for (int n = 0; n < NI; n += 2)
                    store2(__builtin_bit_cast(u32x4, v[m][n]), __builtin_bit_cast(u32x4, v[m][n + 1]), 64 * n);
            }
            off_a += 16 * stride_b;
            off_b += 16 * stride_b;
            __builtin_amdgcn_sched_barrier(0);
        }
        return MI * NI / (kPair ? 2 : 1);
    }
    int off = il * stride_b;
#pragma unroll
    for (int m = 0; m < MI; ++m) {
#pragma unroll
        for (int n = 0; n < NI; ++n)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int j = 16 * n + 4 * g4 + r;
                store_at<TO>((TO)v[m][n][r], rs, j0 + j < J ? off + j * (int)sizeof(TO) : kOutside);
            }
        off += 16 * stride_b;
        __builtin_amdgcn_sched_barrier(0);
    }
    return MI * NI;
}

// Whether all sums of a wave's block are finite; writes the flags of its 64 x 64 blocks.
template <int MI, int NI>
__device__ __forceinline__ bool all_finite(int* flags, const f32x4 (&acc)[MI][NI], long long i0, int j0, long long I, int J, int lane) {
    static_assert(MI % 4 == 0 && NI == 4, "whole blocks of flags");
    float worst = 0.0f;                                      // 0 x finite = 0, 0 x (infinity or NaN) = NaN
#pragma unroll
    for (int m = 0; m < MI; ++m)
#pragma unroll
        for (int n = 0; n < NI; ++n)
#pragma unroll
            for (int r = 0; r < 4; ++r) worst = fmaf(acc[m][n][r], 0.0f, worst);
    const bool bad = __any(worst != 0.0f);
    const int per_row = (J + 63) / 64;
    if (lane < MI / 4 && i0 + 64 * lane < I && j0 < J) flags[(i0 / 64 + lane) * per_row + j0 / 64] = bad;
    return !bad;
}

// SEG 3: a wave's sums in the operands' own scale, plus the bias.  False: some of them are not to be had from planes (never
// so for parts of the contraction, whose join decides); with flags, writes those of its 64 x 64 blocks.
template <typename TB, int MI, int NI>
__device__ __forceinline__ bool unscale(const Out& o, f32x4 (&acc)[MI][NI], long long i0, int j0, long long I, int J, float nq, int lane) {
    static_assert(MI % 4 == 0 && NI == 4, "whole blocks of flags");
    const int il = lane & 15, g4 = lane >> 4;
    const int rows = max(0, (int)min(I - i0, (long long)16 * MI)), cols = max(0, min(J - j0, 16 * NI));
    const __amdgpu_buffer_rsrc_t rp = __builtin_amdgcn_make_buffer_rsrc((void*)(o.scale_p + (rows ? i0 : 0)), 0, rows * 4, kFlags);
    const __amdgpu_buffer_rsrc_t rq = __builtin_amdgcn_make_buffer_rsrc((void*)(o.scale_q + (cols ? j0 : 0)), 0, cols * 4, kFlags);
    typename vec<TB, 4>::type bias[NI];
    load_bias<TB, NI>(o, bias, j0, J, lane);
    int qs[NI][4];
#pragma unroll
    for (int n = 0; n < NI; ++n)
#pragma unroll
        for (int r = 0; r < 4; ++r) qs[n][r] = __builtin_amdgcn_raw_buffer_load_b32(rq, (16 * n + 4 * g4 + r) * 4, 0, 0);
    bool good = true;
#pragma unroll
    for (int m = 0; m < MI; ++m) {
        const gl_scale p = {(int)__builtin_amdgcn_raw_buffer_load_b32(rp, (16 * m + il) * 4, 0, 0)};
#pragma unroll
        for (int n = 0; n < NI; ++n)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const gl_scale q = {qs[n][r]};
                good &= gl_halves_give(acc[m][n][r], p, q, nq);
                acc[m][n][r] = ldexpf(acc[m][n][r], -(p.e() + q.e())) + gl_to_f32(bias[n][r]);
            }
    }
    if (!o.flags) return true;
    const bool bad = !__all(good);
    const int per_row = (J + 63) / 64;
    if (lane < MI / 4 && i0 + 64 * lane < I && j0 < J) o.flags[(i0 / 64 + lane) * per_row + j0 / 64] = bad;
    return !bad;
}

// Writes a wave's block at (i0, j0): activation, residual and one rounding.  All loads come before the
// results' stores: the memory counter runs in order, a load behind a store would wait for it.
// EXTRA: there may be a residual or a preactivation.
template <typename T, typename TO, int ACT, bool EXTRA, bool TAIL, bool LINES, int MI, int NI>
__device__ __forceinline__ int epilogue(const Out& o, f32x4 (&acc)[MI][NI], long long i0, int j0, long long I, int J,
                                        int part, int lane) {
    const int il = lane & 15, g4 = lane >> 4;
    if (EXTRA && o.z) put_block<TO, TAIL, LINES, MI, NI>((TO*)o.z, o.z_stride, acc, i0, j0, I, J, lane, o.odd);
    auto activate = [&](auto act) {
#pragma unroll
        for (int m = 0; m < MI; ++m)
#pragma unroll
            for (int n = 0; n < NI; ++n) {
#pragma unroll
                for (int r = 0; r < 4; ++r) acc[m][n][r] = gl_act<TO>(acc[m][n][r], decltype(act)::value);
                if (n & 1) __builtin_amdgcn_sched_barrier(0);    // keeps the block's temporaries few
            }
    };
    if constexpr (ACT < 0) gl_with_act(o.act, activate);
    else activate(gl_int<ACT>());
    if (EXTRA && o.residual) {
        const __amdgpu_buffer_rsrc_t rs = block_of<TO, MI, NI>(o.residual, o.r_stride, i0, j0, I, J);
        const int stride_b = (int)o.r_stride * (int)sizeof(TO);
        int off = il * stride_b + 4 * g4 * (int)sizeof(TO);
        const bool whole = !TAIL || (j0 + 16 * NI <= J && !o.odd);
#pragma unroll
        for (int m = 0; m < MI; ++m) {
#pragma unroll
            for (int n = 0; n < NI; ++n) {
                typename vec<TO, 4>::type rv;
                if (whole) {
                    if constexpr (sizeof(TO) == 4)
                        rv = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, off + 64 * n, 0, 0));
                    else
                        rv = __builtin_bit_cast(typename vec<TO, 4>::type, __builtin_amdgcn_raw_buffer_load_b64(rs, off + 32 * n, 0, 0));
                } else {
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        rv[r] = load_at<TO>(rs, j0 + 16 * n + 4 * g4 + r < J ? off + (16 * n + r) * (int)sizeof(TO) : kOutside);
                }
#pragma unroll
                for (int r = 0; r < 4; ++r) acc[m][n][r] += gl_to_f32(rv[r]);
            }
            off += 16 * stride_b;
            __builtin_amdgcn_sched_barrier(0);
        }
    }
    return put_block<TO, TAIL, LINES, MI, NI>((TO*)o.y + part * o.part_stride, o.y_stride, acc, i0, j0, I, J, lane, o.odd);
}

// The sums of the lower planes, which count `step`, before the highest ones' are added: SEG 3, h l + l h, 2^-12; SEG 2, kSplitStep
template <int SEG, typename T> constexpr float kLower = SEG == 3 ? 0x1p-12f : SEG == 2 ? kSplitStep<T> : 1.0f;
template <int MI, int NI>
__device__ __forceinline__ void lower(f32x4 (&acc)[MI][NI], float step) {
#pragma unroll
    for (int m = 0; m < MI; ++m)
#pragma unroll
        for (int n = 0; n < NI; ++n)
#pragma unroll
            for (int r = 0; r < 4; ++r) acc[m][n][r] *= step;
}

// A tile a workgroup, for products too small for the walk below: two stages of 64 contraction indexes, two workgroups a CU
// that cover each other's waits.  Bound by LDS reads (a wave of 64 x 64 reads 8 KiB for 16 matrix instructions): float32 as three
// products of 6888 x 1024 x 1024 58 to 66 us (43 GF, 700 TF), gradients as six of 13 776 x 512 x 512 48 to 79 us.
template <typename T, typename TO, typename TB, int SEG, int ACT, int BM, int BN, int WM, int WN, int BK, int ST, bool PT, bool QT, int WPE>
__global__ void __launch_bounds__(64 * (BM / WM) * (BN / WN), WPE)
k_mm16(Side P, Side Q, Out o, long long I, int J, long long nq, long long q_per_part, int tiles_j, int n_tiles) {
    constexpr int WAVES = (BM / WM) * (BN / WN);
    typedef Stage<BM, BK, PT, WAVES, PT || QT> SP;
    typedef Stage<BN, BK, QT, WAVES, PT || QT> SQ;
    constexpr int kStage = SP::kBytes + SQ::kBytes;
    constexpr int MI = WM / 16, NI = WN / 16;
    __shared__ __attribute__((aligned(1024))) char lds[ST * kStage];

    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // consecutive workgroups go to the 8 XCDs in turn: each XCD walks its own run of tiles, j fastest, so the rows of P
    // it reads and all of Q stay in its L2
    const int per = (n_tiles + 7) / 8;
    const int tile = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
    if ((int)(blockIdx.x >> 3) >= per || tile >= n_tiles) return;
    const long long i0 = (long long)(tile / tiles_j) * BM;
    const int j0 = tile % tiles_j * BN;
    const long long q0 = (long long)blockIdx.y * q_per_part;
    const long long q1 = q0 + q_per_part < nq ? q0 + q_per_part : nq;
    const int wi = wave / (BN / WN) * WM, wj = wave % (BN / WN) * WN;

    SP sp;
    SQ sq;
    sp.init(P, i0, q0, wave, lane);
    sq.init(Q, j0, q0, wave, lane);
    sp.base += plane_of(kPlanesP<SEG>, 0) * P.plane * 2;
    sq.base += plane_of(kPlanesQ<SEG>, 0) * Q.plane * 2;
    const int once = (int)((q1 - q0 + BK - 1) / BK), steps = SEG * once;
    const int missing = (int)max(0LL, q1 - (nq - Q.missing));   // at the end of this part
    int krem = (int)(q1 - q0), seg = 0;
    auto load = [&](int slot) {
        sp.load(lds + slot * kStage, krem, wave, lane);
        sq.load(lds + slot * kStage + SP::kBytes, krem - missing, wave, lane);
        krem -= BK;
        if (SEG > 1 && krem <= 0 && ++seg < SEG) {
            krem = (int)(q1 - q0);
            sp.base = sp.start + plane_of(kPlanesP<SEG>, seg) * P.plane * 2;
            sq.base = sq.start + plane_of(kPlanesQ<SEG>, seg) * Q.plane * 2;
        }
    };
#pragma unroll
    for (int s = 0; s < ST - 1; ++s) load(s);

    f32x4 acc[MI][NI];
    typename vec<TB, 4>::type bias[NI];
    load_bias<TB, NI>(o, bias, SEG == 3 ? J : j0 + wj, J, lane);
    start_sums<TB, MI, NI>(acc, bias);

    int slot = 0;
    for (int k = 0; k < steps; ++k) {
        if (kLower<SEG, T> != 1.0f && k == (SEG - 1) * once) lower(acc, kLower<SEG, T>);
        wait_loads((SP::kLoads + SQ::kLoads) * (ST - 2));
        barrier();
        load(slot == 0 ? ST - 1 : slot - 1);
        const char* ps = lds + slot * kStage;
        const char* qs = ps + SP::kBytes;
#pragma unroll
        for (int ks = 0; ks < BK / 32; ++ks) {
            s16x8 a[NI], b[MI];
#pragma unroll
            for (int n = 0; n < NI; ++n) a[n] = SQ::frag(qs, wj + 16 * n, ks, lane);
#pragma unroll
            for (int m = 0; m < MI; ++m) b[m] = SP::frag(ps, wi + 16 * m, ks, lane);
#pragma unroll
            for (int m = 0; m < MI; ++m)
#pragma unroll
                for (int n = 0; n < NI; ++n) acc[m][n] = mfma16<T>(a[n], b[m], acc[m][n]);
        }
        slot = slot + 1 == ST ? 0 : slot + 1;
    }
    wait_loads(0);                                           // nothing may be on its way into LDS when the wave ends

    if constexpr (SEG == 3) {
        if (!unscale<TB, MI, NI>(o, acc, i0 + wi, j0 + wj, I, J, (float)nq, lane)) return;
    } else if constexpr (SEG > 2) {
        if (o.flags && !all_finite<MI, NI>(o.flags, acc, i0 + wi, j0 + wj, I, J, lane)) return;
    }
    epilogue<T, TO, ACT, true, true, false, MI, NI>(o, acc, i0 + wi, j0 + wj, I, J, blockIdx.y, lane);
}

// The same product for many tiles.  Persistent: one workgroup a CU walks over the tiles, the ring running on into the next
// tile's first stages while a tile's results are written.  A step's fragments are read, and the loads of the step RING
// ahead started, between the products of the step before.
// A contraction that one side is contiguous in is a multiple of 32 here, J a multiple of BN.
// 256 x 256 tiles of 8 waves: a wave of 128 x 64 needs 12 KiB of LDS reads for 32 matrix instructions, which leaves room under
// the LDS rate; 4 stages, one barrier a step.  Two workgroups a CU on 256 x 128 tiles, to cover the epilogue, read half again
// as much from the L2s: 150 us where this one takes 124, and 181 with gelu where this one takes 179.
// Measured, bf16: 55 104 x 512 x 2048 124 us (930 TF; 1200 without results), with gelu 151 to 163 (two transcendental
// and fifteen other operations a result, which no product runs under: the wave of both SIMD slots is in its epilogue then);
// x 1025 exp to float32 89 us for the first 1024; gradients: dx 55 104 x 2048 x 512 115 us (1000 TF), dweight in 16 parts 114 to 124.
template <typename T, typename TO, typename TB, int SEG, int ACT, bool EXTRA, bool LINES, int BM, int BN, int WM, int WN, int RING, bool PT, bool QT>
__global__ void __launch_bounds__(64 * (BM / WM) * (BN / WN), (BM / WM) * (BN / WN) / 4)
k_mm16_walk(Side P, Side Q, Out o, long long I, int J, long long nq, long long q_per_part, int tiles_j, int n_tiles) {
    constexpr int BK = 32, WAVES = (BM / WM) * (BN / WN);
    typedef Stage<BM, BK, PT, WAVES, PT || QT> SP;
    typedef Stage<BN, BK, QT, WAVES, PT || QT> SQ;
    constexpr int kStage = SP::kBytes + SQ::kBytes, kLoads = SP::kLoads + SQ::kLoads;
    constexpr int MI = WM / 16, NI = WN / 16;
    __shared__ __attribute__((aligned(1024))) char lds[RING * kStage];

    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wi = wave / (BN / WN) * WM, wj = wave % (BN / WN) * WN;
    // consecutive workgroups go to the 8 XCDs in turn: each XCD walks its own run of tiles, j fastest
    const int per = (n_tiles + 7) / 8, walkers = gridDim.x / 8;
    const int first = (blockIdx.x & 7) * per, end = min(first + per, n_tiles);
    const long long q0 = (long long)blockIdx.y * q_per_part;
    const int nk = (int)(nq - q0 < q_per_part ? nq - q0 : q_per_part);
    const int missing = (int)max(0LL, q0 + nk - (nq - Q.missing));           // of them on Q's side
    const int once = (nk + BK - 1) / BK, steps = SEG * once;
    const int pairs = max(RING / 2, (steps + 1) / 2);        // steps run in twos, at least RING of them: the extra ones add zeros
    static_assert(RING % 2 == 0, "a tile's first load is a pair's first");
    int tile = first + (blockIdx.x >> 3);
    if (tile >= end) return;
    SP sp;
    SQ sq;
    int krem = 0, seg = 0;                                   // what is left of the tile (its product) the loads are in
    auto move = [&] {
        krem -= BK;
        if (SEG > 1 && krem <= 0 && ++seg < SEG) {
            krem = nk;
            sp.base = sp.start + plane_of(kPlanesP<SEG>, seg) * P.plane * 2;
            sq.base = sq.start + plane_of(kPlanesQ<SEG>, seg) * Q.plane * 2;
        }
    };
    auto enter = [&](int t) {
        seg = 0;
        if (t < end) {
            sp.init(P, (long long)(t / tiles_j) * BM, q0, wave, lane);
            sq.init(Q, (long long)(t % tiles_j) * BN, q0, wave, lane);
            sp.base += plane_of(kPlanesP<SEG>, 0) * P.plane * 2;
            sq.base += plane_of(kPlanesQ<SEG>, 0) * Q.plane * 2;
        }
        krem = t < end ? nk : 0;                             // past the last tile: zeros
    };
    enter(tile);
#pragma unroll
    for (int s = 0; s < RING; ++s) {
        sp.load(lds + s * kStage, krem, wave, lane);
        sq.load(lds + s * kStage + SP::kBytes, krem - missing, wave, lane);
        move();
    }
    wait_loads(kLoads * (RING - 1));
    int slot = 0, left = 2 * pairs - RING;                   // loads left in the tile they are in
    f32x4 acc[MI][NI];
    s16x8 a[2][NI], b[MI];
    typename vec<TB, 4>::type bias[NI];
    load_bias<TB, NI>(o, bias, SEG == 3 ? J : tile % tiles_j * BN + wj, J, lane);
    // Stores of the last tile's results are newer than the first RING stages of this one: while those are waited for
    // (RING - 1 steps) they may stay outstanding; `old` is how many there are at least, rounded down to 16 or 32.
    int old = 0, grace = 0;
    auto step = [&](const s16x8 (&ca)[NI], s16x8 (&na)[NI]) {
        if (grace > 0 && old >= 32) wait_loads(kLoads * (RING - 2) + 32);
        else if (grace > 0 && old >= 16) wait_loads(kLoads * (RING - 2) + 16);
        else wait_loads(kLoads * (RING - 2));
        --grace;
        barrier();                                           // step k + 1 has landed, step k has been read by all
        char* into = lds + slot * kStage;
        slot = slot + 1 == RING ? 0 : slot + 1;
        const char* ps = lds + slot * kStage;
        const __amdgpu_buffer_rsrc_t rp = sp.buffer(krem), rq = sq.buffer(krem - missing);
#pragma unroll
        for (int m = 0; m < MI; ++m) {
#pragma unroll
            for (int i = m * kLoads / MI; i < (m + 1) * kLoads / MI; ++i) {
                if (i < SP::kLoads) sp.load_one(rp, into, i, sp.voff[i < SP::kLoads ? i : 0], wave);
                else sq.load_one(rq, into + SP::kBytes, i - SP::kLoads, sq.voff[i < SP::kLoads ? 0 : i - SP::kLoads], wave);
            }
#pragma unroll
            for (int n = m * NI / MI; n < (m + 1) * NI / MI; ++n) na[n] = SQ::frag(ps + SP::kBytes, wj + 16 * n, 0, lane);
#pragma unroll
            for (int n = 0; n < NI; ++n) acc[m][n] = mfma16<T>(ca[n], b[m], acc[m][n]);
            b[m] = SP::frag(ps, wi + 16 * m, 0, lane);
            __builtin_amdgcn_sched_barrier(0);
        }
        sp.advance();
        sq.advance();
        move();
    };
    for (; tile < end; tile += walkers) {
        barrier();                                           // the tile's first stage has landed
#pragma unroll
        for (int n = 0; n < NI; ++n) a[0][n] = SQ::frag(lds + slot * kStage + SP::kBytes, wj + 16 * n, 0, lane);
#pragma unroll
        for (int m = 0; m < MI; ++m) b[m] = SP::frag(lds + slot * kStage, wi + 16 * m, 0, lane);
        start_sums<TB, MI, NI>(acc, bias);
#pragma unroll 1
        for (int k = pairs; k > 0; --k) {
            const int at = 2 * (pairs - k), from = (SEG - 1) * once;
            if (kLower<SEG, T> != 1.0f && at == from) lower(acc, kLower<SEG, T>);
            if (left == 0) enter(tile + walkers);
            step(a[0], a[1]);
            left -= 2;
            if (kLower<SEG, T> != 1.0f && SEG == 2 && at + 1 == from) lower(acc, kLower<SEG, T>);
            step(a[1], a[0]);
        }
        left = 2 * pairs - RING;
        wait_loads(kLoads * (RING - 1));
        if constexpr (SEG != 3) {
            if (tile + walkers < end) load_bias<TB, NI>(o, bias, (tile + walkers) % tiles_j * BN + wj, J, lane);
#pragma unroll
            for (int n = 0; n < NI; ++n) {                   // arrived before the stores below are issued
                typedef unsigned uB __attribute__((ext_vector_type(sizeof(TB))));
                uB t = __builtin_bit_cast(uB, bias[n]);
                asm volatile("" : "+v"(t) : : "memory");
                bias[n] = __builtin_bit_cast(typename vec<TB, 4>::type, t);
            }
        }
        grace = RING - 1;
        if constexpr (SEG == 3) {
            if (!unscale<TB, MI, NI>(o, acc, (long long)(tile / tiles_j) * BM + wi, tile % tiles_j * BN + wj, I, J, (float)nq, lane)) {
                old = 0;
                continue;
            }
        } else if constexpr (SEG > 2) {
            if (o.flags && !all_finite<MI, NI>(o.flags, acc, (long long)(tile / tiles_j) * BM + wi, tile % tiles_j * BN + wj, I, J, lane)) {
                old = 0;
                continue;
            }
        }
        old = epilogue<T, TO, ACT, EXTRA, false, LINES, MI, NI>(o, acc, (long long)(tile / tiles_j) * BM + wi, tile % tiles_j * BN + wj, I, J, blockIdx.y, lane);
    }
    wait_loads(0);                                           // nothing may be on its way into LDS when the wave ends
}

}  // namespace gl_mm
