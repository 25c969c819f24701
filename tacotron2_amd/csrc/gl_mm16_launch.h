// Launches of the 16-bit products (gl_mm16.h), instantiated once per element type (gl_dense_bf16.hip, gl_dense_f16.hip,
// gl_dense_f32.hip: its planes).
#pragma once
#include "gl_dense.h"
#include "gl_mm16.h"

namespace gl_mm {

// rows: of C on this side.  A padded operand contiguous in the contraction has nq rounded up to kPadded of it, one contiguous
// across it may be read in whole chunks of 8.
static inline Side side(const gl_operand& o, long long rows, long long nq, long long nq_padded) {
    const bool across = o.across();
    return {o.base, across ? o.qs : o.is, across && o.padded ? (rows + 7) / 8 * 8 : rows, o.plane,
            across ? (int)(nq_padded - nq) : 0};
}

static inline long long padded_q(const gl_operand& P, long long nq) {
    return P.padded && !P.across() ? (nq + kPadded - 1) / kPadded * kPadded : nq;
}

template <typename T, typename TO, typename TB, int SEG, int ACT, bool EXTRA, bool LINES, int BM, bool PT, bool QT>
int walk_as(const gl_operand& P, const gl_operand& Q, const Out& o, long long I, int J, long long nq, const gl_mm_plan& p, hipStream_t st) {
    const long long pad = padded_q(P, nq);
    const int tiles_j = J / 256;
    const long long tiles = gl_ceil_div(I, BM) * tiles_j;
    long long walkers = 256 / p.parts / 8 * 8;               // one workgroup a CU in all, whole rounds of the 8 XCDs
    if (walkers > (tiles + 7) / 8 * 8) walkers = (tiles + 7) / 8 * 8;
    if (walkers < 8) walkers = 8;
    hipLaunchKernelGGL((k_mm16_walk<T, TO, TB, SEG, ACT, EXTRA, LINES, BM, 256, BM / 2, 64, 4, PT, QT>), dim3((unsigned)walkers, p.parts), dim3(512),
                       0, st, side(P, I, nq, pad), side(Q, J, nq, pad), o, I, J, pad, p.per, tiles_j, (int)tiles);
    GL_HIP_CHECK(hipGetLastError());
    return 0;
}

template <typename T, typename TO, typename TB, int SEG, int ACT, bool EXTRA, bool PT, bool QT>
int walk(const gl_operand& P, const gl_operand& Q, const Out& o, long long I, int J, long long nq, const gl_mm_plan& p, hipStream_t st) {
    auto on_lines = [](const void* q, long long stride) { return !q || ((uintptr_t)q % 128 == 0 && stride * (long long)sizeof(TO) % 128 == 0); };
    const bool lines = p.parts == 1 && on_lines(o.y, o.y_stride) && on_lines(o.z, o.z_stride);
    if constexpr (!PT && SEG <= 2) {
        // Tiles of 224 rows where the chip's rounds of them are shorter than of 256: 55 104 x 512 (of 2048) are 1.7 rounds of 256,
        // 136 us, and 1.9 of 224, 123 us.  Not for rows read transposed (whole powers of two) or flagged in blocks of 64.
        auto rounds = [&](int rows) { return gl_ceil_div(gl_ceil_div(I, rows) * (J / 256), 256) * rows; };
        if (p.parts == 1 && rounds(224) < rounds(256))
            return lines ? walk_as<T, TO, TB, SEG, ACT, EXTRA, true, 224, PT, QT>(P, Q, o, I, J, nq, p, st)
                         : walk_as<T, TO, TB, SEG, ACT, EXTRA, false, 224, PT, QT>(P, Q, o, I, J, nq, p, st);
    }
    return lines ? walk_as<T, TO, TB, SEG, ACT, EXTRA, true, 256, PT, QT>(P, Q, o, I, J, nq, p, st)
                 : walk_as<T, TO, TB, SEG, ACT, EXTRA, false, 256, PT, QT>(P, Q, o, I, J, nq, p, st);
}

template <typename T, typename TO, typename TB, int SEG, int B, int W, bool PT, bool QT>
int tiles(const gl_operand& P, const gl_operand& Q, const Out& o, long long I, int J, long long nq, const gl_mm_plan& p, hipStream_t st) {
    const long long pad = padded_q(P, nq);
    const int tiles_j = (int)gl_ceil_div(J, B);
    const long long n = gl_ceil_div(I, B) * tiles_j;
    hipLaunchKernelGGL((k_mm16<T, TO, TB, SEG, -1, B, B, W, W, 64, 2, PT, QT, 2>), dim3((unsigned)((n + 7) / 8 * 8), p.parts), dim3(256), 0, st,
                       side(P, I, nq, pad), side(Q, J, nq, pad), o, I, J, pad, p.per, tiles_j, (int)n);
    GL_HIP_CHECK(hipGetLastError());
    return 0;
}

// 64 x 64 tiles: their waves are smaller than a block of flags, so float32 planes take 128 x 128 instead
template <typename T, typename TO, typename TB, int SEG, bool PT, bool QT>
int small(const gl_operand& P, const gl_operand& Q, const Out& o, long long I, int J, long long nq, const gl_mm_plan& p, hipStream_t st) {
    if constexpr (SEG > 2) return tiles<T, TO, TB, SEG, 128, 64, PT, QT>(P, Q, o, I, J, nq, p, st);
    else return tiles<T, TO, TB, SEG, 64, 32, PT, QT>(P, Q, o, I, J, nq, p, st);
}

template <typename T, typename TO, typename TB, int SEG, bool PT, bool QT>
int one(const gl_operand& P, const gl_operand& Q, const gl_epilogue& e, long long I, int J, long long nq, const gl_mm_plan& p,
        float* partial, hipStream_t st) {
    if (p.parts > 1) {
        const Out o = {nullptr, nullptr, 0, partial, J, nullptr, 0, GL_ACT_NONE, nullptr, I * J, 0, e.scale_p, e.scale_q};
        const int rc = p.kind == 2 ? walk<T, float, TB, SEG, GL_ACT_NONE, false, PT, QT>(P, Q, o, I, J, nq, p, st)
                     : p.kind == 1 ? tiles<T, float, TB, SEG, 128, 64, PT, QT>(P, Q, o, I, J, nq, p, st)
                                   : small<T, float, TB, SEG, PT, QT>(P, Q, o, I, J, nq, p, st);
        if (rc) return rc;
        gl_epilogue j = e;
        j.partial = partial;
        if constexpr (SEG > 2) return gl_dense_join_planes(j, I, J, nq, p, st);
        else return gl_dense_join<TB, TO>(j, I, J, p.parts, st);
    }
    auto off4 = [](const void* q, long long stride) { return q && (stride % 2 || (uintptr_t)q % 4); };
    const int odd = sizeof(TO) == 2 && (off4(e.y, e.y_stride) || off4(e.z, e.z_stride) || off4(e.residual, e.r_stride));
    const Out o = {e.bias, e.residual, e.r_stride, e.y, e.y_stride, e.z, e.z_stride, e.act, e.flags, 0, odd, e.scale_p, e.scale_q};
    if (p.kind == 0) return small<T, TO, TB, SEG, PT, QT>(P, Q, o, I, J, nq, p, st);
    if (p.kind == 1) return tiles<T, TO, TB, SEG, 128, 64, PT, QT>(P, Q, o, I, J, nq, p, st);
    if constexpr (PT || QT) return walk<T, TO, TB, SEG, GL_ACT_NONE, false, PT, QT>(P, Q, o, I, J, nq, p, st);   // gradients: no epilogue
    else {
        const bool extra = e.residual || e.z;
#define GL_WALK(A)                                                                                                          \
    case A:                                                                                                                 \
        return extra ? walk<T, TO, TB, SEG, A, true, false, false>(P, Q, o, I, J, nq, p, st)                                         \
                     : walk<T, TO, TB, SEG, A, false, false, false>(P, Q, o, I, J, nq, p, st);
        switch (e.act) {
            GL_WALK(GL_ACT_RELU) GL_WALK(GL_ACT_SILU) GL_WALK(GL_ACT_GELU) GL_WALK(GL_ACT_TANH) GL_WALK(GL_ACT_EXP)
            default: return extra ? walk<T, TO, TB, SEG, GL_ACT_NONE, true, false, false>(P, Q, o, I, J, nq, p, st)
                                  : walk<T, TO, TB, SEG, GL_ACT_NONE, false, false, false>(P, Q, o, I, J, nq, p, st);
        }
#undef GL_WALK
    }
}

}  // namespace gl_mm

template <typename T, typename TO, typename TB, int SEG>
int gl_mm16(const gl_operand& P, const gl_operand& Q, gl_epilogue e, long long I, int J, long long nq, float* partial, hipStream_t st) {
    const bool pt = P.across(), qt = Q.across();
    const long long pad = gl_mm::padded_q(P, nq);
    const int first = gl_mm_first_columns(I, J, pad, pt && qt, (int)sizeof(TO));
    for (int j = 0; j < J; j += first) {
        const int n = j ? J - j : first;
        gl_operand q = Q;
        gl_epilogue f = e;
        q.base = (const T*)Q.base + j * Q.is;
        if (e.bias) f.bias = (const TB*)e.bias + j;
        if (e.residual) f.residual = (const TO*)e.residual + j;
        f.y = (TO*)e.y + j;
        if (e.z) f.z = (TO*)e.z + j;
        if (e.exact_q) f.exact_q = e.exact_q + j * e.exact_q_is;
        if (e.scale_q) f.scale_q = e.scale_q + j;
        const gl_mm_plan p = gl_mm_plan_for(I, n, pad, pt && qt);
        int rc = 0;
        bool along = SEG == 3;                               // both sides contiguous in the contraction: no gradients
        if constexpr (SEG != 2) {
            along |= !pt && !qt;
            if (along) rc = gl_mm::one<T, TO, TB, SEG, false, false>(P, q, f, I, n, nq, p, partial, st);
        }
        if constexpr (SEG != 3) {
            if (!along) rc = !pt ? gl_mm::one<T, TO, TB, SEG, false, true>(P, q, f, I, n, nq, p, partial, st)
                     : gl_mm::one<T, TO, TB, SEG, true, true>(P, q, f, I, n, nq, p, partial, st);
        }
        if (rc) return rc;
        if (SEG > 2 && p.parts == 1) {                       // the blocks that were left out, if any
            const int rf = gl_dense_flagged(f, I, n, nq, st);
            if (rf) return rf;
        }
        if (j) break;                                        // two launches at most
    }
    return 0;
}
