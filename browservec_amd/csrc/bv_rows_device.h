// Rows in the registers of a few waves: sums over a row's threads, the norms'
// statistics, weights (bv_rows.hip, bv_add_norm.hip).  Chunk j of a row's thread i
// holds the eight elements from (j * 64 * WAVES + i) * 8 on, zeros past the row's
// end.
#pragma once

#include "bv_embed.h"
#include "bv_embed_device.h"

namespace bvk {
namespace {

template <int WAVES>
constexpr int BLOCK = WAVES <= 4 ? 256 : 64 * WAVES;

// Sums over a row's threads, of up to R rows at once.  Waves exchange theirs
// through two places in turn, with one barrier a sum: a place is written again
// after the next sum's barrier, which every reader has reached by then.  That
// holds for sums of fewer rows too, since the places lie WAVES * R apart whatever
// a sum's rows: all sums of a workgroup go through one of these.
template <int WAVES, int R>
struct RowSums {
    static constexpr int PLACE = WAVES * R, FLOATS = 2 * PLACE;
    float *lds;
    int turn = 0;
    template <int K>
    __device__ __forceinline__ void operator()(float (&x)[K]) {
        static_assert(WAVES * K <= PLACE, "a sum stays within its place");
#pragma unroll
        for (int k = 0; k < K; k++) x[k] = wave_sum(x[k]);
        if (WAVES == 1) return;
        float *p = lds + turn * PLACE;
        turn ^= 1;
        if ((threadIdx.x & 63) == 0)
#pragma unroll
            for (int k = 0; k < K; k++) p[(threadIdx.x >> 6) * K + k] = x[k];
        __syncthreads();
#pragma unroll
        for (int k = 0; k < K; k++) x[k] = 0;
#pragma unroll
        for (int w = 0; w < WAVES; w++)
#pragma unroll
            for (int k = 0; k < K; k++) x[k] += p[w * K + k];
    }
};

// weights and biases: of any of the three types
__device__ __forceinline__ void load8_of(int type, const void *p, uint32_t at, uint32_t n, bool tail, float (&f)[8]) {
    if (type == T_F32) load8((const float *)p, at, n, tail, f);
    else if (type == T_F16) load8((const f16 *)p, at, n, tail, f);
    else load8((const bf16 *)p, at, n, tail, f);
}

// What the norm does to each row: (f - mean) * r.
template <int WAVES, int CH, int R, class Args>
__device__ __forceinline__ void norm_stats(const Args &a, const int norm, uint32_t i, RowSums<WAVES, R> &sums,
                                           const float (&f)[R][CH][8], float (&mean)[R], float (&r)[R]) {
#pragma unroll
    for (int k = 0; k < R; k++) mean[k] = 0.0f, r[k] = 1.0f;
    if (norm == 1) {
        float sum[R] = {};
#pragma unroll
        for (int k = 0; k < R; k++)
#pragma unroll
            for (int j = 0; j < CH; j++)
#pragma unroll
                for (int e = 0; e < 8; e++) sum[k] += f[k][j][e];
        sums(sum);
#pragma unroll
        for (int k = 0; k < R; k++) mean[k] = sum[k] / (float)a.dim;
    }
    if (norm) {  // the squares about the mean, after it: no cancellation
        float sq[R] = {};
#pragma unroll
        for (int k = 0; k < R; k++)
#pragma unroll
            for (int j = 0; j < CH; j++)
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    float d = f[k][j][e];
                    if (norm == 1) d = (j * 64 * WAVES + i) * 8 + e < a.dim ? d - mean[k] : 0.0f;
                    sq[k] = fmaf(d, d, sq[k]);
                }
        sums(sq);
#pragma unroll
        for (int k = 0; k < R; k++) r[k] = 1.0f / sqrtf(sq[k] / (float)a.dim + a.eps);
    }
}

// f times the weights plus the biases, zeros past the row's end.
template <int WAVES, int CH, int R, class Args>
__device__ __forceinline__ void weighted(const Args &a, uint32_t i, float (&f)[R][CH][8]) {
    const bool tail = a.dim % 8 != 0;
#pragma unroll
    for (int j = 0; j < CH; j++) {
        const uint32_t at = (j * 64 * WAVES + i) * 8;
        float w[8], b[8];
#pragma unroll
        for (int e = 0; e < 8; e++) w[e] = 1.0f, b[e] = 0.0f;
        if (a.w) load8_of(a.wtype, a.w, at, a.dim, tail, w);
        if (a.b) load8_of(a.wtype, a.b, at, a.dim, tail, b);
#pragma unroll
        for (int k = 0; k < R; k++)
#pragma unroll
            for (int e = 0; e < 8; e++) f[k][j][e] = at + e < a.dim ? fmaf(f[k][j][e], w[e], b[e]) : 0.0f;
    }
}

}  // namespace
}  // namespace bvk
