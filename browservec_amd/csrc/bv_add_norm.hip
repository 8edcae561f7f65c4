// t = x + r and the norm of t, in one pass: to a float type, or to codes of 8
// bits and a scale a row, as the products of bv_linear_q8.hip take them.
#include "bv_embed.h"
#include "bv_embed_device.h"
#include "bv_rows_device.h"

#include <algorithm>

namespace bvk {
namespace {

// as in bv_rows.hip: launches of at most 2^31 threads
constexpr uint32_t GRID_MOST = 1u << 21;

// A row's waves are a workgroup of their own, rows of one wave go by fours.
template <int WAVES>
constexpr int ADD_BLOCK = WAVES == 1 ? 256 : 64 * WAVES;

// Rows' codes: q = rint(f 127 / top) and the scale top / 127, in 32 bits each.
//   top 0 (a row of zeros): codes and scale 0.
//   top infinite or NaN: codes 0 and a scale of NaN, so that what is made of the
//     row is NaN.
//   tops below 2^-100 go through a factor of 2^100: 127 / top would pass 2^128.
template <int WAVES, int CH, int R>
__device__ __forceinline__ void store_codes(const AddNormArgs &a, uint64_t row0, uint64_t rows, uint32_t i, float *lds,
                                            const float (&f)[R][CH][8]) {
    float top[R];
#pragma unroll
    for (int k = 0; k < R; k++) {
        top[k] = 0;
#pragma unroll
        for (int j = 0; j < CH; j++)
#pragma unroll
            for (int e = 0; e < 8; e++) top[k] = top_of(top[k], fabsf(f[k][j][e]));
        top[k] = wave_top(top[k]);
    }
    if (WAVES > 1) {
        if ((threadIdx.x & 63) == 0)
#pragma unroll
            for (int k = 0; k < R; k++) lds[(threadIdx.x >> 6) * R + k] = top[k];
        __syncthreads();
#pragma unroll
        for (int w = 0; w < WAVES; w++)
#pragma unroll
            for (int k = 0; k < R; k++) top[k] = top_of(top[k], lds[w * R + k]);
    }
#pragma unroll
    for (int k = 0; k < R; k++) {
        if (k >= rows) break;
        const bool fine = top[k] <= 3.402823466e38f, none = top[k] == 0.0f;
        const float up = top[k] < 0x1p-100f ? 0x1p100f : 1.0f;
        const float inv = none || !fine ? 0.0f : 127.0f / (top[k] * up);
        int8_t *y = (int8_t *)a.y + (row0 + k) * a.ldy;
#pragma unroll
        for (int j = 0; j < CH; j++) {
            const uint32_t at = (j * 64 * WAVES + i) * 8;
            if (at >= a.dim) continue;
            union {
                int8_t b[8];
                uint64_t all;
            } q;
#pragma unroll
            for (int e = 0; e < 8; e++) q.b[e] = fine ? (int8_t)(int)__builtin_rintf(f[k][j][e] * up * inv) : 0;
            typedef uint64_t u64_any __attribute__((aligned(1)));
            if (at + 8 <= a.dim) {
                *(u64_any *)(y + at) = q.all;
            } else {
#pragma unroll
                for (int e = 0; e < 8; e++)
                    if (at + e < a.dim) y[at + e] = q.b[e];
            }
        }
        if (i == 0) a.scales[row0 + k] = fine ? top[k] / 127.0f : __builtin_nanf("");
    }
}

template <class O, int WAVES, int CH, int R>
__device__ __forceinline__ void store_floats(void *y0, uint64_t ld, uint32_t dim, uint64_t row0, uint64_t rows, uint32_t i,
                                             const float (&f)[R][CH][8]) {
#pragma unroll
    for (int k = 0; k < R; k++)
        if (k < rows)
#pragma unroll
            for (int j = 0; j < CH; j++) {
                const uint32_t at = (j * 64 * WAVES + i) * 8;
                if (at < dim) store8((O *)y0 + (row0 + k) * ld + at, (int)min(8u, dim - at), f[k][j]);
            }
}

// R rows' chunks of eight elements: chunk j of thread i from (j * 64 * WAVES + i) * 8 on.
template <bool ONCE, int WAVES, int CH, int R, class T>
__device__ __forceinline__ void load_rows(const T *x, uint64_t ld, uint32_t dim, uint64_t row0, uint64_t tokens, uint32_t i,
                                          float (&f)[R][CH][8]) {
#pragma unroll
    for (int k = 0; k < R; k++)
#pragma unroll
        for (int j = 0; j < CH; j++)
            load8<ONCE>(x + min(row0 + k, tokens - 1) * ld, (j * 64 * WAVES + i) * 8, dim, dim % 8 != 0, f[k][j]);
}

// R rows per WAVES waves.  The sum is kept as it is rounded to r's type; the norm
// is of the sum in 32 bits.  Everything is read and written once, which is the
// bound: 30011 x 768 with a residual (bf16, layer) 37.5 us, 4.9 TB/s of 5.1 that a copy
// reaches; 20011 x 4096 to codes 47 us, 5.2.
template <class T, class TR, bool Q8, int WAVES, int CH, int R>
__global__ __launch_bounds__(ADD_BLOCK<WAVES>) void add_norm_rows(AddNormArgs a, uint64_t first) {
    __shared__ float lds[RowSums<WAVES, R>::FLOATS], tops[Q8 ? WAVES * R : 1];
    RowSums<WAVES, R> sums{lds};
    const uint32_t i = WAVES == 1 ? threadIdx.x & 63 : threadIdx.x;
    const uint64_t row0 = first + (WAVES == 1 ? (uint64_t)blockIdx.x * 4 + (threadIdx.x >> 6) : blockIdx.x) * R;
    if (row0 >= a.tokens) return;
    const uint64_t rows = a.tokens - row0;
    float f[R][CH][8];
    if (a.once) load_rows<true, WAVES>((const T *)a.x, a.ldx, a.dim, row0, a.tokens, i, f);
    else load_rows<false, WAVES>((const T *)a.x, a.ldx, a.dim, row0, a.tokens, i, f);
    if (a.r) {
        float g[R][CH][8];
        if (a.once) load_rows<true, WAVES>((const TR *)a.r, a.ldr, a.dim, row0, a.tokens, i, g);
        else load_rows<false, WAVES>((const TR *)a.r, a.ldr, a.dim, row0, a.tokens, i, g);
#pragma unroll
        for (int k = 0; k < R; k++)
#pragma unroll
            for (int j = 0; j < CH; j++)
#pragma unroll
                for (int e = 0; e < 8; e++) f[k][j][e] += g[k][j][e];
        if (a.total) {
            // it may lie where x or r does: a row's last chunk is loaded from
            // elements that another thread stores
            if (a.dim % 8) {
                asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
                if (WAVES > 1) __syncthreads();
            }
            store_floats<TR, WAVES, CH, R>(a.total, a.ldt, a.dim, row0, rows, i, f);
        }
    }
    float mean[R], r[R];
    norm_stats<WAVES, CH, R>(a, a.norm, i, sums, f, mean, r);
#pragma unroll
    for (int k = 0; k < R; k++)
#pragma unroll
        for (int j = 0; j < CH; j++)
#pragma unroll
            for (int e = 0; e < 8; e++) f[k][j][e] = (f[k][j][e] - mean[k]) * r[k];
    weighted<WAVES, CH, R>(a, i, f);
    if (Q8) {
        store_codes<WAVES, CH, R>(a, row0, rows, i, tops, f);
        return;
    }
    if (WAVES > 1) __syncthreads();  // y may be x: every thread has its elements
    if (a.out_dtype == T_F32) store_floats<float, WAVES, CH, R>(a.y, a.ldy, a.dim, row0, rows, i, f);
    else if (a.out_dtype == T_F16) store_floats<f16, WAVES, CH, R>(a.y, a.ldy, a.dim, row0, rows, i, f);
    else store_floats<bf16, WAVES, CH, R>(a.y, a.ldy, a.dim, row0, rows, i, f);
}

template <class T, class TR, bool Q8, int WAVES, int CH, int R>
hipError_t add_norm_of(const AddNormArgs &a, hipStream_t s) {
    constexpr uint64_t each = R * (ADD_BLOCK<WAVES> / 64 / WAVES);
    for (uint64_t r = 0; r < a.tokens; r += GRID_MOST * each) {
        const uint64_t blocks = (a.tokens - r + each - 1) / each;
        add_norm_rows<T, TR, Q8, WAVES, CH, R><<<(uint32_t)std::min<uint64_t>(blocks, GRID_MOST), ADD_BLOCK<WAVES>, 0, s>>>(a, r);
    }
    return hipGetLastError();
}

// 30011 x 768: two waves of one chunk, two rows at a time 40.4 us, one 43.1, four
// 48.9; one wave of two chunks 43.5 and 46.0; 20011 x 4096: four waves of two chunks, one row
// 47, two 52; eight of one 62.
template <class T, class TR, bool Q8>
hipError_t add_norm_sized(const AddNormArgs &a, hipStream_t s) {
    if (a.dim <= 512) return add_norm_of<T, TR, Q8, 1, 1, 2>(a, s);
    if (a.dim <= 1024) return add_norm_of<T, TR, Q8, 2, 1, 2>(a, s);
    if (a.dim <= 2048) return add_norm_of<T, TR, Q8, 4, 1, 2>(a, s);
    if (a.dim <= 4096) return add_norm_of<T, TR, Q8, 4, 2, 1>(a, s);
    if (a.dim <= 8192) return add_norm_of<T, TR, Q8, 16, 1, 1>(a, s);
    return add_norm_of<T, TR, Q8, 16, 2, 1>(a, s);
}
template <class T, class TR>
hipError_t add_norm_typed(const AddNormArgs &a, hipStream_t s) {
    return a.out_dtype == T_I8 ? add_norm_sized<T, TR, true>(a, s) : add_norm_sized<T, TR, false>(a, s);
}

}  // namespace

// r is of x's type or of 32 bits.
hipError_t launch_add_norm(const AddNormArgs &given, hipStream_t s) {
    AddNormArgs a = given;
    const bool wide = a.r && a.r_dtype == T_F32;
    // Rows that the card's caches (256 MB) do not hold together with the results do not
    // go there: 30011 x 768 with a residual, 184 MB in all, 40.4 -> 37.5 us; 8192 x 1024, 67
    // MB, 13.0 plainly and 14.6.
    const uint64_t each = (a.dtype == T_F32 ? 4 : 2) + (a.out_dtype == T_F32 ? 4 : a.out_dtype == T_I8 ? 1 : 2) +
                          (a.r ? 2 * (wide || a.dtype == T_F32 ? 4 : 2) : 0);
    a.once = a.tokens * a.dim * each > (128u << 20);
    switch (a.dtype) {
    case T_F16: return wide ? add_norm_typed<f16, float>(a, s) : add_norm_typed<f16, f16>(a, s);
    case T_BF16: return wide ? add_norm_typed<bf16, float>(a, s) : add_norm_typed<bf16, bf16>(a, s);
    default: return add_norm_typed<float, float>(a, s);
    }
}

}  // namespace bvk
