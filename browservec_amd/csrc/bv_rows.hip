// Row operators of an embedding model: rotary positions, norms, pooling.
#include "bv_embed.h"
#include "bv_embed_device.h"
#include "bv_rows_device.h"

#include <algorithm>

namespace bvk {
namespace {

// workgroups of a launch: of 2^32 threads and more a dimension it runs the low 32
// bits, so with up to 1024 a workgroup more work is launched in pieces
constexpr uint32_t GRID_MOST = 1u << 21;

// ---------------------------------------------------------------- rotary --
// A thread turns (or copies) one unit of a token's heads: eight pairs, whose
// cosines and sines it keeps in registers, of every `groups`-th head:
//   (x, y) -> (x cos - y sin, y cos + x sin).
// Bound by HBM: every element is read and written once.  65536 x 20 heads of 64
// (bf16): 79.5 us, 4.3 TB/s of 5.2 that a copy reaches.  Small calls (17 tokens,
// 6 us) are one chain of position, table, heads.
constexpr uint32_t ROT_HEADS = 4;  // heads per thread: 79.9 us, with 1, 2, 8: 94, 81, 83

template <class T, bool INTERLEAVED>
__global__ __launch_bounds__(256) void rotary_rows(RotaryArgs a, uint64_t first, uint32_t turned, uint32_t units,
                                                   uint32_t groups, uint32_t per_block) {
    const uint32_t per_token = units * groups;
    uint32_t r = threadIdx.x, t = 0;
    if (per_token <= 256) {
        t = r / per_token;
        r -= t * per_token;
        if (t >= per_block) return;
    } else {
        r += blockIdx.y * 256;
        if (r >= per_token) return;
    }
    const uint64_t token = first + (uint64_t)blockIdx.x * per_block + t;
    if (token >= a.tokens) return;
    const uint32_t unit = r % units, group = r / units, half = a.rot / 2;
    float c[8], s[8];
    const bool turn = unit < turned;
    const uint32_t p0 = unit * 8;                                  // first pair
    const uint32_t e0 = a.rot + (turn ? 0 : (unit - turned) * 8);  // first copied element
    const int n = turn ? (int)min(8u, half - p0) : (int)min(8u, a.d - e0);
    if (turn) {
        const int64_t pos = a.pos ? (int64_t)a.pos[token] : (int64_t)token;
        const bool in = pos >= 0 && pos < (int64_t)a.rows;
        const float *row = a.table + (in ? (uint64_t)pos * a.rot : 0) + 2 * p0;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const bool ok = i < n && in;
            c[i] = ok ? row[2 * i] : __builtin_nanf("");
            s[i] = ok ? row[2 * i + 1] : __builtin_nanf("");
        }
    }
    for (uint32_t h = group; h < a.hq + a.hk; h += groups) {
        const bool key = h >= a.hq;
        const uint32_t hh = key ? h - a.hq : h;
        const T *x = (const T *)(key ? a.k : a.q) + token * (key ? a.sk : a.sq) + hh * (key ? a.skh : a.sqh);
        T *y = (T *)(key ? a.ko : a.qo) + token * (key ? a.sko : a.sqo) + hh * (key ? a.skoh : a.sqoh);
        float u[8], v[8];
        if (!turn) {
            load8(x + a.rot, e0 - a.rot, a.d - a.rot, (a.d - a.rot) % 8 != 0, u);
            store8(y + e0, n, u);
        } else if (INTERLEAVED) {
            const int n1 = min(8, 2 * n), n2 = 2 * n - n1;
            load8(x, 2 * p0, a.rot, a.rot % 8 != 0, u);
            load8(x, 2 * p0 + 8, a.rot, a.rot % 8 != 0, v);
            float f[8], g[8];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                f[2 * i] = u[2 * i] * c[i] - u[2 * i + 1] * s[i];
                f[2 * i + 1] = u[2 * i + 1] * c[i] + u[2 * i] * s[i];
                g[2 * i] = v[2 * i] * c[i + 4] - v[2 * i + 1] * s[i + 4];
                g[2 * i + 1] = v[2 * i + 1] * c[i + 4] + v[2 * i] * s[i + 4];
            }
            store8(y + 2 * p0, n1, f);
            store8(y + 2 * p0 + (n2 ? 8 : 0), n2, g);
        } else {
            load8(x, p0, half, half % 8 != 0, u);
            load8(x + half, p0, half, half % 8 != 0, v);
            float f[8], g[8];
#pragma unroll
            for (int i = 0; i < 8; i++) {
                f[i] = u[i] * c[i] - v[i] * s[i];
                g[i] = v[i] * c[i] + u[i] * s[i];
            }
            store8(y + p0, n, f);
            store8(y + half + p0, n, g);
        }
    }
}

template <class T>
hipError_t rotary_of(const RotaryArgs &a, hipStream_t s) {
    const bool copy = a.q != a.qo || (a.hk && a.k != a.ko);
    const uint32_t turned = (a.rot / 2 + 7) / 8;
    const uint32_t units = turned + (copy ? (a.d - a.rot + 7) / 8 : 0);
    const uint32_t heads = a.hq + a.hk, groups = (heads + ROT_HEADS - 1) / ROT_HEADS;
    const uint32_t per_token = units * groups;
    if (!per_token) return hipSuccess;
    const uint32_t per_block = per_token <= 256 ? 256 / per_token : 1;
    for (uint64_t t = 0; t < a.tokens; t += (uint64_t)GRID_MOST * per_block) {
        const uint64_t blocks = (a.tokens - t + per_block - 1) / per_block;
        const dim3 grid((uint32_t)std::min<uint64_t>(blocks, GRID_MOST), per_token <= 256 ? 1 : (per_token + 255) / 256);
        if (a.interleaved) rotary_rows<T, true><<<grid, 256, 0, s>>>(a, t, turned, units, groups, per_block);
        else rotary_rows<T, false><<<grid, 256, 0, s>>>(a, t, turned, units, groups, per_block);
    }
    return hipGetLastError();
}

// ----------------------------------------------------------------- norms --
// R rows in the registers of WAVES waves, CH chunks of eight elements a thread
// and row: chunk j of thread i holds elements (j * 64 * WAVES + i) * 8 onwards,
// and zeros past the row's end.  Several rows at a time: their loads are in
// flight together and their reductions interleave.  The mean first and then the
// squares about it, both from registers: one read, one write, which is the
// bound.  30011 x 768 (bf16, layer): 22.4 us, 4.1 TB/s of 5.2 that a copy
// reaches, two rows at a time (one 26.5, four 28.7); 131072 x 768 in 32 bits 167,
// 4.8 TB/s.
// Rows y0 on, `rows` of them: y = f, unit: f times 1 / |f| (a zero row stays).
template <class O, int WAVES, int CH, int R, int MOST>
__device__ __forceinline__ void store_rows(const NormArgs &a, O *y0, uint64_t rows, uint32_t i, RowSums<WAVES, MOST> &sums,
                                           float (&f)[R][CH][8]) {
    if (a.unit) {
        float sq[R] = {};
#pragma unroll
        for (int k = 0; k < R; k++)
#pragma unroll
            for (int j = 0; j < CH; j++)
#pragma unroll
                for (int e = 0; e < 8; e++) sq[k] = fmaf(f[k][j][e], f[k][j][e], sq[k]);
        sums(sq);
#pragma unroll
        for (int k = 0; k < R; k++) {
            const float norm = sqrtf(sq[k]);
            const float r = norm == 0.0f ? 1.0f : 1.0f / norm;
#pragma unroll
            for (int j = 0; j < CH; j++)
#pragma unroll
                for (int e = 0; e < 8; e++) f[k][j][e] *= r;
        }
    }
#pragma unroll
    for (int k = 0; k < R; k++)
        if (k < rows)
#pragma unroll
            for (int j = 0; j < CH; j++) {
                const uint32_t at = (j * 64 * WAVES + i) * 8;
                if (at < a.dim) store8(y0 + k * a.ldy + at, (int)min(8u, a.dim - at), f[k][j]);
            }
}

// R output rows per WAVES waves: tokens' (no pooling), or the first or last of
// each sequence's.
template <class T, class O, int WAVES, int CH, int R>
__global__ __launch_bounds__(BLOCK<WAVES>) void norm_rows(NormArgs a, uint64_t first) {
    __shared__ float lds[RowSums<WAVES, R>::FLOATS];
    RowSums<WAVES, R> sums{lds};
    const uint32_t i = WAVES == 1 ? threadIdx.x & 63 : threadIdx.x;
    const uint64_t row0 = first + (WAVES == 1 ? (uint64_t)blockIdx.x * 4 + (threadIdx.x >> 6) : blockIdx.x) * R;
    const uint64_t rows = a.pool ? a.batch : a.tokens;
    if (row0 >= rows) return;
    const bool tail = a.dim % 8 != 0;
    float f[R][CH][8];
    bool empty[R];
#pragma unroll
    for (int k = 0; k < R; k++) {
        const uint64_t row = min(row0 + k, rows - 1);
        int64_t from = row;
        empty[k] = false;
        if (a.pool) {
            const int64_t b = clip_cu(a.cu, row, a.tokens), e = clip_cu(a.cu, row + 1, a.tokens);
            empty[k] = e <= b;
            from = empty[k] ? 0 : a.pool == 2 ? b : e - 1;
        }
        if (a.tokens == 0) {
#pragma unroll
            for (int j = 0; j < CH; j++)
#pragma unroll
                for (int e = 0; e < 8; e++) f[k][j][e] = 0.0f;
        } else {
#pragma unroll
            for (int j = 0; j < CH; j++)
                load8((const T *)a.x + from * a.ldx, (j * 64 * WAVES + i) * 8, a.dim, tail, f[k][j]);
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
    if (WAVES > 1) __syncthreads();  // y may be x: every thread has its elements
#pragma unroll
    for (int k = 0; k < R; k++)
        if (empty[k])
#pragma unroll
            for (int j = 0; j < CH; j++)
#pragma unroll
                for (int e = 0; e < 8; e++) f[k][j][e] = 0.0f;
    store_rows<O, WAVES, CH, R>(a, (O *)a.y + row0 * a.ldy, rows - row0, i, sums, f);
}

// --------------------------------------------------------------- pooling --
// The mean in two launches: a workgroup sums a chunk of one sequence's rows (its
// slot, see slot_sequence), WAVES waves taking R rows at a time in turn with
// the others, and writes a partial sum, or the result where the sequence has no
// more rows; a second launch joins the partial sums of longer sequences in their
// order.  Weights and biases are applied to the mean: they are the same for
// every row.  Bound by the read of the rows: 3000 x 1..256 x 1024 (bf16, RMS
// norm) 182 us, 4.4 TB/s, of which the join takes 12.

// The sums of a workgroup's GROUPS groups of waves, by halves: group 0's.
template <int WAVES, int CH, int GROUPS>
__device__ __forceinline__ void join_groups(uint32_t group, uint32_t i, float *lds, float (&acc)[1][CH][8]) {
    constexpr uint32_t SPAN = CH * 512 * WAVES;
#pragma unroll
    for (int h = GROUPS / 2; h; h /= 2) {
        if ((int)group >= h && (int)group < 2 * h)
#pragma unroll
            for (int j = 0; j < CH; j++)
#pragma unroll
                for (int x = 0; x < 8; x++) lds[(group - h) * SPAN + (j * 8 + x) * 64 * WAVES + i] = acc[0][j][x];
        __syncthreads();
        if ((int)group < h)
#pragma unroll
            for (int j = 0; j < CH; j++)
#pragma unroll
                for (int x = 0; x < 8; x++) acc[0][j][x] += lds[group * SPAN + (j * 8 + x) * 64 * WAVES + i];
        __syncthreads();
    }
}

template <class T, int WAVES, int CH, int R, int NORM>
__global__ __launch_bounds__(BLOCK<WAVES>) void pool_chunk(NormArgs a, uint64_t first, uint32_t shift) {
    constexpr int GROUPS = BLOCK<WAVES> / 64 / WAVES;  // waves with rows of their own
    __shared__ float acc_lds[GROUPS > 1 ? GROUPS / 2 * CH * 512 * WAVES : 1], lds[RowSums<WAVES, R>::FLOATS];
    RowSums<WAVES, R> sums{lds};
    const uint64_t slot = first + spread(blockIdx.x, gridDim.x, 1);
    const uint32_t rows = 1u << shift;
    const uint32_t s = __builtin_amdgcn_readfirstlane(slot_sequence(a.cu, a.batch, a.tokens, 1, rows, slot));
    const int64_t b = clip_cu(a.cu, s, a.tokens), e = clip_cu(a.cu, s + 1, a.tokens);
    const int64_t chunk = (int64_t)slot - (b >> shift) - s;
    const int64_t r0 = b + chunk * rows, r1 = min(e, r0 + rows);
    if (chunk < 0 || (chunk && r0 >= e)) return;  // chunk 0 of an empty sequence writes its zeros
    const uint32_t group = GROUPS == 1 ? 0 : threadIdx.x / (64 * WAVES), i = threadIdx.x % (64 * WAVES);
    const bool tail = a.dim % 8 != 0;
    float acc[1][CH][8] = {};
    for (int64_t row = r0 + group * R; row < r1; row += GROUPS * R) {
        float f[R][CH][8], mean[R], r[R];
#pragma unroll
        for (int k = 0; k < R; k++)
#pragma unroll
            for (int j = 0; j < CH; j++)
                load8<true>((const T *)a.x + min(row + k, r1 - 1) * a.ldx, (j * 64 * WAVES + i) * 8, a.dim, tail, f[k][j]);
        norm_stats<WAVES, CH, R>(a, NORM, i, sums, f, mean, r);
#pragma unroll
        for (int k = 0; k < R; k++)
            if (row + k < r1)
#pragma unroll
                for (int j = 0; j < CH; j++)
#pragma unroll
                    for (int x = 0; x < 8; x++)
                        acc[0][j][x] = fmaf(NORM == 1 ? f[k][j][x] - mean[k] : f[k][j][x], r[k], acc[0][j][x]);
    }
    join_groups<WAVES, CH, GROUPS>(group, i, acc_lds, acc);
    if (group) return;
    if (e - b > rows) {
        float *p = a.part + slot * a.dim;
#pragma unroll
        for (int j = 0; j < CH; j++) {
            const uint32_t at = (j * 64 * WAVES + i) * 8;
            if (at < a.dim) store8(p + at, (int)min(8u, a.dim - at), acc[0][j]);
        }
        return;
    }
    const float inv = e > b ? 1.0f / (float)(e - b) : 0.0f;
#pragma unroll
    for (int j = 0; j < CH; j++)
#pragma unroll
        for (int x = 0; x < 8; x++) acc[0][j][x] *= inv;
    if (e > b) weighted<WAVES, CH, 1>(a, i, acc);
    store_rows<float, WAVES, CH, 1>(a, (float *)a.y + (uint64_t)s * a.ldy, 1, i, sums, acc);
}

// A sequence a workgroup of JOIN waves, of which groups of WAVES take the parts
// in turn.
template <int WAVES, int CH, int JOIN>
__global__ __launch_bounds__(64 * JOIN) void pool_join(NormArgs a, uint32_t first, uint32_t shift) {
    constexpr int GROUPS = JOIN / WAVES;
    __shared__ float acc_lds[GROUPS > 1 ? GROUPS / 2 * CH * 512 * WAVES : 1], lds[RowSums<WAVES, 1>::FLOATS];
    const uint32_t s = first + blockIdx.x;
    const int64_t b = clip_cu(a.cu, s, a.tokens), e = clip_cu(a.cu, s + 1, a.tokens);
    const uint32_t rows = 1u << shift;
    if (e - b <= rows) return;
    const uint32_t group = GROUPS == 1 ? 0 : threadIdx.x / (64 * WAVES), i = threadIdx.x % (64 * WAVES);
    const uint64_t p0 = (b >> shift) + s;
    const uint32_t n = (uint32_t)((e - b + rows - 1) >> shift);
    const bool tail = a.dim % 8 != 0;
    float acc[1][CH][8] = {};
#pragma unroll 8
    for (uint32_t c = group; c < n; c += GROUPS) {
        const float *p = a.part + (p0 + c) * a.dim;
#pragma unroll
        for (int j = 0; j < CH; j++) {
            float f[8];
            load8(p, (j * 64 * WAVES + i) * 8, a.dim, tail, f);
#pragma unroll
            for (int x = 0; x < 8; x++) acc[0][j][x] += f[x];
        }
    }
    join_groups<WAVES, CH, GROUPS>(group, i, acc_lds, acc);
    if (group) return;
    const float inv = 1.0f / (float)(e - b);
#pragma unroll
    for (int j = 0; j < CH; j++)
#pragma unroll
        for (int x = 0; x < 8; x++) acc[0][j][x] *= inv;
    weighted<WAVES, CH, 1>(a, i, acc);
    RowSums<WAVES, 1> sums{lds};
    store_rows<float, WAVES, CH, 1>(a, (float *)a.y + (uint64_t)s * a.ldy, 1, i, sums, acc);
}

// Rows of a chunk, a power of two's exponent: 64 (3000 x 256 rows of 1024: 183
// us, with 32 or 128 more), fewer where that leaves compute units idle (32 x
// 100..500 rows of 768: 16.5 us, with 32 rows 20.6, with 64 28).
uint32_t pool_shift(uint64_t tokens) {
    uint32_t shift = 6;
    while (shift > 4 && tokens > 64 && tokens >> shift < 1024) shift--;
    return shift;
}

template <class T, int WAVES, int CH, int R>
hipError_t pool_of(const NormArgs &a, hipStream_t s) {
    const uint64_t chunks = pool_chunks(a.tokens, a.batch);
    const uint32_t shift = pool_shift(a.tokens);
    for (uint64_t c = 0; c < chunks; c += GRID_MOST) {
        const uint32_t n = (uint32_t)std::min<uint64_t>(chunks - c, GRID_MOST);
        switch (a.norm) {
        case 0: pool_chunk<T, WAVES, CH, R, 0><<<n, BLOCK<WAVES>, 0, s>>>(a, c, shift); break;
        case 1: pool_chunk<T, WAVES, CH, R, 1><<<n, BLOCK<WAVES>, 0, s>>>(a, c, shift); break;
        default: pool_chunk<T, WAVES, CH, R, 2><<<n, BLOCK<WAVES>, 0, s>>>(a, c, shift);
        }
    }
    if (a.tokens >> shift == 0 || a.tokens == 1ull << shift) return hipGetLastError();  // every sequence fits one chunk
    // 16 waves a sequence up to one a compute unit, four (or a row's) for more,
    // most of which have nothing to join: 4096 x 1..16 rows of 768
    // 34.5 us against 39.7
    for (uint64_t b = 0; b < a.batch; b += GRID_MOST) {
        const uint32_t n = (uint32_t)std::min<uint64_t>(a.batch - b, GRID_MOST);
        if (a.batch <= 256) pool_join<WAVES, CH, 16><<<n, 1024, 0, s>>>(a, b, shift);
        else pool_join<WAVES, CH, std::max(WAVES, 4)><<<n, 64 * std::max(WAVES, 4), 0, s>>>(a, b, shift);
    }
    return hipGetLastError();
}
template <class T, class O, int WAVES, int CH, int R>
hipError_t norm_of(const NormArgs &a, hipStream_t s) {
    const uint64_t rows = a.pool ? a.batch : a.tokens;
    constexpr uint64_t each = R * (BLOCK<WAVES> / 64 / WAVES);
    for (uint64_t r = 0; r < rows; r += GRID_MOST * each) {
        const uint64_t blocks = (rows - r + each - 1) / each;
        norm_rows<T, O, WAVES, CH, R><<<(uint32_t)std::min<uint64_t>(blocks, GRID_MOST), BLOCK<WAVES>, 0, s>>>(a, r);
    }
    return hipGetLastError();
}
// A row's waves: one up to 1024 elements, 16 elements a thread at most beyond
// (a wave with 64 a thread fills its registers, one wave a SIMD: 300 x 64 rows of
// 3904, layer norm, mean, 258 us against 60; norm of 40000 x 3901 374 against 173).
template <class T>
hipError_t pool_sized(const NormArgs &a, hipStream_t s) {
    if (a.dim <= 512) return pool_of<T, 1, 1, 2>(a, s);
    if (a.dim <= 1024) return pool_of<T, 1, 2, 1>(a, s);
    if (a.dim <= 2048) return pool_of<T, 4, 1, 2>(a, s);
    if (a.dim <= 4096) return pool_of<T, 4, 2, 2>(a, s);
    if (a.dim <= 8192) return pool_of<T, 16, 1, 2>(a, s);
    return pool_of<T, 16, 2, 1>(a, s);
}
template <class T, class O>
hipError_t norm_sized(const NormArgs &a, hipStream_t s) {
    if (a.dim <= 512) return norm_of<T, O, 1, 1, 2>(a, s);
    if (a.dim <= 1024) return norm_of<T, O, 1, 2, 2>(a, s);
    if (a.dim <= 2048) return norm_of<T, O, 4, 1, 2>(a, s);
    if (a.dim <= 4096) return norm_of<T, O, 4, 2, 2>(a, s);
    if (a.dim <= 8192) return norm_of<T, O, 16, 1, 1>(a, s);
    return norm_of<T, O, 16, 2, 1>(a, s);
}
template <class T>
hipError_t norm_typed(const NormArgs &a, hipStream_t s) {
    if (a.pool == 1) return pool_sized<T>(a, s);
    switch (a.out_dtype) {
    case T_F16: return norm_sized<T, f16>(a, s);
    case T_BF16: return norm_sized<T, bf16>(a, s);
    default: return norm_sized<T, float>(a, s);
    }
}

}  // namespace

hipError_t launch_rotary(const RotaryArgs &a, hipStream_t s) {
    switch (a.dtype) {
    case T_F16: return rotary_of<f16>(a, s);
    case T_BF16: return rotary_of<bf16>(a, s);
    default: return rotary_of<float>(a, s);
    }
}

uint64_t pool_chunks(uint64_t tokens, uint32_t batch) { return (tokens >> pool_shift(tokens)) + batch; }

hipError_t launch_norm(const NormArgs &a, hipStream_t s) {
    switch (a.dtype) {
    case T_F16: return norm_typed<f16>(a, s);
    case T_BF16: return norm_typed<bf16>(a, s);
    default: return norm_typed<float>(a, s);
    }
}

}  // namespace bvk
