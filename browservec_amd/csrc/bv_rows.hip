// Row operators of an embedding model: rotary positions, norms, pooling.
#include "bv_embed.h"
#include "bv_embed_device.h"

#include <algorithm>

namespace bvk {
namespace {

// workgroups of a launch: a grid holds fewer than 2^32 threads a dimension, more
// work is launched in pieces
constexpr uint32_t GRID_MOST = 1u << 23;

// ---------------------------------------------------------------- rotary --
// A thread turns (or copies) one unit of a token's heads: eight pairs, whose
// cosines and sines it keeps in registers, of every `groups`-th head.
constexpr uint32_t ROT_HEADS = 4;  // heads per thread

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
// flight together and their reductions interleave.
template <int WAVES>
__device__ __forceinline__ float row_sum(float x, float *lds) {
    x = wave_sum(x);
    if (WAVES == 1) return x;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = x;
    __syncthreads();
    x = 0;
#pragma unroll
    for (int i = 0; i < WAVES; i++) x += lds[i];
    return x;
}

// weights and biases: of any of the three types
__device__ __forceinline__ void load8_of(int type, const void *p, uint32_t at, uint32_t n, bool tail, float (&f)[8]) {
    if (type == T_F32) load8((const float *)p, at, n, tail, f);
    else if (type == T_F16) load8((const f16 *)p, at, n, tail, f);
    else load8((const bf16 *)p, at, n, tail, f);
}

// What the norm does to each row: (f - mean) * r.
template <int WAVES, int CH, int R>
__device__ __forceinline__ void norm_stats(const NormArgs &a, const int norm, uint32_t i, float *lds,
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
#pragma unroll
        for (int k = 0; k < R; k++) mean[k] = row_sum<WAVES>(sum[k], lds) / (float)a.dim;
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
#pragma unroll
        for (int k = 0; k < R; k++) r[k] = 1.0f / sqrtf(row_sum<WAVES>(sq[k], lds) / (float)a.dim + a.eps);
    }
}

// f times the weights plus the biases, zeros past the row's end.
template <int WAVES, int CH, int R>
__device__ __forceinline__ void weighted(const NormArgs &a, uint32_t i, float (&f)[R][CH][8]) {
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

// y = f times 1 / |f| (unit; a zero row stays)
template <class O, int WAVES, int CH>
__device__ __forceinline__ void store_row(const NormArgs &a, O *y, uint32_t i, float *lds, float (&f)[CH][8]) {
    if (a.unit) {
        float sq = 0;
#pragma unroll
        for (int j = 0; j < CH; j++)
#pragma unroll
            for (int e = 0; e < 8; e++) sq = fmaf(f[j][e], f[j][e], sq);
        const float norm = sqrtf(row_sum<WAVES>(sq, lds));
        const float r = norm == 0.0f ? 1.0f : 1.0f / norm;
#pragma unroll
        for (int j = 0; j < CH; j++)
#pragma unroll
            for (int e = 0; e < 8; e++) f[j][e] *= r;
    }
#pragma unroll
    for (int j = 0; j < CH; j++) {
        const uint32_t at = (j * 64 * WAVES + i) * 8;
        if (at < a.dim) store8(y + at, (int)min(8u, a.dim - at), f[j]);
    }
}

// R output rows per WAVES waves: tokens' (no pooling), or the first or last of
// each sequence's.
template <class T, class O, int WAVES, int CH, int R>
__global__ __launch_bounds__(256) void norm_rows(NormArgs a, uint64_t first) {
    __shared__ float lds[4];
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
    norm_stats<WAVES, CH, R>(a, a.norm, i, lds, f, mean, r);
#pragma unroll
    for (int k = 0; k < R; k++)
#pragma unroll
        for (int j = 0; j < CH; j++)
#pragma unroll
            for (int e = 0; e < 8; e++) f[k][j][e] = (f[k][j][e] - mean[k]) * r[k];
    weighted<WAVES, CH, R>(a, i, f);
    if (WAVES > 1) __syncthreads();  // y may be x: every thread has its elements
#pragma unroll
    for (int k = 0; k < R; k++) {
        if (empty[k])
#pragma unroll
            for (int j = 0; j < CH; j++)
#pragma unroll
                for (int e = 0; e < 8; e++) f[k][j][e] = 0.0f;
        if (row0 + k < rows) store_row<O, WAVES, CH>(a, (O *)a.y + (row0 + k) * a.ldy, i, lds, f[k]);
    }
}

// --------------------------------------------------------------- pooling --
// The mean in two launches: a workgroup sums a chunk of POOL_CHUNK rows of one
// sequence (its slot, see slot_sequence), waves taking rows in turn, and
// writes a partial sum, or the result where the sequence has no more rows; a
// second launch joins the partial sums of longer sequences in their order.
// Weights and biases are applied to the mean: they are the same for every row.
constexpr uint32_t POOL_CHUNK = 64;

template <class T, int WAVES, int CH, int NORM>
__global__ __launch_bounds__(256) void pool_chunk(NormArgs a, uint64_t first) {
    constexpr int ROWS = 4 / WAVES;  // waves with rows of their own
    extern __shared__ float acc_lds[];
    __shared__ float lds[4];
    const uint64_t slot = first + blockIdx.x;
    const uint32_t s = __builtin_amdgcn_readfirstlane(slot_sequence(a.cu, a.batch, a.tokens, 1, POOL_CHUNK, slot));
    const int64_t b = clip_cu(a.cu, s, a.tokens), e = clip_cu(a.cu, s + 1, a.tokens);
    const int64_t chunk = (int64_t)slot - b / POOL_CHUNK - s;
    const int64_t r0 = b + chunk * POOL_CHUNK, r1 = min(e, r0 + POOL_CHUNK);
    if (chunk < 0 || (chunk && r0 >= e)) return;  // chunk 0 of an empty sequence writes its zeros
    const uint32_t i = WAVES == 1 ? threadIdx.x & 63 : threadIdx.x, wave = WAVES == 1 ? threadIdx.x >> 6 : 0;
    const bool tail = a.dim % 8 != 0;
    float acc[1][CH][8] = {};
    for (int64_t row = r0 + wave; row < r1; row += ROWS) {
        float f[1][CH][8], mean[1], r[1];
#pragma unroll
        for (int j = 0; j < CH; j++)
            load8<true>((const T *)a.x + row * a.ldx, (j * 64 * WAVES + i) * 8, a.dim, tail, f[0][j]);
        norm_stats<WAVES, CH, 1>(a, NORM, i, lds, f, mean, r);
#pragma unroll
        for (int j = 0; j < CH; j++)
#pragma unroll
            for (int x = 0; x < 8; x++)
                acc[0][j][x] = fmaf(NORM == 1 ? f[0][j][x] - mean[0] : f[0][j][x], r[0], acc[0][j][x]);
    }
    if (ROWS > 1) {  // the waves' sums, by halves
        const uint32_t span = CH * 512;
        for (int h = ROWS / 2; h; h /= 2) {
            if ((int)wave >= h && (int)wave < 2 * h)
#pragma unroll
                for (int j = 0; j < CH; j++)
#pragma unroll
                    for (int x = 0; x < 8; x++) acc_lds[(wave - h) * span + (j * 8 + x) * 64 + i] = acc[0][j][x];
            __syncthreads();
            if ((int)wave < h)
#pragma unroll
                for (int j = 0; j < CH; j++)
#pragma unroll
                    for (int x = 0; x < 8; x++) acc[0][j][x] += acc_lds[wave * span + (j * 8 + x) * 64 + i];
            __syncthreads();
        }
        if (wave) return;
    }
    if (e - b > POOL_CHUNK) {
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
    store_row<float, WAVES, CH>(a, (float *)a.y + (uint64_t)s * a.ldy, i, lds, acc[0]);
}

template <int CH>
__global__ __launch_bounds__(256) void pool_join(NormArgs a, uint32_t first) {
    __shared__ float lds[4];
    const uint32_t s = first + blockIdx.x;
    const int64_t b = clip_cu(a.cu, s, a.tokens), e = clip_cu(a.cu, s + 1, a.tokens);
    if (e - b <= POOL_CHUNK) return;
    const uint32_t i = threadIdx.x;
    const uint64_t p0 = b / POOL_CHUNK + s;
    const uint32_t n = (uint32_t)((e - b + POOL_CHUNK - 1) / POOL_CHUNK);
    float acc[1][CH][8] = {};
    for (uint32_t c = 0; c < n; c++) {
        const float *p = a.part + (p0 + c) * a.dim;
#pragma unroll
        for (int j = 0; j < CH; j++) {
            float f[8];
            load8(p, (j * 256 + i) * 8, a.dim, a.dim % 8 != 0, f);
#pragma unroll
            for (int x = 0; x < 8; x++) acc[0][j][x] += f[x];
        }
    }
    const float inv = 1.0f / (float)(e - b);
#pragma unroll
    for (int j = 0; j < CH; j++)
#pragma unroll
        for (int x = 0; x < 8; x++) acc[0][j][x] *= inv;
    weighted<4, CH, 1>(a, i, acc);
    store_row<float, 4, CH>(a, (float *)a.y + (uint64_t)s * a.ldy, i, lds, acc[0]);
}

template <class T, class O, int WAVES, int CH, int R>
hipError_t norm_of(const NormArgs &a, hipStream_t s) {
    if (a.pool == 1) {
        const uint64_t chunks = pool_chunks(a.tokens, a.batch);
        const size_t lds = WAVES == 1 ? (size_t)2 * CH * 512 * 4 : 0;
        for (uint64_t c = 0; c < chunks; c += GRID_MOST)
            switch (a.norm) {
            case 0: pool_chunk<T, WAVES, CH, 0><<<(uint32_t)std::min<uint64_t>(chunks - c, GRID_MOST), 256, lds, s>>>(a, c); break;
            case 1: pool_chunk<T, WAVES, CH, 1><<<(uint32_t)std::min<uint64_t>(chunks - c, GRID_MOST), 256, lds, s>>>(a, c); break;
            default: pool_chunk<T, WAVES, CH, 2><<<(uint32_t)std::min<uint64_t>(chunks - c, GRID_MOST), 256, lds, s>>>(a, c);
            }
        if (a.tokens <= POOL_CHUNK) return hipGetLastError();  // every sequence fits one chunk
        for (uint64_t b = 0; b < a.batch; b += GRID_MOST) {
            const uint32_t n = (uint32_t)std::min<uint64_t>(a.batch - b, GRID_MOST);
            if (a.dim <= 2048) pool_join<1><<<n, 256, 0, s>>>(a, b);
            else pool_join<8><<<n, 256, 0, s>>>(a, b);
        }
        return hipGetLastError();
    }
    const uint64_t rows = a.pool ? a.batch : a.tokens;
    constexpr uint64_t each = R * (4 / WAVES);
    for (uint64_t r = 0; r < rows; r += GRID_MOST * each) {
        const uint64_t blocks = (rows - r + each - 1) / each;
        norm_rows<T, O, WAVES, CH, R><<<(uint32_t)std::min<uint64_t>(blocks, GRID_MOST), 256, 0, s>>>(a, r);
    }
    return hipGetLastError();
}
template <class T, class O>
hipError_t norm_sized(const NormArgs &a, hipStream_t s) {
    if (a.dim <= 512) return norm_of<T, O, 1, 1, 2>(a, s);
    if (a.dim <= 1024) return norm_of<T, O, 1, 2, 2>(a, s);
    if (a.dim <= 2048) return norm_of<T, O, 1, 4, 2>(a, s);
    if (a.dim <= 4096) return norm_of<T, O, 1, 8, 1>(a, s);
    if (a.dim <= 8192) return norm_of<T, O, 4, 4, 1>(a, s);
    return norm_of<T, O, 4, 8, 1>(a, s);
}
template <class T>
hipError_t norm_typed(const NormArgs &a, hipStream_t s) {
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

uint64_t pool_chunks(uint64_t tokens, uint32_t batch) { return tokens / POOL_CHUNK + batch; }

hipError_t launch_norm(const NormArgs &a, hipStream_t s) {
    switch (a.dtype) {
    case T_F16: return norm_typed<f16>(a, s);
    case T_BF16: return norm_typed<bf16>(a, s);
    default: return norm_typed<float>(a, s);
    }
}

}  // namespace bvk
