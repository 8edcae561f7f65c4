// Softmax attention over packed sequences with grouped heads, on the matrix
// cores.
//
// A sequence's rows are its queries times the heads that share a key head
// (row r: query r / group, head r % group), so that one read of keys and
// values serves all of them.  A workgroup takes a tile of rows and goes over
// the keys once, with the running maximum and sum of the softmax.
//
// Scores are computed transposed, keys as the matrix instructions' first
// operand: a lane then holds scores of one row alone (lane & 31), its maximum
// and sum need one exchange between the wave's halves, and the weights are
// already where the second product, values^T weights^T, takes them.
#include "bv_embed.h"
#include "bv_embed_device.h"
#include "bv_mfma.h"

#include <algorithm>
#include <cmath>

namespace bvk {
namespace {

typedef float v4f __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

__device__ __forceinline__ v16f mfma32(Vec8<f16>::type a, Vec8<f16>::type b, v16f c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ v16f mfma32(Vec8<bf16>::type a, Vec8<bf16>::type b, v16f c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

// What a call's kernels share beside its arguments: the split of the keys and
// where partial results go.
struct AttentionPlan {
    float c;          // |scale| * log2(e): weights are powers of two
    int negate;       // scale < 0: the queries are negated
    uint32_t splits;  // parts of every sequence's keys, each a workgroup's
    float *part_o;    // [split][query][head][d], not yet divided by the sum
    float2 *part_ml;  // [split][query][head]: maximum (log2) and sum
    const void *zeros;  // 16 bytes of zeros that loads past an end read
};

// A tile's place: sequence, rows, keys.
struct Place {
    int64_t qb, kb;      // first query and key of the sequence
    int32_t lq, lk;      // its lengths
    int64_t rows, row0;  // its rows, the tile's first
};
__device__ __forceinline__ bool place_of(const AttentionArgs &a, uint32_t group, uint32_t tile, uint64_t slot, Place &p) {
    const uint32_t s = __builtin_amdgcn_readfirstlane(slot_sequence(a.cu_q, a.batch, a.tq, group, tile, slot));
    p.qb = clip_cu(a.cu_q, s, a.tq);
    p.kb = clip_cu(a.cu_k, s, a.tk);
    p.lq = (int32_t)max((int64_t)0, clip_cu(a.cu_q, s + 1, a.tq) - p.qb);
    p.lk = (int32_t)max((int64_t)0, clip_cu(a.cu_k, s + 1, a.tk) - p.kb);
    const int64_t nth = (int64_t)slot - p.qb * group / tile - s;
    p.rows = (int64_t)p.lq * group;
    p.row0 = nth * tile;
    return nth >= 0 && p.row0 < p.rows;
}
// How many of the sequence's keys a query sees: the first ones.
__device__ __forceinline__ int32_t seen_by(const AttentionArgs &a, const Place &p, int32_t query) {
    return a.causal ? max(0, min(p.lk, p.lk - p.lq + query + 1)) : p.lk;
}

// LDS rows of D elements in 16-byte chunks; chunk c of row r lies at
// c ^ swizzle.  Keys: eight lanes read the same chunk of consecutive rows and
// cover all banks.  Values: sixteen lanes read 32 bytes of four consecutive
// rows (a transposing read), which cover all banks.
template <int D>
__device__ __forceinline__ uint32_t key_swizzle(uint32_t row) {
    return D % 64 == 0 ? row & 7 : (row >> 1) & 3;
}
template <int D>
__device__ __forceinline__ uint32_t value_swizzle(uint32_t row) {
    return D % 64 == 0 ? (row & 3) << 1 : (row >> 1 & 1) << 1;
}

// Eight elements from at on of a row of d, zeros past its end, in the type
// itself; `any`: the row may be read at all.
template <class T>
__device__ __forceinline__ typename Vec8<T>::type raw8(const T *row, uint32_t at, uint32_t d, bool any, const T *zeros) {
    typedef typename Vec8<T>::type V;
    if (d % 8 == 0) {
        const T *p = any && at < d ? row + at : zeros;
        return *(const typename Vec8<T>::unaligned *)p;
    }
    V v;
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = *(any && at + i < d ? row + at + i : zeros);
    return v;
}

__device__ __forceinline__ bool any_not_finite(v4i v, uint32_t exponent) {
    bool bad = false;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t x = (uint32_t)v[i];
        bad |= (x & exponent) == exponent || (x >> 16 & exponent) == exponent;
    }
    return bad;
}
template <class T>
constexpr uint32_t EXPONENT = sizeof(T) && __is_same(T, f16) ? 0x7c00 : 0x7f80;

// One row by one wave, reading only keys that it sees: for the rows of tiles
// in which a value that some rows see and others do not is not finite (it
// would reach those as 0 * inf in a matrix product).
template <class T>
__device__ __forceinline__ void row_alone(const AttentionArgs &a, const AttentionPlan &pl, const Place &p, uint32_t group,
                                       uint32_t hk, int64_t row, int32_t j0, int32_t j1, uint32_t split, float *qs,
                                       float *ps) {
    const uint32_t lane = threadIdx.x & 63;
    const int32_t query = (int32_t)(row / group);
    const int64_t token = p.qb + query, h = hk * group + row % group;
    const T *q = (const T *)a.q + token * a.sq + h * a.sqh;
    for (uint32_t i = lane; i < a.d; i += 64) qs[i] = (float)q[i] * (pl.negate ? -pl.c : pl.c);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    const int32_t all = seen_by(a, p, query), seen = min(all, j1);
    float top = -INFINITY, sum = 0, acc[4] = {};
    for (int32_t j = j0; j < seen; j += 64) {
        float s = -INFINITY;
        if (j + (int32_t)lane < seen) {
            const T *k = (const T *)a.k + (p.kb + j + lane) * a.sk + hk * a.skh;
            float dot = 0;
            for (uint32_t i = 0; i < a.d; i++) dot = fmaf(qs[i], (float)k[i], dot);
            s = dot;
        }
        const float best = fmaxf(top, wave_max(s));
        const float keep = top == best ? 1.0f : exp2f(top - best);
        const float w = j + (int32_t)lane < seen ? exp2f(s - best) : 0.0f;
        top = best;
        sum = sum * keep + wave_sum(w);
        ps[lane] = w;
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        const int n = min(64, seen - j);
#pragma unroll
        for (int c = 0; c < 4; c++) acc[c] *= keep;
        for (int i = 0; i < n; i++) {
            const T *v = (const T *)a.v + (p.kb + j + i) * a.sv + hk * a.svh;
#pragma unroll
            for (int c = 0; c < 4; c++)
                if (c * 64 + lane < a.d) acc[c] = fmaf(ps[i], (float)v[c * 64 + lane], acc[c]);
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
    if (pl.splits > 1) {
        const uint64_t at = ((uint64_t)split * a.tq + token) * a.hq + h;
        if (lane == 0) pl.part_ml[at] = make_float2(top, sum);
        for (int c = 0; c < 4; c++)
            if (c * 64 + lane < a.d) pl.part_o[at * a.d + c * 64 + lane] = acc[c];
    } else {
        T *o = (T *)a.o + token * a.so + h * a.soh;
        for (int c = 0; c < 4; c++)
            if (c * 64 + lane < a.d) o[c * 64 + lane] = (T)(all > 0 ? acc[c] / sum : 0.0f);
    }
}

// QB blocks of 32 rows a wave, four waves; tiles of KT keys and values through
// ST buffers in LDS, loaded straight into it where DIRECT (16-byte aligned rows
// of whole chunks), through registers otherwise.  One barrier a tile: after a
// wave's wait for its share of the oldest tile, and before the loads of the
// next one go where the tile before was.
template <class T, int D, int QB, int KT, int ST, bool DIRECT>
__global__ __launch_bounds__(256, D <= 128 ? 2 : 1) void attention_tile(AttentionArgs a, AttentionPlan pl, uint64_t first) {
    typedef typename Vec8<T>::type V;
    constexpr int CH = D / 8, NL = KT * CH / 256, KB = KT / 32, DB = D / 32;
    constexpr int STAGE = 2 * KT * D * 2;
    constexpr uint32_t ROWS = 128 * QB;
    __shared__ __align__(1024) unsigned char lds[ST * STAGE];
    const uint32_t group = a.hq / a.hk, hk = blockIdx.y, split = blockIdx.z;
    Place p;
    if (!place_of(a, group, ROWS, first + gridDim.x - 1 - blockIdx.x, p)) return;
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t lo = lane & 31, hi = lane >> 5;

    const int64_t row_end = min(p.rows, p.row0 + ROWS);
    const int32_t seen_first = seen_by(a, p, (int32_t)(p.row0 / group));
    const int32_t seen_last = seen_by(a, p, (int32_t)((row_end - 1) / group));
    const int32_t per = ((p.lk + KT - 1) / KT + pl.splits - 1) / pl.splits;
    const int32_t t0 = split * per, t1 = min((seen_last + KT - 1) / KT, t0 + per);

    // this wave's rows
    const int64_t wrow = p.row0 + wave * 32 * QB, wend = min(p.rows, wrow + 32 * QB);
    const bool works = wrow < p.rows;
    const int32_t wave_all = works ? seen_by(a, p, (int32_t)(wrow / group)) : 0;          // every row sees these
    const int32_t wave_any = works ? seen_by(a, p, (int32_t)((wend - 1) / group)) : 0;    // some row sees these
    int32_t seen[QB];
    int64_t token[QB], head[QB];
    V q[QB][D / 16];
    const T *zeros = (const T *)pl.zeros;
#pragma unroll
    for (int b = 0; b < QB; b++) {
        const int64_t row = wrow + b * 32 + lo;
        const bool in = row < p.rows;
        const int32_t query = in ? (int32_t)(row / group) : 0;
        token[b] = p.qb + query;
        head[b] = hk * group + (in ? row - (int64_t)query * group : 0);
        seen[b] = in ? seen_by(a, p, query) : 0;
        const T *src = (const T *)a.q + token[b] * a.sq + head[b] * a.sqh;
#pragma unroll
        for (int i = 0; i < D / 16; i++) {
            q[b][i] = raw8(src, i * 16 + hi * 8, a.d, in, zeros);
            if (pl.negate) q[b][i] = -q[b][i];
        }
    }

    const T *kp = (const T *)a.k + p.kb * a.sk + hk * a.skh, *vp = (const T *)a.v + p.kb * a.sv + hk * a.svh;
    const uint32_t lds0 = lds_addr(lds) + wave * 1024;
    auto load = [&](int32_t t) {
        const uint32_t buf = (uint32_t)(t - t0) % ST * STAGE;
#pragma unroll
        for (int i = 0; i < NL; i++) {
            const uint32_t idx = i * 256 + tid, row = idx / CH, slot = idx % CH;
            const uint32_t kc = (slot ^ key_swizzle<D>(row)) * 8, vc = (slot ^ value_swizzle<D>(row)) * 8;
            const int32_t j = t * KT + row;
            const T *kr = kp + (int64_t)j * a.sk, *vr = vp + (int64_t)j * a.sv;
            const bool in = j < p.lk;
            if (DIRECT) {
                const T *ks = in && kc < a.d ? kr + kc : zeros, *vs = in && vc < a.d ? vr + vc : zeros;
                lds_dma16(ks, __builtin_amdgcn_readfirstlane(lds0 + buf + i * 4096));
                lds_dma16(vs, __builtin_amdgcn_readfirstlane(lds0 + buf + STAGE / 2 + i * 4096));
            } else {
                *(V *)(lds + buf + idx * 16) = raw8(kr, kc, a.d, in, zeros);
                *(V *)(lds + buf + STAGE / 2 + idx * 16) = raw8(vr, vc, a.d, in, zeros);
            }
        }
    };

    v16f o[DB][QB];
    float top[QB], sum[QB];
#pragma unroll
    for (int b = 0; b < QB; b++) {
        top[b] = -INFINITY;
        sum[b] = 0;
#pragma unroll
        for (int d = 0; d < DB; d++)
#pragma unroll
            for (int e = 0; e < 16; e++) o[d][b][e] = 0.0f;
    }
    bool not_finite = false;

#pragma unroll
    for (int s = 0; s < ST - 1; s++)
        if (t0 + s < t1) load(t0 + s);
    for (int32_t t = t0; t < t1; t++) {
        if (DIRECT) {
            if (t + ST - 1 <= t1) __builtin_amdgcn_s_waitcnt(vmcnt_imm((ST - 2) * 2 * NL));
            else __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
        }
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        if (t + ST - 1 < t1) load(t + ST - 1);
        const unsigned char *kbuf = lds + (uint32_t)(t - t0) % ST * STAGE, *vbuf = kbuf + STAGE / 2;
        if (a.causal && (t + 1) * KT > seen_first) {
#pragma unroll
            for (int i = 0; i < NL; i++)
                not_finite |= any_not_finite(*(const v4i *)(vbuf + (i * 256 + tid) * 16), EXPONENT<T>);
        }
        if (t * KT >= wave_any) continue;

        v16f s[KB][QB];
#pragma unroll
        for (int k = 0; k < KB; k++) {
#pragma unroll
            for (int b = 0; b < QB; b++)
#pragma unroll
                for (int e = 0; e < 16; e++) s[k][b][e] = 0.0f;
            const uint32_t r = k * 32 + lo;
#pragma unroll
            for (int i = 0; i < D / 16; i++) {
                const V kv = *(const V *)(kbuf + r * D * 2 + (((i * 2 + hi) ^ key_swizzle<D>(r)) * 16));
#pragma unroll
                for (int b = 0; b < QB; b++) s[k][b] = mfma32(kv, q[b][i], s[k][b]);
            }
        }
        if ((t + 1) * KT > wave_all) {
#pragma unroll
            for (int k = 0; k < KB; k++)
#pragma unroll
                for (int b = 0; b < QB; b++)
#pragma unroll
                    for (int e = 0; e < 16; e++) {
                        const int32_t j = t * KT + k * 32 + e / 4 * 8 + (int)hi * 4 + e % 4;
                        s[k][b][e] = j < seen[b] ? s[k][b][e] : -INFINITY;
                    }
        }
        V w[QB][KT / 16];
#pragma unroll
        for (int b = 0; b < QB; b++) {
            float best = -INFINITY;
#pragma unroll
            for (int k = 0; k < KB; k++)
#pragma unroll
                for (int e = 0; e < 16; e++) best = fmaxf(best, s[k][b][e]);
            best = halves_max(best) * pl.c;
            // The maximum that weights refer to follows when one passes it by
            // 2^8: until then weights stay below 2^8, and nothing is rescaled.
            if (__any(best > top[b] + 8.0f)) {
                const float next = fmaxf(top[b], best);
                const float keep = top[b] == next ? 1.0f : __builtin_amdgcn_exp2f(top[b] - next);
                top[b] = next;
                sum[b] *= keep;
#pragma unroll
                for (int d = 0; d < DB; d++)
#pragma unroll
                    for (int e = 0; e < 16; e++) o[d][b][e] *= keep;
            }
            const float m = top[b] == -INFINITY ? 0.0f : top[b];
#pragma unroll
            for (int k = 0; k < KB; k++)
#pragma unroll
                for (int e = 0; e < 16; e++) {
                    const float x = __builtin_amdgcn_exp2f(fmaf(s[k][b][e], pl.c, -m));
                    sum[b] += x;
                    w[b][k * 2 + e / 8][e % 8] = (T)x;
                }
        }
        // values: 4 keys of 16 elements are read by 16 lanes and come back
        // transposed, lane i with element i of the four keys.  Which eight keys a
        // lane's half of an operand stands for is free as long as both operands
        // agree: keys 4 hi + 0..3 and 8 + 4 hi + 0..3 of sixteen, as the scores lie.
#pragma unroll
        for (int k = 0; k < KT / 16; k++)
#pragma unroll
            for (int d = 0; d < DB; d++) {
                union {
                    s16x4 half[2];
                    V all;
                } v;
#pragma unroll
                for (int x = 0; x < 2; x++) {
                    const uint32_t r = k * 16 + x * 8 + hi * 4 + ((lane & 15) >> 2);
                    const uint32_t e = d * 32 + (lane & 16) + (lane & 3) * 4;
                    const uint32_t at = r * D * 2 + (((e >> 3) ^ value_swizzle<D>(r)) * 16) + (e & 7) * 2;
                    v.half[x] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(vbuf + at));
                }
#pragma unroll
                for (int b = 0; b < QB; b++) o[d][b] = mfma32(v.all, w[b][k], o[d][b]);
            }
    }

    if (__syncthreads_or(not_finite)) {
        float *own = (float *)lds + wave * 320;
        for (int64_t row = wrow; row < wend; row++)
            row_alone<T>(a, pl, p, group, hk, row, t0 * KT, (t0 + per) * KT, split, own, own + 256);
        return;
    }
#pragma unroll
    for (int b = 0; b < QB; b++) {
        const float total = halves_sum(sum[b]);
        if (wrow + b * 32 + lo >= p.rows) continue;
        if (pl.splits > 1) {
            const uint64_t at = ((uint64_t)split * a.tq + token[b]) * a.hq + head[b];
            if (hi == 0) pl.part_ml[at] = make_float2(top[b], total);
            if (t0 >= t1) continue;
            float *out = pl.part_o + at * a.d;
#pragma unroll
            for (int d = 0; d < DB; d++)
#pragma unroll
                for (int e = 0; e < 16; e += 4) {
                    const uint32_t i = d * 32 + e * 2 + hi * 4;
#pragma unroll
                    for (int x = 0; x < 4; x++)
                        if (i + x < a.d) out[i + x] = o[d][b][e + x];
                }
            continue;
        }
        const float r = 1.0f / total;
        T *out = (T *)a.o + token[b] * a.so + head[b] * a.soh;
#pragma unroll
        for (int d = 0; d < DB; d++)
#pragma unroll
            for (int e = 0; e < 16; e += 4) {
                const uint32_t i = d * 32 + e * 2 + hi * 4;
                typedef T V4 __attribute__((ext_vector_type(4)));
                typedef V4 V4U __attribute__((aligned(sizeof(T))));
                V4 f;
#pragma unroll
                for (int x = 0; x < 4; x++) f[x] = (T)(seen[b] > 0 ? o[d][b][e + x] * r : 0.0f);
                if (i + 4 <= a.d) {
                    *(V4U *)(out + i) = f;
                } else {
#pragma unroll
                    for (int x = 0; x < 4; x++)
                        if (i + x < a.d) out[i + x] = f[x];
                }
            }
    }
}

// Joins the parts of a row, a wave each, in their order.
template <class T>
__global__ __launch_bounds__(256) void attention_join(AttentionArgs a, AttentionPlan pl, uint64_t first) {
    const uint32_t group = a.hq / a.hk, lane = threadIdx.x & 63;
    Place p;
    if (!place_of(a, group, 4, first + blockIdx.x, p)) return;
    const int64_t row = p.row0 + (threadIdx.x >> 6);
    if (row >= p.rows) return;
    const int32_t query = (int32_t)(row / group);
    const int64_t token = p.qb + query, h = blockIdx.y * group + row % group;
    const uint64_t at = (uint64_t)token * a.hq + h, step = (uint64_t)a.tq * a.hq;
    float top = -INFINITY;
    for (uint32_t s = lane; s < pl.splits; s += 64) top = fmaxf(top, pl.part_ml[at + s * step].x);
    top = wave_max(top);
    float sum = 0, acc[4] = {};
    for (uint32_t s = 0; s < pl.splits; s++) {
        const float2 ml = pl.part_ml[at + s * step];
        if (ml.x == -INFINITY && ml.y == 0.0f) continue;  // a part with no key
        const float keep = ml.x == top ? 1.0f : exp2f(ml.x - top);
        sum = fmaf(ml.y, keep, sum);
        const float *o = pl.part_o + (at + s * step) * a.d;
#pragma unroll
        for (int c = 0; c < 4; c++)
            if (c * 64 + lane < a.d) acc[c] = fmaf(o[c * 64 + lane], keep, acc[c]);
    }
    T *o = (T *)a.o + token * a.so + h * a.soh;
#pragma unroll
    for (int c = 0; c < 4; c++)
        if (c * 64 + lane < a.d) o[c * 64 + lane] = (T)(seen_by(a, p, query) > 0 ? acc[c] / sum : 0.0f);
}

// The shape of a head dimension's tiles.
template <int D>
struct Shape {
    static constexpr int QB = 1, KT = D <= 128 ? 64 : 32, ST = 2;
};
uint32_t rows_of_tile(uint32_t d) { return 128; }
uint32_t keys_of_tile(uint32_t d) { return d <= 128 ? 64 : 32; }

// Parts of the keys: where tiles of rows alone leave most of the card idle, and
// no more than tiles of keys.
uint32_t splits_of(const AttentionArgs &a) {
    const uint64_t tiles = (a.tq * (a.hq / a.hk) / rows_of_tile(a.d) + a.batch) * a.hk;
    const uint64_t keys = a.max_k ? std::min<uint64_t>(a.max_k, a.tk) : a.tk;
    const uint64_t most = (keys + 4 * keys_of_tile(a.d) - 1) / (4 * keys_of_tile(a.d));
    return (uint32_t)std::max<uint64_t>(1, std::min<uint64_t>({512 / tiles, most, 256}));
}

template <class T, int D, bool DIRECT>
hipError_t attention_sized(const AttentionArgs &a, const AttentionPlan &pl, hipStream_t s) {
    typedef Shape<D> S;
    const uint64_t slots = a.tq * (a.hq / a.hk) / (128 * S::QB) + a.batch;
    for (uint64_t f = 0; f < slots; f += 1u << 23) {
        const dim3 grid((uint32_t)std::min<uint64_t>(slots - f, 1u << 23), a.hk, pl.splits);
        attention_tile<T, D, S::QB, S::KT, S::ST, DIRECT><<<grid, 256, 0, s>>>(a, pl, f);
    }
    if (pl.splits > 1) {
        const uint64_t rows = a.tq * (a.hq / a.hk) / 4 + a.batch;
        for (uint64_t f = 0; f < rows; f += 1u << 23)
            attention_join<T><<<dim3((uint32_t)std::min<uint64_t>(rows - f, 1u << 23), a.hk), 256, 0, s>>>(a, pl, f);
    }
    return hipGetLastError();
}

template <class T>
hipError_t attention_of(const AttentionArgs &a, const AttentionPlan &pl, hipStream_t s) {
    const bool direct = a.d % 8 == 0 && ((uintptr_t)a.k | (uintptr_t)a.v) % 16 == 0 && (a.sk | a.skh | a.sv | a.svh) % 8 == 0;
    if (!direct) {
        if (a.d <= 64) return attention_sized<T, 64, false>(a, pl, s);
        if (a.d <= 128) return attention_sized<T, 128, false>(a, pl, s);
        return attention_sized<T, 256, false>(a, pl, s);
    }
    if (a.d <= 32) return attention_sized<T, 32, true>(a, pl, s);
    if (a.d <= 64) return attention_sized<T, 64, true>(a, pl, s);
    if (a.d <= 96) return attention_sized<T, 96, true>(a, pl, s);
    if (a.d <= 128) return attention_sized<T, 128, true>(a, pl, s);
    return attention_sized<T, 256, true>(a, pl, s);
}

}  // namespace

size_t attention_workspace(const AttentionArgs &a) {
    const uint32_t splits = splits_of(a);
    return splits > 1 ? (size_t)splits * a.tq * a.hq * (a.d + 2) * 4 : 0;
}

hipError_t launch_attention(const AttentionArgs &a, void *ws, hipStream_t s) {
    AttentionPlan pl{};
    pl.c = std::fabs(a.scale) * 1.44269504f;
    pl.negate = a.scale < 0;
    pl.splits = splits_of(a);
    pl.part_ml = (float2 *)ws;
    pl.part_o = (float *)ws + (size_t)pl.splits * a.tq * a.hq * 2;
    pl.zeros = a.zeros;
    return a.dtype == T_F16 ? attention_of<f16>(a, pl, s) : attention_of<bf16>(a, pl, s);
}

}  // namespace bvk
