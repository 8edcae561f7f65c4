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
    uint32_t splits;  // parts of every sequence's keys, each a workgroup's or wave's
    uint32_t chunk;   // keys of a part, whole tiles; the last part takes the rest
    float *part_o;    // [split][query][head][d], not yet divided by the sum
    float2 *part_ml;  // [split][query][head]: maximum (log2) and sum
    const void *zeros;  // 16 bytes of zeros that loads past an end read
};

// A tile's place: sequence, rows, keys.
struct Place {
    int64_t qb, kb;      // first query and key of the sequence
    int32_t lq, lk;      // its lengths
    int32_t rows, row0;  // its rows, the tile's first (all rows are fewer than 2^31)
};
__device__ __forceinline__ bool place_of(const AttentionArgs &a, uint32_t group, uint32_t tile, uint64_t slot, Place &p) {
    const uint32_t s = __builtin_amdgcn_readfirstlane(slot_sequence(a.cu_q, a.batch, a.tq, group, tile, slot));
    p.qb = clip_cu(a.cu_q, s, a.tq);
    p.kb = clip_cu(a.cu_k, s, a.tk);
    p.lq = (int32_t)max((int64_t)0, clip_cu(a.cu_q, s + 1, a.tq) - p.qb);
    p.lk = (int32_t)max((int64_t)0, clip_cu(a.cu_k, s + 1, a.tk) - p.kb);
    const int64_t nth = (int64_t)slot - (uint32_t)p.qb * group / tile - s;
    p.rows = p.lq * (int32_t)group;
    if (nth < 0 || nth * tile >= p.rows) return false;
    p.row0 = (int32_t)nth * (int32_t)tile;
    return true;
}
// How many of the sequence's keys a query sees: the first ones.
__device__ __forceinline__ int32_t seen_by(const AttentionArgs &a, const Place &p, int32_t query) {
    return a.causal ? max(0, min(p.lk, p.lk - p.lq + query + 1)) : p.lk;
}

// The tiles of KT keys of a part: t0 up to the result.
template <int KT>
__device__ __forceinline__ int32_t part_of(const AttentionPlan &pl, uint32_t split, int32_t keys, int32_t &t0) {
    const int32_t tiles = (keys + KT - 1) / KT, each = pl.chunk / KT;
    t0 = (int32_t)min((int64_t)split * each, (int64_t)tiles);
    return split + 1 == pl.splits ? tiles : min(tiles, t0 + each);
}

// LDS rows of D elements in 16-byte chunks; chunk c of row r lies at
// c ^ swizzle.  LDS serves 256 bytes a cycle.  Keys: sixteen lanes read the same
// chunk of consecutive rows and cover all banks.  Values: 32 lanes read 64
// bytes of four consecutive rows (a transposing read), which cover all banks.
// (Swizzles that covered 128 bytes spent half of LDS's time on conflicts.)
template <int D>
__device__ __forceinline__ uint32_t key_swizzle(uint32_t row) {
    return D % 128 == 0 ? row & 15 : D == 64 ? row >> 1 & 7 : row >> 2 & 3;
}
template <int D>
__device__ __forceinline__ uint32_t value_swizzle(uint32_t row) {
    return D % 128 == 0 ? (row & 3) << 2 : D == 64 ? (row >> 1 & 1) << 2 : 0;
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

// Whether one of eight elements is infinite or NaN: an exponent of ones carries
// into the sign's place.
template <class T>
__device__ __forceinline__ bool any_not_finite(v4i v) {
    constexpr uint32_t EXPONENT = __is_same(T, f16) ? 0x7c007c00u : 0x7f807f80u, ONE = __is_same(T, f16) ? 0x04000400u : 0x00800080u;
    uint32_t bad = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) bad |= ((uint32_t)v[i] & EXPONENT) + ONE;
    return bad & 0x80008000u;
}

// One row by one wave, reading only keys that it sees: for the rows of tiles
// in which a value that some rows see and others do not is not finite (it
// would reach those as 0 * inf in a matrix product).
template <class T>
__device__ __forceinline__ void row_alone(const AttentionArgs &a, const AttentionPlan &pl, const Place &p, uint32_t group,
                                       uint32_t hk, int32_t row, int32_t j0, int32_t j1, uint32_t split, float *qs,
                                       float *ps) {
    const uint32_t lane = threadIdx.x & 63;
    const int32_t query = (uint32_t)row / group;
    const int64_t token = p.qb + query, h = hk * group + (uint32_t)row % group;
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
        const float m = best == -INFINITY ? 0.0f : best;  // keys that score -inf weigh nothing, as in the tiles
        const float w = j + (int32_t)lane < seen ? exp2f(s - m) : 0.0f;
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

// A wave's 32 rows: the result, or a part of it that attention_join takes up
// (any: it saw keys).
template <class T, int D>
__device__ __forceinline__ void store_rows(const AttentionArgs &a, const AttentionPlan &pl, const v16f (&o)[D / 32],
                                           float top, float sum, bool in, int32_t seen, int64_t token, int64_t head,
                                           uint32_t split, bool any) {
    const uint32_t hi = (threadIdx.x & 63) >> 5;
    const float total = halves_sum(sum);
    if (!in) return;
    if (pl.splits > 1) {
        const uint64_t at = ((uint64_t)split * a.tq + token) * a.hq + head;
        if (hi == 0) pl.part_ml[at] = make_float2(top, total);
        if (!any) return;
        float *out = pl.part_o + at * a.d;
#pragma unroll
        for (int d = 0; d < D / 32; d++)
#pragma unroll
            for (int e = 0; e < 16; e += 4) {
                const uint32_t i = d * 32 + e * 2 + hi * 4;
#pragma unroll
                for (int x = 0; x < 4; x++)
                    if (i + x < a.d) out[i + x] = o[d][e + x];
            }
        return;
    }
    const float scale = 1.0f / total;
    T *out = (T *)a.o + token * a.so + head * a.soh;
#pragma unroll
    for (int d = 0; d < D / 32; d++)
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
            const uint32_t i = d * 32 + e * 2 + hi * 4;
            typedef T V4 __attribute__((ext_vector_type(4)));
            typedef V4 V4U __attribute__((aligned(sizeof(T))));
            V4 f;
#pragma unroll
            for (int x = 0; x < 4; x++) f[x] = (T)(seen > 0 ? o[d][e + x] * scale : 0.0f);
            if (i + 4 <= a.d) {
                *(V4U *)(out + i) = f;
            } else {
#pragma unroll
                for (int x = 0; x < 4; x++)
                    if (i + x < a.d) out[i + x] = f[x];
            }
        }
}

// 32 rows a wave; keys and values in tiles of KT, two of each in LDS, loaded
// straight into it where DIRECT (16-byte aligned rows of whole chunks), through
// registers otherwise.
//
// A tile takes a wave two phases: products (the values of the tile before and
// the scores of this one; matrix cores) and softmax (vector unit).
//   GROUPS 1: four waves, phase after phase, one barrier a tile.  What overlaps
//     are the waves of other workgroups; four of them fit a CU up to D = 64.
//   GROUPS 2: eight waves, two a SIMD, of which one multiplies while the other
//     does its softmax, held apart by a barrier a phase.  (Two workgroups of
//     GROUPS 1 that share a CU fall into step, both waves of a SIMD multiplying
//     and then both computing weights: 2300 cycles a tile and wave at D = 128
//     where the products take 1024.)
// At D = 128 (9001 and 16001 tokens, 8 heads over 2, causal, f16: 857 us, 1020
// TFLOP/s; on another card 902) the matrix cores are busy for 53% of the cycles
// and the vector unit, beside issuing to them, for 40%: the counters do not say
// how much of that lies side by side, and so not whether the rest is turns or
// waiting.  At D = 64 (96 x 1..512 tokens, 12 heads over 4: 46 us causal, 58
// without a mask) they are busy for 12 and 38%: what is left is the chain at a
// workgroup's start, offsets, queries and first keys one after the other.
//   Registers spilled by a lane: with turns 2 at D = 128 and 23 at D = 256; where
// not DIRECT 83 at D = 128 and 33 at D = 256.  4 x 4096 tokens, 8 heads, no mask:
// d = 128 335 us, at odd addresses 749; d = 104 331, d = 100, whose elements are
// loaded one by one, 2216; d = 256 1213, at odd addresses 2582.
template <class T, int D, int KT, int GROUPS, bool DIRECT>
__global__ __launch_bounds__(256 * GROUPS, D <= 128 ? 2 : 1) void attention_tile(AttentionArgs a, AttentionPlan pl,
                                                                                 uint64_t first) {
    typedef typename Vec8<T>::type V;
    constexpr int THREADS = 256 * GROUPS, CH = D / 8, CHUNKS = KT * CH, NL = (CHUNKS + THREADS - 1) / THREADS;
    constexpr int KB = KT / 32, DB = D / 32, TILE = KT * D * 2;
    constexpr uint32_t ROWS = 128 * GROUPS;
    __shared__ __align__(1024) unsigned char lds[4 * TILE];  // keys, values, keys, values
    // The last tiles of rows first: with a causal mask they take longest.  Key
    // heads side by side: workgroups that run together spread over them, and
    // where 8 is a multiple of their number, an XCD reads those of one.
    const uint32_t group = a.hq / a.hk, nth = blockIdx.x / a.hk, hk = blockIdx.x - nth * a.hk, split = blockIdx.z;
    Place p;
    const uint32_t slots = gridDim.x / a.hk;
    if (!place_of(a, group, ROWS, first + slots - 1 - spread(nth, slots, a.hk), p)) return;
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t lo = lane & 31, hi = lane >> 5;

    const int32_t row_end = min(p.rows, p.row0 + (int32_t)ROWS);
    const int32_t seen_first = seen_by(a, p, (uint32_t)p.row0 / group);
    const int32_t seen_last = seen_by(a, p, (uint32_t)(row_end - 1) / group);
    int32_t t0;
    const int32_t t1 = part_of<KT>(pl, split, seen_last, t0);

    // this wave's rows, and the tiles that some of them see
    const int32_t wrow = p.row0 + wave * 32, wend = min(p.rows, wrow + 32);
    const int32_t wave_all = wrow < p.rows ? seen_by(a, p, (uint32_t)wrow / group) : 0;
    const int32_t wave_any = wrow < p.rows ? seen_by(a, p, (uint32_t)(wend - 1) / group) : 0;
    const int32_t tw = min(t1, (wave_any + KT - 1) / KT);
    const T *zeros = (const T *)pl.zeros;
    const int32_t row = wrow + lo;
    const bool in = row < p.rows;
    const int32_t query = in ? (uint32_t)row / group : 0;
    const int64_t token = p.qb + query, head = hk * group + (in ? row - query * (int32_t)group : 0);
    const int32_t seen = in ? seen_by(a, p, query) : 0;
    V q[D / 16];
#pragma unroll
    for (int i = 0; i < D / 16; i++) {
        q[i] = raw8((const T *)a.q + token * a.sq + head * a.sqh, i * 16 + hi * 8, a.d, in, zeros);
        if (pl.negate) q[i] = -q[i];
    }

    // A tile of keys or values to a place in LDS.  Rows past the last key repeat
    // it: they get no weight, and a value that is not finite is looked for
    // below.  Elements past d stay the zeros that the buffers begin with.
    const char *kp = (const char *)((const T *)a.k + p.kb * a.sk + hk * a.skh);
    const char *vp = (const char *)((const T *)a.v + p.kb * a.sv + hk * a.svh);
    const uint32_t lds0 = lds_addr(lds) + wave * 1024;
    // Where rows have 4, 8 or 16 chunks, a thread's chunks of a tile lie at the
    // same place of every THREADS / CH-th row.
    constexpr bool REGULAR = THREADS % CH == 0 && CHUNKS % THREADS == 0 && CH <= 16;
    const uint32_t r0 = tid / CH;
    const uint32_t kc = ((tid % CH) ^ key_swizzle<D>(r0)) * 8, vc = ((tid % CH) ^ value_swizzle<D>(r0)) * 8;
    const uint32_t koff = (r0 * (uint32_t)a.sk + kc) * 2, voff = (r0 * (uint32_t)a.sv + vc) * 2;
    auto load = [&](int32_t t, uint32_t to, bool values) {
        const uint64_t step = values ? a.sv : a.sk;
        const char *base = (values ? vp : kp) + (uint64_t)t * KT * step * 2;
        if (DIRECT && REGULAR && (t + 1) * KT <= p.lk) {
            if ((values ? vc : kc) < a.d)
#pragma unroll
                for (int i = 0; i < NL; i++)
                    lds_load16(base + i * (THREADS / CH) * step * 2, values ? voff : koff,
                               __builtin_amdgcn_readfirstlane(lds0 + to + i * THREADS * 16));
            return;
        }
        const uint32_t last = p.lk - 1 - t * KT;
#pragma unroll
        for (int i = 0; i < NL; i++) {
            if (CHUNKS % THREADS && i * THREADS + wave * 64 >= CHUNKS) break;
            const uint32_t idx = i * THREADS + tid, r = idx / CH;
            const uint32_t c = ((idx % CH) ^ (values ? value_swizzle<D>(r) : key_swizzle<D>(r))) * 8;
            const uint32_t from = min(r, last);
            if (DIRECT) {
                if (c < a.d)
                    lds_load16(base, (from * (uint32_t)step + c) * 2,
                               __builtin_amdgcn_readfirstlane(lds0 + to + i * THREADS * 16));
            } else {
                *(V *)(lds + to + idx * 16) = raw8((const T *)base + from * step, c, a.d, true, zeros);
            }
        }
    };
    auto wait_and_meet = [&] {  // this wave's loads have arrived, its reads are done
        if (DIRECT) __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    };
    auto keys_at = [&](int32_t t) { return ((uint32_t)(t - t0) & 1) * 2 * TILE; };

    v16f o[DB], s[KB];
#pragma unroll
    for (int d = 0; d < DB; d++)
#pragma unroll
        for (int e = 0; e < 16; e++) o[d][e] = 0.0f;
    V w[KT / 16];
    float top = -INFINITY, sum = 0;
    bool not_finite = false;

    // Both products read their operands from LDS a batch ahead of the matrix
    // instructions that take them, in an order that the compiler is held to: left
    // to itself it saves the registers and waits for every read.
    //
    // Tile t's weights times its values.  4 keys of 16 elements are read by 16
    // lanes and come back transposed, lane i with element i of the four keys.
    // Which eight keys a lane's half of an operand stands for is free as long as
    // both operands agree: keys 4 hi + 0..3 and 8 + 4 hi + 0..3 of sixteen, as the
    // scores lie.
    const uint32_t vrow = hi * 4 + ((lane & 15) >> 2);
    const uint32_t vat = TILE + vrow * D * 2 + ((((lane & 16) >> 3 | (lane & 2) >> 1) ^ value_swizzle<D>(vrow)) << 4) + (lane & 1) * 8;
    constexpr int VB = DB < 4 ? DB : 4, VBATCHES = KT / 16 * DB / VB;
    auto read_values = [&](uint32_t at, int b, V(&v)[VB]) {
        const int k = b * VB / DB;
#pragma unroll
        for (int i = 0; i < VB; i++) {
            const int d = b * VB % DB + i;
            union {
                s16x4 half[2];
                V all;
            } u;
#pragma unroll
            for (int x = 0; x < 2; x++) {
                const uint32_t from = D % 64 == 0 ? (vat + at) ^ (d * 64) : vat + at + d * 64;
                u.half[x] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(lds + from + (k * 16 + x * 8) * D * 2));
            }
            v[i] = u.all;
        }
    };
    auto weigh_values = [&](int32_t t) {
        const uint32_t at = keys_at(t);
        if ((t + 1) * KT > seen_first) {  // some rows do not see all of these values
#pragma unroll
            for (int i = 0; i < NL; i++)
                if (CHUNKS % THREADS == 0 || i * THREADS + wave * 64 < CHUNKS)
                    not_finite |= any_not_finite<T>(*(const v4i *)(lds + at + TILE + (i * THREADS + tid) * 16));
        }
        if (t >= tw) return;
        V v[2][VB];
        read_values(at, 0, v[0]);
#pragma unroll
        for (int b = 0; b < VBATCHES; b++) {
            if (b + 1 < VBATCHES) read_values(at, b + 1, v[(b + 1) & 1]);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < VB; i++) {
                const int d = b * VB % DB + i;
                o[d] = mfma32(v[b & 1][i], w[b * VB / DB], o[d]);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    // Scores of tile t.  Chunk 2 i + hi of row lo: rows of a power of two of bytes
    // take i * 32 by exclusive or, others (swizzled within four chunks) from two
    // places.
    const uint32_t kat = lo * D * 2 + ((hi ^ key_swizzle<D>(lo)) << 4);
    const uint32_t kat2 = lo * D * 2 + (((2 | hi) ^ key_swizzle<D>(lo)) << 4);
    constexpr int BATCH = 4, BATCHES = KB * (D / 16) / BATCH;
    auto read_keys = [&](uint32_t at, int b, V(&f)[BATCH]) {
#pragma unroll
        for (int x = 0; x < BATCH; x++) {
            const int k = (b * BATCH + x) % KB, i = (b * BATCH + x) / KB;
            const uint32_t from = D == 96 ? (i & 1 ? kat2 : kat) + at + i / 2 * 64 : (kat + at) ^ (i * 32);
            f[x] = *(const V *)(lds + from + k * 32 * D * 2);
        }
    };
    auto scores = [&](int32_t t) {
        if (t >= tw) return;
        const uint32_t at = keys_at(t);
        V f[2][BATCH];
        read_keys(at, 0, f[0]);
#pragma unroll
        for (int k = 0; k < KB; k++)
#pragma unroll
            for (int e = 0; e < 16; e++) s[k][e] = 0.0f;
#pragma unroll
        for (int b = 0; b < BATCHES; b++) {
            if (b + 1 < BATCHES) read_keys(at, b + 1, f[(b + 1) & 1]);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < BATCH; i++) {
                const int k = (b * BATCH + i) % KB;  // neighbours do not wait for each other's sum
                s[k] = mfma32(f[b & 1][i], q[(b * BATCH + i) / KB], s[k]);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    // Scores to weights, after the values of the tiles before.
    auto softmax = [&](int32_t t) {
        if (t >= tw) return;
        if ((t + 1) * KT > wave_all) {
            const int32_t left = seen - t * KT - (int)hi * 4;  // keys that the row sees, from this lane's first
#pragma unroll
            for (int k = 0; k < KB; k++)
#pragma unroll
                for (int e = 0; e < 16; e++) s[k][e] = k * 32 + e / 4 * 8 + e % 4 < left ? s[k][e] : -INFINITY;
        }
        float best = -INFINITY;
#pragma unroll
        for (int k = 0; k < KB; k++)
#pragma unroll
            for (int e = 0; e < 16; e++) best = fmaxf(best, s[k][e]);
        best = halves_max(best) * pl.c;
        // The maximum that weights refer to follows when one passes it by 2^8:
        // until then weights stay below 2^8, and nothing is rescaled.
        if (__any(best > top + 8.0f)) {
            const float now = fmaxf(top, best);
            const float keep = top == now ? 1.0f : __builtin_amdgcn_exp2f(top - now);
            top = now;
            sum *= keep;
#pragma unroll
            for (int d = 0; d < DB; d++)
#pragma unroll
                for (int e = 0; e < 16; e++) o[d][e] *= keep;
        }
        // Weights are rounded to T here, as the second product takes them, while
        // their sum has all bits: rounding errors of up to half a unit in T's last
        // place a weight, averaged over the keys (2.6e-4 of the result's size in
        // f16 against 2.0e-4 with weights of 32 bits, 1.9e-3 against 1.6e-3 in bf16).
        const float m = top == -INFINITY ? 0.0f : top;
#pragma unroll
        for (int k = 0; k < KB; k++)
#pragma unroll
            for (int e = 0; e < 16; e++) {
                const float x = __builtin_amdgcn_exp2f(fmaf(s[k][e], pl.c, -m));
                sum += x;
                w[k * 2 + e / 8][e % 8] = (T)x;
            }
        if (GROUPS == 2)
#pragma unroll
            for (int k = 0; k < KT / 16; k++) asm volatile("" : "+v"(w[k]));  // in this phase
    };

    if (t0 < t1) {
        if (DIRECT && a.d < D) {  // what lies past d
            for (uint32_t i = tid; i < 4 * TILE / 16; i += THREADS) *(v4i *)(lds + i * 16) = v4i{0, 0, 0, 0};
            __syncthreads();
        }
        load(t0, 0, false);
    }
    if (GROUPS == 1) {
        if (t0 < t1) load(t0, TILE, true);
        for (int32_t t = t0; t < t1; t++) {
            wait_and_meet();
            if (t + 1 < t1) {
                load(t + 1, keys_at(t + 1), false);
                load(t + 1, keys_at(t + 1) + TILE, true);
            }
            scores(t);
            softmax(t);
            weigh_values(t);
        }
    } else if (t0 < t1) {
        // Phase 2 (t - t0) + g: group g multiplies for tile t, the next phase is its
        // softmax.  At even phases everyone starts the loads of the next tile's
        // keys and this one's values, which are waited for two phases later.
        const uint32_t g = wave >> 2;
        auto load_next = [&](int32_t t) {
            if (t + 1 < t1) load(t + 1, keys_at(t + 1), false);
            if (t < t1) load(t, keys_at(t) + TILE, true);
        };
        if (g) {
            wait_and_meet();
            load_next(t0);
        }
        for (int32_t t = t0; t <= t1; t++) {
            if (g) {
                asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
            } else {
                wait_and_meet();
                load_next(t);
            }
            if (t > t0) weigh_values(t - 1);
            scores(t);
            if (g) {
                wait_and_meet();
                load_next(t + 1);
            } else {
                asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
            }
            softmax(t);
        }
        if (!g) asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    }

    if (__syncthreads_or(not_finite)) {
        float *own = (float *)lds + wave * 320;
        for (int32_t i = wrow; i < wend; i++)
            row_alone<T>(a, pl, p, group, hk, i, t0 * KT, t1 * KT, split, own, own + 256);
        return;
    }
    store_rows<T, D>(a, pl, o, top, sum, in, seen, token, head, split, t0 < t1);
}

// Few rows a sequence (the next tokens over kept keys): what counts is to
// stream keys and values.  Each wave works alone: 32 rows of one key head over
// its part of the keys, 32 at a time through two tiles of its own in LDS, one on
// its way; no barriers.  Neighbouring waves take the key heads side by side in
// memory.  Bound by the read of keys and values and the start of their chain:
// 8 sequences of up to 32768 keys, 4 key heads of 64, one new token each: 25 us, and
// 6 to join.
template <class T, int D>
__global__ __launch_bounds__(256, 1) void attention_few(AttentionArgs a, AttentionPlan pl, uint64_t first, uint64_t units) {
    typedef typename Vec8<T>::type V;
    constexpr int KT = 32, CH = D / 8, NL = KT * CH / 64, DB = D / 32, TILE = KT * D * 2, ST = 2;
    __shared__ __align__(1024) unsigned char all_lds[4 * ST * 2 * TILE];
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t lo = lane & 31, hi = lane >> 5;
    unsigned char *lds = all_lds + wave * ST * 2 * TILE;
    // unit: key head, then part of the keys, then tile of rows
    const uint64_t unit = first + (uint64_t)blockIdx.x * 4 + wave;
    if (unit >= units) return;
    const uint32_t group = a.hq / a.hk, hk = (uint32_t)(unit % a.hk), split = (uint32_t)(unit / a.hk % pl.splits);
    Place p;
    if (!place_of(a, group, 32, unit / a.hk / pl.splits, p)) return;
    const int32_t row = p.row0 + lo, wend = min(p.rows, p.row0 + 32);
    const int32_t all = seen_by(a, p, (uint32_t)p.row0 / group), any = seen_by(a, p, (uint32_t)(wend - 1) / group);
    int32_t t0;
    const int32_t t1 = part_of<KT>(pl, split, any, t0);
    const bool in = row < p.rows;
    const int32_t query = in ? (uint32_t)row / group : 0;
    const int64_t token = p.qb + query, head = hk * group + (in ? row - query * (int32_t)group : 0);
    const int32_t seen = in ? seen_by(a, p, query) : 0;
    V q[D / 16];
#pragma unroll
    for (int i = 0; i < D / 16; i++) {
        q[i] = raw8((const T *)a.q + token * a.sq + head * a.sqh, i * 16 + hi * 8, a.d, in, (const T *)pl.zeros);
        if (pl.negate) q[i] = -q[i];
    }
    const char *kp = (const char *)((const T *)a.k + p.kb * a.sk + hk * a.skh);
    const char *vp = (const char *)((const T *)a.v + p.kb * a.sv + hk * a.svh);
    const uint32_t lds0 = lds_addr(lds);
    auto load = [&](int32_t t) {
        const uint32_t to = lds0 + (uint32_t)(t - t0) % ST * 2 * TILE;
        const char *kb = kp + (uint64_t)t * KT * a.sk * 2, *vb = vp + (uint64_t)t * KT * a.sv * 2;
        const uint32_t last = p.lk - 1 - t * KT;
#pragma unroll
        for (int i = 0; i < NL; i++) {
            const uint32_t idx = i * 64 + lane, r = idx / CH, from = min(r, last);
            const uint32_t kc = ((idx % CH) ^ key_swizzle<D>(r)) * 8, vc = ((idx % CH) ^ value_swizzle<D>(r)) * 8;
            if (kc < a.d)
                lds_load16(kb, (from * (uint32_t)a.sk + kc) * 2, __builtin_amdgcn_readfirstlane(to + i * 1024));
            if (vc < a.d)
                lds_load16(vb, (from * (uint32_t)a.sv + vc) * 2, __builtin_amdgcn_readfirstlane(to + TILE + i * 1024));
        }
    };
    v16f o[DB];
#pragma unroll
    for (int d = 0; d < DB; d++)
#pragma unroll
        for (int e = 0; e < 16; e++) o[d][e] = 0.0f;
    float top = -INFINITY, sum = 0;
    bool not_finite = false;
    const uint32_t vrow = hi * 4 + ((lane & 15) >> 2);
    const uint32_t kat = lo * D * 2, vat = TILE + vrow * D * 2 + (lane & 1) * 8;
    if (a.d < D) {  // what lies past d
        for (uint32_t i = lane; i < ST * 2 * TILE / 16; i += 64) *(v4i *)(lds + i * 16) = v4i{0, 0, 0, 0};
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
#pragma unroll
    for (int i = 0; i < ST - 1; i++)
        if (t0 + i < t1) load(t0 + i);
    for (int32_t t = t0; t < t1; t++) {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the reads of the tile that the load replaces
        if (t + ST - 1 < t1) {
            load(t + ST - 1);
            __builtin_amdgcn_s_waitcnt(vmcnt_imm((ST - 1) * 2 * NL));
        } else {
            __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
        }
        asm volatile("" ::: "memory");
        const unsigned char *buf = lds + (uint32_t)(t - t0) % ST * 2 * TILE;
        if ((t + 1) * KT > all) {
#pragma unroll
            for (int i = 0; i < NL; i++)
                not_finite |= any_not_finite<T>(*(const v4i *)(buf + TILE + (i * 64 + lane) * 16));
        }
        v16f s;
#pragma unroll
        for (int e = 0; e < 16; e++) s[e] = 0.0f;
        V f[D / 16];
#pragma unroll
        for (int i = 0; i < D / 16; i++) f[i] = *(const V *)(buf + kat + (((i * 2 + hi) ^ key_swizzle<D>(lo)) << 4));
#pragma unroll
        for (int i = 0; i < D / 16; i++) s = mfma32(f[i], q[i], s);
        if ((t + 1) * KT > all) {
            const int32_t left = seen - t * KT - (int)hi * 4;
#pragma unroll
            for (int e = 0; e < 16; e++) s[e] = e / 4 * 8 + e % 4 < left ? s[e] : -INFINITY;
        }
        float best = -INFINITY;
#pragma unroll
        for (int e = 0; e < 16; e++) best = fmaxf(best, s[e]);
        best = halves_max(best) * pl.c;
        if (__any(best > top + 8.0f)) {
            const float now = fmaxf(top, best);
            const float keep = top == now ? 1.0f : __builtin_amdgcn_exp2f(top - now);
            top = now;
            sum *= keep;
#pragma unroll
            for (int d = 0; d < DB; d++)
#pragma unroll
                for (int e = 0; e < 16; e++) o[d][e] *= keep;
        }
        const float m = top == -INFINITY ? 0.0f : top;
        V w[2];  // rounded to T, as in attention_tile (bf16: 2.3e-3 against 1.6e-3)
#pragma unroll
        for (int e = 0; e < 16; e++) {
            const float x = __builtin_amdgcn_exp2f(fmaf(s[e], pl.c, -m));
            sum += x;
            w[e / 8][e % 8] = (T)x;
        }
#pragma unroll
        for (int k = 0; k < 2; k++)
#pragma unroll
            for (int d = 0; d < DB; d++) {
                union {
                    s16x4 half[2];
                    V v;
                } u;
#pragma unroll
                for (int x = 0; x < 2; x++) {
                    const uint32_t c = (d * 4 + ((lane & 16) >> 3 | (lane & 2) >> 1)) ^ value_swizzle<D>(vrow);
                    u.half[x] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                        (lds_s16x4 *)(buf + vat + (c << 4) + (k * 16 + x * 8) * D * 2));
                }
                o[d] = mfma32(u.v, w[k], o[d]);
            }
    }
    if (__any(not_finite)) {
        float *own = (float *)lds;
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        for (int32_t i = p.row0; i < wend; i++)
            row_alone<T>(a, pl, p, group, hk, i, t0 * KT, t1 * KT, split, own, own + 256);
        return;
    }
    store_rows<T, D>(a, pl, o, top, sum, in, seen, token, head, split, t0 < t1);
}

// Joins the parts of a row, a workgroup each: a wave takes every fourth part.
constexpr uint32_t MAX_SPLITS = 128;
template <class T>
__global__ __launch_bounds__(256) void attention_join(AttentionArgs a, AttentionPlan pl, uint64_t first) {
    __shared__ float part[4][256];
    const uint32_t group = a.hq / a.hk, lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    Place p;
    if (!place_of(a, group, 1, first + blockIdx.x, p)) return;
    const int32_t query = (uint32_t)p.row0 / group;
    const int64_t token = p.qb + query, h = blockIdx.y * group + (uint32_t)p.row0 % group;
    const uint64_t at = (uint64_t)token * a.hq + h, step = (uint64_t)a.tq * a.hq;
    // lane s holds part s (and 64 + s)
    constexpr int MANY = MAX_SPLITS / 64;
    float2 ml[MANY];
    float top = -INFINITY, sum = 0, acc[4] = {};
#pragma unroll
    for (int i = 0; i < MANY; i++) {
        const uint32_t s = i * 64 + lane;
        ml[i] = s < pl.splits ? pl.part_ml[at + s * step] : make_float2(-INFINITY, 0.0f);
        top = fmaxf(top, ml[i].x);
    }
    top = wave_max(top);
#pragma unroll
    for (int i = 0; i < MANY; i++) {
        // a part with no key weighs nothing, and what its place holds is not used
        const float keep = ml[i].x == top ? 1.0f : exp2f(ml[i].x - top);
        ml[i].x = ml[i].x == -INFINITY && ml[i].y == 0.0f ? 0.0f : keep;
        sum += ml[i].x * ml[i].y;
    }
    sum = wave_sum(sum);
    for (uint32_t s0 = wave; s0 < pl.splits; s0 += 32) {  // eight parts' loads in flight
        float x[8][4], keep[8];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const uint32_t s = min(s0 + i * 4, pl.splits - 1);
            keep[i] = __shfl(s < 64 ? ml[0].x : ml[1].x, s & 63);
            keep[i] = s0 + i * 4 < pl.splits ? keep[i] : 0.0f;
#pragma unroll
            for (int c = 0; c < 4; c++)
                if (c * 64 < a.d) x[i][c] = pl.part_o[(at + s * step) * a.d + min(c * 64 + lane, a.d - 1)];
        }
#pragma unroll
        for (int i = 0; i < 8; i++)
#pragma unroll
            for (int c = 0; c < 4; c++)
                if (c * 64 < a.d) acc[c] += keep[i] == 0.0f ? 0.0f : x[i][c] * keep[i];
    }
#pragma unroll
    for (int c = 0; c < 4; c++) part[wave][c * 64 + lane] = acc[c];
    __syncthreads();
    const uint32_t i = threadIdx.x;
    if (i >= a.d) return;
    const float o = part[0][i] + part[1][i] + part[2][i] + part[3][i];
    ((T *)a.o)[token * a.so + h * a.soh + i] = (T)(seen_by(a, p, query) > 0 ? o / sum : 0.0f);
}

// Waves that are wanted: as many as the card holds at D = 128 (four a CU, one
// round of 16 x 8192..16384 keys 51 us, two 56).
constexpr uint64_t FEW_WAVES = 1024;

// Keys of a tile: what two of keys and two of values leave of LDS and what a
// wave's scores leave of its registers.  With turns between products and softmax
// 128 keys a phase beat 64 by 3 to 5% (D = 128).
constexpr uint32_t tile_keys(uint32_t d, uint32_t groups = 1) { return d > 128 ? 32 : groups == 2 && d >= 96 ? 128 : 64; }

// Rows of whole chunks at 16-byte addresses, near enough for 32-bit offsets.
bool direct(const AttentionArgs &a) {
    return a.d % 8 == 0 && std::max(a.sk, a.sv) < (1u << 24) && ((uintptr_t)a.k | (uintptr_t)a.v) % 16 == 0 &&
           (a.sk | a.skh | a.sv | a.svh) % 8 == 0;
}
// Whether a sequence's rows fit 32, as far as the caller says, or on average.
bool few_rows(const AttentionArgs &a) {
    const uint64_t queries = a.max_q ? a.max_q : (a.tq + a.batch - 1) / a.batch;
    return queries * (a.hq / a.hk) <= 32 && a.d <= 128 && direct(a);
}

// Bytes of the partial results of one part of the keys.
size_t part_bytes(const AttentionArgs &a) { return a.tq * a.hq * (a.d + 2) * 4; }

// Parts of the keys, where tiles of rows alone leave most of the card idle:
// chunks of one length over all sequences, so that each part is as much work,
// as long as `wanted` workgroups or waves need for all of them.
uint32_t splits_of(const AttentionArgs &a, uint32_t *chunk) {
    const bool few = few_rows(a);
    const uint64_t rows = a.tq * (a.hq / a.hk) / (few ? 32 : 128) + a.batch, wanted = few ? FEW_WAVES : 512;
    const uint64_t keys = a.max_k ? std::min<uint64_t>(a.max_k, a.tk) : a.tk;
    *chunk = 0;
    if (wanted / (rows * a.hk) < (few ? 4 : 2)) return 1;  // (few: joining costs what it saves)
    auto up = [](uint64_t x) { return (x + 127) / 128 * 128; };  // whole tiles, and not less than one of any kernel
    uint64_t c = up(a.tk * (rows / a.batch) * a.hk / wanted);
    c = std::max<uint64_t>({c, few ? 128u : 256u, up((keys + MAX_SPLITS - 1) / MAX_SPLITS)});
    *chunk = (uint32_t)std::min<uint64_t>(c, 1u << 30);
    uint64_t parts = std::max<uint64_t>(1, (keys + c - 1) / c);
    // Where the longest length is not known, any sequence might have all keys, but
    // most parts hold none where there are many sequences: as many as 256 MB of
    // partial results are, or twice a sequence's share of the keys takes (64 x 12
    // queries of 32 heads of 256, 600 keys each: 254 MB instead of 2.5 GB).  A
    // sequence's last part takes what is left.
    if (!a.max_k && a.batch > 1) {
        const uint64_t part = part_bytes(a), share = (2 * a.tk / a.batch + c) / c;
        parts = std::min(parts, std::max(share, (256u << 20) / part));
    }
    return (uint32_t)parts;
}

template <class T, int D, int GROUPS, bool DIRECT>
void launch_tiles(const AttentionArgs &a, const AttentionPlan &pl, hipStream_t s) {
    const uint64_t slots = a.tq * (a.hq / a.hk) / (128 * GROUPS) + a.batch;
    const uint64_t most = std::max<uint64_t>(1, (1u << 22) / a.hk);  // a grid's dimension holds fewer than 2^32 threads
    for (uint64_t f = 0; f < slots; f += most) {
        const dim3 grid((uint32_t)std::min<uint64_t>(slots - f, most) * a.hk, 1, pl.splits);
        attention_tile<T, D, tile_keys(D, GROUPS), GROUPS, DIRECT><<<grid, 256 * GROUPS, 0, s>>>(a, pl, f);
    }
}

template <class T, int D, bool DIRECT>
hipError_t attention_sized(const AttentionArgs &a, const AttentionPlan &pl, hipStream_t s) {
    // Turns pay where the products are as long as the softmax (D >= 96) and the
    // larger tiles of rows still fill the card: 16384 x 8 x 128 966 us against
    // 1028, D = 96 393 against 434, but D = 64 1250 against 1158.
    if (DIRECT && D <= 128 && few_rows(a)) {
        const uint64_t units = (a.tq * (a.hq / a.hk) / 32 + a.batch) * a.hk * pl.splits;
        for (uint64_t f = 0; f < units; f += 4u << 23)
            attention_few<T, D <= 128 ? D : 128><<<(uint32_t)std::min<uint64_t>((units - f + 3) / 4, 1u << 23), 256, 0, s>>>(a, pl, f, units);
    } else if (DIRECT && D >= 96 && a.tq * (a.hq / a.hk) / 256 * a.hk >= 256)
        launch_tiles<T, D, DIRECT && D >= 96 ? 2 : 1, DIRECT>(a, pl, s);
    else launch_tiles<T, D, 1, DIRECT>(a, pl, s);
    if (pl.splits > 1) {
        const uint64_t rows = a.tq * (a.hq / a.hk) + a.batch;
        for (uint64_t f = 0; f < rows; f += 1u << 23)
            attention_join<T><<<dim3((uint32_t)std::min<uint64_t>(rows - f, 1u << 23), a.hk), 256, 0, s>>>(a, pl, f);
    }
    return hipGetLastError();
}

template <class T>
hipError_t attention_of(const AttentionArgs &a, const AttentionPlan &pl, hipStream_t s) {
    if (!direct(a)) {
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
    uint32_t chunk;
    const uint32_t splits = splits_of(a, &chunk);
    return splits > 1 ? splits * part_bytes(a) : 0;
}

hipError_t launch_attention(const AttentionArgs &a, void *ws, hipStream_t s) {
    AttentionPlan pl{};
    pl.c = std::fabs(a.scale) * 1.44269504f;
    pl.negate = a.scale < 0;
    pl.splits = splits_of(a, &pl.chunk);
    pl.part_ml = (float2 *)ws;
    pl.part_o = (float *)ws + (size_t)pl.splits * a.tq * a.hq * 2;
    pl.zeros = a.zeros;
    return a.dtype == T_F16 ? attention_of<f16>(a, pl, s) : attention_of<bf16>(a, pl, s);
}

}  // namespace bvk
