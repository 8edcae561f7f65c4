// Attention over a window of keys about a query's place and a few first keys: the
// kernels of bv_attention_device.h, and one for windows whose scores a wave holds
// at once.
#include "bv_attention_device.h"

namespace bvk {
namespace {

// ---------------------------------------------------------- short windows --
// Four waves of 32 rows.  The keys that their 128 rows see are loaded into LDS at
// once, and when every wave has its scores, up to NT tiles of 32 keys, all of them
// in its registers, the values take the keys' place while the softmax is computed:
// three waits for memory (offsets; queries and keys; values) and none a tile, no
// running maximum, no rescaling.  A wave's tiles begin at its own first key, so that
// it computes no more of the neighbours' keys than fill its last one.
//   Bound by the waits and HBM: 6 x 4001..8192 tokens, 12 heads of 64, 64 on both sides, 57
// us, 3.8 TB/s of 5.1 that a copy reaches (vector unit busy for 42% of the cycles, matrix
// cores for 11; attention_tile 79).  Four workgroups a CU: with keys and values in LDS side by side
// there are two, 71; weights made tile by tile, which saves registers, 63.
// FIRSTS: the sequence's first keys are a tile of their own, in which keys of the window
// do not count.  They lie in LDS before the window's, as many rows as `sinks` and a
// wave's whole loads of 1024 bytes take; the tile's other rows are the window's, without
// weight.
template <int D>
constexpr uint32_t whole_rows(uint32_t n) {
    constexpr uint32_t of = D == 128 ? 4 : D == 64 ? 8 : 16;
    return (n + of - 1) / of * of;
}
template <class T, int D, int NT, bool FIRSTS>
__global__ __launch_bounds__(256, NT <= 5 && D <= 64 ? 4 : 2) void attention_window(AttentionArgs a, AttentionPlan pl, uint64_t first,
                                                                          uint32_t slots, uint32_t lds_rows) {
    typedef typename Vec8<T>::type V;
    constexpr int CH = D / 8, FR = D / 16, DB = D / 32, ALL = NT + FIRSTS;
    extern __shared__ __align__(1024) unsigned char lds[];
    // An XCD takes neighbouring tiles of a head, which share most of their keys.
    const uint32_t group = a.hq / a.hk, all = slots * a.hk, xcd = blockIdx.x & 7, per = (all + 7) / 8;
    const uint32_t id = xcd * per + (blockIdx.x >> 3);
    if ((blockIdx.x >> 3) >= per || id >= all) return;
    const uint32_t hk = id / slots;
    Place p;
    if (!place_of(a, group, 128, first + (id - hk * slots), p)) return;
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t lo = lane & 31, hi = lane >> 5;
    const int32_t row_end = min(p.rows, p.row0 + 128);
    const View from = view_of(a, p, (uint32_t)p.row0 / group), to = view_of(a, p, (uint32_t)(row_end - 1) / group);
    const int32_t wrow = p.row0 + wave * 32, wend = min(p.rows, wrow + 32);
    const bool work = wrow < p.rows;
    const View wfrom = work ? view_of(a, p, (uint32_t)wrow / group) : View{to.hi, to.hi, 0};
    const View wto = work ? view_of(a, p, (uint32_t)(wend - 1) / group) : View{to.hi, to.hi, 0};
    const int32_t row = wrow + lo;
    const bool in = row < p.rows;
    const int32_t query = in ? (uint32_t)row / group : 0;
    const int64_t token = p.qb + query, head = hk * group + (in ? row - query * (int32_t)group : 0);
    const View view = in ? view_of(a, p, query) : View{0, 0, 0};
    const T *zeros = (const T *)pl.zeros;
    V q[FR];
#pragma unroll
    for (int i = 0; i < FR; i++) {
        q[i] = raw8((const T *)a.q + token * a.sq + head * a.sqh, i * 16 + hi * 8, a.d, in, zeros);
        if (pl.negate) q[i] = -q[i];
    }
    // LDS row first_rows + r is key from.lo + r.  Rows past the last key repeat it: they
    // get no weight, and a value that is not finite is found in the results.
    const char *kp = (const char *)((const T *)a.k + p.kb * a.sk + hk * a.skh);
    const char *vp = (const char *)((const T *)a.v + p.kb * a.sv + hk * a.svh);
    const uint32_t lds0 = lds_addr(lds) + wave * 1024;
    const int32_t first_rows = FIRSTS ? whole_rows<D>(a.sinks) : 0;
    const int32_t rows = min((int32_t)lds_rows - first_rows, (to.hi - from.lo + 31 + 31) & ~31);  // loaded: what the waves' tiles reach
    // Where rows have 4, 8 or 16 chunks a thread's chunks lie at the same place of
    // every PASS-th row, whose swizzle is the same.
    constexpr int PASS = 256 / CH;
    constexpr bool REGULAR = 256 % CH == 0;
    auto load_rows = [&](const char *base, uint64_t step, bool values, int32_t k0, int32_t rows, uint32_t row0) {
        const int32_t chunks = rows * CH;
        const uint32_t to = row0 * D * 2, r0 = tid / CH;
        const uint32_t c0 = ((tid % CH) ^ (values ? value_swizzle<D>(row0 + r0) : key_swizzle<D>(row0 + r0))) * 8;
        const uint32_t off = (r0 * (uint32_t)step + c0) * 2;
        const char *at = base + (uint64_t)k0 * step * 2;
        for (int32_t i = 0; i < chunks; i += 256) {
            if (i + (int32_t)wave * 64 >= chunks) break;
            const uint32_t into = __builtin_amdgcn_readfirstlane(lds0 + to + i * 16);
            if (REGULAR && k0 + PASS <= p.lk) {
                if (c0 < a.d) lds_load16(at, off, into);
            } else {
                const uint32_t idx = i + tid, r = idx / CH;
                const uint32_t c = REGULAR ? c0 : ((idx % CH) ^ (values ? value_swizzle<D>(row0 + r) : key_swizzle<D>(row0 + r))) * 8;
                const uint64_t key = (uint32_t)min(REGULAR ? k0 + (int32_t)r0 : k0 + (int32_t)r, p.lk - 1);
                if (c < a.d) lds_dma16(base + (key * step + c) * 2, into);
            }
            if (REGULAR) {
                k0 += PASS;
                at += PASS * step * 2;
            }
        }
    };
    auto load = [&](const char *base, uint64_t step, bool values) {
        if (to.hi > from.lo || (FIRSTS && to.first > 0)) load_rows(base, step, values, from.lo, rows, first_rows);
        if (FIRSTS && to.first > 0) load_rows(base, step, values, 0, first_rows, 0);
    };
    if (a.d < D) {  // what lies past d
        for (uint32_t i = tid; i < lds_rows * CH; i += 256) *(v4i *)(lds + i * 16) = v4i{0, 0, 0, 0};
        __syncthreads();
    }
    load(kp, a.sk, false);
    const int32_t w0 = wfrom.lo - from.lo;                   // the wave's first LDS row
    const int32_t nt = min(NT, (wto.hi - wfrom.lo + 31) / 32);  // its tiles of the window
    __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");

    // Scores, tile after tile; other waves multiply while this one reads.
    v16f s[ALL];
    V f[FR];
    const bool firsts = FIRSTS && wto.first > 0;
    auto any = [&](int t) { return t < NT ? t < nt : firsts; };
    auto lds_row = [&](int t) { return (uint32_t)(t < NT ? first_rows + w0 + t * 32 : 0); };
    auto read_keys = [&](int t, V(&f)[FR]) {
        const uint32_t r = lds_row(t) + lo;
        const uint32_t at = r * D * 2, sw = key_swizzle<D>(r);
#pragma unroll
        for (int i = 0; i < FR; i++) f[i] = *(const V *)(lds + at + (((i * 2 + hi) ^ sw) << 4));
    };
#pragma unroll
    for (int t = 0; t < ALL; t++)
        if (any(t)) {
            read_keys(t, f);
#pragma unroll
            for (int e = 0; e < 16; e++) s[t][e] = 0.0f;
#pragma unroll
            for (int i = 0; i < FR; i++) s[t] = mfma32(f[i], q[i], s[t]);
        }
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    load(vp, a.sv, true);

    // -inf for what the row does not see, the maximum, weights
    float best = -INFINITY;
#pragma unroll
    for (int t = 0; t < ALL; t++) {
        if (!any(t)) continue;
        const int32_t k0 = t < NT ? wfrom.lo + t * 32 : 0;
        const int32_t begin = view.lo - k0 - (int)hi * 4, end = view.hi - k0 - (int)hi * 4;
        if (t == NT) {
            const int32_t count = view.first - (int)hi * 4;
#pragma unroll
            for (int e = 0; e < 16; e++) {
                const int at = e / 4 * 8 + e % 4;
                s[t][e] = at < count && (at < begin || at >= end) ? s[t][e] : -INFINITY;
            }
        } else {
            if (k0 < wto.lo)
#pragma unroll
                for (int e = 0; e < 16; e++) s[t][e] = e / 4 * 8 + e % 4 >= begin ? s[t][e] : -INFINITY;
            if (k0 + 32 > wfrom.hi)
#pragma unroll
                for (int e = 0; e < 16; e++) s[t][e] = e / 4 * 8 + e % 4 < end ? s[t][e] : -INFINITY;
        }
#pragma unroll
        for (int e = 0; e < 16; e++) best = fmaxf(best, s[t][e]);
    }
    best = halves_max(best) * pl.c;
    const float m = best == -INFINITY ? 0.0f : best;
    // rounded to T, as in attention_tile, while their sum has all bits
    V w[ALL * 2];
    float sum = 0;
#pragma unroll
    for (int t = 0; t < ALL; t++)
        if (any(t))
#pragma unroll
            for (int e = 0; e < 16; e++) {
                const float x = __builtin_amdgcn_exp2f(fmaf(s[t][e], pl.c, -m));
                sum += x;
                w[t * 2 + e / 8][e % 8] = (T)x;
            }

    __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    v16f o[DB];
#pragma unroll
    for (int d = 0; d < DB; d++)
#pragma unroll
        for (int e = 0; e < 16; e++) o[d][e] = 0.0f;
    // values^T weights^T, as in attention_tile: 4 keys of 16 elements come back
    // transposed
    const uint32_t vrow = hi * 4 + ((lane & 15) >> 2);
    V v[2][DB];
    auto read_values = [&](int k, V(&v)[DB]) {
        const uint32_t r0 = lds_row(k / 2) + k % 2 * 16 + vrow;
#pragma unroll
        for (int d = 0; d < DB; d++) {
            union {
                s16x4 half[2];
                V all;
            } u;
#pragma unroll
            for (int x = 0; x < 2; x++) {
                const uint32_t r = r0 + x * 8, c = (d * 4 + ((lane & 16) >> 3 | (lane & 2) >> 1)) ^ value_swizzle<D>(r);
                u.half[x] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(lds + r * D * 2 + (c << 4) + (lane & 1) * 8));
            }
            v[d] = u.all;
        }
    };
    if (any(0)) read_values(0, v[0]);
#pragma unroll
    for (int k = 0; k < ALL * 2; k++) {
        if (k + 1 < ALL * 2 && any((k + 1) / 2)) read_values(k + 1, v[(k + 1) & 1]);
        if (k == NT * 2 && !any(NT - 1) && any(NT)) read_values(k, v[k & 1]);
        __builtin_amdgcn_sched_barrier(0);
        if (any(k / 2))
#pragma unroll
            for (int d = 0; d < DB; d++) o[d] = mfma32(v[k & 1][d], w[k], o[d]);
        __builtin_amdgcn_sched_barrier(0);
    }
    // A value that is not finite reaches rows that do not see it as 0 * inf: where a
    // result is not finite, the rows are done one by one, but for those whose weights
    // have no finite sum (as in attention_tile).
    float check = 0;
#pragma unroll
    for (int d = 0; d < DB; d++)
#pragma unroll
        for (int e = 0; e < 16; e++) check = fmaf(o[d][e], 0.0f, check);
    const bool not_finite = in && !(check == 0.0f);
    bool alone = __syncthreads_or(not_finite);
    if (alone) {
        const float total = halves_sum(sum);
        alone = __syncthreads_or(not_finite && total == total);
    }
    if (alone) {
        float *own = (float *)lds + wave * 320;
        const Tiles<32> tiles(from, to);
        for (int32_t i = wrow; i < wend; i++)
            row_alone<T, 32, true>(a, pl, p, group, hk, i, tiles, 0, tiles.tiles, 0, own, own + 256);
        return;
    }
    store_by_rows<T, D>(a, p, group, hk, o, sum, wrow, view.any(), lds + wave * 32 * D * 2);
}

// The keys that a wave's 32 rows see in a window.
uint64_t keys_of_wave(const AttentionArgs &a) {
    const uint64_t group = a.hq / a.hk;
    return (31 + group - 1) / group + (uint64_t)a.left + (a.causal ? 0 : a.right) + 1;
}
// A wave's tiles of a window's keys, or 0 for attention_tile: the window, or the first
// keys, are too many, or nine tiles' scores leave a SIMD too few waves (128 on
// both sides, 16 heads over 4, 8 x 2000..4096 tokens: d = 64 79 us against 69, with 4
// first keys 87 against 85; d = 32 45 against 50 but with first keys 63 against 60; d = 96 101
// against 137, d = 128 119 against 157).
int window_tiles(const AttentionArgs &a) {
    const uint64_t keys = keys_of_wave(a);
    if (a.sinks > 32 || keys > 288) return 0;
    return keys <= 160 ? 5 : a.d > 64 || (a.d <= 32 && !a.sinks) ? 9 : 0;
}

// (A tile's offsets within 64 rows have 32 bits.)
bool by_window(const AttentionArgs &a) {
    return direct(a) && std::max(a.sk, a.sv) < (1u << 22) && a.d <= 128 && !few_rows(a) && window_tiles(a);
}

template <class T, int D, int NT, bool FIRSTS>
hipError_t window_of(const AttentionArgs &a, const AttentionPlan &pl, hipStream_t s) {
    const uint32_t group = a.hq / a.hk;
    const uint64_t slots = a.tq * group / 128 + a.batch;
    // The waves' first rows lie at most 96 rows apart, and each reads the tiles that its
    // keys reach, not NT: as little LDS as a call needs (d = 128, 16 heads over 4, the last 201
    // keys and 4 first ones, 8 x 2000..4096 tokens: two workgroups a CU, 123 us, one 194).  The
    // results take 128 rows.
    const uint32_t span = (96 + group - 1) / group + (uint32_t)(keys_of_wave(a) + 31) / 32 * 32;
    const uint32_t rows = std::max(128u, whole_rows<D>(span) + (FIRSTS ? whole_rows<D>(a.sinks) : 0));
    const uint32_t bytes = rows * D * 2;
    const uint64_t most = std::max<uint64_t>(1, (1u << 22) / a.hk);  // launches of fewer than 2^32 threads
    for (uint64_t f = 0; f < slots; f += most) {
        const uint32_t n = (uint32_t)std::min<uint64_t>(slots - f, most);
        attention_window<T, D, NT, FIRSTS><<<(n * a.hk + 7) / 8 * 8, 256, bytes, s>>>(a, pl, f, n, rows);
    }
    return hipGetLastError();
}
// window_tiles says 9 for D > 64, and for D = 32 where there are no first keys.
template <class T, int D>
hipError_t window_sized(const AttentionArgs &a, const AttentionPlan &pl, hipStream_t s) {
    if constexpr (D != 64)
        if (window_tiles(a) == 9) {
            if constexpr (D > 64)
                if (a.sinks) return window_of<T, D, 9, true>(a, pl, s);
            return window_of<T, D, 9, false>(a, pl, s);
        }
    return a.sinks ? window_of<T, D, 5, true>(a, pl, s) : window_of<T, D, 5, false>(a, pl, s);
}
template <class T>
hipError_t window_typed(const AttentionArgs &a, const AttentionPlan &pl, hipStream_t s) {
    if (a.d <= 32) return window_sized<T, 32>(a, pl, s);
    if (a.d <= 64) return window_sized<T, 64>(a, pl, s);
    if (a.d <= 96) return window_sized<T, 96>(a, pl, s);
    return window_sized<T, 128>(a, pl, s);
}

}  // namespace

hipError_t launch_attention_local(const AttentionArgs &a, void *ws, hipStream_t s) {
    if (by_window(a)) {
        const AttentionPlan pl = whole_plan(a);
        return a.dtype == T_F16 ? window_typed<f16>(a, pl, s) : window_typed<bf16>(a, pl, s);
    }
    return launch_attention_as<true>(a, ws, s);
}

}  // namespace bvk
