// Softmax attention over packed sequences with grouped heads.
#include "bv_embed.h"
#include "bv_embed_device.h"

#include <algorithm>

namespace bvk {
namespace {

// One wave per query row (a token's head; a sequence's rows are its tokens
// times the heads of a key head's group): keys 64 at a time, a lane each, with
// the running maximum and sum of the softmax; only keys the row sees are read.
constexpr uint32_t ROWS = 4;  // a workgroup's tile

template <class T>
__global__ __launch_bounds__(256) void attention_rows(AttentionArgs a, uint64_t first) {
    __shared__ float qs[4][256], ps[4][64];
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, group = a.hq / a.hk, hk = blockIdx.y;
    const uint64_t slot = first + blockIdx.x;
    const uint32_t s = slot_sequence(a.cu_q, a.batch, a.tq, group, ROWS, slot);
    const int64_t qb = clip_cu(a.cu_q, s, a.tq), qe = clip_cu(a.cu_q, s + 1, a.tq);
    const int64_t kb = clip_cu(a.cu_k, s, a.tk), ke = clip_cu(a.cu_k, s + 1, a.tk);
    const int64_t tile = (int64_t)slot - qb * group / ROWS - s;
    const int64_t row = tile * ROWS + wave;
    if (tile < 0 || row >= (qe - qb) * (int64_t)group) return;
    const int64_t token = row / group, h = hk * group + row % group;
    const T *q = (const T *)a.q + (qb + token) * a.sq + h * a.sqh;
    for (uint32_t i = lane; i < a.d; i += 64) qs[wave][i] = (float)q[i];
    const int64_t lk = max((int64_t)0, ke - kb);
    const int64_t seen = a.causal ? min(lk, lk - (qe - qb) + token + 1) : lk;
    float top = -INFINITY, sum = 0, acc[4] = {};
    for (int64_t j0 = 0; j0 < seen; j0 += 64) {
        const int64_t j = j0 + lane;
        float sc = -INFINITY;
        if (j < seen) {
            const T *k = (const T *)a.k + (kb + j) * a.sk + hk * a.skh;
            float dot = 0;
            for (uint32_t i = 0; i < a.d; i++) dot = fmaf(qs[wave][i], (float)k[i], dot);
            sc = dot * a.scale;
        }
        const float best = fmaxf(top, wave_max(sc));
        const float keep = top == best ? 1.0f : __expf(top - best);
        const float p = j < seen ? __expf(sc - best) : 0.0f;
        top = best;
        sum = sum * keep + wave_sum(p);
        ps[wave][lane] = p;
        const int n = (int)min((int64_t)64, seen - j0);
#pragma unroll
        for (int c = 0; c < 4; c++) acc[c] *= keep;
        for (int i = 0; i < n; i++) {
            const T *v = (const T *)a.v + (kb + j0 + i) * a.sv + hk * a.svh;
#pragma unroll
            for (int c = 0; c < 4; c++)
                if (c * 64 + lane < a.d) acc[c] = fmaf(ps[wave][i], (float)v[c * 64 + lane], acc[c]);
        }
    }
    T *o = (T *)a.o + (qb + token) * a.so + h * a.soh;
#pragma unroll
    for (int c = 0; c < 4; c++)
        if (c * 64 + lane < a.d) o[c * 64 + lane] = (T)(seen > 0 ? acc[c] / sum : 0.0f);
}

template <class T>
hipError_t attention_of(const AttentionArgs &a, hipStream_t s) {
    const uint64_t slots = a.tq * (a.hq / a.hk) / ROWS + a.batch;
    for (uint64_t f = 0; f < slots; f += 1u << 23)
        attention_rows<T><<<dim3((uint32_t)std::min<uint64_t>(slots - f, 1u << 23), a.hk), 256, 0, s>>>(a, f);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_attention(const AttentionArgs &a, hipStream_t s) {
    return a.dtype == T_F16 ? attention_of<f16>(a, s) : attention_of<bf16>(a, s);
}

}  // namespace bvk
