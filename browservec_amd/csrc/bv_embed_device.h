// Device helpers of the embedding operators' kernels: loads and stores of
// eight elements of a type as 32-bit floats, wave reductions, and the place of
// a workgroup's tile in packed sequences.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace bvk {
namespace {

typedef _Float16 f16;
typedef __bf16 bf16;

// Rows may start at any element, so eight elements are loaded and stored at
// the type's own alignment: gfx950 takes a 16-byte access at any address.
template <class T>
struct Vec8 {
    typedef T type __attribute__((ext_vector_type(8)));
    typedef type unaligned __attribute__((aligned(sizeof(T))));
};

// ONCE: read once in all, not kept in the caches before other data
template <bool ONCE = false, class T>
__device__ __forceinline__ void load8(const T *p, float (&f)[8]) {
    typename Vec8<T>::type v;
    if (ONCE) v = __builtin_nontemporal_load((const typename Vec8<T>::unaligned *)p);
    else v = *(const typename Vec8<T>::unaligned *)p;
#pragma unroll
    for (int i = 0; i < 8; i++) f[i] = (float)v[i];
}
// Elements at..at+7 of a row of n, zeros past its end, without a branch per
// lane: the load stays inside the row (ends with it) and its elements move down
// by what it was too early.  tail: whether n is no multiple of 8.
template <bool ONCE = false, class T>
__device__ __forceinline__ void load8(const T *row, uint32_t at, uint32_t n, bool tail, float (&f)[8]) {
    if (tail && n < 8) {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const float x = (float)row[min(at + i, n - 1)];
            f[i] = at + i < n ? x : 0.0f;
        }
        return;
    }
    const uint32_t from = min(at, n - 8), early = at - from;
    load8<ONCE>(row + from, f);
    if (tail) {
#pragma unroll
        for (int step = 4; step; step /= 2)
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float next = i + step < 8 ? f[i + step] : 0.0f;
                f[i] = early & step ? next : f[i];
            }
    }
#pragma unroll
    for (int i = 0; i < 8; i++) f[i] = early < 8 ? f[i] : 0.0f;
}
template <bool ONCE = false, class T>
__device__ __forceinline__ void store8(T *p, int n, const float (&f)[8]) {
    if (n >= 8) {
        typename Vec8<T>::type v;
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = (T)f[i];
        if (ONCE) __builtin_nontemporal_store(v, (typename Vec8<T>::unaligned *)p);
        else *(typename Vec8<T>::unaligned *)p = v;
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; i++)
        if (i < n) p[i] = (T)f[i];
}

// Over the wave, the result in every lane, in the VALU alone: within rows of 16
// lanes by permutations of quads and mirrors, across rows by swaps (a swap of x
// with itself gives a lane its own value and its partner's).
template <int CTRL>
__device__ __forceinline__ float dpp(float x) {
    return __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(x), CTRL, 0xf, 0xf, true));
}
#define BV_OVER_WAVE(x, OP)                                                                              \
    x = OP(x, dpp<0xb1>(x));  /* quads: 1 0 3 2 */                                                       \
    x = OP(x, dpp<0x4e>(x));  /* quads: 2 3 0 1 */                                                       \
    x = OP(x, dpp<0x141>(x)); /* halves of a row mirrored */                                             \
    x = OP(x, dpp<0x140>(x)); /* rows mirrored */                                                        \
    {                                                                                                    \
        auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false); \
        x = OP(__uint_as_float(r[0]), __uint_as_float(r[1]));                                            \
        r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);      \
        x = OP(__uint_as_float(r[0]), __uint_as_float(r[1]));                                            \
    }
__device__ __forceinline__ float add_f32(float a, float b) { return a + b; }
__device__ __forceinline__ float wave_sum(float x) {
    BV_OVER_WAVE(x, add_f32)
    return x;
}
__device__ __forceinline__ float wave_max(float x) {
    BV_OVER_WAVE(x, fmaxf)
    return x;
}
// Of values without a sign the largest of their bits: infinity is above every
// number, NaN above that.
__device__ __forceinline__ float top_of(float a, float b) { return __uint_as_float(max(__float_as_uint(a), __float_as_uint(b))); }
__device__ __forceinline__ float wave_top(float x) {
    BV_OVER_WAVE(x, top_of)
    return x;
}
#undef BV_OVER_WAVE
// A lane's value and that of lane ^ 32.
__device__ __forceinline__ float halves_sum(float x) {
    auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float halves_max(float x) {
    auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// Packed sequences in tiles of `tile` places without a list of tiles: sequence
// s, places [at(s), at(s+1)), takes the slots from floor(at(s) / tile) + s on.
// That many follow until the next sequence's first: ceil(n / tile) <=
// floor(b / tile) - floor(a / tile) + 1 for n = b - a.  All slots are
// floor(at(batch) / tile) + batch; some hold no tile.  A slot's sequence is
// the last one whose first slot is not past it, found 64 sequences at a time.
__device__ __forceinline__ int64_t clip_cu(const int32_t *cu, uint32_t i, uint64_t tokens) {
    const int64_t c = cu[i];
    return c < 0 ? 0 : c > (int64_t)tokens ? (int64_t)tokens : c;
}
// All lanes of a wave call it with the same arguments.
__device__ __forceinline__ uint32_t slot_sequence(const int32_t *cu, uint32_t batch, uint64_t tokens, uint32_t group,
                                                  uint32_t tile, uint64_t slot) {
    const uint32_t lane = threadIdx.x & 63;
    uint32_t lo = 0, n = batch;  // the sequence is in [lo, lo + n)
    while (n > 1) {
        const uint32_t step = (n + 63) / 64;
        const uint32_t at = lane * step;
        // tokens * group fits 32 bits
        const bool past = at >= n || (uint64_t)((uint32_t)clip_cu(cu, lo + at, tokens) * group / tile) + lo + at > slot;
        const uint64_t not_past = __ballot(!past);
        // ascending offsets: the lanes not past are the first ones
        const uint32_t last = not_past ? 63 - __builtin_clzll(not_past) : 0;
        lo += last * step;
        n = n - last * step < step ? n - last * step : step;
    }
    return lo;
}

// Slots without a tile come at steps that the lengths give, every second one
// where sequences fill a tile each, and workgroups go to XCDs, and there to
// shader engines, in turn: taken in order, half of the card would idle.  So of
// `each` workgroups a slot, i-th of n slots: an XCD takes two neighbouring ones,
// in an order that changes from two to two.  Attention over 512 x 128 tokens, 8
// heads of 64: 81 us, in order 133; pooling 1111 x 16 rows of 3904 66 and 103.
__device__ __forceinline__ uint32_t spread(uint32_t i, uint32_t n, uint32_t each) {
    const uint32_t lg = 3 - min(3, (int)__builtin_ctz(each));  // after 2^lg slots XCDs repeat
    const uint32_t group = i >> (1 + lg), l = i & ((2 << lg) - 1);
    if ((group + 1) << (1 + lg) > n) return i;
    return (group << (1 + lg)) + 2 * (l & ((1 << lg) - 1)) + ((l >> lg) ^ (group * 0x9e3779b9u >> 31));
}

}  // namespace
}  // namespace bvk
