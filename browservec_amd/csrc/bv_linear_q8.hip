// y = act(sx_i sw_j sum_k x_ik w_jk + bias_j) + residual_ij of codes of 8 bits, on
// the matrix cores.  The sums are whole numbers of 32 bits and exact (the host
// refuses a k at which they might not be); they are rounded to 32-bit floats
// once, on their way to the scales.
//
// As in bv_linear.hip the products are computed transposed, w's rows as the matrix
// instructions' first operand: a lane holds four neighbouring columns of a row.
#include "bv_embed.h"
#include "bv_embed_device.h"
#include "bv_finish.h"
#include "bv_linear_q8_plan.h"
#include "bv_mfma.h"

#include <algorithm>

namespace bvk {
namespace {

typedef float v4f __attribute__((ext_vector_type(4)));
typedef v4i v4i_any __attribute__((aligned(1)));  // 16 codes at any address

__device__ __forceinline__ v16i mfma32(v4i a, v4i b, v16i c) { return __builtin_amdgcn_mfma_i32_32x32x32_i8(a, b, c, 0, 0, 0); }
__device__ __forceinline__ v4i mfma16(v4i a, v4i b, v4i c) { return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0); }

__device__ __forceinline__ float bias_at(const LinearQ8Args &a, uint32_t n) {
    if (!a.bias) return 0.0f;
    if (a.bias_dtype == T_F32) return ((const float *)a.bias)[n];
    return a.bias_dtype == T_F16 ? (float)((const f16 *)a.bias)[n] : (float)((const bf16 *)a.bias)[n];
}

// ------------------------------------------------------------------ tiles --
// A workgroup of 2 x WN waves computes BM x BN results, a wave BM/2 x BN/WN of
// them; KG such groups share the columns of every tile and join their sums at
// the end.  Tiles of BK columns of x and w stream through ST buffers in LDS,
// loaded straight into it; a wave reads the operands of 32 columns while it
// multiplies those of the 32 before, and waits for the next tile before it
// multiplies a tile's last 32, already in registers.
//
// Bound by the card's power and the end of a tile.  8192 x 8192 x 8192: 470 to 490 us by
// card, 2.3 POP/s (the library's bare product 450): the matrix cores are busy for 60% of the
// cycles at 1.8 GHz; without loads 385, without LDS reads as well 324.  32768 x 4096, k 1024,
// bf16: the loop takes 127 us, all of it 166 (the library's bare product 194), with
// bias and GELU 195 to 215, of which the activation's 13 instructions a result are 30 to 50.
// 20011 x 1024, k 4096, onto a residual of 32 bits: 114 to 126 in two launches.  Tried and
// slower: groups of waves that take turns between LDS and matrix cores (482), four waves of
// 128 x 128 (539), 192 x 128 tiles two a CU (535); steps of 64 codes ask the L2 for half lines
// and are bound by its requests (580), but two such workgroups a CU cover each other's ends.
//
// LDS rows hold BK codes, in 16-byte chunks; chunk c of row r lies at
// c ^ swizzle(r), so that sixteen lanes that read the same chunk of consecutive
// rows cover all banks (256 bytes).  Loads put lane i's chunk at a fixed place, so the
// swizzle is applied to the address they load from.
template <int BK>
__device__ __forceinline__ uint32_t swizzle(uint32_t row) {
    return BK >= 256 ? row & 15 : BK == 128 ? row >> 1 & 7 : row >> 2 & 3;
}

template <class O, int BM, int BN, int WN, int BK, int ST, int KG = 1>
__global__ __launch_bounds__(128 * WN * KG, BM * BN / WN > 16384 ? 1 : 2) void linear_q8_tile(LinearQ8Args a, uint32_t tiles_m,
                                                                                              uint32_t tiles_n) {
    constexpr int THREADS = 128 * WN * KG, WB = BN / WN;  // KG times 2 x WN waves, of WB columns each
    constexpr int MI = BM / 64, NI = WB / 32;             // 32 x 32 blocks of a wave
    constexpr int CH = BK / 16;                           // chunks of a row
    constexpr int STAGE = (BM + BN) * BK;                 // bytes of a tile
    constexpr int NL = (BM + BN) * CH / THREADS;          // loads of a thread for a tile
    constexpr int KK = BK / 32 / KG;                      // of a tile, for each group
    constexpr int PITCH = WB + 4;                         // floats of a row in the epilogue
    constexpr int ROWS_END = 2 * WN * 32 * PITCH * 4;     // bytes of those rows; after them, the other groups' sums
    static_assert(ROWS_END + (KG - 1) * 2 * WN * MI * NI * 4096 <= ST * STAGE, "the epilogue's data fits the buffers");
    static_assert(KK % 2 == 0 && BM * CH % THREADS == 0 && BN * CH % THREADS == 0, "whole loads, two sets of operands");
    __shared__ __align__(1024) unsigned char lds[ST * STAGE];
    __shared__ __align__(16) float bias[BN], scale_w[BN], scale_x[BM];

    // Workgroups go to the 8 XCDs in turn: each takes a run of tiles of its own,
    // in columns of 8 tiles of rows, so that what its workgroups read at a time
    // stays in its L2.
    const uint32_t tiles = tiles_m * tiles_n, xcd = blockIdx.x & 7, nth = blockIdx.x >> 3;
    const uint32_t per = tiles / 8, more = tiles % 8;
    const uint32_t tile = xcd * per + min(xcd, more) + nth;
    const uint32_t group = tile / (8 * tiles_n), in = tile % (8 * tiles_n);
    const uint32_t rows = min(8u, tiles_m - group * 8);
    const uint64_t m0 = (uint64_t)(group * 8 + in % rows) * BM;
    const uint32_t n0 = (in / rows) * BN;

    const uint32_t tid = threadIdx.x, lane = tid & 63, any_wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t wave = any_wave % (2 * WN), kg = any_wave / (2 * WN);
    const uint32_t lo = lane & 31, hi = lane >> 5;
    for (uint32_t i = tid; i < BN; i += THREADS) {
        const uint32_t n = min(n0 + i, a.n - 1);
        bias[i] = bias_at(a, n);
        scale_w[i] = a.w_scales[n];
    }
    for (uint32_t i = tid; i < BM; i += THREADS) scale_x[i] = a.x_scales[min(m0 + i, a.m - 1)];

    // this thread's chunks: rows 0..BM-1 are x's, BM.. are w's; rows past the
    // end repeat the last one, their results are not stored
    const char *xb = (const char *)a.x + m0 * a.ldx, *wb = (const char *)a.w + (uint64_t)n0 * a.ldw;
    auto chunk = [&](int i) { return (i * THREADS + tid) % CH ^ swizzle<BK>((i * THREADS + tid) / CH); };
    uint32_t off[NL];
#pragma unroll
    for (int i = 0; i < NL; i++) {
        const uint32_t row = (i * THREADS + tid) / CH;
        off[i] = (row < (uint32_t)BM ? (uint32_t)(min((uint64_t)row, a.m - 1 - m0) * a.ldx)
                                     : (uint32_t)(min(row - BM, a.n - 1 - n0) * a.ldw)) + chunk(i) * 16;
    }
    const uint32_t lds0 = lds_addr(lds) + any_wave * 1024;
    const uint32_t steps = (a.k + BK - 1) / BK;
    auto load_one = [&](uint32_t step, int i) {
        constexpr int XL = BM * CH / THREADS;
        const uint32_t k0 = step * BK;
        const char *base = (i < XL ? xb : wb) + k0;
        const uint32_t to = __builtin_amdgcn_readfirstlane(lds0 + step % ST * STAGE + i * THREADS * 16);
        if (k0 + BK <= a.k) lds_load16(base, off[i], to);
        else lds_load16(base, k0 + chunk(i) * 16 < a.k ? off[i] : off[i] - chunk(i) * 16, to);  // cleared in arrive()
    };
    auto load = [&](uint32_t step) {
#pragma unroll
        for (int i = 0; i < NL; i++) load_one(step, i);
    };

    v16i acc[NI][MI];
#pragma unroll
    for (int n = 0; n < NI; n++)
#pragma unroll
        for (int m = 0; m < MI; m++)
#pragma unroll
            for (int e = 0; e < 16; e++) acc[n][m][e] = 0;

    // where this lane's results go
    constexpr uint32_t LANES = WB / 8, RI = 64 / LANES;  // lanes of a row, rows of a turn
    static_assert(64 % LANES == 0, "a lane keeps its columns");
    const uint32_t mr = (wave & 1) * (BM / 2), lrow = lane / LANES, col = lane % LANES * 8, nc = (wave >> 1) * WB + col;
    const int left = n0 + nc < a.n ? (int)min(8u, a.n - n0 - nc) : 0;
    const uint32_t rows_left = left && m0 + mr < a.m ? (uint32_t)min((uint64_t)BM / 2, a.m - m0 - mr) : 0;
    const O *res = (const O *)a.residual + (a.residual ? (m0 + mr + lrow) * a.ldr + n0 + nc : 0);
    // Small tiles take their residuals to registers during the first step: there is
    // nothing else to wait beside (2037 x 768, k 768, tiles of 64 x 128: 7.2 us, later 8.2).
    constexpr uint32_t TURNS = MI * 32 / RI;
    constexpr bool EARLY = ST == 2 && TURNS <= 4;
    typename Vec8<O>::type early[EARLY ? TURNS : 1];

    const uint32_t mrow = (wave & 1) * (BM / 2) + lo, nrow = BM + (wave >> 1) * WB + lo;
    v4i x[2][MI], w[2][NI];
    auto read = [&](uint32_t step, int k, v4i(&xs)[MI], v4i(&ws)[NI]) {
        const uint32_t kk = kg * KK + k;
        const unsigned char *buf = lds + step % ST * STAGE;
#pragma unroll
        for (int n = 0; n < NI; n++) {
            const uint32_t r = nrow + n * 32;
            ws[n] = *(const v4i *)(buf + r * BK + (((kk * 2 + hi) ^ swizzle<BK>(r)) * 16));
        }
#pragma unroll
        for (int m = 0; m < MI; m++) {
            const uint32_t r = mrow + m * 32;
            xs[m] = *(const v4i *)(buf + r * BK + (((kk * 2 + hi) ^ swizzle<BK>(r)) * 16));
        }
    };
    // tile `step` is in LDS, for every wave
    auto arrive = [&](uint32_t step) {
        if (step + ST - 2 < steps) __builtin_amdgcn_s_waitcnt(vmcnt_imm((ST - 2) * NL));
        else __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        if ((step + 1) * BK > a.k) {  // chunks past k: zeros in both operands
#pragma unroll
            for (int i = 0; i < NL; i++)
                if (step * BK + chunk(i) * 16 >= a.k)
                    *(v4i *)(lds + step % ST * STAGE + (i * THREADS + tid) * 16) = v4i{0, 0, 0, 0};
            __syncthreads();
        }
    };
#pragma unroll
    for (int s = 0; s < ST - 1; s++)
        if ((uint32_t)s < steps) load(s);
    if (steps) {
        arrive(0);
        if (ST - 1 < steps) load(ST - 1);
        read(0, 0, x[0], w[0]);
    }
    if (EARLY && a.residual && left == 8 && !kg)
#pragma unroll
        for (uint32_t i = 0; i < TURNS; i++)
            if (i * RI + lrow < rows_left) early[i] = *(const typename Vec8<O>::unaligned *)(res + (uint64_t)i * RI * a.ldr);
    for (uint32_t step = 0; step < steps; step++) {
#pragma unroll
        for (int kk = 0; kk < KK; kk++) {
            if (kk + 1 < KK) {
                read(step, kk + 1, x[(kk + 1) & 1], w[(kk + 1) & 1]);
            } else if (step + 1 < steps) {
                arrive(step + 1);
                read(step + 1, 0, x[0], w[0]);
            }
            __builtin_amdgcn_sched_barrier(0);
            const bool loads = kk + 1 == KK && step + ST < steps;
#pragma unroll
            for (int n = 0; n < NI; n++)
#pragma unroll
                for (int m = 0; m < MI; m++) {
                    acc[n][m] = mfma32(w[kk & 1][n], x[kk & 1][m], acc[n][m]);
                    constexpr int EACH = (NL + MI * NI - 1) / (MI * NI);
                    if (loads)  // between matrix instructions, where issue is idle
#pragma unroll
                        for (int i = 0; i < EACH; i++)
                            if ((n * MI + m) * EACH + i < NL) load_one(step + ST, (n * MI + m) * EACH + i);
                    __builtin_amdgcn_sched_barrier(0);
                }
        }
    }
    __syncthreads();
    if (KG > 1) {  // the groups' sums
        int *sums = (int *)(lds + ROWS_END) + (wave * 64 + lane) * 4;
        constexpr int QUADS = MI * NI * 4, GROUP = 2 * WN * 64 * 4;  // sums from a quad to the next
        if (kg)
#pragma unroll
            for (int i = 0; i < QUADS; i++) {
                const v16i &f = acc[i / 4 / MI][i / 4 % MI];
                *(v4i *)(sums + ((kg - 1) * QUADS + i) * GROUP) = v4i{f[i % 4 * 4], f[i % 4 * 4 + 1], f[i % 4 * 4 + 2], f[i % 4 * 4 + 3]};
            }
        __syncthreads();
        if (kg) return;
#pragma unroll
        for (int g = 0; g < KG - 1; g++)
#pragma unroll
            for (int i = 0; i < QUADS; i++) {
                const v4i f = *(const v4i *)(sums + (g * QUADS + i) * GROUP);
#pragma unroll
                for (int e = 0; e < 4; e++) acc[i / 4 / MI][i / 4 % MI][i % 4 * 4 + e] += f[e];
            }
    }

    // Results by rows: 32 of a wave's rows at a time go through LDS as 32-bit
    // floats, so that residuals are read and results written 16 bytes a lane
    // along the rows.  A lane's columns are the same in every row.
    float *rows32 = (float *)lds + wave * 32 * PITCH;
    O *y = (O *)a.y + (m0 + mr + lrow) * a.ldy + n0 + nc;
    float b[8], s[8];
#pragma unroll
    for (int e = 0; e < 8; e += 4) *(v4f *)(b + e) = *(const v4f *)(bias + nc + e), *(v4f *)(s + e) = *(const v4f *)(scale_w + nc + e);
#pragma unroll
    for (int m = 0; m < MI; m++) {
        const float sx = scale_x[mr + m * 32 + lo];
#pragma unroll
        for (int n = 0; n < NI; n++)
#pragma unroll
            for (int q = 0; q < 4; q++) {
                v4f f;
#pragma unroll
                for (int e = 0; e < 4; e++) f[e] = (float)acc[n][m][q * 4 + e] * sx;
                *(v4f *)(rows32 + lo * PITCH + n * 32 + q * 8 + hi * 4) = f;
            }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the wave's own rows
#pragma unroll 4
        for (uint32_t i = 0; i < 32 / RI; i++) {
            float f[8];
            const float *from = rows32 + (i * RI + lrow) * PITCH + col;
            *(v4f *)f = *(const v4f *)from;
            *(v4f *)(f + 4) = *(const v4f *)(from + 4);
#pragma unroll
            for (int e = 0; e < 8; e++) f[e] = fmaf(f[e], s[e], b[e]);
            activate8(f, a.act);
            if (m * 32 + i * RI + lrow < rows_left) {
                if (a.residual) {
                    if (left == 8) {
                        float g[8];
                        if (EARLY) {
#pragma unroll
                            for (int e = 0; e < 8; e++) g[e] = (float)early[EARLY ? m * (32 / RI) + i : 0][e];
                        } else {
                            load8(res, g);
                        }
#pragma unroll
                        for (int e = 0; e < 8; e++) f[e] += g[e];
                    } else {
#pragma unroll
                        for (int e = 0; e < 8; e++) f[e] += (float)res[min(e, left - 1)];
                    }
                }
                if (a.once) store8<true>(y, left, f);
                else store8(y, left, f);
            }
            y += RI * a.ldy;
            res += RI * a.ldr;
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
}

// --------------------------------------------------------------- few rows --
// Up to 16 * MF rows of x (one question, a few): w is read once, straight into
// the matrix instructions' registers, 16 of its rows a workgroup; the waves
// split k and join their sums in LDS.  Bound by latency: a wave waits for four
// steps' loads before it starts the next four (9 x 1536, k 384: 3.7 us; 8 x 4096, k 4096, 6.3:
// 16.8 MB of w at 2.7 TB/s).
constexpr uint32_t ROW_WAVES = 8;
template <class O, int MF>
__global__ __launch_bounds__(ROW_WAVES * 64) void linear_q8_rows(LinearQ8Args a) {
    constexpr uint32_t waves = ROW_WAVES;
    __shared__ __align__(16) int red[waves * MF * 256];
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t n0 = blockIdx.x * 16, lo = lane & 15, kc = lane >> 4 << 4;
    const int8_t *w = a.w + (uint64_t)min(n0 + lo, a.n - 1) * a.ldw + kc;
    const int8_t *x[MF];
    v4i acc[MF];
#pragma unroll
    for (int m = 0; m < MF; m++) {
        x[m] = a.x + min((uint64_t)m * 16 + lo, a.m - 1) * a.ldx + kc;
        acc[m] = v4i{0, 0, 0, 0};
    }
    const uint32_t steps = a.k / 64, each = (steps + waves - 1) / waves;
    const uint32_t s0 = min(steps, wave * each), s1 = min(steps, s0 + each);
    uint32_t s = s0;
    for (; s + 4 <= s1; s += 4) {  // four steps' loads in flight
        v4i wv[4], xv[4][MF];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            wv[i] = *(const v4i_any *)(w + (s + i) * 64);
#pragma unroll
            for (int m = 0; m < MF; m++) xv[i][m] = *(const v4i_any *)(x[m] + (s + i) * 64);
        }
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int m = 0; m < MF; m++) acc[m] = mfma16(wv[i], xv[i][m], acc[m]);
    }
    for (; s < s1; s++) {
        const v4i wv = *(const v4i_any *)(w + s * 64);
#pragma unroll
        for (int m = 0; m < MF; m++) acc[m] = mfma16(wv, (v4i) * (const v4i_any *)(x[m] + s * 64), acc[m]);
    }
    if (steps * 64 < a.k && wave == waves - 1) {  // the rest of k, code by code
        const uint32_t k = steps * 64, left = a.k - k;
        union {
            int8_t b[16];
            v4i v;
        } wv, xv;
#pragma unroll
        for (int i = 0; i < 16; i++) {
            const int8_t e = w[kc + i < left ? (int64_t)(k + i) : -(int64_t)kc];
            wv.b[i] = kc + i < left ? e : 0;
        }
#pragma unroll
        for (int m = 0; m < MF; m++) {
#pragma unroll
            for (int i = 0; i < 16; i++) {
                const int8_t e = x[m][kc + i < left ? (int64_t)(k + i) : -(int64_t)kc];
                xv.b[i] = kc + i < left ? e : 0;
            }
            acc[m] = mfma16(wv.v, xv.v, acc[m]);
        }
    }
#pragma unroll
    for (int m = 0; m < MF; m++) *(v4i *)(red + (wave * MF + m) * 256 + lo * 16 + (lane >> 4) * 4) = acc[m];
    __syncthreads();
    // red[wave][row][column]: eight columns of a row a thread
    for (uint32_t i = threadIdx.x; i < MF * 32; i += waves * 64) {
        int t[8] = {};
        for (uint32_t v = 0; v < waves; v++) {
            const v4i *r = (const v4i *)(red + v * MF * 256 + i * 8);
            const v4i p = r[0], q = r[1];
#pragma unroll
            for (int e = 0; e < 4; e++) t[e] += p[e], t[e + 4] += q[e];
        }
        const uint32_t row = i / 2, n = n0 + i % 2 * 8;
        if (row >= a.m || n >= a.n) continue;
        const float sx = a.x_scales[row];
        float f[8];
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const uint32_t at = min(n + e, a.n - 1);
            f[e] = fmaf((float)t[e] * sx, a.w_scales[at], bias_at(a, at));
        }
        activate8(f, a.act);
        finish8<O>(a, row, n, f);
    }
}

// ---------------------------------------------------------------- packing --
// Rows for linear_q8_tile, which loads 16 bytes at 16-byte addresses: k rounded
// up to 16 with zeros, by every call: nothing is kept.  x's and w's in one launch (114 x
// 1000, k 820: 8.5 us, 2 more in two).  20011 x 1024, k 4090, onto a residual of 32 bits: 150
// us, k 4096 114; of w alone 120; 32768 x 4096, k 1000, GELU: 224, k 1008 209.
struct PackJob {
    const int8_t *from;
    int8_t *to;
    uint64_t ld, count;  // chunks of 16 codes in all
};
__global__ __launch_bounds__(256) void pack_codes(PackJob a, PackJob b, uint32_t k, uint32_t chunks) {
    const uint64_t step = (uint64_t)gridDim.x * 256;
    for (uint64_t n = (uint64_t)blockIdx.x * 256 + threadIdx.x; n < a.count + b.count; n += step) {
        const PackJob &j = n < a.count ? a : b;
        const uint64_t i = n < a.count ? n : n - a.count, row = i / chunks;
        const uint32_t at = (uint32_t)(i - row * chunks) * 16;
        const int8_t *p = j.from + row * j.ld + at;
        union {
            int8_t b[16];
            v4i v;
        } u;
        if (at + 16 <= k) {
            u.v = *(const v4i_any *)p;
        } else {
#pragma unroll
            for (int e = 0; e < 16; e++) {
                const int8_t z = p[at + e < k ? e : 0];
                u.b[e] = at + e < k ? z : 0;
            }
        }
        *(v4i *)(j.to + i * 16) = u.v;
    }
}

// Rows up to which w goes straight to the registers: 32 rows of 4096 x 4096 8.3 us,
// 33 by tiles 10.8; of 768 x 768 3.4 and 4.3.
constexpr uint64_t FEW_ROWS = 32;
// A tile's loads have 32-bit offsets: 256 rows of as many codes reach 2^31
// bytes.  Rows further apart are packed; k itself is far below.
constexpr uint64_t FAR_ROWS = 1u << 23;
static_assert(LINEAR_Q8_MAX_K < FAR_ROWS, "packed rows are near enough");

bool aligned(const void *p, uint64_t ld) { return (uintptr_t)p % 16 == 0 && ld % 16 == 0; }
bool packs(const LinearQ8Args &a, const void *p, uint64_t ld) {
    return a.m > FEW_ROWS && a.k && (a.k % 16 || !aligned(p, ld) || ld >= FAR_ROWS);
}
uint64_t packed_bytes(uint64_t rows, uint32_t k) { return (rows * ((k + 15) / 16) * 16 + 255) & ~255ull; }

// Workgroups of a launch: of 2^32 threads and more it runs the low 32 bits, so
// with up to 1024 a workgroup more work is launched in pieces.
constexpr uint32_t GRID_MOST = 1u << 21;

// The part of a call that makes rows m to m + rows and columns n to n + cols.
template <class O>
LinearQ8Args part_of(const LinearQ8Args &a, uint64_t m, uint64_t rows, uint64_t n, uint64_t cols) {
    LinearQ8Args b = a;
    b.m = std::min(a.m - m, rows);
    b.n = (uint32_t)std::min(a.n - n, cols);
    b.x = a.x + m * a.ldx;
    b.w = a.w + n * a.ldw;
    b.x_scales = a.x_scales + m;
    b.w_scales = a.w_scales + n;
    b.y = (O *)a.y + m * a.ldy + n;
    if (a.bias) b.bias = (const char *)a.bias + n * (a.bias_dtype == T_F32 ? 4 : 2);
    if (a.residual) b.residual = (const O *)a.residual + m * a.ldr + n;
    return b;
}

template <class O, int BM, int BN, int WN, int BK, int ST, int KG = 1>
hipError_t tile_of(const LinearQ8Args &a, hipStream_t s) {
    static_assert(128 * WN * KG <= 1024, "GRID_MOST is for 1024 threads");
    for (uint64_t n = 0; n < a.n; n += (uint64_t)GRID_MOST * BN) {
        const uint32_t tn = (uint32_t)((std::min<uint64_t>(a.n - n, (uint64_t)GRID_MOST * BN) + BN - 1) / BN);
        const uint64_t most = GRID_MOST / tn;
        for (uint64_t m = 0; m < a.m; m += most * BM) {
            const LinearQ8Args b = part_of<O>(a, m, most * BM, n, (uint64_t)GRID_MOST * BN);
            const uint32_t tm = (uint32_t)((b.m + BM - 1) / BM);
            linear_q8_tile<O, BM, BN, WN, BK, ST, KG><<<tm * tn, 128 * WN * KG, 0, s>>>(b, tm, tn);
        }
    }
    return hipGetLastError();
}

template <class O, int MF>
hipError_t rows_of(const LinearQ8Args &a, hipStream_t s) {
    linear_q8_rows<O, MF><<<(a.n - 1) / 16 + 1, ROW_WAVES * 64, 0, s>>>(a);
    return hipGetLastError();
}

// Shape I's tiles: its rows, columns and step from the plan's table, waves across, buffers, groups.
template <class O, int I, int WN, int ST, int KG = 1>
hipError_t shape(const LinearQ8Args &a, hipStream_t s) {
    constexpr Q8Shape t = q8_shapes[I];
    return tile_of<O, t.bm, t.bn, WN, t.bk, ST, KG>(a, s);
}
template <class O>
hipError_t shape_of(const LinearQ8Args &a, int i, hipStream_t s) {
    switch (i) {
    case 0: return shape<O, 0, 2, 2, 4>(a, s);
    case 1: return shape<O, 1, 2, 2, 2>(a, s);
    case 2: return shape<O, 2, 2, 2, 2>(a, s);
    case 3: return shape<O, 3, 4, 4>(a, s);
    case 4: return shape<O, 4, 4, 3>(a, s);
    case 5: return shape<O, 5, 4, 2>(a, s);
    case 6: return shape<O, 6, 4, 3>(a, s);
    default: return shape<O, 7, 4, 2>(a, s);
    }
}

template <class O>
hipError_t linear_q8_of(LinearQ8Args a, void *ws, hipStream_t s) {
    if (a.m <= FEW_ROWS) {
        static_assert(ROW_WAVES * 64 <= 1024, "GRID_MOST is for 1024 threads");
        for (uint64_t n = 0; n < a.n; n += GRID_MOST * 16) {
            const LinearQ8Args b = part_of<O>(a, 0, a.m, n, GRID_MOST * 16);
            const hipError_t e = b.m <= 16 ? rows_of<O, 1>(b, s) : rows_of<O, 2>(b, s);
            if (e != hipSuccess) return e;
        }
        return hipSuccess;
    }
    const uint32_t chunks = (a.k + 15) / 16;
    PackJob jobs[2] = {};
    int n = 0;
    auto pack = [&](const int8_t *&p, uint64_t &ld, uint64_t rows) {
        if (!packs(a, p, ld)) return;
        jobs[n++] = {p, (int8_t *)ws, ld, rows * chunks};
        p = (const int8_t *)ws;
        ld = (uint64_t)chunks * 16;
        ws = (char *)ws + packed_bytes(rows, a.k);
    };
    pack(a.x, a.ldx, a.m);
    pack(a.w, a.ldw, a.n);
    if (n) {
        const uint64_t count = jobs[0].count + jobs[1].count;
        pack_codes<<<(uint32_t)std::min<uint64_t>((count + 255) / 256, 8192), 256, 0, s>>>(jobs[0], jobs[1], a.k, chunks);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    a.k = (a.k + 15) / 16 * 16;
    // Results that pass the L2s' 32 MB twice over go by them, and leave them to x and w:
    // 32768 x 4096, k 1024, bf16 192 -> 176 us, with GELU 251 -> 226.
    a.once = a.m * a.n * sizeof(O) > (64u << 20);
    const Q8Plan p = q8_plan(a.m, a.n, a.k, a.act);
    const hipError_t e = shape_of<O>(part_of<O>(a, 0, p.rows, 0, a.n), p.shape, s);
    return e != hipSuccess || p.rows == a.m ? e : shape_of<O>(part_of<O>(a, p.rows, a.m - p.rows, 0, a.n), p.then, s);
}

}  // namespace

size_t linear_q8_workspace(const LinearQ8Args &a) {
    return (packs(a, a.x, a.ldx) ? packed_bytes(a.m, a.k) : 0) + (packs(a, a.w, a.ldw) ? packed_bytes(a.n, a.k) : 0);
}

hipError_t launch_linear_q8(const LinearQ8Args &a, void *ws, hipStream_t s) {
    switch (a.out_dtype) {
    case T_F16: return linear_q8_of<f16>(a, ws, s);
    case T_BF16: return linear_q8_of<bf16>(a, ws, s);
    default: return linear_q8_of<float>(a, ws, s);
    }
}

}  // namespace bvk
