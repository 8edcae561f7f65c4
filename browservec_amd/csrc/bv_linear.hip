// y = act(x w^T + bias) + residual for an embedding model's layers, on the
// matrix cores.
//
// The products are computed transposed, w's rows as the matrix instructions'
// first operand and x's as their second: a lane then holds four neighbouring
// columns of one of y's rows, which leave it as one piece.
#include "bv_embed.h"
#include "bv_embed_device.h"
#include "bv_finish.h"
#include "bv_mfma.h"

#include <algorithm>

namespace bvk {
namespace {

typedef float v4f __attribute__((ext_vector_type(4)));
typedef f16 f16x8 __attribute__((ext_vector_type(8)));
typedef bf16 bf16x8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ v16f mfma32(f16x8 a, f16x8 b, v16f c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ v16f mfma32(bf16x8 a, bf16x8 b, v16f c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ v4f mfma16(f16x8 a, f16x8 b, v4f c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ v4f mfma16(bf16x8 a, bf16x8 b, v4f c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// ------------------------------------------------------------------ tiles --
// A workgroup of 2 x WN waves computes BM x BN results, a wave BM/2 x BN/WN of
// them; KG such groups share the columns of every tile and join their sums at
// the end, where tiles are few and what counts is the number of steps.  Tiles of
// BK columns of x and w stream through ST buffers in LDS, loaded straight into it.
// A wave reads the operands of 16 columns while it multiplies those of the 16
// before.  Before it multiplies a tile's last 16, already in registers, it waits
// for its share of the next tile and meets the others at a barrier: the next
// tile's first operands can then be read, and the tile's buffer takes the tile ST
// steps ahead, while the matrix cores are busy.
//
// Bound by the matrix cores where k is long (8192 x 8192 x 8192 bf16: 881 us, 1250
// TFLOP/s; matrix instructions and barriers alone take 655 at the clock they leave),
// and beside them by the epilogue where it is short: 32768 x 4096, k 1024, with
// bias and GELU 316 to 327 us, 840 to 870 TFLOP/s (on another card 343, 802), 66 of
// it the epilogue (the library's bare product, without it, takes 218); 335 with
// results of 32 bits.  2037 x 768 x 768 (8.9 us): start, steps one
// after the other and end of one round of tiles.
//
// LDS rows hold BK elements, in 16-byte chunks; chunk c of row r lies at
// c ^ swizzle(r), so that sixteen lanes that read the same chunk of consecutive
// rows cover all banks (256 bytes).  Loads put lane i's chunk at a fixed place, so the
// swizzle is applied to the address they load from.
template <int BK>
__device__ __forceinline__ uint32_t swizzle(uint32_t row) {
    return BK >= 128 ? row & 15 : BK == 64 ? row >> 1 & 7 : row >> 2 & 3;
}

template <class T, class O, int BM, int BN, int WN, int BK, int ST, int KG = 1>
__global__ __launch_bounds__(128 * WN * KG, BM * BN / WN > 16384 ? 1 : 2) void linear_tile(LinearArgs a, uint32_t tiles_m,
                                                                                           uint32_t tiles_n) {
    constexpr int THREADS = 128 * WN * KG, WB = BN / WN;  // KG times 2 x WN waves, of WB columns each
    constexpr int MI = BM / 64, NI = WB / 32;         // 32 x 32 blocks of a wave
    constexpr int CH = BK / 8;                        // chunks of a row
    constexpr int STAGE = (BM + BN) * BK * 2;         // bytes of a tile
    constexpr int NL = (BM + BN) * CH / THREADS;        // loads of a thread for a tile
    constexpr int PITCH = WB + 4;                     // floats of a row in the epilogue
    constexpr int ROWS_END = 2 * WN * 32 * PITCH * 4;  // bytes of those rows; after them, the other groups' sums
    static_assert(ROWS_END + (KG - 1) * 2 * WN * MI * NI * 4096 <= ST * STAGE, "the epilogue's data fits the buffers");
    typedef typename Vec8<T>::type V;
    __shared__ __align__(1024) unsigned char lds[ST * STAGE];
    __shared__ __align__(16) float bias[BN];

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
    for (uint32_t i = tid; i < BN; i += THREADS)
        bias[i] = a.bias && n0 + i < a.n ? (float)((const T *)a.bias)[n0 + i] : 0.0f;

    // this thread's chunks: rows 0..BM-1 are x's, BM.. are w's; rows past the
    // end repeat the last one, their results are not stored
    const char *xb = (const char *)((const T *)a.x + m0 * a.ldx), *wb = (const char *)((const T *)a.w + (uint64_t)n0 * a.ldw);
    auto chunk = [&](int i) { return (i * THREADS + tid) % CH ^ swizzle<BK>((i * THREADS + tid) / CH); };
    uint32_t off[NL];
#pragma unroll
    for (int i = 0; i < NL; i++) {
        const uint32_t row = (i * THREADS + tid) / CH;
        off[i] = (row < (uint32_t)BM ? (uint32_t)(min((uint64_t)row, a.m - 1 - m0) * a.ldx)
                                     : (uint32_t)(min(row - BM, a.n - 1 - n0) * a.ldw)) * 2 + chunk(i) * 16;
    }
    const uint32_t lds0 = lds_addr(lds) + any_wave * 1024;
    const uint32_t steps = (a.k + BK - 1) / BK;
    auto load_one = [&](uint32_t step, int i) {
        constexpr int XL = BM * CH / THREADS;
        const uint32_t k0 = step * BK;
        const char *base = (i < XL ? xb : wb) + (uint64_t)k0 * 2;
        const uint32_t to = __builtin_amdgcn_readfirstlane(lds0 + step % ST * STAGE + i * THREADS * 16);
        if (k0 + BK <= a.k) lds_load16(base, off[i], to);
        else lds_load16(base, k0 + chunk(i) * 8 < a.k ? off[i] : off[i] - chunk(i) * 16, to);  // cleared in arrive()
    };
    auto load = [&](uint32_t step) {
#pragma unroll
        for (int i = 0; i < NL; i++) load_one(step, i);
    };

    v16f acc[NI][MI];
#pragma unroll
    for (int n = 0; n < NI; n++)
#pragma unroll
        for (int m = 0; m < MI; m++)
#pragma unroll
            for (int e = 0; e < 16; e++) acc[n][m][e] = 0.0f;

    const uint32_t mrow = (wave & 1) * (BM / 2) + lo, nrow = BM + (wave >> 1) * WB + lo;
    constexpr int KK = BK / 16 / KG;  // of a tile, for each group
    V x[2][MI], w[2][NI];
    auto read = [&](uint32_t step, int k, V(&xs)[MI], V(&ws)[NI]) {
        const uint32_t kk = kg * KK + k;
        const unsigned char *buf = lds + step % ST * STAGE;
#pragma unroll
        for (int n = 0; n < NI; n++) {
            const uint32_t r = nrow + n * 32;
            ws[n] = *(const V *)(buf + r * BK * 2 + (((kk * 2 + hi) ^ swizzle<BK>(r)) * 16));
        }
#pragma unroll
        for (int m = 0; m < MI; m++) {
            const uint32_t r = mrow + m * 32;
            xs[m] = *(const V *)(buf + r * BK * 2 + (((kk * 2 + hi) ^ swizzle<BK>(r)) * 16));
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
                if (step * BK + chunk(i) * 8 >= a.k)
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
    if (KG > 1) {  // the groups' sums, in their order
        float *sums = (float *)(lds + ROWS_END) + (wave * 64 + lane) * 4;
        constexpr int QUADS = MI * NI * 4, GROUP = 2 * WN * 64 * 4;  // floats from a quad to the next
        if (kg)
#pragma unroll
            for (int i = 0; i < QUADS; i++) {
                const v16f &f = acc[i / 4 / MI][i / 4 % MI];
                *(v4f *)(sums + ((kg - 1) * QUADS + i) * GROUP) = v4f{f[i % 4 * 4], f[i % 4 * 4 + 1], f[i % 4 * 4 + 2], f[i % 4 * 4 + 3]};
            }
        __syncthreads();
        if (kg) return;
#pragma unroll
        for (int g = 0; g < KG - 1; g++)
#pragma unroll
            for (int i = 0; i < QUADS; i++) {
                const v4f f = *(const v4f *)(sums + (g * QUADS + i) * GROUP);
#pragma unroll
                for (int e = 0; e < 4; e++) acc[i / 4 / MI][i / 4 % MI][i % 4 * 4 + e] += f[e];
            }
    }

    // Results by rows: 32 of a wave's rows at a time go through LDS as 32-bit
    // floats, so that residuals are read and results written 16 bytes a lane
    // along the rows.
    float *rows32 = (float *)lds + wave * 32 * PITCH;
    const uint32_t nw = (wave >> 1) * WB;
#pragma unroll
    for (int m = 0; m < MI; m++) {
#pragma unroll
        for (int n = 0; n < NI; n++)
#pragma unroll
            for (int q = 0; q < 4; q++) {
                const uint32_t col = n * 32 + q * 8 + hi * 4;
                *(v4f *)(rows32 + lo * PITCH + col) =
                    v4f{acc[n][m][q * 4], acc[n][m][q * 4 + 1], acc[n][m][q * 4 + 2], acc[n][m][q * 4 + 3]};
            }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the wave's own rows
        const uint64_t mw = m0 + (wave & 1) * (BM / 2) + m * 32;
        for (int i = 0; i < 32 * WB / 8 / 64; i++) {
            const uint32_t idx = i * 64 + lane, row = idx / (WB / 8), col = idx % (WB / 8) * 8;
            float f[8];
            *(v4f *)f = *(const v4f *)(rows32 + row * PITCH + col);
            *(v4f *)(f + 4) = *(const v4f *)(rows32 + row * PITCH + col + 4);
            float b[8];
            *(v4f *)b = *(const v4f *)(bias + nw + col);
            *(v4f *)(b + 4) = *(const v4f *)(bias + nw + col + 4);
#pragma unroll
            for (int e = 0; e < 8; e++) f[e] += b[e];
            activate8(f, a.act);
            if (mw + row < a.m && n0 + nw + col < a.n) finish8<O>(a, mw + row, n0 + nw + col, f);
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
}

// --------------------------------------------------------------- few rows --
// Up to 16 * MF rows of x (one question, a few): w is read once, straight into
// the matrix instructions' registers, 16 of its rows a workgroup; the waves
// split k and join their sums in LDS.  Bound by latency: a wave waits for four
// steps' loads before it starts the next four, and 32 x 4096 x 4096 reads its 33.6
// MB of w in 13.6 us, 2.5 TB/s; 9 x 384 x 1536 3.5, one chain.
constexpr uint32_t ROW_WAVES = 8;
template <class T, class O, int MF>
__global__ __launch_bounds__(ROW_WAVES * 64) void linear_rows(LinearArgs a) {
    typedef typename Vec8<T>::type V;
    typedef typename Vec8<T>::unaligned VU;
    constexpr uint32_t waves = ROW_WAVES;
    __shared__ __align__(16) float red[waves * MF * 256];
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t n0 = blockIdx.x * 16, lo = lane & 15, kc = lane >> 4 << 3;
    const T *w = (const T *)a.w + (uint64_t)min(n0 + lo, a.n - 1) * a.ldw + kc;
    const T *x[MF];
    v4f acc[MF];
#pragma unroll
    for (int m = 0; m < MF; m++) {
        x[m] = (const T *)a.x + min((uint64_t)m * 16 + lo, a.m - 1) * a.ldx + kc;
        acc[m] = v4f{0, 0, 0, 0};
    }
    const uint32_t steps = a.k / 32, each = (steps + waves - 1) / waves;
    const uint32_t s0 = min(steps, wave * each), s1 = min(steps, s0 + each);
    uint32_t s = s0;
    for (; s + 4 <= s1; s += 4) {  // four steps' loads in flight
        V wv[4], xv[4][MF];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            wv[i] = *(const VU *)(w + (s + i) * 32);
#pragma unroll
            for (int m = 0; m < MF; m++) xv[i][m] = *(const VU *)(x[m] + (s + i) * 32);
        }
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int m = 0; m < MF; m++) acc[m] = mfma16(wv[i], xv[i][m], acc[m]);
    }
    for (; s < s1; s++) {
        const V wv = *(const VU *)(w + s * 32);
#pragma unroll
        for (int m = 0; m < MF; m++) acc[m] = mfma16(wv, (V) * (const VU *)(x[m] + s * 32), acc[m]);
    }
    if (steps * 32 < a.k && wave == waves - 1) {  // the rest of k, element by element
        const uint32_t k = steps * 32, left = a.k - k;
        V wv, xv;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const T e = w[kc + i < left ? (int64_t)(k + i) : -(int64_t)kc];
            wv[i] = kc + i < left ? e : (T)0.0f;
        }
#pragma unroll
        for (int m = 0; m < MF; m++) {
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const T e = x[m][kc + i < left ? (int64_t)(k + i) : -(int64_t)kc];
                xv[i] = kc + i < left ? e : (T)0.0f;
            }
            acc[m] = mfma16(wv, xv, acc[m]);
        }
    }
#pragma unroll
    for (int m = 0; m < MF; m++) *(v4f *)(red + (wave * MF + m) * 256 + lo * 16 + (lane >> 4) * 4) = acc[m];
    __syncthreads();
    // red[wave][row][column]: eight columns of a row a thread
    for (uint32_t i = threadIdx.x; i < MF * 32; i += waves * 64) {
        float f[8] = {};
        for (uint32_t v = 0; v < waves; v++) {
            const v4f *r = (const v4f *)(red + v * MF * 256 + i * 8);
            const v4f p = r[0], q = r[1];
#pragma unroll
            for (int e = 0; e < 4; e++) f[e] += p[e], f[e + 4] += q[e];
        }
        const uint32_t row = i / 2, n = n0 + i % 2 * 8;
        if (row >= a.m || n >= a.n) continue;
        if (a.bias)
#pragma unroll
            for (int e = 0; e < 8; e++) f[e] += (float)((const T *)a.bias)[min(n + e, a.n - 1)];
        activate8(f, a.act);
        finish8<O>(a, row, n, f);
    }
}

// ---------------------------------------------------------------- packing --
// Rows for linear_tile, which loads 16 bytes at 16-byte addresses: k rounded
// up to 8 with zeros.
template <class T>
__global__ __launch_bounds__(256) void pack_rows(const T *x, uint64_t ldx, uint32_t k, uint32_t chunks, uint64_t count, T *y) {
    const uint64_t step = (uint64_t)gridDim.x * 256;
    for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < count; i += step) {
        const uint64_t row = i / chunks;
        const uint32_t at = (uint32_t)(i - row * chunks) * 8;
        const T *p = x + row * ldx + at;
        typename Vec8<T>::type v;
        if (at + 8 <= k) {
            v = *(const typename Vec8<T>::unaligned *)p;
        } else {
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const T z = p[at + e < k ? e : 0];
                v[e] = at + e < k ? z : (T)0.0f;
            }
        }
        *(typename Vec8<T>::type *)(y + i * 8) = v;
    }
}

// Rows up to which w goes straight to the registers: 32 rows, 4096 x 4096: 15.8
// us, by tiles 17.7; 64 rows 21.7 and 19.2.
constexpr uint64_t FEW_ROWS = 32;
// A tile's loads have 32-bit offsets: 256 rows of as many elements reach 2^31
// bytes.  Rows further apart are packed, longer rows go 32 at a time.
constexpr uint64_t FAR_ROWS = 1u << 22;

bool aligned(const void *p, uint64_t ld) { return (uintptr_t)p % 16 == 0 && ld % 8 == 0; }
bool by_rows(const LinearArgs &a) { return a.m <= FEW_ROWS || a.k >= FAR_ROWS; }
bool packs(const LinearArgs &a, const void *p, uint64_t ld) {
    return !by_rows(a) && a.k && (a.k % 8 || !aligned(p, ld) || ld >= FAR_ROWS);
}
uint64_t packed_bytes(uint64_t rows, uint32_t k) { return (rows * ((k + 7) / 8) * 16 + 255) & ~255ull; }

template <class T>
hipError_t pack(const void *&p, uint64_t &ld, uint64_t rows, uint32_t k, void *to, hipStream_t s) {
    const uint32_t chunks = (k + 7) / 8;
    const uint64_t count = rows * chunks;
    pack_rows<T><<<(uint32_t)std::min<uint64_t>((count + 255) / 256, 8192), 256, 0, s>>>((const T *)p, ld, k, chunks, count, (T *)to);
    p = to;
    ld = (uint64_t)chunks * 8;
    return hipGetLastError();
}

// Workgroups of a launch: of 2^32 threads and more it runs the low 32 bits, so
// with up to 1024 a workgroup more work is launched in pieces.
constexpr uint32_t GRID_MOST = 1u << 21;

// The part of a call that makes rows m to m + rows and columns n to n + cols.
template <class T, class O>
LinearArgs part_of(const LinearArgs &a, uint64_t m, uint64_t rows, uint64_t n, uint64_t cols) {
    LinearArgs b = a;
    b.m = std::min(a.m - m, rows);
    b.n = (uint32_t)std::min(a.n - n, cols);
    b.x = (const T *)a.x + m * a.ldx;
    b.w = (const T *)a.w + n * a.ldw;
    b.y = (O *)a.y + m * a.ldy + n;
    if (a.bias) b.bias = (const T *)a.bias + n;
    if (a.residual) b.residual = (const O *)a.residual + m * a.ldr + n;
    return b;
}

template <class T, class O, int BM, int BN, int WN, int BK, int ST, int KG = 1>
hipError_t tile_of(const LinearArgs &a, hipStream_t s) {
    static_assert(128 * WN * KG <= 1024, "GRID_MOST is for 1024 threads");
    for (uint64_t n = 0; n < a.n; n += (uint64_t)GRID_MOST * BN) {
        const uint32_t tn = (uint32_t)((std::min<uint64_t>(a.n - n, (uint64_t)GRID_MOST * BN) + BN - 1) / BN);
        const uint64_t most = GRID_MOST / tn;
        for (uint64_t m = 0; m < a.m; m += most * BM) {
            const LinearArgs b = part_of<T, O>(a, m, most * BM, n, (uint64_t)GRID_MOST * BN);
            const uint32_t tm = (uint32_t)((b.m + BM - 1) / BM);
            linear_tile<T, O, BM, BN, WN, BK, ST, KG><<<tm * tn, 128 * WN * KG, 0, s>>>(b, tm, tn);
        }
    }
    return hipGetLastError();
}

template <class T, class O, int MF>
hipError_t rows_of(const LinearArgs &a, hipStream_t s) {
    // 8 waves: k 384 to 4096 within 0.1 us of the best of 4, 8 and 16
    linear_rows<T, O, MF><<<(a.n - 1) / 16 + 1, ROW_WAVES * 64, 0, s>>>(a);
    return hipGetLastError();
}

template <class T, class O>
hipError_t linear_of(LinearArgs a, void *ws, hipStream_t s) {
    if (by_rows(a)) {
        static_assert(ROW_WAVES * 64 <= 1024, "GRID_MOST is for 1024 threads");
        for (uint64_t n = 0; n < a.n; n += GRID_MOST * 16)
            for (uint64_t m = 0; m < a.m; m += FEW_ROWS) {
                const LinearArgs b = part_of<T, O>(a, m, FEW_ROWS, n, GRID_MOST * 16);
                const hipError_t e = b.m <= 16 ? rows_of<T, O, 1>(b, s) : rows_of<T, O, 2>(b, s);
                if (e != hipSuccess) return e;
            }
        return hipSuccess;
    }
    const bool px = packs(a, a.x, a.ldx), pw = packs(a, a.w, a.ldw);
    if (px) {
        const hipError_t e = pack<T>(a.x, a.ldx, a.m, a.k, ws, s);
        if (e != hipSuccess) return e;
        ws = (char *)ws + packed_bytes(a.m, a.k);
    }
    if (pw) {
        const hipError_t e = pack<T>(a.w, a.ldw, a.n, a.k, ws, s);
        if (e != hipSuccess) return e;
    }
    if (a.k % 8) a.k = (a.k + 7) / 8 * 8;
    // The shape that is done first: rounds of the tiles that the card holds at a
    // time, each a + b k long (ns, fitted to 100..32768 x 384..8192 x 384..8192).
    // 2037 x 768 x 768 (k 768): 8.6 us in the first, 11.2 in the second, 14.2 and
    // 24.4 in the others; 4096 x 768: 14.7, 11.9, 14.7, 25.1; 8192 x 768: 23.4, 20.7,
    // 18.5, 26.5; 16384 x 768: 42.9, 34.0, 31.3, 28.2.
    struct {
        uint32_t bm, bn, at_a_time, a, b;
    } const shapes[4] = {{64, 64, 512, 2400, 73}, {128, 128, 256, 4700, 94}, {128, 128, 512, 3600, 174}, {256, 256, 256, 9800, 198}};
    int best = 0;
    uint64_t least = ~0ull;
    for (int i = 0; i < 4; i++) {
        const auto &t = shapes[i];
        const uint64_t tiles = ((a.m + t.bm - 1) / t.bm) * ((a.n + t.bn - 1) / t.bn);
        const uint64_t ns = (tiles + t.at_a_time - 1) / t.at_a_time * (t.a + (uint64_t)t.b * a.k / 10);
        if (ns < least) least = ns, best = i;
    }
    switch (best) {
    case 0:  // four groups where a CU has one tile (300 x 384, k 1536: 8.1 us against 9.5)
        if (a.k >= 1024 && ((a.m + 63) / 64) * ((a.n + 63) / 64) <= 256) return tile_of<T, O, 64, 64, 2, 256, 2, 4>(a, s);
        return tile_of<T, O, 64, 64, 2, 128, 2, 2>(a, s);
    case 1: return tile_of<T, O, 128, 128, 4, 64, 4>(a, s);
    case 2: return tile_of<T, O, 128, 128, 2, 64, 2>(a, s);
    default: return tile_of<T, O, 256, 256, 4, 64, 2>(a, s);
    }
}

}  // namespace

size_t linear_workspace(const LinearArgs &a) {
    return (packs(a, a.x, a.ldx) ? packed_bytes(a.m, a.k) : 0) + (packs(a, a.w, a.ldw) ? packed_bytes(a.n, a.k) : 0);
}

hipError_t launch_linear(const LinearArgs &a, void *ws, hipStream_t s) {
    if (a.dtype == T_F16) return a.out_dtype == T_F32 ? linear_of<f16, float>(a, ws, s) : linear_of<f16, f16>(a, ws, s);
    return a.out_dtype == T_F32 ? linear_of<bf16, float>(a, ws, s) : linear_of<bf16, bf16>(a, ws, s);
}

}  // namespace bvk
