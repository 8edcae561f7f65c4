// Launchers of an embedding model's operators (bv_linear.hip, bv_linear_q8.hip,
// bv_attention.hip, bv_rows.hip, bv_add_norm.hip), called by bv_embed.cpp with checked arguments: every stride is
// set, sizes fit the types below.  Strides are in elements.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace bvk {

enum { T_F32 = 0, T_F16 = 1, T_BF16 = 2 };  // BV_F32, BV_F16, BV_BF16

// ---------------------------------------------------------------- linear --
struct LinearArgs {
    int dtype, out_dtype, act;
    uint64_t m;
    uint32_t n, k;
    const void *x, *w, *bias, *residual;
    void *y;
    uint64_t ldx, ldw, ldr, ldy;
};
// Bytes of workspace that a call needs (rows laid out for the matrix cores).
size_t linear_workspace(const LinearArgs &a);
hipError_t launch_linear(const LinearArgs &a, void *ws, hipStream_t s);

// ------------------------------------------------------------- linear_q8 --
// Sums of k products of codes, each at most 2^14, stay below 2^31.
constexpr uint32_t LINEAR_Q8_MAX_K = 131071;
struct LinearQ8Args {
    int out_dtype, act, bias_dtype;
    uint64_t m;
    uint32_t n, k;
    const int8_t *x, *w;
    const float *x_scales, *w_scales;
    const void *bias, *residual;
    void *y;
    uint64_t ldx, ldw, ldr, ldy;
    bool once;  // the launcher's: y goes past the caches
};
// Bytes of workspace that a call needs (rows laid out for the matrix cores).
size_t linear_q8_workspace(const LinearQ8Args &a);
hipError_t launch_linear_q8(const LinearQ8Args &a, void *ws, hipStream_t s);

// ------------------------------------------------------------- attention --
struct AttentionArgs {
    int dtype, causal;
    uint32_t hq, hk, d, batch, max_q, max_k;
    float scale;
    uint64_t tq, tk;
    const void *q, *k, *v;
    void *o;
    const int32_t *cu_q, *cu_k;
    uint64_t sq, sqh, sk, skh, sv, svh, so, soh;  // token and head strides
    const void *zeros;                            // 16 bytes of zeros
    int local;  // a query sees `left` keys before its place, `right` after it and the first `sinks`
    uint32_t left, right, sinks;                  // at most 2^31 - 1
};
// Bytes of workspace that a call needs (partial results of split keys).
size_t attention_workspace(const AttentionArgs &a);
hipError_t launch_attention(const AttentionArgs &a, void *ws, hipStream_t s);
hipError_t launch_attention_local(const AttentionArgs &a, void *ws, hipStream_t s);

// ------------------------------------------------------------------ rows --
struct RotaryArgs {
    int dtype, interleaved;
    uint32_t hq, hk, d, rot, rows;
    uint64_t tokens;
    const float *table;
    const int32_t *pos;
    const void *q, *k;
    void *qo, *ko;
    uint64_t sq, sqh, sk, skh, sqo, sqoh, sko, skoh;
};
hipError_t launch_rotary(const RotaryArgs &a, hipStream_t s);

constexpr uint32_t NORM_MAX_DIM = 16384;
struct NormArgs {
    int dtype, out_dtype, wtype, norm, pool, unit;
    uint32_t batch, dim;
    float eps;
    uint64_t tokens;
    const void *x, *w, *b;
    const int32_t *cu;
    void *y;
    uint64_t ldx, ldy;
    float *part;  // mean pooling: partial sums, pool_chunks() rows of dim floats
};
// Workgroups that sum a chunk of one sequence's rows each: rows of NormArgs::part.
uint64_t pool_chunks(uint64_t tokens, uint32_t batch);
hipError_t launch_norm(const NormArgs &a, hipStream_t s);

// Norm of x, or of x + r, to a float type or to codes of 8 bits and scales.
enum { T_I8 = 3 };  // BV_I8
struct AddNormArgs {
    int dtype, r_dtype, out_dtype, wtype, norm;
    uint32_t dim;
    float eps;
    uint64_t tokens;
    const void *x, *r, *w, *b;
    void *total, *y;
    float *scales;
    uint64_t ldx, ldr, ldt, ldy;
    bool once;  // the launcher's: x and r are read past the caches
};
hipError_t launch_add_norm(const AddNormArgs &a, hipStream_t s);

}  // namespace bvk
