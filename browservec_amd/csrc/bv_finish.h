// What the products of a layer share once their sums are made: activation,
// residual, rounding, store (bv_linear.hip, bv_linear_q8.hip).
#pragma once

#include "bv_embed_device.h"

namespace bvk {
namespace {

// The activations are y * sigmoid(t), with t / log(2) = y q(y^2):
//   SILU       q = log2(e)
//   GELU_TANH  q = log2(e) 2 sqrt(2/pi) (1 + 0.044715 y^2)
//   GELU       Phi(y) = sigmoid(log(Phi(y) / Phi(-y))), whose argument over y is
//              smooth in y^2: a polynomial of degree 6 fitted on |y| <= 5.5 so
//              that the result is within 1.7e-7 max(1, |y|) everywhere (y^2 is
//              clamped past it, where Phi is 0 or 1 to 2e-8)
// One exponential and one reciprocal each: with 64 columns of 32 rows a lane,
// the epilogue's arithmetic is a third of the time of a product with k = 1024
// (erff took as long as the product).
__device__ __forceinline__ float times_sigmoid(float y, float q) {
    return y * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-y * q));
}
__device__ __forceinline__ float gelu(float y) {
    const float u = fminf(y * y, 30.25f);
    float q = 5.209913833681412e-09f;
    q = fmaf(q, u, -3.8504521171489614e-07f);
    q = fmaf(q, u, 1.1452433682279661e-05f);
    q = fmaf(q, u, -1.5938944125082344e-04f);
    q = fmaf(q, u, -9.559283353155479e-05f);
    q = fmaf(q, u, 1.0483857989311218e-01f);
    q = fmaf(q, u, 2.3022072315216064f);
    return times_sigmoid(y, q);
}
__device__ __forceinline__ void activate8(float (&f)[8], int act) {
    switch (act) {  // the same for the whole launch
    case 1:
#pragma unroll
        for (int i = 0; i < 8; i++) f[i] = f[i] < 0.0f ? 0.0f : f[i];
        break;
    case 2:
#pragma unroll
        for (int i = 0; i < 8; i++) f[i] = gelu(f[i]);
        break;
    case 3:
#pragma unroll
        for (int i = 0; i < 8; i++) f[i] = times_sigmoid(f[i], fmaf(f[i] * f[i], 0.10294324f, 2.3022082f));
        break;
    case 4:
#pragma unroll
        for (int i = 0; i < 8; i++) f[i] = times_sigmoid(f[i], 1.44269504f);
        break;
    default: break;
    }
}

// The end of eight neighbouring results of a row, columns n on: residual,
// rounding, store.
template <class O, class Args>
__device__ __forceinline__ void finish8(const Args &a, uint64_t m, uint32_t n, float (&f)[8]) {
    const int left = (int)min(8u, a.n - n);
    if (a.residual) {
        const O *r = (const O *)a.residual + m * a.ldr + n;
        if (left == 8) {
            float g[8];
            load8(r, g);
#pragma unroll
            for (int i = 0; i < 8; i++) f[i] += g[i];
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++) f[i] += (float)r[min(i, left - 1)];
        }
    }
    store8((O *)a.y + m * a.ldy + n, left, f);
}

}  // namespace
}  // namespace bvk
