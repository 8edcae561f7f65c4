// y = act(x w^T + bias) + residual for an embedding model's layers.
#include "bv_embed.h"
#include "bv_embed_device.h"

#include <algorithm>

namespace bvk {
namespace {

__device__ __forceinline__ float activate(float y, int act) {
    switch (act) {
    case 1: return fmaxf(y, 0.0f) + (y != y ? y : 0.0f);
    case 2: return 0.5f * y * (1.0f + erff(y * 0.70710678118654752f));
    case 3: return 0.5f * y * (1.0f + tanhf(0.79788456080286536f * (y + 0.044715f * y * y * y)));
    case 4: return y / (1.0f + expf(-y));
    default: return y;
    }
}

// 16 x 16 results a workgroup, the operands in tiles of 16 through LDS.
template <class T, class O>
__global__ __launch_bounds__(256) void linear_tile(LinearArgs a, uint64_t first) {
    __shared__ float xs[16][17], ws[16][17];
    const uint32_t tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    const uint64_t m0 = first + (uint64_t)blockIdx.y * 16, n0 = (uint64_t)blockIdx.x * 16;
    const T *x = (const T *)a.x, *w = (const T *)a.w;
    float acc = 0;
    for (uint32_t k0 = 0; k0 < a.k; k0 += 16) {
        const bool in = k0 + tx < a.k;
        xs[ty][tx] = in && m0 + ty < a.m ? (float)x[(m0 + ty) * a.ldx + k0 + tx] : 0.0f;
        ws[ty][tx] = in && n0 + ty < a.n ? (float)w[(n0 + ty) * a.ldw + k0 + tx] : 0.0f;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 16; i++) acc = fmaf(xs[ty][i], ws[tx][i], acc);
        __syncthreads();
    }
    const uint64_t m = m0 + ty, n = n0 + tx;
    if (m >= a.m || n >= a.n) return;
    if (a.bias) acc += (float)((const T *)a.bias)[n];
    acc = activate(acc, a.act);
    if (a.residual) acc += (float)((const O *)a.residual)[m * a.ldr + n];
    ((O *)a.y)[m * a.ldy + n] = (O)acc;
}

template <class T, class O>
hipError_t linear_of(const LinearArgs &a, hipStream_t s) {
    for (uint64_t m = 0; m < a.m; m += 16 * 32768) {
        const dim3 grid((a.n + 15) / 16, (uint32_t)std::min<uint64_t>((a.m - m + 15) / 16, 32768));
        linear_tile<T, O><<<grid, 256, 0, s>>>(a, m);
    }
    return hipGetLastError();
}

}  // namespace

hipError_t launch_linear(const LinearArgs &a, hipStream_t s) {
    if (a.dtype == T_F16) return a.out_dtype == T_F32 ? linear_of<f16, float>(a, s) : linear_of<f16, f16>(a, s);
    return a.out_dtype == T_F32 ? linear_of<bf16, float>(a, s) : linear_of<bf16, bf16>(a, s);
}

}  // namespace bvk
