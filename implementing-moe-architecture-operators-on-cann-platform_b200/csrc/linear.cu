// linear.cu -- MoeLinear on sm_100a: a matrix product with bias, activation, gate and
// residual in its epilogue.
//
//   plain: y[t, n] = act(sum_k x[t, k] w[n, k] + bias[n]) + residual[t, n]
//   gated: y[t, n] = act(sum_k x[t, k] w[n, k] + bias[n]) *
//                    (sum_k x[t, k] w[N + n, k] + bias[N + n]) + residual[t, n]
// x [T, K], w [N or 2N, K], fp16 or bf16; sums, bias, activation, product and residual
// are taken in fp32 and rounded once, to the type of y.
#include <cuda_bf16.h>

#include "../../include/moe_ops.h"
#include "moe_common.cuh"
#include "moe_kernels.h"

namespace moe {

__device__ __forceinline__ float lin_act(float z, int act)
{
    switch (act) {
        case MOE_ACT_RELU: return z > 0.0f ? z : (z != z ? z : 0.0f);
        case MOE_ACT_GELU: return z * normcdff(z);
        case MOE_ACT_GELU_TANH: {
            // 0.5 z (1 + tanh(u)) = z / (1 + exp(-2u)), u = sqrt(2/pi) (z + 0.044715 z^3)
            const float u2 = 1.5957691216057308f * (z + 0.044715f * z * z * z);
            return z / (1.0f + expf(-u2));
        }
        case MOE_ACT_SILU: return z / (1.0f + expf(-z));
        case MOE_ACT_SIGMOID: return 1.0f / (1.0f + expf(-z));
        default: return z;
    }
}

__device__ __forceinline__ float lin_load(const void* p, size_t i, int type)
{
    if (type == MOE_DT_FLOAT) return static_cast<const float*>(p)[i];
    if (type == MOE_DT_FLOAT16) return __half2float(static_cast<const __half*>(p)[i]);
    return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}
__device__ __forceinline__ void lin_store(void* p, size_t i, float v, int type)
{
    if (type == MOE_DT_FLOAT)
        static_cast<float*>(p)[i] = v;
    else if (type == MOE_DT_FLOAT16)
        static_cast<__half*>(p)[i] = __float2half_rn(v);
    else
        static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
}

constexpr int LS_TILE = 64;
constexpr int LS_BK = 16;

// 64 x 64 outputs per block, 4 x 4 per thread, operands through shared memory.
__global__ void __launch_bounds__(256) linear_simple_kernel(const LinearArgs a)
{
    __shared__ float sx[LS_BK][LS_TILE + 1];
    __shared__ float sw[2][LS_BK][LS_TILE + 1];
    pdl_wait();
    const int t0 = blockIdx.y * LS_TILE, n0 = blockIdx.x * LS_TILE;
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    float acc[2][4][4] = {};
    const int parts = a.gated ? 2 : 1;
    for (int k0 = 0; k0 < a.K; k0 += LS_BK) {
        for (int i = threadIdx.x; i < LS_TILE * LS_BK; i += 256) {
            const int r = i / LS_BK, k = i % LS_BK;
            const bool kin = k0 + k < a.K;
            sx[k][r] = (kin && t0 + r < a.T) ? lin_load(a.x, (size_t)(t0 + r) * a.ldx + k0 + k, a.type) : 0.0f;
            for (int p = 0; p < parts; p++)
                sw[p][k][r] = (kin && n0 + r < a.N)
                                  ? lin_load(a.w, ((size_t)p * a.N + n0 + r) * a.ldw + k0 + k, a.type) : 0.0f;
        }
        __syncthreads();
        for (int k = 0; k < LS_BK; k++)
            for (int p = 0; p < parts; p++)
#pragma unroll
                for (int i = 0; i < 4; i++)
#pragma unroll
                    for (int j = 0; j < 4; j++) acc[p][i][j] += sx[k][ty * 4 + i] * sw[p][k][tx + 16 * j];
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int t = t0 + ty * 4 + i, n = n0 + tx + 16 * j;
            if (t >= a.T || n >= a.N) continue;
            float z = acc[0][i][j] + (a.bias ? lin_load(a.bias, n, a.type) : 0.0f);
            float v = lin_act(z, a.act);
            if (a.gated) v *= acc[1][i][j] + (a.bias ? lin_load(a.bias, (size_t)a.N + n, a.type) : 0.0f);
            if (a.residual) v += lin_load(a.residual, (size_t)t * a.ldr + n, a.otype);
            lin_store(a.y, (size_t)t * a.ldy + n, v, a.otype);
        }
}

cudaError_t launch_linear(const LinearArgs& a, cudaStream_t s)
{
    const dim3 grid((unsigned)((a.N + LS_TILE - 1) / LS_TILE), (unsigned)((a.T + LS_TILE - 1) / LS_TILE));
    return launch_pdl(linear_simple_kernel, grid, dim3(256), 0, s, a);
}

}  // namespace moe
