// select.cu -- MoeRouterSelect on sm_100a: router logits -> expert ids and weights.
//
// Per token, with logits l[0..E):
//   score   s_e = exp(l_e) / sum_j exp(l_j)   or   1 / (1 + exp(-l_e))
//   key     k_e = s_e + bias_e (no bias: k_e = s_e)
//   groups  E experts in G consecutive groups; a group's value is its largest key,
//           or the sum of its two largest; the topG best groups stay
//   ids     the K largest keys of the groups that stay, larger first, ties to the
//           lower id
//   weight  w = s (not k), divided by the sum over the K chosen when renormalising,
//           times scale
// An expert is closed when its logit or its bias is -inf or NaN, or its group did not
// stay.  Closed experts fill the slots that no open expert is left for, in ascending id
// order, with weight 0.
//
// The choice is that of keys in 64 bits: two scores may lie closer together than 32
// bits tell apart, and the id is a whole number that is right or wrong.  Without a bias
// scores order as their logits do, so the logits themselves are the keys.
#include <math_constants.h>

#include <cuda_bf16.h>

#include "../../include/moe_ops.h"
#include "moe_common.cuh"
#include "moe_kernels.h"

namespace moe {

constexpr int SEL_MAX_E = 256;
constexpr int SEL_MAX_G = 32;
constexpr int SEL_WARPS = 4;

__device__ __forceinline__ float sel_load(const float* p, int i) { return p[i]; }
__device__ __forceinline__ float sel_load(const __half* p, int i) { return __half2float(p[i]); }
__device__ __forceinline__ float sel_load(const __nv_bfloat16* p, int i) { return __bfloat162float(p[i]); }

// false for -inf and NaN
__device__ __forceinline__ bool sel_open(float v) { return v > -CUDART_INF_F; }

__device__ __forceinline__ float warp_max(float v)
{
    for (int d = 16; d; d >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, d));
    return v;
}
__device__ __forceinline__ float warp_sum(float v)
{
    for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    return v;
}

struct ExactScratch {
    double key[SEL_MAX_E];
    double group[SEL_MAX_G];
};

// The K chosen experts of one token, by one warp, with keys in 64 bits.  Lane r < K
// gets slot r's expert; `closed` tells whether that slot had no open expert left.
template <typename LT>
__device__ __noinline__ int select_exact(const SelectArgs& a, const LT* row, ExactScratch& s, bool& closed)
{
    const int lane = threadIdx.x & 31;
    const int E = a.E, size = a.E / a.G;
    const double NINF = -CUDART_INF;
    // keys: the logits order like their scores, so scores are only needed where they
    // are added to something
    const bool use_score = a.bias != nullptr || (a.G > 1 && a.groupTop > 1);
    float mx = -CUDART_INF_F;
    double total = 0.0;
    if (use_score && !a.sigmoid) {
        for (int e = lane; e < E; e += 32) {
            const float l = sel_load(row, e);
            if (sel_open(l)) mx = fmaxf(mx, l);
        }
        mx = warp_max(mx);
        for (int e = lane; e < E; e += 32) {
            const float l = sel_load(row, e);
            if (sel_open(l)) total += l == mx ? 1.0 : exp((double)l - (double)mx);
        }
        for (int d = 16; d; d >>= 1) total += __shfl_xor_sync(0xffffffffu, total, d);
    }
    for (int e = lane; e < E; e += 32) {
        const float l = sel_load(row, e);
        double k = NINF;
        if (sel_open(l)) {
            k = (double)l;
            if (use_score) {
                k = a.sigmoid ? 1.0 / (1.0 + exp(-(double)l)) : (l == mx ? 1.0 : exp((double)l - (double)mx)) / total;
                if (a.bias) {
                    const float b = a.bias[e];
                    k = sel_open(b) ? k + (double)b : NINF;
                }
            }
        }
        s.key[e] = k;
    }
    __syncwarp();
    if (a.G > 1) {
        if (lane < a.G) {
            double m1 = NINF, m2 = NINF;
            for (int i = 0; i < size; i++) {
                const double k = s.key[lane * size + i];
                m2 = fmax(m2, fmin(m1, k));
                m1 = fmax(m1, k);
            }
            s.group[lane] = (a.groupTop > 1 && m2 > NINF) ? m1 + m2 : m1;
        }
        __syncwarp();
        bool drop = false;
        if (lane < a.G) {
            const double v = s.group[lane];
            int before = 0;
            for (int g = 0; g < a.G; g++) before += (s.group[g] > v || (s.group[g] == v && g < lane)) ? 1 : 0;
            drop = before >= a.topG;
        }
        const unsigned dropped = __ballot_sync(0xffffffffu, drop);
        for (int e = lane; e < E; e += 32)
            if ((dropped >> (e / size)) & 1u) s.key[e] = NINF;
        __syncwarp();
    }
    // K times the largest key, lowest id first; a taken expert's key becomes NaN
    int mine = 0;
    closed = false;
    for (int r = 0; r < a.K; r++) {
        double best = NINF;
        int at = SEL_MAX_E;
        for (int e = lane; e < E; e += 32) {
            const double k = s.key[e];
            if (k > best || (k == best && e < at)) {
                best = k;
                at = e;
            }
        }
        for (int d = 16; d; d >>= 1) {
            const double ob = __shfl_xor_sync(0xffffffffu, best, d);
            const int oa = __shfl_xor_sync(0xffffffffu, at, d);
            if (ob > best || (ob == best && oa < at)) {
                best = ob;
                at = oa;
            }
        }
        if (lane == r) {
            mine = at;
            closed = best == NINF;
        }
        if (lane == (at & 31)) s.key[at] = CUDART_NAN;
        __syncwarp();
    }
    return mine;
}

// The weight of this lane's slot (lanes >= K return 0).  mx, total: softmax maximum and
// sum over the row (used without renormalisation only).
//   renormalised softmax: e^(l - m) / sum, m the largest chosen logit
//   renormalised sigmoid: s_k / sum s = r_k / sum r with r = e^(l - c) / (1 + e^l)
//     (l <= 0) or e^(-c) / (1 + e^-l) (l > 0) and c = min(0, largest chosen logit): no
//     common factor underflows, however small the scores are.
__device__ __forceinline__ float sel_weight(const SelectArgs& a, float l, bool open, float mx, float total)
{
    float w = 0.0f;
    if (a.renorm) {
        const float top = warp_max(open ? l : -CUDART_INF_F);
        if (open) {
            if (a.sigmoid) {
                const float c = fminf(0.0f, top);
                w = l > 0.0f ? 1.0f / (1.0f + expf(-l)) : expf(l - c) / (1.0f + expf(l));
            } else {
                w = l == top ? 1.0f : expf(l - top);
            }
        }
        const float sum = warp_sum(w);
        if (open) w = w / sum;
    } else if (open) {
        w = a.sigmoid ? 1.0f / (1.0f + expf(-l)) : (l == mx ? 1.0f : expf(l - mx)) / total;
    }
    return w * a.scale;
}

template <typename LT>
__global__ void __launch_bounds__(SEL_WARPS * 32) select_kernel(const SelectArgs a)
{
    __shared__ ExactScratch scratch[SEL_WARPS];
    pdl_trigger();
    pdl_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int t = blockIdx.x * SEL_WARPS + warp;
    if (t >= a.T) return;
    const LT* row = static_cast<const LT*>(a.logits) + (size_t)t * a.ldl;
    bool closed;
    const int e = select_exact<LT>(a, row, scratch[warp], closed);
    float mx = -CUDART_INF_F, total = 0.0f;
    if (!a.sigmoid && !a.renorm) {
        for (int i = lane; i < a.E; i += 32) {
            const float l = sel_load(row, i);
            if (sel_open(l)) mx = fmaxf(mx, l);
        }
        mx = warp_max(mx);
        for (int i = lane; i < a.E; i += 32) {
            const float l = sel_load(row, i);
            if (sel_open(l)) total += l == mx ? 1.0f : expf(l - mx);
        }
        total = warp_sum(total);
    }
    const bool open = lane < a.K && !closed;
    const float w = sel_weight(a, open ? sel_load(row, e) : 0.0f, open, mx, total);
    if (lane < a.K) {
        const size_t o = (size_t)t * a.K + lane;
        a.ids[o] = e;
        if (a.wtype == MOE_DT_FLOAT)
            static_cast<float*>(a.weights)[o] = w;
        else
            static_cast<__half*>(a.weights)[o] = __float2half_rn(w);
    }
}

cudaError_t launch_select(const SelectArgs& a, int ltype, cudaStream_t s)
{
    const dim3 grid((unsigned)((a.T + SEL_WARPS - 1) / SEL_WARPS)), block(SEL_WARPS * 32);
    if (ltype == MOE_DT_FLOAT) return launch_pdl(select_kernel<float>, grid, block, 0, s, a);
    if (ltype == MOE_DT_FLOAT16) return launch_pdl(select_kernel<__half>, grid, block, 0, s, a);
    return launch_pdl(select_kernel<__nv_bfloat16>, grid, block, 0, s, a);
}

}  // namespace moe
