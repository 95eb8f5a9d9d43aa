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

// ---------------------------------------------------------------------- fast path
// LPT lanes per token (8: four tokens to a warp, 32: one).  Group g belongs to L = LPT / G'
// lanes, G' the next power of two; each holds up to C consecutive experts of it.  A key is
// one fp32 number whose lowest 8 bits give way to 255 - e, so that sorting and comparing move
// one register per expert.  What that rounding, or the fast exp and quotient, may have turned
// around is noticed: neighbours among the K + 1 best, or a group that stays and one that does
// not, closer than the bounds below send the token to select_exact.  About one token in a
// hundred goes there, and so do those with too few open experts.
// Closed experts have the key -inf; open ones a finite one (+-SEL_MAX at most).
constexpr float SEL_MAX = 3.4028235e38f;
#define SEL_NINF (-CUDART_INF_F)

template <int LPT>
__device__ __forceinline__ float sub_max(float v)
{
    if constexpr (LPT == 32) {
        float r;
        asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
        return r;
    }
#pragma unroll
    for (int d = LPT / 2; d; d >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, d));
    return v;
}
template <int LPT>
__device__ __forceinline__ float sub_sum(float v)
{
#pragma unroll
    for (int d = LPT / 2; d; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    return v;
}

__device__ __forceinline__ void sel_order(float& a, float& b)  // a >= b afterwards
{
    const float hi = fmaxf(a, b), lo = fminf(a, b);
    a = hi;
    b = lo;
}

// Sorts v[0..N) in descending order (Batcher's odd-even merge sort).
template <int N>
__device__ __forceinline__ void sel_sort(float* v)
{
#pragma unroll
    for (int p = 1; p < N; p *= 2)
#pragma unroll
        for (int k = p; k >= 1; k /= 2)
#pragma unroll
            for (int j = k % p; j + k < N; j += 2 * k)
#pragma unroll
                for (int i = 0; i < k; i++)
                    if (i + j + k < N && (i + j) / (2 * p) == (i + j + k) / (2 * p)) sel_order(v[i + j], v[i + j + k]);
}

// a[0..8) becomes the 8 largest of a and b (both descending), descending.
__device__ __forceinline__ void sel_merge8(float* a, const float* b)
{
#pragma unroll
    for (int i = 0; i < 8; i++) a[i] = fmaxf(a[i], b[7 - i]);  // a bitonic sequence of the 8 largest
#pragma unroll
    for (int d = 4; d; d >>= 1)
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (!(i & d)) sel_order(a[i], a[i + d]);
}

// The weight of this lane's slot (lanes whose slot does not exist or is closed return 0).
// mx, total: softmax maximum and sum over the row (used without renormalisation only).
//   renormalised softmax: e^(l - m) / sum, m the largest chosen logit
//   renormalised sigmoid: s_k / sum s = r_k / sum r with r = e^(l - c) / (1 + e^l)
//     (l <= 0) or e^(-c) / (1 + e^-l) (l > 0) and c = min(0, largest chosen logit): no
//     common factor underflows, however small the scores are.
template <int LPT>
__device__ __forceinline__ float sel_weight(const SelectArgs& a, float l, bool open, float mx, float total)
{
    float w = 0.0f;
    if (a.renorm) {
        const float top = sub_max<LPT>(open ? l : -CUDART_INF_F);
        if (open) {
            if (a.sigmoid) {
                const float c = fminf(0.0f, top);
                w = l > 0.0f ? 1.0f / (1.0f + expf(-l)) : expf(l - c) / (1.0f + expf(l));
            } else {
                w = l == top ? 1.0f : expf(l - top);
            }
        }
        const float sum = sub_sum<LPT>(w);
        if (open) w = w / sum;
    } else if (open) {
        w = a.sigmoid ? 1.0f / (1.0f + expf(-l)) : (l == mx ? 1.0f : expf(l - mx)) / total;
    }
    return w * a.scale;
}

// Position of expert e in a staged row: 4 floats of padding after every 32, so that lanes
// that read 16 bytes at strides of 4, 8, 16 or 32 floats meet different banks.
__device__ __forceinline__ int sel_at(int e) { return e + ((e >> 5) << 2); }
constexpr int SEL_ROW = SEL_MAX_E + SEL_MAX_E / 32 * 4;

// A row of logits into shared memory as floats, NaN as -inf, by the LPT lanes of a token.
template <int LPT, typename LT>
__device__ __forceinline__ void sel_stage(const LT* row, float* dst, int E, int sub, bool vec)
{
    constexpr int V = 16 / (int)sizeof(LT);
    if (vec) {
        constexpr int MAXV = SEL_MAX_E / V / LPT;  // 16-byte pieces per lane
        uint4 q[MAXV];
#pragma unroll
        for (int i = 0; i < MAXV; i++) {
            const int e = (i * LPT + sub) * V;
            if (e < E) q[i] = *reinterpret_cast<const uint4*>(row + e);
        }
#pragma unroll
        for (int i = 0; i < MAXV; i++) {
            const int e = (i * LPT + sub) * V;
            if (e < E) {
                const LT* x = reinterpret_cast<const LT*>(&q[i]);
#pragma unroll
                for (int j = 0; j < V; j += 4)
                    *reinterpret_cast<float4*>(dst + sel_at(e + j)) =
                        make_float4(fmaxf(sel_load(x, j), -CUDART_INF_F), fmaxf(sel_load(x, j + 1), -CUDART_INF_F),
                                    fmaxf(sel_load(x, j + 2), -CUDART_INF_F), fmaxf(sel_load(x, j + 3), -CUDART_INF_F));
            }
        }
    } else {
#pragma unroll 8
        for (int e = sub; e < E; e += LPT) dst[sel_at(e)] = fmaxf(sel_load(row, e), -CUDART_INF_F);
    }
}

struct SelectPlan {
    int lanes_shift;  // log2 of the lanes per group
    int per_lane;     // experts per lane, at most C
    bool whole;       // per_lane == C everywhere: 16-byte reads of the staged row
    bool vec;         // rows of logits start on 16-byte boundaries and hold whole 16 bytes
    bool by_logit;    // no bias and no sums of scores: the logits order as their scores do
};

template <typename LT, int LPT, int C>
__global__ void __launch_bounds__(SEL_WARPS * 32, C == 32 ? 4 : 6) select_kernel(const SelectArgs a, const SelectPlan p)
{
    constexpr int TPW = 32 / LPT;  // tokens per warp
    constexpr int KEEP = C < 8 ? C : 8;
    constexpr bool EXACT16 = sizeof(LT) == 2;  // a 16-bit logit is whole in the upper 24 bits
    __shared__ __align__(16) float rows[SEL_WARPS][TPW][SEL_ROW];
    __shared__ __align__(16) float sbias[SEL_ROW];
    __shared__ ExactScratch scratch[SEL_WARPS];
    pdl_trigger();
    pdl_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int sub = lane & (LPT - 1), tok = lane / LPT;
    if (a.bias) {
        for (int e = threadIdx.x; e < a.E; e += SEL_WARPS * 32) sbias[sel_at(e)] = fmaxf(a.bias[e], -CUDART_INF_F);
        __syncthreads();
    }
    const int size = a.E / a.G;
    const int grp = sub >> p.lanes_shift;
    const int first = grp * size + (sub & ((1 << p.lanes_shift) - 1)) * p.per_lane;
    const int mine = grp < a.G ? max(0, min(p.per_lane, (grp + 1) * size - first)) : 0;
    const int step = gridDim.x * SEL_WARPS * TPW;
    float* const row = rows[warp][tok];
    for (int t0 = (blockIdx.x * SEL_WARPS + warp) * TPW; t0 < a.T; t0 += step) {
        const int t = min(t0 + tok, a.T - 1);  // the last warp's spare tokens repeat the last one
        const LT* src = static_cast<const LT*>(a.logits) + (size_t)t * a.ldl;
        sel_stage<LPT, LT>(src, row, a.E, sub, p.vec);
        __syncwarp();
        // ---- keys
        float v[C];
        if (p.whole) {
#pragma unroll
            for (int i = 0; i < C; i += 4) {
                const float4 q = *reinterpret_cast<const float4*>(row + sel_at(first + i));
                v[i] = q.x;
                v[i + 1] = q.y;
                v[i + 2] = q.z;
                v[i + 3] = q.w;
            }
        } else {
#pragma unroll
            for (int i = 0; i < C; i++) v[i] = i < mine ? row[sel_at(first + i)] : -CUDART_INF_F;
        }
        float mx = -CUDART_INF_F, total = 0.0f;
        if (!a.sigmoid && !(p.by_logit && a.renorm)) {
#pragma unroll
            for (int i = 0; i < C; i++) mx = fmaxf(mx, v[i]);
            mx = sub_max<LPT>(mx);
#pragma unroll
            for (int i = 0; i < C; i++) {
                // -inf: 0 (also where the whole row is -inf); +inf: 1
                total += v[i] > SEL_NINF ? (v[i] == mx ? 1.0f : __expf(v[i] - mx)) : 0.0f;
            }
            total = sub_sum<LPT>(total);
        }
        if (p.by_logit) {
#pragma unroll
            for (int i = 0; i < C; i++) {
                // the lower id ahead: more in the low bits of a positive number is more, of
                // a negative one less; + 0 makes one zero of two
                const int b = __float_as_int(fminf(fmaxf(v[i] + 0.0f, -SEL_MAX), SEL_MAX));
                const float k = __int_as_float((b & ~255) | (((b >> 31) ^ (255 - (first + i))) & 255));
                v[i] = v[i] > SEL_NINF ? k : SEL_NINF;
            }
        } else {
            const float inv = __fdividef(1.0f, total);
#pragma unroll
            for (int i = 0; i < C; i++) {
                const float l = v[i];
                float s = a.sigmoid ? __fdividef(1.0f, 1.0f + __expf(-l)) : (l == mx ? 1.0f : __expf(l - mx)) * inv;
                if (a.bias) s += i < mine ? sbias[sel_at(first + i)] : 0.0f;
                const int b = __float_as_int(fminf(fmaxf(s, -SEL_MAX), SEL_MAX));
                const float k = __int_as_float((b & ~255) | (255 - (first + i)));
                v[i] = l > SEL_NINF && s > SEL_NINF ? k : SEL_NINF;
            }
        }
        // ---- this lane's largest, in order
        if constexpr (C <= 8) {
            sel_sort<C>(v);
        } else {
            sel_sort<8>(v);
#pragma unroll
            for (int i = 8; i < C; i += 8) {
                sel_sort<8>(v + i);
                sel_merge8(v, v + i);
            }
        }
        bool unsure = false;
        // ---- groups
        if (a.G > 1) {
            float m1 = v[0], m2 = KEEP > 1 ? v[KEEP > 1 ? 1 : 0] : SEL_NINF;
            for (int d = (1 << p.lanes_shift) >> 1; d; d >>= 1) {
                const float o1 = __shfl_xor_sync(0xffffffffu, m1, d), o2 = __shfl_xor_sync(0xffffffffu, m2, d);
                m2 = fmaxf(fminf(m1, o1), fmaxf(m2, o2));
                m1 = fmaxf(m1, o1);
            }
            // the low bits must not count: they are ids
            const float k1 = __int_as_float(__float_as_int(m1) & ~255);
            const float k2 = a.groupTop > 1 && m2 > SEL_NINF ? __int_as_float(__float_as_int(m2) & ~255) : 0.0f;
            const float val = m1 > SEL_NINF ? fmaxf(k1 + k2, -SEL_MAX) : SEL_NINF;
            int before = 0;
            for (int d = 1 << p.lanes_shift; d < LPT; d += 1 << p.lanes_shift) {
                const int from = sub ^ d;
                const float o = __shfl_xor_sync(0xffffffffu, val, d);
                before += (o > val || (o == val && (from >> p.lanes_shift) < grp)) ? 1 : 0;
            }
            const bool stay = before < a.topG;
            if (!(EXACT16 && p.by_logit)) {
                const float in = -sub_max<LPT>(stay ? -val : SEL_NINF);  // the least that stays
                const float out = sub_max<LPT>(stay ? SEL_NINF : val);   // the most that does not
                // Each key is off by 2^-15 of its size (the bits given to ids) and by its
                // score's error: 2^-15 of it, and 2e-6 at most (see below).
                float tol;
                if (a.bias)
                    tol = sub_max<LPT>(val > SEL_NINF ? fabsf(k1) + fabsf(k2) : 0.0f) * 6.2e-5f + 8e-6f;
                else
                    tol = (fabsf(in) + fabsf(out)) * 6.6e-5f + 1e-37f;
                unsure = out > SEL_NINF && !(in - out > tol);
            }
            if (!stay) {
#pragma unroll
                for (int i = 0; i < KEEP; i++) v[i] = SEL_NINF;
            }
        }
        // ---- the K + 1 largest: the largest head K + 1 times
        float win = SEL_NINF, last = SEL_NINF;
        for (int r = 0; r <= a.K; r++) {
            const float m = sub_max<LPT>(v[0]);
            if (sub == r) win = m;
            last = m;
            if (__float_as_int(v[0]) == __float_as_int(m)) {  // (bits: -0 is not +0)
#pragma unroll
                for (int i = 0; i + 1 < KEEP; i++) v[i] = v[i + 1];
                v[KEEP - 1] = SEL_NINF;
            }
        }
        float next = __shfl_down_sync(0xffffffffu, win, 1);
        if (sub == a.K - 1) next = last;
        const bool slot = sub < a.K;
        int e = 0;
        if (slot && win > SEL_NINF) {
            const int b = __float_as_int(win);
            e = p.by_logit && b < 0 ? b & 255 : 255 - (b & 255);
            if (next > SEL_NINF && !(EXACT16 && p.by_logit)) {
                const float k0 = __int_as_float(b & ~255), k1 = __int_as_float(__float_as_int(next) & ~255);
                const float big = fmaxf(fabsf(k0), fabsf(k1));
                // Two keys with truncated values this far apart are in order: a step of the
                // truncation (2^-15 of the key) and twice a score's error.  A sigmoid is off
                // by s (1 - s) (1.44 |l| + 4) 2^-23 + 2^-22 s < 4e-7, a softmax by
                // (3 |l - m| + 31) 2^-24 s < 2e-6; relative to s, both by less than 2^-15 down
                // to where fp32 ends.
                if (p.by_logit)
                    unsure |= k0 == k1;
                else
                    unsure |= !(k0 - k1 > (a.bias ? big * 3.08e-5f + 4e-6f : big * 9.2e-5f + 1e-37f));
            }
        } else if (slot) {
            unsure = true;  // too few open experts
        }
        bool closed = false;
        // ---- tokens to be told apart exactly, by the whole warp
        for (unsigned todo = __ballot_sync(0xffffffffu, unsure); todo;) {
            const int which = (__ffs(todo) - 1) / LPT;
            const int tt = __shfl_sync(0xffffffffu, t, which * LPT);
            bool shut;
            const int got = select_exact<LT>(a, static_cast<const LT*>(a.logits) + (size_t)tt * a.ldl, scratch[warp], shut);
            const int ge = __shfl_sync(0xffffffffu, got, sub);
            const bool gs = __shfl_sync(0xffffffffu, (int)shut, sub) != 0;
            if (tok == which) {
                e = slot ? ge : 0;
                closed = slot && gs;
            }
            todo &= ~((LPT == 32 ? 0xffffffffu : ((1u << (LPT & 31)) - 1u)) << (which * (LPT & 31)));
            if (LPT == 32) todo = 0;
        }
        const bool open = slot && !closed;
        const float w = sel_weight<LPT>(a, open ? row[sel_at(e)] : 0.0f, open, mx, total);
        if (slot && t0 + tok < a.T) {
            const size_t o = (size_t)t * a.K + sub;
            a.ids[o] = e;
            if (a.wtype == MOE_DT_FLOAT)
                static_cast<float*>(a.weights)[o] = w;
            else
                static_cast<__half*>(a.weights)[o] = __float2half_rn(w);
        }
        __syncwarp();
    }
}

namespace {

template <typename LT, int LPT, int C>
cudaError_t launch_select_as(const SelectArgs& a, SelectPlan p, cudaStream_t s)
{
    int groups = 1, shift = 0;
    while (groups < a.G) groups *= 2;
    while ((LPT / groups) >> (shift + 1)) shift++;
    const int size = a.E / a.G, lanes = 1 << shift;
    p.lanes_shift = shift;
    p.per_lane = (size + lanes - 1) / lanes;
    p.whole = a.G == groups && size == lanes * C;
    constexpr int per_block = SEL_WARPS * (32 / LPT);
    const long long blocks = ((long long)a.T + per_block - 1) / per_block;
    return launch_pdl(select_kernel<LT, LPT, C>, dim3((unsigned)(blocks < 148 * 6 ? blocks : 148 * 6)),
                      dim3(SEL_WARPS * 32), 0, s, a, p);
}

template <typename LT>
cudaError_t launch_select_type(const SelectArgs& a, cudaStream_t s)
{
    SelectPlan p = {};
    p.vec = reinterpret_cast<uintptr_t>(a.logits) % 16 == 0 && (a.ldl * sizeof(LT)) % 16 == 0 &&
            (a.E * sizeof(LT)) % 16 == 0;
    p.by_logit = !a.bias && (a.G == 1 || a.groupTop == 1);
    int groups = 1;
    while (groups < a.G) groups *= 2;
    const int size = a.E / a.G;
    if (groups <= 8 && a.T >= 1024) {
        const int per = (size + 8 / groups - 1) / (8 / groups);
        if (per <= 4) return launch_select_as<LT, 8, 4>(a, p, s);
        if (per <= 8) return launch_select_as<LT, 8, 8>(a, p, s);
        if (per <= 16) return launch_select_as<LT, 8, 16>(a, p, s);
        if (per <= 32) return launch_select_as<LT, 8, 32>(a, p, s);
    }
    const int per = (size + 32 / groups - 1) / (32 / groups);
    if (per <= 8) return launch_select_as<LT, 32, 8>(a, p, s);
    return launch_select_as<LT, 32, 16>(a, p, s);
}

}  // namespace

cudaError_t launch_select(const SelectArgs& a, int ltype, cudaStream_t s)
{
    if (ltype == MOE_DT_FLOAT) return launch_select_type<float>(a, s);
    if (ltype == MOE_DT_FLOAT16) return launch_select_type<__half>(a, s);
    return launch_select_type<__nv_bfloat16>(a, s);
}

}  // namespace moe
