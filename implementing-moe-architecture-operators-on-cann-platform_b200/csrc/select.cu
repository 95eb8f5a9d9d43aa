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
// bits tell apart, and the id is a whole number that is right or wrong.  Scores order as
// their logits do, so where nothing is added to them (no bias, and one group or groupTop 1)
// the logits themselves are the keys.
//
// Measured, 65536 x 256 fp32 logits, sigmoid, bias, 4 of 8 groups, K = 8: 50 us, 1.4 TB/s.  It
// reads its 67 MB once.  No unit is full: 422 instructions per token take 61% of the issue
// slots, and the 207 of them on the ALU pipe (where a min or max takes two cycles) 57% of it.
// What bounds it is latency with few warps: 96 registers leave 4.5 per scheduler, of which at
// each issue 2.1 wait for a result of fixed latency, 1.2 for shared memory, a shuffle or a
// special function, and 0.7 for the pipe.
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
    float r;
    asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
    return r;
}

struct ExactScratch {
    double key[SEL_MAX_E];
    double group[SEL_MAX_G];
};

// Doubles as unsigned integers in the same order, none of them 0 (NaN does not occur).
__device__ __forceinline__ unsigned long long sel_ordered(double v)
{
    const long long b = __double_as_longlong(v + 0.0);  // one zero of two
    return (unsigned long long)(b ^ ((b >> 63) | (long long)0x8000000000000000ull));
}

// Called, not inlined: fetched once per call site, the code took longer than it runs.
__device__ __noinline__ double sel_sigmoid64(float l) { return 1.0 / (1.0 + exp(-(double)l)); }
__device__ __noinline__ double sel_exp64(float l, float mx) { return l == mx ? 1.0 : exp((double)l - (double)mx); }

// The K chosen experts of one token, by one warp, with keys in 64 bits.  Returns to lane
// r < K slot r's expert, plus 256 where no open expert was left for that slot.
template <typename LT>
__device__ __noinline__ int select_exact(const SelectArgs& a, const LT* row, ExactScratch& s)
{
    constexpr int N = SEL_MAX_E / 32;  // expert lane + 32 i is this lane's i-th
    const int lane = threadIdx.x & 31;
    const int E = a.E, size = a.E / a.G;
    const double NINF = -CUDART_INF;
    // the logits order like their scores, so scores are only needed where something is added
    const bool use_score = a.bias != nullptr || (a.G > 1 && a.groupTop > 1);
    float l[N];
    double key[N];
#pragma unroll
    for (int i = 0; i < N; i++) l[i] = lane + 32 * i < E ? fmaxf(sel_load(row, lane + 32 * i), -CUDART_INF_F) : -CUDART_INF_F;
    if (!use_score) {
#pragma unroll
        for (int i = 0; i < N; i++) key[i] = (double)l[i];
    } else if (a.sigmoid) {
#pragma unroll
        for (int i = 0; i < N; i++) key[i] = sel_sigmoid64(l[i]);
    } else {
        float mx = -CUDART_INF_F;
#pragma unroll
        for (int i = 0; i < N; i++) mx = fmaxf(mx, l[i]);
        mx = warp_max(mx);
        double total = 0.0;
#pragma unroll
        for (int i = 0; i < N; i++) {
            key[i] = sel_open(l[i]) ? sel_exp64(l[i], mx) : 0.0;
            total += key[i];
        }
        for (int d = 16; d; d >>= 1) total += __shfl_xor_sync(0xffffffffu, total, d);
#pragma unroll
        for (int i = 0; i < N; i++) key[i] /= total;
    }
#pragma unroll
    for (int i = 0; i < N; i++) {
        bool open = sel_open(l[i]);
        if (a.bias && open) {
            const float b = a.bias[lane + 32 * i];
            open = sel_open(b);
            key[i] += (double)b;
        }
        if (!open) key[i] = NINF;
    }
    if (a.G > 1) {
        __syncwarp();
#pragma unroll
        for (int i = 0; i < N; i++)
            if (lane + 32 * i < E) s.key[lane + 32 * i] = key[i];
        __syncwarp();
        // the two largest keys of each group, by 32 / G' lanes (G' the next power of two)
        int shift = 5;
        while ((a.G - 1) >> (5 - shift)) shift--;
        const int grp = lane >> shift;
        double m1 = NINF, m2 = NINF;
        if (grp < a.G)
            for (int i = lane & ((1 << shift) - 1); i < size; i += 1 << shift) {
                const double k = s.key[grp * size + i];
                m2 = fmax(m2, fmin(m1, k));
                m1 = fmax(m1, k);
            }
        for (int d = (1 << shift) >> 1; d; d >>= 1) {
            const double o1 = __shfl_xor_sync(0xffffffffu, m1, d), o2 = __shfl_xor_sync(0xffffffffu, m2, d);
            m2 = fmax(fmin(m1, o1), fmax(m2, o2));
            m1 = fmax(m1, o1);
        }
        if (grp < a.G) s.group[grp] = (a.groupTop > 1 && m2 > NINF) ? m1 + m2 : m1;
        __syncwarp();
        bool drop = false;
        if (lane < a.G) {
            const double v = s.group[lane];
            int before = 0;
            for (int g = 0; g < a.G; g++) before += (s.group[g] > v || (s.group[g] == v && g < lane)) ? 1 : 0;
            drop = before >= a.topG;
        }
        const unsigned dropped = __ballot_sync(0xffffffffu, drop);
#pragma unroll
        for (int i = 0; i < N; i++)
            if (lane + 32 * i < E && ((dropped >> ((lane + 32 * i) / size)) & 1u)) key[i] = NINF;
    }
    // K times the largest key, lowest id first; a taken expert, or one that does not exist,
    // is 0
    unsigned long long u[N];
#pragma unroll
    for (int i = 0; i < N; i++) u[i] = lane + 32 * i < E ? sel_ordered(key[i]) : 0ull;
    const unsigned long long shut = sel_ordered(NINF);
    int mine = 0;
    for (int r = 0; r < a.K; r++) {
        unsigned long long best = u[0];
        int at = lane;
#pragma unroll
        for (int i = 1; i < N; i++)
            if (u[i] > best) {
                best = u[i];
                at = lane + 32 * i;
            }
        const unsigned hi = __reduce_max_sync(0xffffffffu, (unsigned)(best >> 32));
        const bool in = (unsigned)(best >> 32) == hi;
        const unsigned lo = __reduce_max_sync(0xffffffffu, in ? (unsigned)best : 0u);
        const unsigned long long top = (unsigned long long)hi << 32 | lo;
        const int e = (int)__reduce_min_sync(0xffffffffu, best == top ? (unsigned)at : 0xffffu);
        if (lane == r) mine = e + (top == shut ? SEL_MAX_E : 0);
#pragma unroll
        for (int i = 0; i < N; i++)
            if (e == lane + 32 * i) u[i] = 0ull;
    }
    return mine;
}

// ---------------------------------------------------------------------- fast path
// LPT lanes per token (8: four tokens to a warp, 32: one).  Group g belongs to LPT / G' lanes,
// G' the next power of two; each holds consecutive experts of it.  A key is one fp32 number
// whose lowest 8 bits give way to 255 - e, so that sorting and comparing move one register
// per expert; eight keys at a time are sorted by a network and merged into the lane's eight
// largest, and the lanes' lists into the token's.
//
// A sigmoid's keys are taken less 1 where the token's largest logit is positive: the best
// scores are close to 1, and what is left of them is smaller and so finer in its 24 bits.
//
// What the lost bits or the fast exp and quotient may have turned around is noticed.
// Neighbours among the K + 1 best closer than the bounds below are compared once more by the
// difference of their keys (sel_before), which fp32 knows to a few millionths of itself.
// Groups too close, or differences that cancel, send the token to a list, which select_slow
// settles in 64 bits when the warp is through.  Closed experts are looked for only where one
// turns up among the keys that count: the tokens of the warp are then done over, with care.
constexpr float SEL_MAX = 3.4028235e38f;
constexpr float SEL_CLOSED = -3.4e38f;  // keys at or below may be closed experts' 
#define SEL_NINF (-CUDART_INF_F)

template <int LPT>
__device__ __forceinline__ float sub_max(float v)
{
    if constexpr (LPT == 32) {
        return warp_max(v);
    } else {
#pragma unroll
        for (int d = LPT / 2; d; d >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, d));
        return v;
    }
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

// exp2 and 1 / x by the special function unit, what is below fp32's normal range as 0
__device__ __forceinline__ float sel_ex2(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float sel_rcp(float x)
{
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
constexpr float SEL_LOG2E = 1.4426950408889634f;

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

// Staged rows keep their type.  WHOLE (every lane has the same number of experts, a multiple
// of 8): 16 bytes of padding follow every 128, so that lanes that read 16 bytes at strides of
// 16 to 128 bytes meet different banks.
template <bool WHOLE>
__device__ __forceinline__ int sel_at(int byte)
{
    return WHOLE ? byte + ((byte >> 7) << 4) : byte;
}
constexpr int SEL_ROW = SEL_MAX_E * 4 + SEL_MAX_E * 4 / 128 * 16;  // bytes, of floats

template <bool WHOLE, typename LT>
__device__ __forceinline__ float sel_get(const uint8_t* row, int e)
{
    return sel_load(reinterpret_cast<const LT*>(row + sel_at<WHOLE>(e * (int)sizeof(LT))), 0);
}

// Eight experts of a staged row from `first` on, `pad` where i >= n.
template <bool WHOLE, typename LT>
__device__ __forceinline__ void sel_chunk(float (&v)[8], const uint8_t* row, int first, int n, float pad)
{
    if constexpr (WHOLE) {
        uint4 q[sizeof(LT) / 2];
        const uint8_t* src = row + sel_at<true>(first * (int)sizeof(LT));  // (32 bytes never straddle a padding)
#pragma unroll
        for (int i = 0; i < (int)sizeof(LT) / 2; i++) q[i] = *reinterpret_cast<const uint4*>(src + 16 * i);
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = sel_load(reinterpret_cast<const LT*>(q), i);
    } else {
        const LT* src = reinterpret_cast<const LT*>(row) + first;
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = i < n ? sel_load(src, i) : pad;
    }
}

// Starts the copy of a row of logits into shared memory, by the LPT lanes of a token;
// asynchronously, where 16 (vec) or 4 bytes can be.
template <int LPT, bool WHOLE, typename LT>
__device__ __forceinline__ void sel_stage(const LT* row, uint8_t* dst, int E, int sub, bool vec)
{
    const uint32_t d = smem_u32(dst);
    const uint8_t* src = reinterpret_cast<const uint8_t*>(row);
    const int bytes = E * (int)sizeof(LT);
    if (vec) {
        for (int o = sub * 16; o < bytes; o += LPT * 16)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(d + sel_at<WHOLE>(o)), "l"(src + o) : "memory");
    } else if (sizeof(LT) == 4) {
        for (int o = sub * 4; o < bytes; o += LPT * 4)
            asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(d + sel_at<WHOLE>(o)), "l"(src + o) : "memory");
    } else {
#pragma unroll 8
        for (int e = sub; e < E; e += LPT) *reinterpret_cast<LT*>(dst + sel_at<WHOLE>(e * (int)sizeof(LT))) = row[e];
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
}

__device__ __forceinline__ void sel_store(const SelectArgs& a, int t, int k, int e, float w)
{
    const size_t o = (size_t)t * a.K + k;
    a.ids[o] = e;
    if (a.wtype == MOE_DT_FLOAT)
        static_cast<float*>(a.weights)[o] = w;
    else
        static_cast<__half*>(a.weights)[o] = __float2half_rn(w);
}

// Settles a listed token in 64 bits, by the whole warp.
template <typename LT>
__device__ __noinline__ void select_slow(const SelectArgs& a, int t, ExactScratch& scratch)
{
    const int lane = threadIdx.x & 31;
    const LT* row = static_cast<const LT*>(a.logits) + (size_t)t * a.ldl;
    float mx = SEL_NINF, total = 0.0f;
    if (!a.sigmoid && !a.renorm) {
        for (int e = lane; e < a.E; e += 32) mx = fmaxf(mx, sel_load(row, e));
        mx = warp_max(mx);
        for (int e = lane; e < a.E; e += 32) {
            const float l = sel_load(row, e);
            if (sel_open(l)) total += l == mx ? 1.0f : expf(l - mx);
        }
        total = sub_sum<32>(total);
    }
    const int got = select_exact<LT>(a, row, scratch);
    const bool open = lane < a.K && got < SEL_MAX_E;
    const int e = got & (SEL_MAX_E - 1);
    const float w = sel_weight<32>(a, open ? sel_load(row, e) : 0.0f, open, mx, total);
    if (lane < a.K) sel_store(a, t, lane, e, w);
    __syncwarp();
}

// One of the K + 1 best of a token.
struct SelBest {
    float l, b;
    int e;
};

// Whether x comes before y, by the difference of their keys.  With h the one of the larger
// logit, o the other and d = l_h - l_o (nothing here can overflow, and what underflows is
// below 1e-36):
//   sigmoid  s_h - s_o = s_h (1 - s_o) (1 - e^-d)
//   softmax  s_h - s_o = s_h (1 - e^-d)
// plus the difference of their biases.  The first part is known to c of itself (the errors
// of the scores, as bounded in the kernel, and of expm1), the second to 2^-24.  `lost` is
// set where that does not decide, and for differences that 64-bit keys would round away.
__device__ __forceinline__ bool sel_before(const SelectArgs& a, bool by_logit, const SelBest& x, const SelBest& y, float mx,
                                           float inv, bool& lost)
{
    const bool id = x.e < y.e;
    if (by_logit) return x.l > y.l || (x.l == y.l && id);
    if (x.l == y.l && x.b == y.b) return id;
    float A = 0.0f, c = 0.0f;
    if (x.l != y.l) {
        const float h = fmaxf(x.l, y.l), o = fminf(x.l, y.l);
        A = -expm1f(o - h);
        if (a.sigmoid) {
            A *= sel_rcp(1.0f + sel_ex2(h * -SEL_LOG2E)) * sel_rcp(1.0f + sel_ex2(o * SEL_LOG2E));
            c = fmaxf(fabsf(h), fabsf(o)) * 4e-7f + 3e-6f;
        } else {
            A *= h == mx ? inv : sel_ex2((h - mx) * SEL_LOG2E) * inv;
            c = (h == mx ? 0.0f : mx - h) * 2.5e-7f + 3e-6f;
        }
        if (y.l > x.l) A = -A;
    }
    const float B = x.b - y.b, D = A + B;
    lost |= !(fabsf(D) > fabsf(A) * c + fabsf(B) * 2.4e-7f + (1.0f + fmaxf(fabsf(x.b), fabsf(y.b))) * 1e-15f);
    return D > 0.0f;
}

struct SelectPlan {
    int shift;      // log2 of the lanes per group
    int per_lane;   // experts per lane, in chunks of 8
    bool vec;       // rows of logits start on 16-byte boundaries and hold whole 16 bytes
    bool by_logit;  // no bias and no sums of scores: the logits order as their scores do
};

constexpr int SEL_LIST = 32;

template <typename LT, int LPT, bool WHOLE>
__global__ void __launch_bounds__(SEL_WARPS * 32, 5) select_kernel(const __grid_constant__ SelectArgs a, const __grid_constant__ SelectPlan p)
{
    constexpr int TPW = 32 / LPT;              // tokens per warp
    constexpr bool EXACT16 = sizeof(LT) == 2;  // a 16-bit logit is whole in the upper 24 bits
    constexpr unsigned MASK = LPT == 32 ? 0xffffffffu : (1u << (LPT & 31)) - 1u;
    constexpr int BUFS = LPT == 8 ? 2 : 1;     // (32 lanes: few tokens, hardly a second one per warp)
    __shared__ __align__(16) uint8_t rows[SEL_WARPS][BUFS][TPW][SEL_ROW / 4 * sizeof(LT)];
    __shared__ __align__(16) uint8_t sbias[SEL_ROW];
    __shared__ ExactScratch scratch[LPT == 8 ? 1 : SEL_WARPS];  // (8: in the row buffer that is free then)
    static_assert(LPT != 8 || sizeof(rows[0][0]) >= sizeof(ExactScratch), "scratch fits");
    __shared__ int slow[SEL_WARPS][SEL_LIST];  // tokens for select_slow
    pdl_trigger();
    pdl_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int sub = lane & (LPT - 1), tok = lane / LPT, shift = tok * (LPT & 31);
    if (a.bias) {
        for (int e = threadIdx.x; e < a.E; e += SEL_WARPS * 32)
            *reinterpret_cast<float*>(sbias + sel_at<WHOLE>(e * 4)) = sel_open(a.bias[e]) ? fminf(a.bias[e], SEL_MAX) : SEL_NINF;
        __syncthreads();
    }
    const int size = a.E / a.G;
    const int grp = sub >> p.shift;
    const int first = grp * size + (sub & ((1 << p.shift) - 1)) * p.per_lane;
    const int mine = grp < a.G ? max(0, min(p.per_lane, (grp + 1) * size - first)) : 0;
    const uint32_t step = gridDim.x * SEL_WARPS * TPW, T = (uint32_t)a.T;  // (T + step < 2^32)
    // the sum of a softmax: for its scores, or for weights that are not renormalised
    const bool soft = !a.sigmoid && !(p.by_logit && a.renorm);
    const bool exact = EXACT16 && p.by_logit;
    const LT* const logits = static_cast<const LT*>(a.logits);
    auto token = [&](uint32_t from) { return (int)min(from + tok, T - 1); };  // spare tokens repeat the last one
    uint32_t t0 = (blockIdx.x * SEL_WARPS + warp) * TPW;
    int buf = 0;
    if (BUFS > 1 && t0 < T) sel_stage<LPT, WHOLE, LT>(logits + (size_t)token(t0) * a.ldl, rows[warp][0][tok], a.E, sub, p.vec);
    while (t0 < T) {
        int listed = 0;
        for (; t0 < T && listed + TPW <= SEL_LIST; t0 += step) {
            const int t = token(t0);
            const uint8_t* const row = rows[warp][buf][tok];
            if (BUFS > 1) {
                // the next tokens' rows come while these are worked on
                buf ^= BUFS - 1;
                sel_stage<LPT, WHOLE, LT>(logits + (size_t)token(t0 + step < T ? t0 + step : t0) * a.ldl, rows[warp][buf][tok], a.E,
                                   sub, p.vec);
                asm volatile("cp.async.wait_group 1;" ::: "memory");
            } else {
                sel_stage<LPT, WHOLE, LT>(logits + (size_t)t * a.ldl, rows[warp][0][tok], a.E, sub, p.vec);
                asm volatile("cp.async.wait_group 0;" ::: "memory");
            }
            __syncwarp();
            float mx = SEL_NINF, total = 0.0f;
            if (soft || !p.by_logit) {
                // (a sigmoid only asks whether it is positive, which some of them tell)
                float v[8];
                const int upto = soft ? p.per_lane : 8;
#pragma unroll 1
                for (int c = 0; c < upto; c += 8) {
                    sel_chunk<WHOLE, LT>(v, row, first + c, mine - c, SEL_NINF);
#pragma unroll
                    for (int i = 0; i < 8; i++) mx = fmaxf(mx, v[i]);
                }
                mx = sub_max<LPT>(mx);
            }
            if (soft) {
                float v[8];
#pragma unroll 1
                for (int c = 0; c < p.per_lane; c += 8) {
                    sel_chunk<WHOLE, LT>(v, row, first + c, mine - c, SEL_NINF);
                    // (the largest apart: +inf - +inf has no difference; NaN counts as -inf)
#pragma unroll
                    for (int i = 0; i < 8; i++)
                        total += v[i] == mx ? 1.0f : fmaxf(sel_ex2((v[i] - mx) * SEL_LOG2E), 0.0f);
                }
                total = sub_sum<LPT>(total);
            }
            const float inv = soft ? sel_rcp(total) : 1.0f;
            const float sign = mx > 0.0f ? 1.0f : -1.0f;  // a sigmoid's keys: s - 1 or s
            // ---- keys, eight at a time, merged into this lane's eight largest
            float v8[8];
            bool dark = false;  // for select_slow
            bool stay = true;   // this lane's group
            float win, after1, after2;
            // the expert of a key, and the key without its id
            auto expert = [&](float key) {
                const int b = __float_as_int(key);
                return !(key > SEL_NINF) ? 0 : (p.by_logit && b < 0 ? b & 255 : 255 - (b & 255));
            };
            auto value = [&](float key) { return key > SEL_NINF ? __int_as_float(__float_as_int(key) & ~255) : SEL_NINF; };
            // a key that counts may be a closed expert's
            auto suspect = [&](float key) { return !(key > SEL_CLOSED && sel_open(sel_get<WHOLE, LT>(row, expert(key)))); };
            // the largest of the token's keys below x; a lane whose eight are all not below has
            // lost sight of its own next
            auto below = [&](float x) {
                float m = SEL_NINF;
#pragma unroll
                for (int i = 0; i < 8; i++) m = fmaxf(m, v8[i] < x ? v8[i] : SEL_NINF);
                dark |= p.per_lane > 8 && v8[7] > SEL_NINF && v8[7] >= x;
                return sub_max<LPT>(m);
            };
#pragma unroll 1
            for (int careful = 0;; careful++) {
                bool shut = false;
                dark = false;
                win = after1 = after2 = SEL_NINF;
#pragma unroll 1
                for (int c = 0; c < p.per_lane; c += 8) {
                    float v[8];
                    sel_chunk<WHOLE, LT>(v, row, first + c, mine - c, SEL_NINF);
                    const int id = 255 - (first + c);
                    unsigned closed = 0;
                    if (careful) {
#pragma unroll
                        for (int i = 0; i < 8; i++) closed |= (sel_open(v[i]) ? 0u : 1u) << i;
                    }
                    if (p.by_logit) {
#pragma unroll
                        for (int i = 0; i < 8; i++) {
                            // the lower id ahead: more in the low bits of a positive number is
                            // more, of a negative one less; + 0 makes one zero of two
                            const int b = __float_as_int(fminf(fmaxf(v[i] + 0.0f, -SEL_MAX), SEL_MAX));
                            v[i] = __int_as_float((b & ~255) | (((b >> 31) ^ (id - i)) & 255));
                        }
                    } else {
                        if (a.sigmoid) {
#pragma unroll
                            for (int i = 0; i < 8; i++) v[i] = -sign * sel_rcp(1.0f + sel_ex2(v[i] * (sign * SEL_LOG2E)));
                        } else {
#pragma unroll
                            for (int i = 0; i < 8; i++) v[i] = (v[i] == mx ? 1.0f : sel_ex2((v[i] - mx) * SEL_LOG2E)) * inv;
                        }
                        if (a.bias) {
                            float b[8];
                            sel_chunk<WHOLE, float>(b, sbias, first + c, mine - c, 0.0f);
#pragma unroll
                            for (int i = 0; i < 8; i++) v[i] += b[i];
                            if (careful) {
#pragma unroll
                                for (int i = 0; i < 8; i++) closed |= (sel_open(b[i]) ? 0u : 1u) << i;
                            }
                        }
#pragma unroll
                        for (int i = 0; i < 8; i++)  // (NaN becomes -SEL_MAX)
                            v[i] = __int_as_float((__float_as_int(fmaxf(v[i], -SEL_MAX)) & ~255) | ((id - i) & 255));
                    }
                    if (!WHOLE) closed |= 0xffu << max(0, min(mine - c, 8));
                    if (!WHOLE || careful) {
#pragma unroll
                        for (int i = 0; i < 8; i++)
                            if ((closed >> i) & 1u) v[i] = SEL_NINF;
                    }
                    sel_sort<8>(v);
                    if (c == 0) {
#pragma unroll
                        for (int i = 0; i < 8; i++) v8[i] = v[i];
                    } else {
                        sel_merge8(v8, v);
                    }
                }
                // ---- groups
                if (a.G > 1) {
                    float m1 = v8[0], m2 = v8[1];
                    for (int d = (1 << p.shift) >> 1; d; d >>= 1) {
                        const float o1 = __shfl_xor_sync(0xffffffffu, m1, d), o2 = __shfl_xor_sync(0xffffffffu, m2, d);
                        m2 = fmaxf(fminf(m1, o1), fmaxf(m2, o2));
                        m1 = fmaxf(m1, o1);
                    }
                    const float k1 = value(m1), k2 = value(m2);
                    float val = SEL_NINF, mag = 0.0f;
                    if (m1 > SEL_NINF) {
                        const bool two = a.groupTop > 1 && m2 > SEL_NINF;
                        // (one key where others have two: 1 less, if theirs are 1 less each)
                        const float alone = a.groupTop > 1 && !two && a.sigmoid && sign > 0.0f ? 1.0f : 0.0f;
                        val = two ? fmaxf(k1 + k2, -SEL_MAX) : k1 - alone;
                        mag = fabsf(k1) + (two ? fabsf(k2) : alone);
                        shut = suspect(m1) || (two && suspect(m2));
                    }
                    int before = 0;
                    for (int d = 1 << p.shift; d < LPT; d += 1 << p.shift) {
                        const int from = sub ^ d;
                        const float o = __shfl_xor_sync(0xffffffffu, val, d);
                        before += (o > val || (o == val && (from >> p.shift) < grp)) ? 1 : 0;
                    }
                    stay = before < a.topG;
                    if (!exact) {
                        const float in = -sub_max<LPT>(stay ? -val : SEL_NINF);  // the least that stays
                        const float out = sub_max<LPT>(stay ? SEL_NINF : val);   // the most that does not
                        // Each key is off by 2^-15 of its size (the bits given to ids) and by its
                        // score's error: 2^-15 of it, and 2e-6 at most, a sigmoid's 5e-7 (see
                        // below); two keys on either side.
                        float tol;
                        if (a.sigmoid || a.bias)
                            tol = sub_max<LPT>(mag) * 6.2e-5f + (a.sigmoid ? 2e-6f : 8e-6f);
                        else
                            tol = (fabsf(in) + fabsf(out)) * 6.6e-5f + 1e-37f;
                        dark |= out > SEL_NINF && !(in - out > tol);
                    }
                    if (!stay) {
#pragma unroll
                        for (int i = 0; i < 8; i++) v8[i] = SEL_NINF;
                    }
                }
                // ---- slot r's key to lane r, and the two keys after the last slot
                if constexpr (LPT == 32) {
                    // the largest head, K + 2 times; a lane whose list runs out has lost sight of
                    // what comes after it
                    const bool full = p.per_lane > 8 && v8[7] > SEL_NINF;
#pragma unroll 1
                    for (int r = 0; r < a.K + 2; r++) {
                        const float m = warp_max(v8[0]);
                        if (sub == r) win = m;
                        after1 = after2;
                        after2 = m;
                        if (__float_as_int(v8[0]) == __float_as_int(m)) {  // (bits: -0 is not +0)
#pragma unroll
                            for (int i = 0; i < 7; i++) v8[i] = v8[i + 1];
                            v8[7] = SEL_NINF;
                        }
                    }
                    dark |= full && v8[0] == SEL_NINF;
                } else {
                    // lists merge pairwise until every lane has the token's eight largest
                    float t8[8];
#pragma unroll
                    for (int i = 0; i < 8; i++) t8[i] = v8[i];
#pragma unroll 1
                    for (int d = 1; d < LPT; d *= 2) {
                        float o[8];
#pragma unroll
                        for (int i = 0; i < 8; i++) o[i] = __shfl_xor_sync(0xffffffffu, t8[i], d);
                        sel_merge8(t8, o);
                    }
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        if (sub == i) win = t8[i];
                        if (a.K == i) after1 = t8[i];
                        if (a.K + 1 == i) after2 = t8[i];
                    }
                    // the ninth: the largest below the eighth
                    if (a.K == 8) after1 = below(t8[7]);
                    if (a.K == 7) after2 = below(t8[7]);
                }
                if (sub < a.K) shut |= suspect(win);
                if (after1 > SEL_NINF) shut |= suspect(after1);
                if (careful || !__any_sync(0xffffffffu, shut)) break;
            }
            const bool slot = sub < a.K && win > SEL_NINF;
            const int open = __popc((__ballot_sync(0xffffffffu, slot) >> shift) & MASK);  // slots with an open expert
            int e = slot ? expert(win) : 0, at = sub;
            float l = sel_get<WHOLE, LT>(row, e);
            if (!exact) {
                // Two keys with truncated values this far apart are in order: a step of the
                // truncation (2^-15 of the key) and twice a score's error.  A sigmoid is off
                // by s (1 - s) (1.44 |l| + 4) 2^-23 + 2^-22 min(s, 1 - s) < 5e-7, a softmax by
                // (3 |l - m| + 31) 2^-24 s < 2e-6; relative to s, both by less than 2^-15
                // down to where fp32 ends.  A logit is exact.
                const float rel = a.bias || a.sigmoid ? 3.08e-5f : 9.2e-5f;
                const float abs = a.sigmoid ? 1e-6f : (a.bias ? 4e-6f : 1e-37f);
                auto apart = [&](float hi, float lo) {
                    return lo == SEL_NINF || (p.by_logit ? hi != lo : hi - lo > fmaxf(fabsf(hi), fabsf(lo)) * rel + abs);
                };
                const float next = __shfl_down_sync(0xffffffffu, win, 1);
                const bool doubt = slot && !apart(value(win), value(sub == a.K - 1 ? after1 : next));
                if (__any_sync(0xffffffffu, doubt)) {
                    // compare once more, everyone with everyone and with the one after
                    if (LPT == 8 && a.K == 8) after2 = below(after1);
                    if (slot && sub == a.K - 1 && doubt) dark |= !apart(value(after1), value(after2));  // a third at the border
                    const SelBest me = {l, a.bias ? sel_get<WHOLE, float>(sbias, e) : 0.0f, e};
                    SelBest other;
                    bool lost = false, beaten = false;
                    int before = 0;
#pragma unroll 1
                    for (int j = 0; j <= a.K; j++) {
                        if (j < a.K) {
                            other.l = __shfl_sync(0xffffffffu, me.l, shift + j);
                            other.b = __shfl_sync(0xffffffffu, me.b, shift + j);
                            other.e = __shfl_sync(0xffffffffu, me.e, shift + j);
                        } else {
                            other.e = expert(after1);
                            other.l = sel_get<WHOLE, LT>(row, other.e);
                            other.b = a.bias ? sel_get<WHOLE, float>(sbias, other.e) : 0.0f;
                        }
                        beaten = false;
                        if (j != sub && (j < a.K ? j < open : after1 > SEL_NINF))
                            beaten = sel_before(a, p.by_logit, other, me, mx, inv, lost);
                        before += beaten ? 1 : 0;
                    }
                    if (slot) dark |= lost;
                    const unsigned less = __ballot_sync(0xffffffffu, slot && beaten);  // those that the one after beats
                    at = before;
                    if (slot && before >= a.K) {  // it takes the place of the one that falls out
                        e = other.e;
                        l = other.l;
                        at = a.K - __popc((less >> shift) & MASK);
                    }
                    // every slot is taken once, or the comparisons were not of one order
                    unsigned taken = slot ? 1u << at : 0u;
#pragma unroll
                    for (int d = LPT / 2; d; d >>= 1) taken |= __shfl_xor_sync(0xffffffffu, taken, d);
                    dark |= taken != (1u << open) - 1u;
                }
            }
            const float w = sel_weight<LPT>(a, l, slot, mx, total);
            const unsigned darks = __ballot_sync(0xffffffffu, dark);
            const bool done = t0 + tok < T && !((darks >> shift) & MASK);
            if (slot && done) sel_store(a, t, at, e, w);
            if (__any_sync(0xffffffffu, open < a.K)) {
                // closed experts fill the slots that are left, lowest id first
                auto shut = [&](int i) {
                    return !(stay && sel_open(sel_get<WHOLE, LT>(row, first + i)) &&
                             (!a.bias || sel_open(sel_get<WHOLE, float>(sbias, first + i))));
                };
                int n = 0;
                for (int i = 0; i < mine; i++) n += shut(i) ? 1 : 0;
                int m = n;  // those of the lanes up to this one
#pragma unroll
                for (int d = 1; d < LPT; d *= 2) {
                    const int o = __shfl_up_sync(0xffffffffu, m, d, LPT);
                    if (sub >= d) m += o;
                }
                int pos = open + m - n;
                for (int i = 0; i < mine && pos < a.K; i++)
                    if (shut(i)) {
                        if (done) sel_store(a, t, pos, first + i, 0.0f);
                        pos++;
                    }
            }
            if (darks) {
#pragma unroll 1
                for (int k = 0; k < TPW && t0 + k < T; k++)
                    if ((darks >> (k * (LPT & 31))) & MASK) slow[warp][listed++] = (int)t0 + k;
            }
            __syncwarp();
        }
#pragma unroll 1
        for (int i = 0; i < listed; i++)
            select_slow<LT>(a, slow[warp][i],
                            LPT == 8 ? *reinterpret_cast<ExactScratch*>(rows[warp][buf ^ (BUFS - 1)]) : scratch[warp]);
        __syncwarp();
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
}

namespace {

template <typename LT, int LPT>
cudaError_t launch_select_as(const SelectArgs& a, SelectPlan p, int groups, cudaStream_t s)
{
    const int size = a.E / a.G, lanes = LPT / groups;
    p.shift = 0;
    while (lanes >> (p.shift + 1)) p.shift++;
    p.per_lane = (size + lanes - 1) / lanes;
    const bool whole = a.G == groups && size == lanes * p.per_lane && p.per_lane % 8 == 0;
    constexpr int per_block = SEL_WARPS * (32 / LPT);
    const long long blocks = ((long long)a.T + per_block - 1) / per_block;
    const long long most = 148 * 5;  // as many as run at once; each then takes several sets of tokens
    return launch_pdl(whole ? select_kernel<LT, LPT, true> : select_kernel<LT, LPT, false>,
                      dim3((unsigned)(blocks < most ? blocks : most)), dim3(SEL_WARPS * 32), 0, s, a, p);
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
    // Eight lanes per token need a quarter of the merges over lanes, 32 have a quarter of the
    // chain.  Measured (us, 8 / 32 lanes), 256 experts in 8 groups, T = 256
    // 7.0 / 5.7, 512 9.1 / 8.3, 1024 11.4 / 11.1, 4096 14.7 / 14.6, 16384 24.0 / 33.5, 65536
    // 50.1 / 101.5; 64 experts: 512 3.1 / 3.1, 1024 3.1 / 3.8, 4096 4.0 / 6.7, 65536 18 / 68.
    if (groups <= 8 && a.T >= 1024) return launch_select_as<LT, 8>(a, p, groups, s);
    return launch_select_as<LT, 32>(a, p, groups, s);
}

}  // namespace

cudaError_t launch_select(const SelectArgs& a, int ltype, cudaStream_t s)
{
    if (ltype == MOE_DT_FLOAT) return launch_select_type<float>(a, s);
    if (ltype == MOE_DT_FLOAT16) return launch_select_type<__half>(a, s);
    return launch_select_type<__nv_bfloat16>(a, s);
}

}  // namespace moe
