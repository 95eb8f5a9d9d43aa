// linear.cu -- MoeLinear on sm_100a: a matrix product with bias, activation, gate and
// residual in its epilogue.
//
//   plain: y[t, n] = act(sum_k x[t, k] w[n, k] + bias[n]) + residual[t, n]
//   gated: y[t, n] = act(sum_k x[t, k] w[n, k] + bias[n]) *
//                    (sum_k x[t, k] w[N + n, k] + bias[N + n]) + residual[t, n]
// x [T, K], w [N or 2N, K], fp16 or bf16; sums, bias, activation, product and residual
// are taken in fp32 and rounded once, to the type of y.
//
// Three kernels:
//   linear_gemm_kernel<PAIR, BN>  many tokens: persistent tcgen05 tiles of 128 tokens
//       (256 over a CTA pair) x BN accumulator columns; x and w by TMA into a ring of
//       128-byte-swizzled stages, fp32 accumulators double-buffered in TMEM, so that the
//       epilogue of one tile runs under the products of the next;
//   linear_split_kernel           few tiles: the same products, with k divided over the
//       CTAs of a cluster; each CTA sends every other one its slice of columns through
//       distributed shared memory, and each adds its own slice in rank order;
//   linear_few_kernel             a few tokens: w is streamed once, straight into the
//       registers of mma.sync fragments; bound by HBM (by latency for small w).
// No atomics, no workspace: the same inputs give the same bits, and calls on different
// streams share nothing.
#include <cstdlib>
#include <cstring>

#include <cuda_bf16.h>

#include "../../include/moe_ops.h"
#include "moe_common.cuh"
#include "moe_kernels.h"

namespace moe {

// Bounded waits record here when they give up (MoeLinearGetDeviceError; the layer call
// moves it into its workspace's error word).
__device__ int g_linear_err;

// ---------------------------------------------------------------------- epilogue maths
// exp and the quotient by their fast intrinsics: together below 8 + 2|z| half ulps, which
// the fp16 / bf16 rounding of y hides, and of the size of the sum's own roundings for an
// fp32 y.  Results below about 2^-126 become 0.
template <int ACT>
__device__ __forceinline__ float lin_act1(float z)
{
    if (ACT == MOE_ACT_RELU) return z < 0.0f ? 0.0f : z;  // NaN stays
    if (ACT == MOE_ACT_GELU) return z * normcdff(z);
    if (ACT == MOE_ACT_GELU_TANH) {
        // 0.5 z (1 + tanh(u)) = z / (1 + exp(-2u)), u = sqrt(2/pi) (z + 0.044715 z^3)
        const float u2 = 1.5957691216057308f * (z + 0.044715f * z * z * z);
        return __fdividef(z, 1.0f + __expf(-u2));
    }
    if (ACT == MOE_ACT_SILU) return __fdividef(z, 1.0f + __expf(-z));
    if (ACT == MOE_ACT_SIGMOID) return __fdividef(1.0f, 1.0f + __expf(-z));
    return z;
}

template <int ACT, int NV>
__device__ __forceinline__ void lin_act_all(float (&v)[NV])
{
#pragma unroll
    for (int i = 0; i < NV; i++) v[i] = lin_act1<ACT>(v[i]);
}

template <int NV>
__device__ __forceinline__ void lin_act(float (&v)[NV], int act)
{
    switch (act) {
        case MOE_ACT_RELU: lin_act_all<MOE_ACT_RELU>(v); break;
        case MOE_ACT_GELU: lin_act_all<MOE_ACT_GELU>(v); break;
        case MOE_ACT_GELU_TANH: lin_act_all<MOE_ACT_GELU_TANH>(v); break;
        case MOE_ACT_SILU: lin_act_all<MOE_ACT_SILU>(v); break;
        case MOE_ACT_SIGMOID: lin_act_all<MOE_ACT_SIGMOID>(v); break;
        default: break;
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
__device__ __forceinline__ uint32_t lin_pack(float a, float b, int type)
{
    if (type == MOE_DT_FLOAT16) return pack_half2(a, b);
    __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&h);
}
__device__ __forceinline__ float2 lin_unpack(uint32_t q, int type)
{
    if (type == MOE_DT_FLOAT16) return __half22float2(*reinterpret_cast<const __half2*>(&q));
    return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&q));
}

// ---------------------------------------------------------------------- tensor-core tiles
constexpr int LG_BM = 128;                     // tokens per CTA and tile (UMMA M)
constexpr int LG_BK = 64;                      // k per stage: one 128-byte swizzle row
constexpr int LG_A_BYTES = LG_BM * LG_BK * 2;  // 16 KB
constexpr int LG_THREADS = 192;
constexpr int LG_MAX_STAGES = 8;
constexpr int LG_GROUP_M = 8;                  // m tiles that run together over all n tiles

// PAIR: a 2-CTA cluster runs 256 x 256 tiles with cta_group::2 UMMAs; each CTA stages its
// own 128 tokens and one 128-row half of w.
template <int PAIR, int BN>
struct LinCfg {
    static_assert(BN == 256 || (BN == 128 && !PAIR), "tile");
    static constexpr int B_HALF = (BN / 2) * LG_BK * 2;  // bytes of one box of w
    static constexpr int STAGE_BYTES = LG_A_BYTES + (PAIR ? B_HALF : 2 * B_HALF);
    static constexpr int STAGES = PAIR ? 6 : (BN == 256 ? 4 : 6);
    static constexpr int ROWS = PAIR ? 2 * LG_BM : LG_BM;
    static constexpr uint32_t TMEM_COLS = 2 * BN;
};

struct LinTail {
    uint64_t full[LG_MAX_STAGES];
    uint64_t empty[LG_MAX_STAGES];
    uint64_t tfull[2];
    uint64_t tempty[2];
    uint64_t drain;
    uint32_t tmem_base;
    int abort_flag;
};
constexpr size_t LG_TAIL = (sizeof(LinTail) + 127) & ~(size_t)127;

// Staging of one 32-column chunk per epilogue warp: 32 rows x 32 floats, padded to 144
// bytes so that row-wise writes and transposed reads both hit every bank once.
constexpr int LG_STG_ROW = 144;
constexpr int LG_STG_WARP = 32 * LG_STG_ROW;

template <int PAIR, int BN>
__host__ __device__ constexpr size_t lin_smem_bytes()
{
    return 1024 + (size_t)LinCfg<PAIR, BN>::STAGES * LinCfg<PAIR, BN>::STAGE_BYTES + LG_TAIL + 4 * LG_STG_WARP;
}
static_assert(lin_smem_bytes<1, 256>() <= 227 * 1024 && lin_smem_bytes<0, 256>() <= 227 * 1024 &&
                  lin_smem_bytes<0, 128>() <= 227 * 1024, "smem");

struct LinParams {
    const void* bias;
    const void* residual;
    void* y;
    long long ldr, ldy;
    int* err;
    int T, N, nk;        // nk: k blocks of 64
    int type, otype;
    int act, gated;
    int vec_y, vec_r;    // rows of y / residual start on 16-byte boundaries
    int mt, nt;          // tiles
    int w_evict_first;   // w is read by one m tile only
};

__host__ __device__ constexpr uint32_t lin_idesc(int M, int N, bool bf16)
{
    return umma_idesc_f16_f32(M, N) | (bf16 ? (1u << 7) | (1u << 10) : 0u);
}

// Tile index -> (m, n): LG_GROUP_M m tiles run together over all n tiles, so that a
// group's x stays in L2 while w passes by once per group.
__device__ __forceinline__ void lin_tile(const LinParams& p, long long tile, int& m, int& n)
{
    const long long width = (long long)LG_GROUP_M * p.nt;
    const int g = (int)(tile / width);
    const int r = (int)(tile - g * width);
    const int gm = min(LG_GROUP_M, p.mt - g * LG_GROUP_M);
    n = r / gm;
    m = g * LG_GROUP_M + (r - n * gm);
}

// Writes one 32-column chunk of a warp's 32 rows: v[c] is column col0 + c of this lane's
// row, before the residual.  Through shared memory, so that each store instruction covers
// whole 64-byte (fp32: 128-byte) row segments.  row0: the warp's first row; rows: how many
// of its rows exist.
__device__ __forceinline__ void lin_store_chunk(const LinParams& p, uint8_t* stg, int lane, const float (&v)[32],
                                                int row0, int rows, int col0)
{
    float4* mine = reinterpret_cast<float4*>(stg + lane * LG_STG_ROW);
#pragma unroll
    for (int i = 0; i < 8; i++) mine[i] = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
    __syncwarp();
    if (p.otype == MOE_DT_FLOAT) {
        const int c = (lane & 7) * 4, n = col0 + c;
#pragma unroll 4
        for (int i = 0; i < 8; i++) {
            const int r = 4 * i + (lane >> 3);
            if (r >= rows || n >= p.N) continue;
            float4 q = *reinterpret_cast<const float4*>(stg + r * LG_STG_ROW + c * 4);
            float* dst = static_cast<float*>(p.y) + (size_t)(row0 + r) * p.ldy + n;
            const float* res = p.residual ? static_cast<const float*>(p.residual) + (size_t)(row0 + r) * p.ldr + n : nullptr;
            const int left = p.N - n;
            if (left >= 4 && p.vec_y && (!res || p.vec_r)) {
                if (res) {
                    const float4 a = *reinterpret_cast<const float4*>(res);
                    q = make_float4(q.x + a.x, q.y + a.y, q.z + a.z, q.w + a.w);
                }
                *reinterpret_cast<float4*>(dst) = q;
            } else {
                const float e[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
                for (int j = 0; j < 4; j++)
                    if (j < left) dst[j] = e[j] + (res ? res[j] : 0.0f);
            }
        }
    } else {
        const int c = (lane & 3) * 8, n = col0 + c;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int r = 8 * i + (lane >> 2);
            if (r >= rows || n >= p.N) continue;
            const float4 q0 = *reinterpret_cast<const float4*>(stg + r * LG_STG_ROW + c * 4);
            const float4 q1 = *reinterpret_cast<const float4*>(stg + r * LG_STG_ROW + c * 4 + 16);
            float e[8] = {q0.x, q0.y, q0.z, q0.w, q1.x, q1.y, q1.z, q1.w};
            __half* dst = static_cast<__half*>(p.y) + (size_t)(row0 + r) * p.ldy + n;
            const __half* res = p.residual ? static_cast<const __half*>(p.residual) + (size_t)(row0 + r) * p.ldr + n : nullptr;
            const int left = p.N - n;
            if (left >= 8 && p.vec_y && (!res || p.vec_r)) {
                if (res) {
                    const uint4 a = *reinterpret_cast<const uint4*>(res);
                    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const float2 f = lin_unpack(w[j], p.otype);
                        e[2 * j] += f.x;
                        e[2 * j + 1] += f.y;
                    }
                }
                *reinterpret_cast<uint4*>(dst) = make_uint4(lin_pack(e[0], e[1], p.otype), lin_pack(e[2], e[3], p.otype),
                                                            lin_pack(e[4], e[5], p.otype), lin_pack(e[6], e[7], p.otype));
            } else {
#pragma unroll
                for (int j = 0; j < 8; j++)
                    if (j < left) lin_store(dst, j, e[j] + (res ? lin_load(res, j, p.otype) : 0.0f), p.otype);
            }
        }
    }
    __syncwarp();
}

// v[c] += bias[col + c]: each lane fetches one column's bias, the warp shares them.
__device__ __forceinline__ void lin_add_bias(const LinParams& p, int lane, int n, size_t offset, float (&v)[32])
{
    const float b = (n + lane < p.N) ? lin_load(p.bias, offset + n + lane, p.type) : 0.0f;
#pragma unroll
    for (int c = 0; c < 32; c++) v[c] += __shfl_sync(0xffffffffu, b, c);
}

template <int PAIR, int BN>
__global__ void __launch_bounds__(LG_THREADS, 1)
linear_gemm_kernel(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmW,
                   const LinParams p)
{
    using Cfg = LinCfg<PAIR, BN>;
    constexpr int STAGES = Cfg::STAGES;
    constexpr int STAGE_BYTES = Cfg::STAGE_BYTES;
    constexpr int ROWS = Cfg::ROWS;
    extern __shared__ uint8_t lg_smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>(
        (reinterpret_cast<uintptr_t>(lg_smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    LinTail* tail = reinterpret_cast<LinTail*>(smem + STAGES * STAGE_BYTES);

    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    int* err = p.err ? p.err : &g_linear_err;
    // Pair mode: rank 0 of the cluster issues the UMMAs and owns the barriers they wait on.
    const uint32_t crank = PAIR ? cluster_ctarank() : 0u;
    const bool leader = crank == 0u;
    const int unit = PAIR ? (int)(blockIdx.x >> 1) : (int)blockIdx.x;
    const int nunits = PAIR ? (int)(gridDim.x >> 1) : (int)gridDim.x;

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; s++) {
            mbar_init(smem_u32(&tail->full[s]), 1);
            mbar_init(smem_u32(&tail->empty[s]), 1);
        }
        for (int a = 0; a < 2; a++) {
            mbar_init(smem_u32(&tail->tfull[a]), 1);
            mbar_init(smem_u32(&tail->tempty[a]), PAIR ? 8 : 4);  // one arrival per epilogue warp
        }
        mbar_init(smem_u32(&tail->drain), 1);
        tail->abort_flag = 0;
        fence_barrier_init();
        tma_prefetch_desc(&tmX);
        tma_prefetch_desc(&tmW);
    }
    pdl_trigger();
    if (warp == 1) {
        if (PAIR) {
            tmem_alloc_pair(smem_u32(&tail->tmem_base), Cfg::TMEM_COLS);
            tmem_relinquish_pair();
        } else {
            tmem_alloc(smem_u32(&tail->tmem_base), Cfg::TMEM_COLS);
            tmem_relinquish();
        }
    }
    tc_fence_before();
    if (PAIR)
        cluster_sync_all();  // both CTAs' barriers are initialised before any remote arrival
    else
        __syncthreads();
    tc_fence_after();
    pdl_wait();  // inputs come from, and y may still be read by, the launches before

    const uint32_t tmem_base = tail->tmem_base;
    const long long total = (long long)p.mt * p.nt;
    const int nk = p.nk;
    volatile int* abort_flag = &tail->abort_flag;

    if (warp == 0) {
        // ---------------------------------------------------------------- producer
        if (lane == 0) {
            const uint64_t pol_x = l2_policy_evict_last();
            const uint64_t pol_w = p.w_evict_first ? l2_policy_evict_first() : l2_policy_evict_last();
            uint32_t it = 0;
            bool ok = true;
            for (long long tile = unit; ok && tile < total; tile += nunits) {
                int m, n;
                lin_tile(p, tile, m, n);
                const int x_row = m * ROWS + (int)crank * LG_BM;
                const int w_lo = n * (p.gated ? BN / 2 : BN);
                const int w_hi = p.gated ? p.N + w_lo : w_lo + BN / 2;
                for (int kb = 0; kb < nk; kb++, it++) {
                    const int s = it % STAGES;
                    const uint32_t par = ((it / STAGES) & 1u) ^ 1u;
                    const bool got = PAIR ? mbar_wait_bounded_cluster(smem_u32(&tail->empty[s]), par, err,
                                                                      MOE_DEV_WAIT_TIMEOUT_TMA, abort_flag)
                                          : mbar_wait_bounded(smem_u32(&tail->empty[s]), par, err,
                                                              MOE_DEV_WAIT_TIMEOUT_TMA, abort_flag);
                    if (!got) {
                        ok = false;
                        break;
                    }
                    const uint32_t full = smem_u32(&tail->full[s]);
                    const uint32_t st = smem_u32(smem + s * STAGE_BYTES);
                    if (PAIR) {
                        // both CTAs' copies complete on the leader's barrier, which
                        // expects the bytes of both
                        const uint32_t full_leader = mapa_shared(full, 0);
                        if (leader) mbar_arrive_expect_tx(full, 2 * STAGE_BYTES);
                        tma_load_2d_pair(st, &tmX, full_leader, kb * LG_BK, x_row, pol_x);
                        tma_load_2d_pair(st + LG_A_BYTES, &tmW, full_leader, kb * LG_BK, leader ? w_lo : w_hi, pol_w);
                    } else {
                        mbar_arrive_expect_tx(full, STAGE_BYTES);
                        tma_load_2d(st, &tmX, full, kb * LG_BK, x_row, pol_x);
                        tma_load_2d(st + LG_A_BYTES, &tmW, full, kb * LG_BK, w_lo, pol_w);
                        tma_load_2d(st + LG_A_BYTES + Cfg::B_HALF, &tmW, full, kb * LG_BK, w_hi, pol_w);
                    }
                }
            }
            if (!ok && leader) {
                // giving up: the copies in flight land (bounded wait) before the CTA exits
                const uint32_t first = it > (uint32_t)STAGES ? it - STAGES : 0;
                for (uint32_t j = first; j < it; j++) {
                    const uint64_t t0 = global_timer_ns();
                    while (!(PAIR ? mbar_try_wait_cluster(smem_u32(&tail->full[j % STAGES]), (j / STAGES) & 1u)
                                  : mbar_try_wait(smem_u32(&tail->full[j % STAGES]), (j / STAGES) & 1u)))
                        if (global_timer_ns() - t0 > MOE_WAIT_LIMIT_NS) break;
                }
            }
        }
    } else if (warp == 1) {
        // ---------------------------------------------------------------- UMMA issuer
        if (lane == 0 && leader) {
            const uint32_t idesc = lin_idesc(ROWS, BN, p.type == MOE_DT_BF16);
            uint32_t it = 0, lt = 0;
            bool ok = true;
            for (long long tile = unit; ok && tile < total; tile += nunits, lt++) {
                const uint32_t acc = lt & 1u;
                const uint32_t tpar = ((lt >> 1) & 1u) ^ 1u;
                if (!(PAIR ? mbar_wait_bounded_cluster(smem_u32(&tail->tempty[acc]), tpar, err,
                                                       MOE_DEV_WAIT_TIMEOUT_MMA, abort_flag)
                           : mbar_wait_bounded(smem_u32(&tail->tempty[acc]), tpar, err, MOE_DEV_WAIT_TIMEOUT_MMA,
                                               abort_flag)))
                    break;
                tc_fence_after();
                const uint32_t d = tmem_base + acc * BN;
                for (int kb = 0; kb < nk; kb++, it++) {
                    const int s = it % STAGES;
                    const uint32_t fpar = (it / STAGES) & 1u;
                    if (!(PAIR ? mbar_wait_bounded_cluster(smem_u32(&tail->full[s]), fpar, err,
                                                           MOE_DEV_WAIT_TIMEOUT_MMA, abort_flag)
                               : mbar_wait_bounded(smem_u32(&tail->full[s]), fpar, err, MOE_DEV_WAIT_TIMEOUT_MMA,
                                                   abort_flag))) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const uint32_t a_addr = smem_u32(smem + s * STAGE_BYTES);
                    const uint32_t b_addr = a_addr + LG_A_BYTES;
#pragma unroll
                    for (int k = 0; k < LG_BK / 16; k++) {
                        // k advances by 16 elements = 32 bytes inside the swizzle row
                        if (PAIR)
                            umma_f16_ss_pair(d, umma_desc_sw128(a_addr + k * 32), umma_desc_sw128(b_addr + k * 32),
                                             idesc, (kb | k) != 0);
                        else
                            umma_f16_ss(d, umma_desc_sw128(a_addr + k * 32), umma_desc_sw128(b_addr + k * 32), idesc,
                                        (kb | k) != 0);
                    }
                    if (PAIR) {
                        umma_commit_pair(smem_u32(&tail->empty[s]));
                        umma_commit_pair(mapa_shared(smem_u32(&tail->empty[s]), 1));
                    } else {
                        umma_commit(smem_u32(&tail->empty[s]));
                    }
                }
                if (ok) {
                    if (PAIR) {
                        umma_commit_pair(smem_u32(&tail->tfull[acc]));
                        umma_commit_pair(mapa_shared(smem_u32(&tail->tfull[acc]), 1));
                    } else {
                        umma_commit(smem_u32(&tail->tfull[acc]));
                    }
                }
            }
            // no UMMA of this CTA (pair) runs on when TMEM is freed
            if (PAIR)
                umma_commit_pair(smem_u32(&tail->drain));
            else
                umma_commit(smem_u32(&tail->drain));
            const uint64_t t0 = global_timer_ns();
            while (!(PAIR ? mbar_try_wait_cluster(smem_u32(&tail->drain), 0) : mbar_try_wait(smem_u32(&tail->drain), 0)))
                if (global_timer_ns() - t0 > MOE_WAIT_LIMIT_NS) {
                    atomicOr(err, MOE_DEV_WAIT_TIMEOUT_MMA);
                    break;
                }
        }
    } else {
        // ---------------------------------------------------------------- epilogue
        const int q = warp & 3;  // the TMEM lane quarter this warp may read
        uint8_t* stg = smem + STAGES * STAGE_BYTES + LG_TAIL + (size_t)q * LG_STG_WARP;
        // in pair mode the epilogue warps of both CTAs release the leader's accumulator
        const uint32_t tempty0 = PAIR ? mapa_shared(smem_u32(&tail->tempty[0]), 0) : smem_u32(&tail->tempty[0]);
        uint32_t lt = 0;
        for (long long tile = unit; tile < total; tile += nunits, lt++) {
            int m, n;
            lin_tile(p, tile, m, n);
            const uint32_t acc = lt & 1u;
            const uint32_t tpar = (lt >> 1) & 1u;
            if (!(PAIR ? mbar_wait_bounded_cluster(smem_u32(&tail->tfull[acc]), tpar, err, MOE_DEV_WAIT_TIMEOUT_EPI,
                                                   abort_flag)
                       : mbar_wait_bounded(smem_u32(&tail->tfull[acc]), tpar, err, MOE_DEV_WAIT_TIMEOUT_EPI,
                                           abort_flag)))
                break;
            tc_fence_after();
            const int row0 = m * ROWS + (int)crank * LG_BM + q * 32;
            const int rows = min(32, p.T - row0);  // <= 0: none of this warp's rows exist
            const uint32_t tbase = tmem_base + acc * BN + ((uint32_t)(q * 32) << 16);
            const int cols = p.gated ? BN / 2 : BN;
            const int col0 = n * cols;
            if (rows > 0) {
#pragma unroll 1
                for (int j = 0; j < cols && col0 + j < p.N; j += 32) {
                    uint32_t a[32];
                    float v[32];
                    tmem_ld_32x32b_x32(tbase + j, a);
                    if (p.gated) {
                        uint32_t b[32];
                        float u[32];
                        tmem_ld_32x32b_x32(tbase + BN / 2 + j, b);
                        tmem_ld_wait();
#pragma unroll
                        for (int c = 0; c < 32; c++) {
                            v[c] = __uint_as_float(a[c]);
                            u[c] = __uint_as_float(b[c]);
                        }
                        if (p.bias) {
                            lin_add_bias(p, lane, col0 + j, 0, v);
                            lin_add_bias(p, lane, col0 + j, p.N, u);
                        }
                        lin_act(v, p.act);
#pragma unroll
                        for (int c = 0; c < 32; c++) v[c] *= u[c];
                    } else {
                        tmem_ld_wait();
#pragma unroll
                        for (int c = 0; c < 32; c++) v[c] = __uint_as_float(a[c]);
                        if (p.bias) lin_add_bias(p, lane, col0 + j, 0, v);
                        lin_act(v, p.act);
                    }
                    lin_store_chunk(p, stg, lane, v, row0, rows, col0 + j);
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                const uint32_t bar = tempty0 + acc * (uint32_t)sizeof(uint64_t);
                if (PAIR)
                    mbar_arrive_cluster(bar);
                else
                    mbar_arrive(bar);
            }
        }
    }

    // pair mode: neither CTA frees TMEM or exits while the other may still address it
    __syncwarp();
    if (PAIR)
        cluster_sync_all();
    else
        __syncthreads();
    if (warp == 1) {
        __syncwarp();
        tc_fence_after();
        if (PAIR)
            tmem_dealloc_pair(tmem_base, Cfg::TMEM_COLS);
        else
            tmem_dealloc(tmem_base, Cfg::TMEM_COLS);
    }
}

// ---------------------------------------------------------------------- k split over a cluster
// One 128 x 128 tile per cluster of S CTAs (S = 1, 2, 4, 8).  CTA r multiplies k blocks
// [nk r / S, nk (r + 1) / S), then sends the columns that CTA d finishes to d's receive
// buffer [S][128][W + 4], W = 128 / S (gated: W/2 gate and W/2 up columns), and finishes
// its own columns from the S partial sums in rank order.
constexpr int LS_BN = 128;
constexpr int LS_STAGES = 4;
constexpr int LS_STAGE_BYTES = LG_A_BYTES + LS_BN * LG_BK * 2;  // 32 KB
constexpr int LS_MAX_S = 8;
constexpr int LS_RECV_BYTES = LS_MAX_S * LG_BM * (LS_BN / LS_MAX_S + 4) * 4;  // the largest: 80 KB
constexpr size_t LS_SMEM = 1024 + (size_t)LS_STAGES * LS_STAGE_BYTES + LS_RECV_BYTES + LG_TAIL;
static_assert(LS_SMEM <= 227 * 1024, "smem");

__device__ __forceinline__ void st_cluster_v4(uint32_t addr, float a, float b, float c, float d)
{
    asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "f"(a), "f"(b), "f"(c), "f"(d)
                 : "memory");
}

__global__ void __launch_bounds__(LG_THREADS, 1)
linear_split_kernel(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmW,
                    const LinParams p, const int S)
{
    extern __shared__ uint8_t ls_smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>(
        (reinterpret_cast<uintptr_t>(ls_smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    float* recv = reinterpret_cast<float*>(smem + LS_STAGES * LS_STAGE_BYTES);
    LinTail* tail = reinterpret_cast<LinTail*>(smem + LS_STAGES * LS_STAGE_BYTES + LS_RECV_BYTES);

    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    int* err = p.err ? p.err : &g_linear_err;
    const int rank = (int)cluster_ctarank();
    const int tile = (int)(blockIdx.x / S);

    if (threadIdx.x == 0) {
        for (int s = 0; s < LS_STAGES; s++) {
            mbar_init(smem_u32(&tail->full[s]), 1);
            mbar_init(smem_u32(&tail->empty[s]), 1);
        }
        mbar_init(smem_u32(&tail->drain), 1);
        tail->abort_flag = 0;
        fence_barrier_init();
        tma_prefetch_desc(&tmX);
        tma_prefetch_desc(&tmW);
    }
    pdl_trigger();
    if (warp == 1) {
        tmem_alloc(smem_u32(&tail->tmem_base), LS_BN);
        tmem_relinquish();
    }
    tc_fence_before();
    cluster_sync_all();  // barriers are initialised, and every CTA's shared memory is live
    tc_fence_after();
    pdl_wait();

    const uint32_t tmem_base = tail->tmem_base;
    volatile int* abort_flag = &tail->abort_flag;
    int m, n;
    lin_tile(p, tile, m, n);
    const int kb0 = (int)((long long)p.nk * rank / S), kb1 = (int)((long long)p.nk * (rank + 1) / S);
    const int cols = p.gated ? LS_BN / 2 : LS_BN;
    const int W = LS_BN / S;       // columns a CTA finishes (gated: half of them outputs)
    const int pitch = W + 4;

    if (warp == 0) {
        if (lane == 0) {
            const uint64_t pol_x = l2_policy_evict_last();
            const uint64_t pol_w = p.w_evict_first ? l2_policy_evict_first() : l2_policy_evict_last();
            const int w_lo = n * cols;
            const int w_hi = p.gated ? p.N + w_lo : w_lo + LS_BN / 2;
            uint32_t it = 0;
            bool ok = true;
            for (int kb = kb0; kb < kb1; kb++, it++) {
                const int s = it % LS_STAGES;
                if (!mbar_wait_bounded(smem_u32(&tail->empty[s]), ((it / LS_STAGES) & 1u) ^ 1u, err,
                                       MOE_DEV_WAIT_TIMEOUT_TMA, abort_flag)) {
                    ok = false;
                    break;
                }
                const uint32_t full = smem_u32(&tail->full[s]);
                const uint32_t st = smem_u32(smem + s * LS_STAGE_BYTES);
                mbar_arrive_expect_tx(full, LS_STAGE_BYTES);
                tma_load_2d(st + LG_A_BYTES, &tmW, full, kb * LG_BK, w_lo, pol_w);
                tma_load_2d(st + LG_A_BYTES + LS_BN / 2 * LG_BK * 2, &tmW, full, kb * LG_BK, w_hi, pol_w);
                tma_load_2d(st, &tmX, full, kb * LG_BK, m * LG_BM, pol_x);
            }
            if (!ok) {
                const uint32_t first = it > (uint32_t)LS_STAGES ? it - LS_STAGES : 0;
                for (uint32_t j = first; j < it; j++) {
                    const uint64_t t0 = global_timer_ns();
                    while (!mbar_try_wait(smem_u32(&tail->full[j % LS_STAGES]), (j / LS_STAGES) & 1u))
                        if (global_timer_ns() - t0 > MOE_WAIT_LIMIT_NS) break;
                }
            }
        }
    } else if (warp == 1) {
        if (lane == 0) {
            const uint32_t idesc = lin_idesc(LG_BM, LS_BN, p.type == MOE_DT_BF16);
            uint32_t it = 0;
            for (int kb = kb0; kb < kb1; kb++, it++) {
                const int s = it % LS_STAGES;
                if (!mbar_wait_bounded(smem_u32(&tail->full[s]), (it / LS_STAGES) & 1u, err, MOE_DEV_WAIT_TIMEOUT_MMA,
                                       abort_flag))
                    break;
                tc_fence_after();
                const uint32_t a_addr = smem_u32(smem + s * LS_STAGE_BYTES);
                const uint32_t b_addr = a_addr + LG_A_BYTES;
#pragma unroll
                for (int k = 0; k < LG_BK / 16; k++)
                    umma_f16_ss(tmem_base, umma_desc_sw128(a_addr + k * 32), umma_desc_sw128(b_addr + k * 32), idesc,
                                (kb > kb0 || k > 0) ? 1u : 0u);
                umma_commit(smem_u32(&tail->empty[s]));
            }
            umma_commit(smem_u32(&tail->drain));  // all sums of this CTA are in TMEM
            const uint64_t t0 = global_timer_ns();
            while (!mbar_try_wait(smem_u32(&tail->drain), 0))
                if (global_timer_ns() - t0 > MOE_WAIT_LIMIT_NS) {
                    atomicOr(err, MOE_DEV_WAIT_TIMEOUT_MMA);
                    break;
                }
        }
    } else {
        const int q = warp & 3;
        const int row = q * 32 + lane;
        if (mbar_wait_bounded(smem_u32(&tail->drain), 0, err, MOE_DEV_WAIT_TIMEOUT_EPI, abort_flag)) {
            tc_fence_after();
            if (m * LG_BM + q * 32 < p.T) {
                const uint32_t mine = smem_u32(recv) + (uint32_t)((rank * LG_BM + row) * pitch) * 4u;
#pragma unroll 1
                for (int j = 0; j < LS_BN; j += 32) {
                    uint32_t a[32];
                    tmem_ld_32x32b_x32(tmem_base + ((uint32_t)(q * 32) << 16) + j, a);
                    tmem_ld_wait();
#pragma unroll
                    for (int c = 0; c < 32; c += 4) {
                        const int col = j + c;
                        int d, off;
                        if (p.gated) {
                            const int half = col >> 6, cc = col & 63, hw = W >> 1;
                            d = cc / hw;
                            off = half * hw + (cc - d * hw);
                        } else {
                            d = col / W;
                            off = col - d * W;
                        }
                        st_cluster_v4(mapa_shared(mine + (uint32_t)off * 4u, (uint32_t)d), __uint_as_float(a[c]),
                                      __uint_as_float(a[c + 1]), __uint_as_float(a[c + 2]), __uint_as_float(a[c + 3]));
                    }
                }
            }
        }
        tc_fence_before();
    }
    __syncwarp();
    cluster_sync_all();  // every partial sum has arrived
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem_base, LS_BN);
    }

    // this CTA's columns: 4 outputs per thread and step
    const int outs = p.gated ? W / 2 : W;
    const int groups = outs / 4;
    const int col0 = n * cols + rank * outs;
    for (int i = threadIdx.x; i < LG_BM * groups; i += LG_THREADS) {
        const int row = i / groups, g = i - row * groups;
        const int t = m * LG_BM + row, nn = col0 + 4 * g;
        if (t >= p.T) break;
        if (nn >= p.N) continue;
        float v[4] = {}, u[4] = {};
        for (int s = 0; s < S; s++) {
            const float* src = recv + (size_t)(s * LG_BM + row) * pitch + 4 * g;
            const float4 a = *reinterpret_cast<const float4*>(src);
            v[0] += a.x;
            v[1] += a.y;
            v[2] += a.z;
            v[3] += a.w;
            if (p.gated) {
                const float4 b = *reinterpret_cast<const float4*>(src + outs);
                u[0] += b.x;
                u[1] += b.y;
                u[2] += b.z;
                u[3] += b.w;
            }
        }
        const int left = p.N - nn;
        if (p.bias) {
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (j < left) {
                    v[j] += lin_load(p.bias, nn + j, p.type);
                    if (p.gated) u[j] += lin_load(p.bias, (size_t)p.N + nn + j, p.type);
                }
        }
        lin_act(v, p.act);
        if (p.gated) {
#pragma unroll
            for (int j = 0; j < 4; j++) v[j] *= u[j];
        }
        if (p.residual) {
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (j < left) v[j] += lin_load(p.residual, (size_t)t * p.ldr + nn + j, p.otype);
        }
        const size_t o = (size_t)t * p.ldy + nn;
        if (left >= 4 && p.vec_y) {
            if (p.otype == MOE_DT_FLOAT)
                *reinterpret_cast<float4*>(static_cast<float*>(p.y) + o) = make_float4(v[0], v[1], v[2], v[3]);
            else
                *reinterpret_cast<uint2*>(static_cast<__half*>(p.y) + o) =
                    make_uint2(lin_pack(v[0], v[1], p.otype), lin_pack(v[2], v[3], p.otype));
        } else {
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (j < left) lin_store(p.y, o + j, v[j], p.otype);
        }
    }
}

// ---------------------------------------------------------------------- a few tokens
// A warp holds MT blocks of 16 rows of w (gated: 16 gate rows and their 16 up rows) and
// NT blocks of 8 tokens; the block's warps divide k among them and add up in shared
// memory, in warp order.  w goes from HBM into fragment registers with no stop in shared
// memory: a product does not depend on the order of k, so lane (g, t) takes 8 consecutive
// elements (16 bytes) of rows g and g + 8 at k = 32 c + 8 t, and of token g, and feeds
// them to two m16n8k16 products as if they were the columns those expect.
constexpr int LF_WARPS = 16;
constexpr int LF_U = 2;  // k chunks of 32 per step; the next step's loads are in flight under this one's products

__device__ __forceinline__ uint4 ld_stream16(const void* p)
{
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}

// Volatile, so that it stays behind the wait for the launches before it.
__device__ __forceinline__ uint4 ld_cached16(const void* p)
{
    uint4 v;
    asm volatile("ld.global.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}

template <bool BF16>
__device__ __forceinline__ void mma_16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                          uint32_t b1)
{
    if (BF16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

template <bool BF16, int MT, int NT>
__global__ void __launch_bounds__(LF_WARPS * 32, 1) linear_few_kernel(const LinearArgs a)
{
    __shared__ float red[LF_WARPS][NT * 8][MT * 16 + 1];
    pdl_trigger();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = lane >> 2, t = lane & 3;
    const int n0 = blockIdx.x * (a.gated ? 16 : 16 * MT);
    const uint16_t* w = static_cast<const uint16_t*>(a.w);
    const uint16_t* x = static_cast<const uint16_t*>(a.x);
    // rows of this lane (clamped where they do not exist: read, not used)
    const uint16_t* wr[MT][2];
#pragma unroll
    for (int i = 0; i < MT; i++)
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int r = g + 8 * h;
            const int row = a.gated ? min(n0 + r, a.N - 1) + i * a.N : min(n0 + 16 * i + r, a.N - 1);
            wr[i][h] = w + (size_t)row * a.ldw + 8 * t;
        }
    const uint16_t* xr[NT];
    bool xin[NT];
#pragma unroll
    for (int j = 0; j < NT; j++) {
        xin[j] = g + 8 * j < a.T;
        xr[j] = x + (size_t)(xin[j] ? g + 8 * j : 0) * a.ldx + 8 * t;
    }
    float acc[MT][NT][4] = {};
    uint4 wa[LF_U][MT][2], xb[LF_U][NT];
    const uint4 zero = make_uint4(0, 0, 0, 0);
    constexpr int STEP = 32 * LF_U;
    auto load = [&](int k) {
#pragma unroll
        for (int c = 0; c < LF_U; c++) {
            const int kk = k + 32 * c;
            const bool in = kk + 8 * t < a.K;
#pragma unroll
            for (int i = 0; i < MT; i++)
#pragma unroll
                for (int h = 0; h < 2; h++) wa[c][i][h] = in ? ld_stream16(wr[i][h] + kk) : zero;
#pragma unroll
            for (int j = 0; j < NT; j++)
                xb[c][j] = (in && xin[j]) ? ld_cached16(xr[j] + kk) : zero;
        }
    };
    pdl_wait();
    int k = warp * STEP;
    if (k < a.K) load(k);
    while (k < a.K) {
        uint4 wc[LF_U][MT][2], xc[LF_U][NT];
#pragma unroll
        for (int c = 0; c < LF_U; c++) {
#pragma unroll
            for (int i = 0; i < MT; i++) wc[c][i][0] = wa[c][i][0], wc[c][i][1] = wa[c][i][1];
#pragma unroll
            for (int j = 0; j < NT; j++) xc[c][j] = xb[c][j];
        }
        k += STEP * LF_WARPS;
        if (k < a.K) load(k);
#pragma unroll
        for (int c = 0; c < LF_U; c++)
#pragma unroll
            for (int i = 0; i < MT; i++)
#pragma unroll
                for (int j = 0; j < NT; j++) {
                    const uint4 lo = wc[c][i][0], hi = wc[c][i][1], b = xc[c][j];
                    mma_16816<BF16>(acc[i][j], lo.x, hi.x, lo.y, hi.y, b.x, b.y);
                    mma_16816<BF16>(acc[i][j], lo.z, hi.z, lo.w, hi.w, b.z, b.w);
                }
    }
#pragma unroll
    for (int i = 0; i < MT; i++)
#pragma unroll
        for (int j = 0; j < NT; j++) {
            red[warp][8 * j + 2 * t][16 * i + g] = acc[i][j][0];
            red[warp][8 * j + 2 * t + 1][16 * i + g] = acc[i][j][1];
            red[warp][8 * j + 2 * t][16 * i + g + 8] = acc[i][j][2];
            red[warp][8 * j + 2 * t + 1][16 * i + g + 8] = acc[i][j][3];
        }
    __syncthreads();
    const int outs = a.gated ? 16 : 16 * MT;
    for (int i = threadIdx.x; i < outs * a.T; i += LF_WARPS * 32) {
        const int tok = i / outs, r = i - tok * outs, n = n0 + r;
        if (n >= a.N) continue;
        float v[1] = {0.0f}, u = 0.0f;
        for (int s = 0; s < LF_WARPS; s++) v[0] += red[s][tok][r];
        if (MT == 2 && a.gated)
            for (int s = 0; s < LF_WARPS; s++) u += red[s][tok][16 * (MT - 1) + r];
        if (a.bias) {
            v[0] += lin_load(a.bias, n, a.type);
            if (a.gated) u += lin_load(a.bias, (size_t)a.N + n, a.type);
        }
        lin_act(v, a.act);
        if (a.gated) v[0] *= u;
        if (a.residual) v[0] += lin_load(a.residual, (size_t)tok * a.ldr + n, a.otype);
        lin_store(a.y, (size_t)tok * a.ldy + n, v[0], a.otype);
    }
}

// ---------------------------------------------------------------------- host side
int* linear_error_word()
{
    static int* addr[64] = {nullptr};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return nullptr;
    if (!addr[dev]) {
        void* p = nullptr;
        if (cudaGetSymbolAddress(&p, g_linear_err) != cudaSuccess) {
            cudaGetLastError();
            return nullptr;
        }
        addr[dev] = static_cast<int*>(p);
    }
    return addr[dev];
}

namespace {

typedef CUresult (*LinEncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// [rows, inner] matrix of 2-byte elements, rows ld apart; 64 x box_rows boxes, 128-byte
// swizzle, zeros outside.
bool lin_tmap(CUtensorMap* tm, const void* base, int type, uint64_t inner, uint64_t rows, uint64_t ld, uint32_t box_rows)
{
    static LinEncodeFn fn = nullptr;
    if (!fn) {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess)
            return false;
        fn = reinterpret_cast<LinEncodeFn>(p);
    }
    cuuint64_t dims[2] = {inner, rows};
    cuuint64_t strides[1] = {ld * 2};
    cuuint32_t box[2] = {LG_BK, box_rows};
    cuuint32_t es[2] = {1, 1};
    return fn(tm, type == MOE_DT_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2,
              const_cast<void*>(base), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Once per kernel and device: opt in to the dynamic shared memory.
template <typename Kernel>
cudaError_t lin_smem_attr(Kernel* kernel, size_t bytes, bool (&done)[64], int dev)
{
    if (dev >= 0 && dev < 64 && done[dev]) return cudaSuccess;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    if (e == cudaSuccess && dev >= 0 && dev < 64) done[dev] = true;
    return e;
}

int lin_sm_count(int dev)
{
    static int n[64] = {0};
    if (dev < 0 || dev >= 64) return 148;
    if (!n[dev]) {
        cudaDeviceGetAttribute(&n[dev], cudaDevAttrMultiProcessorCount, dev);
        if (n[dev] <= 0) n[dev] = 148;
    }
    return n[dev];
}

template <typename... KArgs, typename... Args>
cudaError_t lin_launch(void (*kernel)(KArgs...), unsigned grid, unsigned block, size_t smem, unsigned cluster,
                       cudaStream_t s, Args... args)
{
    cudaLaunchConfig_t lc = {};
    lc.gridDim = dim3(grid);
    lc.blockDim = dim3(block);
    lc.dynamicSmemBytes = smem;
    lc.stream = s;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = cluster;
    at[1].val.clusterDim.y = 1;
    at[1].val.clusterDim.z = 1;
    lc.attrs = at;
    lc.numAttrs = cluster > 0 ? 2 : 1;
    return cudaLaunchKernelEx(&lc, kernel, static_cast<KArgs>(args)...);
}

LinParams lin_params(const LinearArgs& a, int rows, int cols)
{
    LinParams p = {};
    const size_t es = a.otype == MOE_DT_FLOAT ? 4 : 2;
    p.bias = a.bias;
    p.residual = a.residual;
    p.y = a.y;
    p.ldr = a.ldr;
    p.ldy = a.ldy;
    p.err = a.err;
    p.T = a.T;
    p.N = a.N;
    p.nk = (a.K + LG_BK - 1) / LG_BK;
    p.type = a.type;
    p.otype = a.otype;
    p.act = a.act;
    p.gated = a.gated;
    p.vec_y = reinterpret_cast<uintptr_t>(a.y) % 16 == 0 && (a.ldy * es) % 16 == 0;
    p.vec_r = reinterpret_cast<uintptr_t>(a.residual) % 16 == 0 && (a.ldr * es) % 16 == 0;
    p.mt = (a.T + rows - 1) / rows;
    p.nt = (a.N + cols - 1) / cols;
    p.w_evict_first = p.mt == 1;
    return p;
}

template <int PAIR, int BN>
cudaError_t launch_tiles(const LinearArgs& a, int dev, cudaStream_t s)
{
    using Cfg = LinCfg<PAIR, BN>;
    static bool done[64] = {false};
    auto* kernel = linear_gemm_kernel<PAIR, BN>;
    cudaError_t e = lin_smem_attr(kernel, lin_smem_bytes<PAIR, BN>(), done, dev);
    if (e != cudaSuccess) return e;
    CUtensorMap tx, tw;
    const uint64_t wrows = (uint64_t)a.N * (a.gated ? 2 : 1);
    if (!lin_tmap(&tx, a.x, a.type, a.K, a.T, a.ldx, LG_BM) || !lin_tmap(&tw, a.w, a.type, a.K, wrows, a.ldw, BN / 2))
        return cudaErrorInvalidValue;
    const LinParams p = lin_params(a, Cfg::ROWS, a.gated ? BN / 2 : BN);
    const long long tiles = (long long)p.mt * p.nt;
    long long units = lin_sm_count(dev);
    if (PAIR) {
        // co-resident pairs: both CTAs of a pair need a free SM of one GPC
        static int resident[64] = {0};
        units = (dev >= 0 && dev < 64) ? resident[dev] : 0;
        if (units <= 0) {
            cudaLaunchConfig_t q = {};
            q.gridDim = dim3(2 * (lin_sm_count(dev) / 2));
            q.blockDim = dim3(LG_THREADS);
            q.dynamicSmemBytes = lin_smem_bytes<PAIR, BN>();
            cudaLaunchAttribute ca;
            ca.id = cudaLaunchAttributeClusterDimension;
            ca.val.clusterDim.x = 2;
            ca.val.clusterDim.y = 1;
            ca.val.clusterDim.z = 1;
            q.attrs = &ca;
            q.numAttrs = 1;
            int n = 0;
            if (cudaOccupancyMaxActiveClusters(&n, kernel, &q) != cudaSuccess || n <= 0) {
                cudaGetLastError();
                n = lin_sm_count(dev) / 2;
            }
            units = n;
            if (dev >= 0 && dev < 64) resident[dev] = n;
        }
    }
    const unsigned grid = (unsigned)(tiles < units ? tiles : units) * (PAIR ? 2 : 1);
    return lin_launch(kernel, grid, LG_THREADS, lin_smem_bytes<PAIR, BN>(), PAIR ? 2 : 0, s, tx, tw, p);
}

cudaError_t launch_split(const LinearArgs& a, int S, int dev, cudaStream_t s)
{
    static bool done[64] = {false};
    cudaError_t e = lin_smem_attr(linear_split_kernel, LS_SMEM, done, dev);
    if (e != cudaSuccess) return e;
    CUtensorMap tx, tw;
    const uint64_t wrows = (uint64_t)a.N * (a.gated ? 2 : 1);
    if (!lin_tmap(&tx, a.x, a.type, a.K, a.T, a.ldx, LG_BM) || !lin_tmap(&tw, a.w, a.type, a.K, wrows, a.ldw, LS_BN / 2))
        return cudaErrorInvalidValue;
    const LinParams p = lin_params(a, LG_BM, a.gated ? LS_BN / 2 : LS_BN);
    const long long tiles = (long long)p.mt * p.nt;
    return lin_launch(linear_split_kernel, (unsigned)(tiles * S), LG_THREADS, LS_SMEM, (unsigned)S, s, tx, tw, p, S);
}

template <bool BF16, int MT>
cudaError_t launch_few_rows(const LinearArgs& a, cudaStream_t s)
{
    const int rows = a.gated ? 16 : 16 * MT;
    const unsigned grid = (unsigned)((a.N + rows - 1) / rows);
    if (a.T <= 8) return lin_launch(linear_few_kernel<BF16, MT, 1>, grid, LF_WARPS * 32, 0, 0, s, a);
    return lin_launch(linear_few_kernel<BF16, MT, 2>, grid, LF_WARPS * 32, 0, 0, s, a);
}

cudaError_t launch_few(const LinearArgs& a, int mt, cudaStream_t s)
{
    if (a.type == MOE_DT_BF16) return mt == 2 ? launch_few_rows<true, 2>(a, s) : launch_few_rows<true, 1>(a, s);
    return mt == 2 ? launch_few_rows<false, 2>(a, s) : launch_few_rows<false, 1>(a, s);
}

// MOE_LINEAR_TILE=pair|wide|narrow|split1|split2|split4|split8|few forces a kernel where
// it can run (few: up to 16 tokens; splitS: as many k blocks as CTAs).
const char* lin_forced()
{
#ifdef MOE_LINEAR_TUNE
    return getenv("MOE_LINEAR_TILE");
#else
    static const char* v = getenv("MOE_LINEAR_TILE");
    return v;
#endif
}

}  // namespace

cudaError_t launch_linear(const LinearArgs& a, cudaStream_t s)
{
    int dev = 0;
    cudaGetDevice(&dev);
    const int sms = lin_sm_count(dev);
    const long long wrows = (long long)a.N * (a.gated ? 2 : 1);
    const int nk = (a.K + LG_BK - 1) / LG_BK;
    const int few_mt = a.gated || wrows >= 32LL * 2 * sms ? 2 : 1;
    const long long mt = (a.T + LG_BM - 1) / LG_BM, nt128 = (wrows + 127) / 128;
    if (const char* f = lin_forced()) {
        if (!strcmp(f, "few") && a.T <= 16) return launch_few(a, few_mt, s);
        if (!strcmp(f, "pair")) return launch_tiles<1, 256>(a, dev, s);
        if (!strcmp(f, "wide")) return launch_tiles<0, 256>(a, dev, s);
        if (!strcmp(f, "narrow")) return launch_tiles<0, 128>(a, dev, s);
        if (!strncmp(f, "split", 5) && f[5] >= '1' && f[5] <= '8' && mt * nt128 * 8 < (1LL << 31)) {
            int S = f[5] - '0';
            while (S > nk || (S & (S - 1))) S--;
            return launch_split(a, S, dev, s);
        }
    }
    if (a.T <= 16) return launch_few(a, few_mt, s);
    const long long t128 = mt * nt128;
    if (2 * t128 <= sms) {
        int S = 8;
        while (S > 1 && (t128 * S > sms || S > nk)) S >>= 1;
        return launch_split(a, S, dev, s);
    }
    if (t128 <= sms) return launch_tiles<0, 128>(a, dev, s);
    if (t128 <= 4 * sms) return launch_tiles<0, 256>(a, dev, s);
    return launch_tiles<1, 256>(a, dev, s);
}

}  // namespace moe
