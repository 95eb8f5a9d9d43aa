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
// Measured, cold L2, the kernel alone, against the 6515 GB/s of a copy and the 1679 TFLOP/s of
// a library product: few 8 x 8192 -> 2048 with residual 9.2 us (3.7 TB/s; 128 blocks on 148
// SMs), split 128 x 2048 -> 2048 7.8 us (latency of the first copies and of the exchange), gemm
// 128 x 2048 -> 8192 gated 15.1 us (4.6 TB/s), 4096 x 8192 -> 2048 102 us (1351 TFLOP/s; 128
// tiles on 74 pairs), 8192 x 4096 -> 14336 gated 1229 us (1565 TFLOP/s; tensor pipe, 92% busy
// on a smaller shape).
// No workspace, and no atomics but on the error word: the same inputs give the same bits.
// Calls on different streams share that word and nothing else.
#include <cstdlib>
#include <cstring>

#include <cuda_bf16.h>

#include "../../include/moe_ops.h"
#include "moe_common.cuh"
#include "moe_kernels.h"

namespace moe {

// The bounded waits of MoeLinear calls record here when they give up
// (MoeLinearGetDeviceError); those of a layer call record in its workspace.
__device__ int g_linear_err;

// ---------------------------------------------------------------------- epilogue maths
// exp and the quotient by their fast intrinsics.  __expf(a) is off by up to 2 + 1.173 |a| ulp
// and carries what a itself is off, so a result is off by, in units of 2^-24 of itself,
//   SiLU, sigmoid   10 + 2.4 |z|                              (a = -z is exact)
//   GELU            28 + 1.7 z^2                              (a = P - z^2 / 2, rounded once)
//   GELU, tanh      9 + 9.4 |u|, u = 1.6 (z + 0.0447 z^3)     (a = -u, seven roundings)
// at most.  An fp16 or bf16 y (half a step: 2^13 or 2^16 units) hides that until a result is
// far below its normal range; of an fp32 y it is the accuracy.  A quotient by more than
// 2^126 is 0: results below |z| 2^-126 (sigmoid: 2^-126) may become 0.
template <int ACT>
__device__ __forceinline__ float lin_act1(float z)
{
    if (ACT == MOE_ACT_RELU) return z < 0.0f ? 0.0f : z;  // NaN stays
    if (ACT == MOE_ACT_GELU) {
        // z Phi(z), with Phi(-|z|) = erfc(|z| / sqrt 2) / 2 by the Chebyshev fit of Press et
        // al., Numerical Recipes (erfcc): erfc(x) = t exp(-x^2 + P(t)), t = 1 / (1 + x / 2),
        // relative error below 1.2e-7 for every x >= 0
        const float t = __fdividef(1.0f, fmaf(0.35355339f, fabsf(z), 1.0f));
        float e = 0.17087277f;
        e = fmaf(e, t, -0.82215223f);
        e = fmaf(e, t, 1.48851587f);
        e = fmaf(e, t, -1.13520398f);
        e = fmaf(e, t, 0.27886807f);
        e = fmaf(e, t, -0.18628806f);
        e = fmaf(e, t, 0.09678418f);
        e = fmaf(e, t, 0.37409196f);
        e = fmaf(e, t, 1.00002368f);
        e = fmaf(e, t, -1.26551223f);
        const float q = 0.5f * t * __expf(fmaf(-0.5f * z, z, e));
        return z * (z > 0.0f ? 1.0f - q : q);
    }
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
// The type of y, fixed at compile time where it is used per element.
template <int OT>
struct LinOut;
template <>
struct LinOut<MOE_DT_FLOAT> {
    typedef float T;
    static __device__ __forceinline__ float to(float v) { return v; }
    static __device__ __forceinline__ float from(float v) { return v; }
};
template <>
struct LinOut<MOE_DT_FLOAT16> {
    typedef __half T;
    static __device__ __forceinline__ __half to(float v) { return __float2half_rn(v); }
    static __device__ __forceinline__ float from(__half v) { return __half2float(v); }
    static __device__ __forceinline__ uint32_t pack(float a, float b) { return pack_half2(a, b); }
    static __device__ __forceinline__ float2 unpack(uint32_t q) { return __half22float2(*reinterpret_cast<__half2*>(&q)); }
};
template <>
struct LinOut<MOE_DT_BF16> {
    typedef __nv_bfloat16 T;
    static __device__ __forceinline__ __nv_bfloat16 to(float v) { return __float2bfloat16_rn(v); }
    static __device__ __forceinline__ float from(__nv_bfloat16 v) { return __bfloat162float(v); }
    static __device__ __forceinline__ uint32_t pack(float a, float b)
    {
        __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<uint32_t*>(&h);
    }
    static __device__ __forceinline__ float2 unpack(uint32_t q)
    {
        return __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&q));
    }
};

// 16 bytes of y <-> floats (8 of a 16-bit type, 4 of fp32)
template <int OT>
__device__ __forceinline__ uint4 lin_pack16(const float* v)
{
    if constexpr (OT == MOE_DT_FLOAT)
        return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
    else
        return make_uint4(LinOut<OT>::pack(v[0], v[1]), LinOut<OT>::pack(v[2], v[3]), LinOut<OT>::pack(v[4], v[5]),
                          LinOut<OT>::pack(v[6], v[7]));
}
template <int OT>
__device__ __forceinline__ void lin_add16(float* v, uint4 q)
{
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if constexpr (OT == MOE_DT_FLOAT) {
            v[i] += __uint_as_float(w[i]);
        } else {
            const float2 f = LinOut<OT>::unpack(w[i]);
            v[2 * i] += f.x;
            v[2 * i + 1] += f.y;
        }
    }
}

// ---------------------------------------------------------------------- waits
// Bounded wait for a phase of an mbarrier (CLUSTER: completed by the peer CTA too).  The
// clock is read only after a first round of tries: reading %globaltimer takes longer than
// most of these waits.
template <bool CLUSTER>
__device__ __forceinline__ bool lin_try(uint32_t bar, uint32_t parity)
{
    return CLUSTER ? mbar_try_wait_cluster(bar, parity) : mbar_try_wait(bar, parity);
}
template <bool CLUSTER>
__device__ __noinline__ bool lin_wait_slow(uint32_t bar, uint32_t parity, int* err, int code, volatile int* abort_flag)
{
    const uint64_t t0 = global_timer_ns();
    for (;;) {
        for (int i = 0; i < 64; i++)
            if (lin_try<CLUSTER>(bar, parity)) return true;
        if (*abort_flag) return false;
        if (global_timer_ns() - t0 > MOE_WAIT_LIMIT_NS) {
            atomicOr(err, code);
            *abort_flag = 1;
            return false;
        }
    }
}
template <bool CLUSTER>
__device__ __forceinline__ bool lin_wait(uint32_t bar, uint32_t parity, int* err, int code, volatile int* abort_flag)
{
    for (int i = 0; i < 64; i++)
        if (lin_try<CLUSTER>(bar, parity)) return true;
    return lin_wait_slow<CLUSTER>(bar, parity, err, code, abort_flag);
}

// The same without a way out but the clock: the UMMAs in flight must be done before TMEM
// is freed, whatever else gave up.
template <bool CLUSTER>
__device__ __forceinline__ void lin_drain(uint32_t bar, int* err)
{
    for (int i = 0; i < 64; i++)
        if (lin_try<CLUSTER>(bar, 0)) return;
    const uint64_t t0 = global_timer_ns();
    while (!lin_try<CLUSTER>(bar, 0))
        if (global_timer_ns() - t0 > MOE_WAIT_LIMIT_NS) {
            atomicOr(err, MOE_DEV_WAIT_TIMEOUT_MMA);
            return;
        }
}

// One lane of a converged warp, the way that lets the compiler know it is one: with
// lane == 0 in its place a stage's three copies took about 500 cycles to issue, and its four
// UMMAs with their commit 600, more than the 256 or 512 cycles that the products take.
__device__ __forceinline__ bool elect_one()
{
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p != 0;
}

// ---------------------------------------------------------------------- tensor-core tiles
constexpr int LG_BM = 128;                     // tokens per CTA and tile (UMMA M)
constexpr int LG_BK = 64;                      // k per stage: one 128-byte swizzle row
constexpr int LG_A_BYTES = LG_BM * LG_BK * 2;  // 16 KB
constexpr int LG_EPI_WARPS = 8;                // two per TMEM lane quarter, taking chunks in turn
constexpr int LG_THREADS = 64 + 32 * LG_EPI_WARPS;  // narrow tiles: one warp more
constexpr int LG_MAX_STAGES = 8;
// The tensor cores add in fp32 but cut off instead of rounding, always towards zero: over
// 2048 products y is 2.5e-6 of its size off (rounded sums: 0.8e-6), and in proportion over
// more; over products of one sign up to 2 units of 2^-24 for every 16 of them.  A 16-bit y
// does not show it; for an fp32 one the accumulator is emptied into registers, which round,
// every 8 k blocks (512 products), in the tiles and in the k split alike: 64 x 14336 -> 8192,
// all positive, is then 40 units off and not 173, and takes 49.8 us and not 50.8.
constexpr int LG_SEGMENT = 8;
constexpr int LG_GROUP_M = 8;                  // m tiles that run together over all n tiles

// PAIR: a 2-CTA cluster runs 256 x 256 tiles with cta_group::2 UMMAs; each CTA stages its
// own 128 tokens and one 128-row half of w.
template <int PAIR, int BN>
struct LinCfg {
    static_assert(BN == 256 || BN == 128, "tile");
    static constexpr int B_HALF = (BN / 2) * LG_BK * 2;  // bytes of one box of w
    static constexpr int KB_BYTES = LG_A_BYTES + (PAIR ? B_HALF : 2 * B_HALF);
    // k blocks per stage: with 128 columns the four UMMAs of one run for 256 cycles, little
    // more than their issue, commit and wait
    static constexpr int KPS = BN == 128 ? 2 : 1;
    static constexpr int STAGE_BYTES = KPS * KB_BYTES;
    static constexpr int STAGES = PAIR ? (BN == 256 ? 6 : 4) : (BN == 256 ? 4 : 3);
    static constexpr int ROWS = PAIR ? 2 * LG_BM : LG_BM;
    static constexpr uint32_t TMEM_COLS = 2 * BN;
    // A copy takes about 95 cycles to issue; a k block of a narrow tile runs 256 and needs
    // three: x then has a warp of its own.
    static constexpr bool X_WARP = BN == 128 && !PAIR;
    static constexpr int THREADS = LG_THREADS + (X_WARP ? 32 : 0);
};

struct LinTail {
    uint64_t full[LG_MAX_STAGES];
    uint64_t empty[LG_MAX_STAGES];
    uint64_t tfull[2];
    uint64_t tempty[2];
    uint64_t drain;
    uint64_t recv;  // (k split) the partial sums of this CTA's columns
    uint32_t tmem_base;
    int abort_flag;
};
constexpr size_t LG_TAIL = (sizeof(LinTail) + 127) & ~(size_t)127;

// Staging for the epilogue's stores, per warp: 32 rows of 64 bytes (32 columns of a 16-bit
// type, 16 of fp32), padded to 80 bytes so that row-wise writes and transposed reads both
// spread over the banks.
constexpr int LG_STG_ROW = 80;
constexpr int LG_STG_WARP = 32 * LG_STG_ROW;

template <int PAIR, int BN>
__host__ __device__ constexpr size_t lin_smem_bytes()
{
    return 1024 + (size_t)LinCfg<PAIR, BN>::STAGES * LinCfg<PAIR, BN>::STAGE_BYTES + LG_TAIL + LG_EPI_WARPS * LG_STG_WARP;
}
static_assert(lin_smem_bytes<1, 256>() <= 227 * 1024 && lin_smem_bytes<0, 256>() <= 227 * 1024 &&
                  lin_smem_bytes<0, 128>() <= 227 * 1024 && lin_smem_bytes<1, 128>() <= 227 * 1024, "smem");

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
    int x_rows;          // tokens per box of x: 128, or fewer when T is smaller
    int w_evict_first;   // w is read by one m tile only
};

__host__ __device__ constexpr uint32_t lin_idesc(int M, int N, bool bf16)
{
    return umma_idesc_f16_f32(M, N) | (bf16 ? (1u << 7) | (1u << 10) : 0u);
}

// Tile index -> (m, n): LG_GROUP_M m tiles run together over all n tiles, so that a
// group's x stays in L2 while w passes by once per group.
__device__ __forceinline__ void lin_tile(const LinParams& p, uint32_t tile, int& m, int& n)
{
    const uint32_t width = LG_GROUP_M * (uint32_t)p.nt;
    uint32_t g = 0, r = tile;
    if (tile >= width) {
        g = tile / width;
        r = tile - g * width;
    }
    const uint32_t gm = min((uint32_t)LG_GROUP_M, (uint32_t)p.mt - g * LG_GROUP_M);
    const uint32_t nn = gm == LG_GROUP_M ? r / LG_GROUP_M : r / gm;
    n = (int)nn;
    m = (int)(g * LG_GROUP_M + (r - nn * gm));
}

// v[c] += bias[col + c]: each lane fetches one column's bias, the warp shares them.
__device__ __forceinline__ void lin_add_bias(const LinParams& p, int lane, int n, size_t offset, float (&v)[32])
{
    const float b = (n + lane < p.N) ? lin_load(p.bias, offset + n + lane, p.type) : 0.0f;
#pragma unroll
    for (int c = 0; c < 32; c++) v[c] += __shfl_sync(0xffffffffu, b, c);
}

// Where one warp's part of a tile goes: 32 rows from row0 (`rows` of them exist), `valid`
// columns from col0.
struct LinWarpTile {
    uint8_t* stg;
    int lane, row0, rows, col0, valid;
};

// Stores 32 columns from column j of the part: v[c] belongs to this lane's row.  Straight
// line: an SM runs two such warps per scheduler, so most dependent instructions are waited
// for.  Stores and residual loads go through shared memory, so that each instruction covers
// whole 64-byte row segments.
template <int OT>
struct LinChunk {
    typedef typename LinOut<OT>::T TO;
    static constexpr int HALVES = OT == MOE_DT_FLOAT ? 2 : 1;  // 64-byte pieces of 32 columns
    static constexpr int HC = 32 / HALVES;                     // columns per piece
    static constexpr int E16 = 16 / (int)sizeof(TO);           // elements of 16 bytes
    uint4 rq[HALVES * 4];
    bool fast;

    // rows r0 + 8 i, 16-byte piece c0 of the 64, are this lane's in the transposed view
    __device__ __forceinline__ void load_residual(const LinParams& p, const LinWarpTile& w, int j)
    {
        fast = p.vec_y && (!p.residual || p.vec_r) && j + 32 <= w.valid;
        if (p.residual && fast) {
            const int r0 = w.lane >> 2, c0 = w.lane & 3;
            const TO* res = static_cast<const TO*>(p.residual) + (size_t)w.row0 * p.ldr + w.col0 + j + c0 * E16;
#pragma unroll
            for (int h = 0; h < HALVES; h++)
#pragma unroll
                for (int i = 0; i < 4; i++)
                    if (r0 + 8 * i < w.rows)
                        rq[h * 4 + i] = *reinterpret_cast<const uint4*>(res + (size_t)(r0 + 8 * i) * p.ldr + h * HC);
        }
    }

    __device__ __forceinline__ void store(const LinParams& p, const LinWarpTile& w, int j, float (&v)[32])
    {
        uint8_t* const stg = w.stg;
        uint4* const mine = reinterpret_cast<uint4*>(stg + w.lane * LG_STG_ROW);
        TO* const y = static_cast<TO*>(p.y) + (size_t)w.row0 * p.ldy + w.col0 + j;
        if (fast) {
            const int r0 = w.lane >> 2, c0 = w.lane & 3;
            uint4* const trans = reinterpret_cast<uint4*>(stg + r0 * LG_STG_ROW + c0 * 16);
            constexpr int STEP = 8 * LG_STG_ROW / 16;
#pragma unroll
            for (int h = 0; h < HALVES; h++) {
                if (p.residual) {
#pragma unroll
                    for (int i = 0; i < 4; i++) trans[i * STEP] = rq[h * 4 + i];
                    __syncwarp();
#pragma unroll
                    for (int i = 0; i < 4; i++) lin_add16<OT>(v + h * HC + i * E16, mine[i]);
                    __syncwarp();
                }
#pragma unroll
                for (int i = 0; i < 4; i++) mine[i] = lin_pack16<OT>(v + h * HC + i * E16);
                __syncwarp();
                uint4 o[4];
#pragma unroll
                for (int i = 0; i < 4; i++) o[i] = trans[i * STEP];
#pragma unroll
                for (int i = 0; i < 4; i++)
                    if (r0 + 8 * i < w.rows)
                        *reinterpret_cast<uint4*>(y + (size_t)(r0 + 8 * i) * p.ldy + h * HC + c0 * E16) = o[i];
                __syncwarp();
            }
        } else {
            // Rows off 16-byte boundaries, or the last columns: an element per lane, so that
            // an instruction still covers whole 64-byte segments (two half rows of them, as
            // this once did, took 1.5 times as long: L2 merges every partial sector).
            constexpr int RPI = 32 / HC;  // rows per instruction
            const int rr = w.lane / HC, c = w.lane % HC;
            const TO* const res =
                p.residual ? static_cast<const TO*>(p.residual) + (size_t)w.row0 * p.ldr + w.col0 + j : nullptr;
#pragma unroll
            for (int h = 0; h < HALVES; h++) {
                const bool in = j + h * HC + c < w.valid;
                if (res) {
                    // every load without a condition (clamped to what exists), all at once
                    const TO* const src = res + (in ? h * HC + c : 0);
                    TO a[32 / RPI];
#pragma unroll
                    for (int i = 0; i < 32 / RPI; i++) a[i] = src[(size_t)min(i * RPI + rr, w.rows - 1) * p.ldr];
#pragma unroll
                    for (int i = 0; i < 32 / RPI; i++)
                        reinterpret_cast<TO*>(stg + (i * RPI + rr) * LG_STG_ROW)[c] = a[i];
                    __syncwarp();
#pragma unroll
                    for (int i = 0; i < 4; i++) lin_add16<OT>(v + h * HC + i * E16, mine[i]);
                    __syncwarp();
                }
#pragma unroll
                for (int i = 0; i < 4; i++) mine[i] = lin_pack16<OT>(v + h * HC + i * E16);
                __syncwarp();
                if (in) {
#pragma unroll 8
                    for (int r = rr; r < w.rows; r += RPI)
                        y[(size_t)r * p.ldy + h * HC + c] = reinterpret_cast<const TO*>(stg + r * LG_STG_ROW)[c];
                }
                __syncwarp();
            }
        }
    }
};

// Brings the residual of a warp's rows on its way while the products still run: a lane per
// row, the lines that its columns touch (the two warps of a quarter take every other one).
__device__ __forceinline__ void lin_prefetch_residual(const LinParams& p, const LinWarpTile& w, int half)
{
    if (!p.residual || w.lane >= w.rows) return;
    const size_t es = p.otype == MOE_DT_FLOAT ? 4 : 2;
    const uintptr_t row = reinterpret_cast<uintptr_t>(p.residual) + ((size_t)(w.row0 + w.lane) * p.ldr + w.col0) * es;
    const uintptr_t end = row + (size_t)w.valid * es;
    for (uintptr_t a = (row & ~(uintptr_t)127) + 128 * half; a < end; a += 256)
        asm volatile("prefetch.global.L1 [%0];" ::"l"(a < row ? row : a));
}

__device__ __forceinline__ void lin_tmem_load(uint32_t taddr, float (&v)[32])
{
    uint32_t a[32];
    tmem_ld_32x32b_x32(taddr, a);
    tmem_ld_wait();
#pragma unroll
    for (int c = 0; c < 32; c++) v[c] = __uint_as_float(a[c]);
}

// A warp's part of a 16-bit tile, every other chunk of 32 columns (`half`): sums from TMEM
// (tbase; the up sums of a gated tile `up` columns further), bias, activation, gate,
// residual, store.
template <int OT>
__device__ __forceinline__ void lin_epilogue(const LinParams& p, uint32_t tbase, int up, const LinWarpTile& w, int half)
{
#pragma unroll 1
    for (int j = 32 * half; j < w.valid; j += 64) {
        float v[32];
        LinChunk<OT> chunk;
        chunk.load_residual(p, w, j);
        if (p.gated) {
            float u[32];
            uint32_t a[32], b[32];
            tmem_ld_32x32b_x32(tbase + j, a);
            tmem_ld_32x32b_x32(tbase + up + j, b);
            tmem_ld_wait();
#pragma unroll
            for (int c = 0; c < 32; c++) {
                v[c] = __uint_as_float(a[c]);
                u[c] = __uint_as_float(b[c]);
            }
            if (p.bias) {
                lin_add_bias(p, w.lane, w.col0 + j, 0, v);
                lin_add_bias(p, w.lane, w.col0 + j, p.N, u);
            }
            lin_act(v, p.act);
#pragma unroll
            for (int c = 0; c < 32; c++) v[c] *= u[c];
        } else {
            lin_tmem_load(tbase + j, v);
            if (p.bias) lin_add_bias(p, w.lane, w.col0 + j, 0, v);
            lin_act(v, p.act);
        }
        chunk.store(p, w, j, v);
    }
}

// F32: y is fp32, and the sums go through registers every LG_SEGMENT k blocks.
template <int PAIR, int BN, bool F32>
__global__ void __launch_bounds__((LinCfg<PAIR, BN>::THREADS), 1)
linear_gemm_kernel(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmW,
                   const LinParams p)
{
    using Cfg = LinCfg<PAIR, BN>;
    static_assert(!F32 || (BN == 128 && !PAIR), "a warp holds two chunks of sums");
    constexpr int STAGES = Cfg::STAGES;
    constexpr int STAGE_BYTES = Cfg::STAGE_BYTES;
    constexpr int ROWS = Cfg::ROWS;
    constexpr int KPS = Cfg::KPS;
    extern __shared__ uint8_t lg_smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>(
        (reinterpret_cast<uintptr_t>(lg_smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    LinTail* tail = reinterpret_cast<LinTail*>(smem + STAGES * STAGE_BYTES);

    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);  // uniform, and known to be
    const int lane = threadIdx.x & 31;
    int* err = p.err ? p.err : &g_linear_err;
    // Pair mode: rank 0 of the cluster issues the UMMAs and owns the barriers they wait on.
    const uint32_t crank = PAIR ? cluster_ctarank() : 0u;
    const bool leader = crank == 0u;
    const int unit = PAIR ? (int)(blockIdx.x >> 1) : (int)blockIdx.x;
    const int nunits = PAIR ? (int)(gridDim.x >> 1) : (int)gridDim.x;

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; s++) {
            mbar_init(smem_u32(&tail->full[s]), Cfg::X_WARP ? 2 : 1);
            mbar_init(smem_u32(&tail->empty[s]), 1);
        }
        for (int a = 0; a < 2; a++) {
            mbar_init(smem_u32(&tail->tfull[a]), 1);
            mbar_init(smem_u32(&tail->tempty[a]), (PAIR ? 2 : 1) * LG_EPI_WARPS);  // one arrival per epilogue warp
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
    // what the producers need first, while TMEM is allocated
    const uint64_t pol_x = l2_policy_evict_last();
    const uint64_t pol_w = p.w_evict_first ? l2_policy_evict_first() : l2_policy_evict_last();
    int m, n;
    lin_tile(p, (uint32_t)unit, m, n);
    tc_fence_before();
    if (PAIR)
        cluster_sync_all();  // both CTAs' barriers are initialised before any remote arrival
    else
        __syncthreads();
    tc_fence_after();
    pdl_wait();  // inputs come from, and y may still be read by, the launches before

    const uint32_t tmem_base = tail->tmem_base;
    const int total = p.mt * p.nt;  // below 2^29: the host checks
    const int nk = p.nk;
    volatile int* abort_flag = &tail->abort_flag;

    if (warp == 0 || (Cfg::X_WARP && warp == 2 + LG_EPI_WARPS)) {
        // ---------------------------------------------------------------- producers
        if (elect_one()) {
            const bool do_w = warp == 0, do_x = !Cfg::X_WARP || warp != 0;
            const uint32_t kb_tx = (do_w ? Cfg::KB_BYTES - LG_A_BYTES : 0) + (do_x ? p.x_rows * LG_BK * 2 : 0);
            uint32_t it = 0;
            bool ok = true;
            for (int tile = unit; ok && tile < total; tile += nunits) {
                if (tile != unit) lin_tile(p, tile, m, n);
                const int x_row = m * ROWS + (int)crank * LG_BM;
                const int w_lo = n * (p.gated ? BN / 2 : BN);
                const int w_hi = p.gated ? p.N + w_lo : w_lo + BN / 2;
                for (int kb = 0; kb < nk; kb += KPS, it++) {
                    const int s = it % STAGES;
                    const uint32_t par = ((it / STAGES) & 1u) ^ 1u;
                    // the first round finds every stage empty
                    const bool got = it < (uint32_t)STAGES || lin_wait<PAIR != 0>(smem_u32(&tail->empty[s]), par, err,
                                                                                MOE_DEV_WAIT_TIMEOUT_TMA, abort_flag);
                    if (!got) {
                        ok = false;
                        break;
                    }
                    const uint32_t full = smem_u32(&tail->full[s]);
                    const uint32_t st = smem_u32(smem + s * STAGE_BYTES);
                    const int nb = min(KPS, nk - kb);
                    if (PAIR) {
                        // both CTAs' copies complete on the leader's barrier, which
                        // expects the bytes of both
                        const uint32_t full_leader = mapa_shared(full, 0);
                        if (leader) mbar_arrive_expect_tx(full, 2 * nb * kb_tx);
#pragma unroll
                        for (int i = 0; i < KPS; i++) {
                            if (i >= nb) break;
                            const uint32_t dst = st + i * Cfg::KB_BYTES;
                            tma_load_2d_pair(dst, &tmX, full_leader, (kb + i) * LG_BK, x_row, pol_x);
                            tma_load_2d_pair(dst + LG_A_BYTES, &tmW, full_leader, (kb + i) * LG_BK, leader ? w_lo : w_hi, pol_w);
                        }
                    } else {
                        mbar_arrive_expect_tx(full, nb * kb_tx);
#pragma unroll
                        for (int i = 0; i < KPS; i++) {
                            if (i >= nb) break;
                            const uint32_t dst = st + i * Cfg::KB_BYTES;
                            if (do_x) tma_load_2d(dst, &tmX, full, (kb + i) * LG_BK, x_row, pol_x);
                            if (do_w) {
                                tma_load_2d(dst + LG_A_BYTES, &tmW, full, (kb + i) * LG_BK, w_lo, pol_w);
                                tma_load_2d(dst + LG_A_BYTES + Cfg::B_HALF, &tmW, full, (kb + i) * LG_BK, w_hi, pol_w);
                            }
                        }
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
        if (leader && elect_one()) {
            const uint32_t idesc = lin_idesc(ROWS, BN, p.type == MOE_DT_BF16);
            const int seg = F32 ? LG_SEGMENT : nk;
            uint32_t it = 0, lt = 0;
            bool ok = true;
            for (int tile = unit; ok && tile < total; tile += nunits) {
                for (int k0 = 0; ok && k0 < nk; k0 += seg, lt++) {
                    const int k1 = min(k0 + seg, nk);
                    const uint32_t acc = lt & 1u;
                    if (!lin_wait<PAIR != 0>(smem_u32(&tail->tempty[acc]), ((lt >> 1) & 1u) ^ 1u, err,
                                             MOE_DEV_WAIT_TIMEOUT_MMA, abort_flag)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const uint32_t d = tmem_base + acc * BN;
                    for (int kb = k0; kb < k1; kb += KPS, it++) {
                        const int s = it % STAGES;
                        if (!lin_wait<PAIR != 0>(smem_u32(&tail->full[s]), (it / STAGES) & 1u, err,
                                                 MOE_DEV_WAIT_TIMEOUT_MMA, abort_flag)) {
                            ok = false;
                            break;
                        }
                        tc_fence_after();
#pragma unroll
                        for (int i = 0; i < KPS; i++) {
                            if (kb + i >= k1) break;
                            const uint32_t a_addr = smem_u32(smem + s * STAGE_BYTES + i * Cfg::KB_BYTES);
                            const uint32_t b_addr = a_addr + LG_A_BYTES;
#pragma unroll
                            for (int k = 0; k < LG_BK / 16; k++) {
                                // k advances by 16 elements = 32 bytes inside the swizzle row
                                const uint64_t da = umma_desc_sw128(a_addr + k * 32), db = umma_desc_sw128(b_addr + k * 32);
                                if (PAIR)
                                    umma_f16_ss_pair(d, da, db, idesc, (kb - k0) | i | k);
                                else
                                    umma_f16_ss(d, da, db, idesc, (kb - k0) | i | k);
                            }
                        }
                        if (PAIR) {
                            umma_commit_pair(smem_u32(&tail->empty[s]));
                            umma_commit_pair(mapa_shared(smem_u32(&tail->empty[s]), 1));
                        } else {
                            umma_commit(smem_u32(&tail->empty[s]));
                        }
                    }
                    if (!ok) break;
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
            lin_drain<PAIR != 0>(smem_u32(&tail->drain), err);
        }
    } else {
        // ---------------------------------------------------------------- epilogue
        const int q = warp & 3;  // the TMEM lane quarter this warp may read
        uint8_t* stg = smem + STAGES * STAGE_BYTES + LG_TAIL + (size_t)(warp - 2) * LG_STG_WARP;
        const int half = (warp - 2) >> 2;
        // in pair mode the epilogue warps of both CTAs release the leader's accumulator
        const uint32_t tempty0 = PAIR ? mapa_shared(smem_u32(&tail->tempty[0]), 0) : smem_u32(&tail->tempty[0]);
        uint32_t lt = 0;
        for (int tile = unit; tile < total; tile += nunits, lt++) {
            if (tile != unit) lin_tile(p, tile, m, n);
            const uint32_t acc = lt & 1u;
            const uint32_t tpar = (lt >> 1) & 1u;
            const int cols = p.gated ? BN / 2 : BN;
            LinWarpTile w = {stg, lane, m * ROWS + (int)crank * LG_BM + q * 32, 0, n * cols, 0};
            w.rows = min(32, p.T - w.row0);  // <= 0: none of this warp's rows exist
            w.valid = min(cols, p.N - w.col0);
            lin_prefetch_residual(p, w, half);
            if (!(lin_wait<PAIR != 0>(smem_u32(&tail->tfull[acc]), tpar, err, MOE_DEV_WAIT_TIMEOUT_EPI, abort_flag)))
                break;
            tc_fence_after();
            const uint32_t quarter = tmem_base + ((uint32_t)(q * 32) << 16);
            if constexpr (F32) {
                // The sums of this warp's two chunks (gated: gate and up of one), added up
                // over the segments in fp32 registers; the accumulator of one segment is
                // read while the next one's products run.
                const int j0 = 32 * half, j1 = p.gated ? BN / 2 + j0 : j0 + 64;
                float v[32], u[32];
                bool ok = true;
                for (int k0 = 0; k0 < nk; k0 += LG_SEGMENT, lt++) {
                    const uint32_t acc = lt & 1u;
                    if (k0 > 0 && !lin_wait<false>(smem_u32(&tail->tfull[acc]), (lt >> 1) & 1u, err,
                                                   MOE_DEV_WAIT_TIMEOUT_EPI, abort_flag)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    if (k0 == 0) {
                        lin_tmem_load(quarter + acc * BN + j0, v);
                        lin_tmem_load(quarter + acc * BN + j1, u);
                    } else {
                        float a[32];
                        lin_tmem_load(quarter + acc * BN + j0, a);
#pragma unroll
                        for (int c = 0; c < 32; c++) v[c] += a[c];
                        lin_tmem_load(quarter + acc * BN + j1, a);
#pragma unroll
                        for (int c = 0; c < 32; c++) u[c] += a[c];
                    }
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(tempty0 + acc * (uint32_t)sizeof(uint64_t));
                }
                if (!ok) break;
                lt--;  // the loop's step counts the last segment
                if (w.rows > 0) {
                    if (p.bias) {
                        lin_add_bias(p, lane, w.col0 + j0, 0, v);
                        lin_add_bias(p, lane, w.col0 + (p.gated ? j0 : j1), p.gated ? (size_t)p.N : 0, u);
                    }
                    lin_act(v, p.act);
                    LinChunk<MOE_DT_FLOAT> chunk;
                    if (p.gated) {
#pragma unroll
                        for (int c = 0; c < 32; c++) v[c] *= u[c];
                    }
                    if (j0 < w.valid) {
                        chunk.load_residual(p, w, j0);
                        chunk.store(p, w, j0, v);
                    }
                    if (!p.gated && j1 < w.valid) {
                        lin_act(u, p.act);
                        chunk.load_residual(p, w, j1);
                        chunk.store(p, w, j1, u);
                    }
                }
            } else if (w.rows > 0) {
                if (p.otype == MOE_DT_FLOAT16)
                    lin_epilogue<MOE_DT_FLOAT16>(p, quarter + acc * BN, BN / 2, w, half);
                else
                    lin_epilogue<MOE_DT_BF16>(p, quarter + acc * BN, BN / 2, w, half);
            }
            if (!F32) {
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
// One 128 x BN tile per cluster of S CTAs.  CTA r multiplies k blocks [nk r / S,
// nk (r + 1) / S), lays its sums out as S blocks [128][W + 4], W = BN / S (gated: W/2 gate
// and W/2 up columns), in the shared memory that its operands no longer need, and sends
// block d to CTA d by bulk copies: stores to distributed shared memory, 16 bytes per lane,
// took 5 us for the 64 KB where these take less than 1.  Each CTA finishes its own columns
// from the S partial sums in rank order.
constexpr int LS_KPS = 2;        // k blocks per stage, as in the narrow tiles
constexpr int LS_THREADS = 256;  // w copies, UMMA, 4 TMEM readers, x copies, 1 more to finish columns

template <int S, int BN>
struct SplitCfg {
    static constexpr int W = BN / S;
    static constexpr int PITCH = W + 4;
    static constexpr int B_HALF = BN / 2 * LG_BK * 2;
    static constexpr int KB_BYTES = LG_A_BYTES + 2 * B_HALF;
    static constexpr int STAGE_BYTES = LS_KPS * KB_BYTES;
    static constexpr int RECV_BYTES = S * LG_BM * PITCH * 4;
    static constexpr int STAGES = BN == 64 ? 3 : 2;  // 128 or 144 KB
    static constexpr size_t SMEM = 1024 + (size_t)STAGES * STAGE_BYTES + RECV_BYTES + LG_TAIL;
    static_assert(W >= 16, "a gated CTA finishes at least 8 outputs");
    static_assert(STAGES * STAGE_BYTES >= RECV_BYTES, "the sums fit the ring");
    static_assert(SMEM <= 227 * 1024, "smem");
};

// Copies `bytes` of this CTA's shared memory to another CTA's (shared::cluster addresses),
// counted on that CTA's mbarrier.
__device__ __forceinline__ void copy_to_cta(uint32_t dst_cluster, uint32_t src, uint32_t bytes, uint32_t bar_cluster)
{
    asm volatile("cp.async.bulk.shared::cluster.shared::cta.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst_cluster),
                 "r"(src), "r"(bytes), "r"(bar_cluster)
                 : "memory");
}

// Finishes this CTA's columns: 8 outputs per thread and step.
template <int S, int BN, bool GATED, int OT>
__device__ __forceinline__ void split_finish(const LinParams& p, const float* recv, int m, int col0)
{
    constexpr int OUTS = GATED ? SplitCfg<S, BN>::W / 2 : SplitCfg<S, BN>::W;
    constexpr int V = 8;
    constexpr int GROUPS = OUTS / V;
    constexpr int PITCH = SplitCfg<S, BN>::PITCH;
    const int rows = min(LG_BM, p.T - m * LG_BM);
#pragma unroll 1
    for (int i = threadIdx.x; i < rows * GROUPS; i += LS_THREADS) {
        const int row = i / GROUPS, g = i % GROUPS;
        const int n = col0 + V * g, left = p.N - n;
        if (left <= 0) continue;
        const float* src = recv + row * PITCH + V * g;
        float v[V] = {}, u[V] = {};
#pragma unroll
        for (int s = 0; s < S; s++)
#pragma unroll
            for (int j = 0; j < V; j += 4) {
                const float4 a = *reinterpret_cast<const float4*>(src + s * LG_BM * PITCH + j);
                v[j] += a.x;
                v[j + 1] += a.y;
                v[j + 2] += a.z;
                v[j + 3] += a.w;
                if (GATED) {
                    const float4 b = *reinterpret_cast<const float4*>(src + s * LG_BM * PITCH + OUTS + j);
                    u[j] += b.x;
                    u[j + 1] += b.y;
                    u[j + 2] += b.z;
                    u[j + 3] += b.w;
                }
            }
        if (p.bias) {
#pragma unroll
            for (int j = 0; j < V; j++)
                if (j < left) {
                    v[j] += lin_load(p.bias, n + j, p.type);
                    if (GATED) u[j] += lin_load(p.bias, (size_t)p.N + n + j, p.type);
                }
        }
        lin_act(v, p.act);
        if (GATED) {
#pragma unroll
            for (int j = 0; j < V; j++) v[j] *= u[j];
        }
        typedef typename LinOut<OT>::T TO;
        constexpr int E16 = 16 / (int)sizeof(TO);
        const size_t t = (size_t)m * LG_BM + row;
        TO* dst = static_cast<TO*>(p.y) + t * p.ldy + n;
        const TO* res = p.residual ? static_cast<const TO*>(p.residual) + t * p.ldr + n : nullptr;
        if (V % E16 == 0 && left >= V && p.vec_y && (!res || p.vec_r)) {
#pragma unroll
            for (int j = 0; j < V; j += E16) {
                if (res) lin_add16<OT>(v + j, *reinterpret_cast<const uint4*>(res + j));
                *reinterpret_cast<uint4*>(dst + j) = lin_pack16<OT>(v + j);
            }
        } else {
#pragma unroll
            for (int j = 0; j < V; j++)
                if (j < left) dst[j] = LinOut<OT>::to(v[j] + (res ? LinOut<OT>::from(res[j]) : 0.0f));
        }
    }
}

template <int S, int BN, int OT>
__device__ __forceinline__ void split_finish_any(const LinParams& p, const float* recv, int m, int col0)
{
    if (p.gated)
        split_finish<S, BN, true, OT>(p, recv, m, col0);
    else
        split_finish<S, BN, false, OT>(p, recv, m, col0);
}

// F32: y is fp32, and every LG_SEGMENT k blocks the accumulator is emptied into registers,
// while the next ones go to a second one.  Compiled apart from a 16-bit y, which has
// one segment: 128 x 2048 -> 2048 takes 7.8 us so, 8.1 with both in one kernel.
template <int S, int BN, bool F32>
__global__ void __launch_bounds__(LS_THREADS, 1)
linear_split_kernel(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmW, const LinParams p)
{
    using Cfg = SplitCfg<S, BN>;
    constexpr int W = Cfg::W;
    constexpr int PITCH = Cfg::PITCH;
    extern __shared__ uint8_t ls_smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>(
        (reinterpret_cast<uintptr_t>(ls_smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    float* recv = reinterpret_cast<float*>(smem + Cfg::STAGES * Cfg::STAGE_BYTES);
    LinTail* tail = reinterpret_cast<LinTail*>(smem + Cfg::STAGES * Cfg::STAGE_BYTES + Cfg::RECV_BYTES);

    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);  // uniform, and known to be
    const int lane = threadIdx.x & 31;
    int* err = p.err ? p.err : &g_linear_err;
    const int rank = (int)cluster_ctarank();
    const int tile = (int)(blockIdx.x / S);
    const int kb0 = (int)((long long)p.nk * rank / S), kb1 = (int)((long long)p.nk * (rank + 1) / S);
    constexpr uint32_t TMEM_COLS = F32 ? 2 * BN : BN;

    if (threadIdx.x == 0) {
        for (int s = 0; s < Cfg::STAGES; s++) {
            mbar_init(smem_u32(&tail->full[s]), 2);  // the copies of w, the copies of x
            mbar_init(smem_u32(&tail->empty[s]), 1);
        }
        if (F32) {
            mbar_init(smem_u32(&tail->tfull[0]), 1);
            mbar_init(smem_u32(&tail->tfull[1]), 1);
        }
        mbar_init(smem_u32(&tail->drain), 1);
        mbar_init(smem_u32(&tail->recv), 1);
        tail->abort_flag = 0;
        fence_barrier_init();
        tma_prefetch_desc(&tmX);
        tma_prefetch_desc(&tmW);
    }
    pdl_trigger();
    if (warp == 1) {
        tmem_alloc(smem_u32(&tail->tmem_base), TMEM_COLS);
        tmem_relinquish();
    }
    int m, n;
    lin_tile(p, tile, m, n);
    // (what the producers need first is made while TMEM is allocated)
    const uint64_t pol_x = l2_policy_evict_last();
    const uint64_t pol_w = p.w_evict_first ? l2_policy_evict_first() : l2_policy_evict_last();
    // S slabs of 32 rows come for each of the tile's row quarters that exist
    constexpr uint32_t SLAB = 32 * PITCH * 4;
    const int quarters = min(4, (p.T - m * LG_BM + 31) / 32);
    if (threadIdx.x == 0) {
        if (F32) {
            mbar_init(smem_u32(&tail->tempty[0]), quarters);  // one arrival per warp that reads sums
            mbar_init(smem_u32(&tail->tempty[1]), quarters);
        }
        mbar_arrive_expect_tx(smem_u32(&tail->recv), S * quarters * SLAB);
    }
    tc_fence_before();
    cluster_sync_all();  // barriers are initialised, and every CTA's shared memory is live
    tc_fence_after();
    pdl_wait();

    const uint32_t tmem_base = tail->tmem_base;
    volatile int* abort_flag = &tail->abort_flag;
    const int cols = p.gated ? BN / 2 : BN;

    if (warp == 0 || warp == 6) {
        // A copy takes about 95 cycles to issue, more than a third of the products it
        // feeds: w (two boxes per k block) and x have a warp each.
        if (elect_one()) {
            const bool is_w = warp == 0;
            const uint64_t pol = is_w ? pol_w : pol_x;
            const uint32_t kb_tx = is_w ? 2 * Cfg::B_HALF : p.x_rows * LG_BK * 2;
            const int w_lo = n * cols;
            const int w_hi = p.gated ? p.N + w_lo : w_lo + BN / 2;
            uint32_t it = 0;
            bool ok = true;
            for (int kb = kb0; kb < kb1; kb += LS_KPS, it++) {
                const int s = it % Cfg::STAGES;
                if (it >= (uint32_t)Cfg::STAGES && !lin_wait<false>(smem_u32(&tail->empty[s]), ((it / Cfg::STAGES) & 1u) ^ 1u,
                                                                  err, MOE_DEV_WAIT_TIMEOUT_TMA, abort_flag)) {
                    ok = false;
                    break;
                }
                const uint32_t full = smem_u32(&tail->full[s]);
                const uint32_t st = smem_u32(smem + s * Cfg::STAGE_BYTES);
                const int nb = min(LS_KPS, kb1 - kb);
                mbar_arrive_expect_tx(full, nb * kb_tx);
#pragma unroll
                for (int i = 0; i < LS_KPS; i++) {
                    if (i >= nb) break;
                    const uint32_t dst = st + i * Cfg::KB_BYTES;
                    if (is_w) {
                        tma_load_2d(dst + LG_A_BYTES, &tmW, full, (kb + i) * LG_BK, w_lo, pol);
                        tma_load_2d(dst + LG_A_BYTES + Cfg::B_HALF, &tmW, full, (kb + i) * LG_BK, w_hi, pol);
                    } else {
                        tma_load_2d(dst, &tmX, full, (kb + i) * LG_BK, m * LG_BM, pol);
                    }
                }
            }
            if (!ok) {
                // giving up: the copies in flight land (bounded wait) before the CTA exits
                const uint32_t first = it > (uint32_t)Cfg::STAGES ? it - Cfg::STAGES : 0;
                for (uint32_t j = first; j < it; j++) {
                    const uint64_t t0 = global_timer_ns();
                    while (!mbar_try_wait(smem_u32(&tail->full[j % Cfg::STAGES]), (j / Cfg::STAGES) & 1u))
                        if (global_timer_ns() - t0 > MOE_WAIT_LIMIT_NS) break;
                }
            }
        }
    } else if (warp == 1) {
        if (elect_one()) {
            const uint32_t idesc = lin_idesc(LG_BM, BN, p.type == MOE_DT_BF16);
            uint32_t it = 0;
            for (int kb = kb0; kb < kb1; kb += LS_KPS, it++) {
                const int s = it % Cfg::STAGES;
                if (!lin_wait<false>(smem_u32(&tail->full[s]), (it / Cfg::STAGES) & 1u, err,
                                               MOE_DEV_WAIT_TIMEOUT_MMA, abort_flag))
                    break;
                const int part = F32 ? (kb - kb0) / LG_SEGMENT : 0, first = kb - kb0 - part * LG_SEGMENT;
                const uint32_t acc = part & 1;
                if (F32 && first == 0 && part >= 2 && !lin_wait<false>(smem_u32(&tail->tempty[acc]), ((part >> 1) & 1u) ^ 1u, err,
                                                               MOE_DEV_WAIT_TIMEOUT_MMA, abort_flag))
                    break;
                tc_fence_after();
                const uint32_t d = tmem_base + acc * BN;
                static_assert(LG_SEGMENT % LS_KPS == 0, "a stage belongs to one segment");
#pragma unroll
                for (int i = 0; i < LS_KPS; i++) {
                    if (kb + i >= kb1) break;
                    const uint32_t a_addr = smem_u32(smem + s * Cfg::STAGE_BYTES + i * Cfg::KB_BYTES);
                    const uint32_t b_addr = a_addr + LG_A_BYTES;
#pragma unroll
                    for (int k = 0; k < LG_BK / 16; k++)
                        umma_f16_ss(d, umma_desc_sw128(a_addr + k * 32), umma_desc_sw128(b_addr + k * 32), idesc,
                                    first | i | k);
                }
                umma_commit(smem_u32(&tail->empty[s]));
                if (F32 && (kb + LS_KPS >= kb1 || first + LS_KPS == LG_SEGMENT)) umma_commit(smem_u32(&tail->tfull[acc]));
            }
            umma_commit(smem_u32(&tail->drain));  // all sums of this CTA are in TMEM
            lin_drain<false>(smem_u32(&tail->drain), err);
        }
    } else if (warp < 6) {
        const int q = warp & 3;
        const uint32_t row = tmem_base + ((uint32_t)(q * 32) << 16);
        const int last = F32 ? (kb1 - kb0 - 1) / LG_SEGMENT : 0;
        float sum[F32 ? BN : 1] = {};  // of the segments before the last
        bool got = q < quarters;
        if constexpr (F32) {
            for (int part = 0; got && part < last; part++) {
                const uint32_t acc = part & 1;
                got = lin_wait<false>(smem_u32(&tail->tfull[acc]), (part >> 1) & 1u, err, MOE_DEV_WAIT_TIMEOUT_EPI, abort_flag);
                if (!got) break;
                tc_fence_after();
#pragma unroll
                for (int j = 0; j < BN; j += 32) {
                    float a[32];
                    lin_tmem_load(row + acc * BN + j, a);
#pragma unroll
                    for (int c = 0; c < 32; c++) sum[j + c] += a[c];
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&tail->tempty[acc]));
            }
        }
        if (got && lin_wait<false>(smem_u32(&tail->drain), 0, err, MOE_DEV_WAIT_TIMEOUT_EPI, abort_flag)) {
            tc_fence_after();
            // block d's row of this lane: the ring's operands have been consumed
            float* const mine = reinterpret_cast<float*>(smem) + (q * 32 + lane) * PITCH;
#pragma unroll
            for (int j = 0; j < BN; j += 32) {
                float a[32];
                lin_tmem_load(row + (last & 1) * BN + j, a);
                if constexpr (F32) {
#pragma unroll
                    for (int c = 0; c < 32; c++) a[c] += sum[j + c];
                }
#pragma unroll
                for (int c = 0; c < 32; c += 4) {
                    const int col = j + c;
                    // gated: the first BN / 2 columns are gate sums, the others up sums
                    const int d = p.gated ? col % (BN / 2) / (W / 2) : col / W;
                    const int off = p.gated ? col / (BN / 2) * (W / 2) + col % (BN / 2) % (W / 2) : col % W;
                    *reinterpret_cast<float4*>(mine + d * LG_BM * PITCH + off) =
                        make_float4(a[c], a[c + 1], a[c + 2], a[c + 3]);
                }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane < S) {
                const uint32_t src = smem_u32(smem) + (uint32_t)((lane * LG_BM + q * 32) * PITCH) * 4u;
                const uint32_t dst = smem_u32(recv) + (uint32_t)((rank * LG_BM + q * 32) * PITCH) * 4u;
                copy_to_cta(mapa_shared(dst, (uint32_t)lane), src, SLAB, mapa_shared(smem_u32(&tail->recv), (uint32_t)lane));
            }
        }
        tc_fence_before();
    }
    __syncwarp();
    // Every partial sum of this CTA's columns has arrived (or a wait gave up).  One thread
    // looks: 256 that poll slow down what they wait for.
    if (threadIdx.x == 0) lin_wait<true>(smem_u32(&tail->recv), 0, err, MOE_DEV_WAIT_TIMEOUT_EPI, abort_flag);
    __syncthreads();
    const bool arrived = *abort_flag == 0;
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem_base, TMEM_COLS);
    }
    // no CTA leaves while its sums may still be read: all have arrived here once all have
    // received
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    const int col0 = n * cols + rank * (cols / S);
    if (arrived) {
        if (F32)
            split_finish_any<S, BN, MOE_DT_FLOAT>(p, recv, m, col0);
        else if (p.otype == MOE_DT_FLOAT16)
            split_finish_any<S, BN, MOE_DT_FLOAT16>(p, recv, m, col0);
        else
            split_finish_any<S, BN, MOE_DT_BF16>(p, recv, m, col0);
    }
    __syncwarp();
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// ---------------------------------------------------------------------- a few tokens
// A warp holds MT blocks of 16 rows of w (gated: 16 gate rows and their 16 up rows) and
// NT blocks of 8 tokens; the block's warps divide k among them and add up in shared
// memory, in warp order.  w goes from HBM into fragment registers with no stop in shared
// memory: a product does not depend on the order of k, so lane (g, t) takes 8 consecutive
// elements (16 bytes) of rows g and g + 8 at k = 32 c + 8 t, and of token g, and feeds
// them to two m16n8k16 products as if they were the columns those expect.
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

// k chunks of 32 in flight per warp: 128 to 256 bytes of w per lane
template <int MT, int NT>
constexpr int lin_few_depth() { return MT == 2 || NT == 2 ? 4 : 8; }

template <bool BF16, int MT, int NT, int WARPS>
__global__ void __launch_bounds__(WARPS * 32, 16 / WARPS) linear_few_kernel(const LinearArgs a)
{
    constexpr int D = lin_few_depth<MT, NT>();
    __shared__ float red[WARPS][NT * 8][MT * 16 + 1];
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
    // A ring of D chunks in registers: chunk c of this warp is k = chunk_k(c), two chunks
    // (128 bytes of a row) to a warp in turn.  A slot is loaded again as soon as its chunk
    // has been multiplied, so D - 1 chunks are always on their way.
    float acc[MT][NT][4] = {};
    uint4 wa[D][MT][2], xb[D][NT];
    const uint4 zero = make_uint4(0, 0, 0, 0);
    auto chunk_k = [&](int c) { return ((c >> 1) * WARPS + warp) * 64 + (c & 1) * 32; };
    auto load = [&](int slot, int kk) {
        const bool in = kk + 8 * t < a.K;
#pragma unroll
        for (int i = 0; i < MT; i++)
#pragma unroll
            for (int h = 0; h < 2; h++) wa[slot][i][h] = in ? ld_stream16(wr[i][h] + kk) : zero;
#pragma unroll
        for (int j = 0; j < NT; j++) xb[slot][j] = (in && xin[j]) ? ld_cached16(xr[j] + kk) : zero;
    };
    pdl_wait();
#pragma unroll
    for (int d = 0; d < D; d++) load(d, chunk_k(d));
    for (int c = 0; chunk_k(c) < a.K; c += D) {
        float sum[MT][NT][4] = {};  // added up here, where sums are rounded (see LG_SEGMENT)
#pragma unroll
        for (int d = 0; d < D; d++) {
#pragma unroll
            for (int i = 0; i < MT; i++)
#pragma unroll
                for (int j = 0; j < NT; j++) {
                    const uint4 lo = wa[d][i][0], hi = wa[d][i][1], b = xb[d][j];
                    mma_16816<BF16>(sum[i][j], lo.x, hi.x, lo.y, hi.y, b.x, b.y);
                    mma_16816<BF16>(sum[i][j], lo.z, hi.z, lo.w, hi.w, b.z, b.w);
                }
            load(d, chunk_k(c + d + D));
        }
#pragma unroll
        for (int i = 0; i < MT; i++)
#pragma unroll
            for (int j = 0; j < NT; j++)
#pragma unroll
                for (int e = 0; e < 4; e++) acc[i][j][e] += sum[i][j][e];
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
    for (int i = threadIdx.x; i < outs * a.T; i += WARPS * 32) {
        const int tok = i / outs, r = i - tok * outs, n = n0 + r;
        if (n >= a.N) continue;
        float v[1] = {0.0f}, u = 0.0f;
#pragma unroll
        for (int s = 0; s < WARPS; s++) v[0] += red[s][tok][r];
        if (MT == 2 && a.gated) {
#pragma unroll
            for (int s = 0; s < WARPS; s++) u += red[s][tok][16 * (MT - 1) + r];
        }
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

// A kernel and not a memset, which holds back the dependent launches on both its sides: a
// layer call of 64 tokens took 226 us without either, 227 with this, 233 with a memset.
__global__ void clear_word_kernel(int* word)
{
    pdl_trigger();
    pdl_wait();
    *word = 0;
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

// Rows of x in one copy.  With fewer than 128 tokens the other rows of the tile's operand
// keep whatever shared memory held: their sums go to accumulator rows that nobody reads.
int lin_box_rows(int T) { return T >= LG_BM ? LG_BM : (T + 7) / 8 * 8; }

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
    p.x_rows = lin_box_rows(a.T);
    p.mt = (a.T + rows - 1) / rows;
    p.nt = (a.N + cols - 1) / cols;
    p.w_evict_first = p.mt == 1;
    return p;
}

template <int PAIR, int BN, bool F32 = false>
cudaError_t launch_tiles(const LinearArgs& a, int dev, cudaStream_t s)
{
    using Cfg = LinCfg<PAIR, BN>;
    static bool done[64] = {false};
    auto* kernel = linear_gemm_kernel<PAIR, BN, F32>;
    cudaError_t e = lin_smem_attr(kernel, lin_smem_bytes<PAIR, BN>(), done, dev);
    if (e != cudaSuccess) return e;
    CUtensorMap tx, tw;
    const uint64_t wrows = (uint64_t)a.N * (a.gated ? 2 : 1);
    if (!lin_tmap(&tx, a.x, a.type, a.K, a.T, a.ldx, lin_box_rows(a.T)) || !lin_tmap(&tw, a.w, a.type, a.K, wrows, a.ldw, BN / 2))
        return cudaErrorInvalidValue;
    const LinParams p = lin_params(a, Cfg::ROWS, a.gated ? BN / 2 : BN);
    const long long tiles = (long long)p.mt * p.nt;
    if (tiles >= (1LL << 29)) return cudaErrorInvalidValue;  // (y would not fit any memory)
    long long units = lin_sm_count(dev);
    if (PAIR) {
        // co-resident pairs: both CTAs of a pair need a free SM of one GPC
        static int resident[64] = {0};
        units = (dev >= 0 && dev < 64) ? resident[dev] : 0;
        if (units <= 0) {
            cudaLaunchConfig_t q = {};
            q.gridDim = dim3(2 * (lin_sm_count(dev) / 2));
            q.blockDim = dim3(Cfg::THREADS);
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
    return lin_launch(kernel, grid, Cfg::THREADS, lin_smem_bytes<PAIR, BN>(), PAIR ? 2 : 0, s, tx, tw, p);
}

template <int S, int BN, bool F32>
cudaError_t launch_split_as(const LinearArgs& a, int dev, cudaStream_t s)
{
    static bool done[64] = {false};
    auto* kernel = linear_split_kernel<S, BN, F32>;
    cudaError_t e = lin_smem_attr(kernel, SplitCfg<S, BN>::SMEM, done, dev);
    if (e != cudaSuccess) return e;
    CUtensorMap tx, tw;
    const uint64_t wrows = (uint64_t)a.N * (a.gated ? 2 : 1);
    if (!lin_tmap(&tx, a.x, a.type, a.K, a.T, a.ldx, lin_box_rows(a.T)) ||
        !lin_tmap(&tw, a.w, a.type, a.K, wrows, a.ldw, BN / 2))
        return cudaErrorInvalidValue;
    const LinParams p = lin_params(a, LG_BM, a.gated ? BN / 2 : BN);
    const long long tiles = (long long)p.mt * p.nt;
    if (tiles >= (1LL << 27)) return cudaErrorInvalidValue;  // (y would not fit any memory)
    return lin_launch(kernel, (unsigned)(tiles * S), LS_THREADS, SplitCfg<S, BN>::SMEM, (unsigned)S, s, tx, tw, p);
}

template <bool F32>
cudaError_t launch_split(const LinearArgs& a, int S, int bn, int dev, cudaStream_t s)
{
    if (S == 8) return launch_split_as<8, 128, F32>(a, dev, s);
    if (S == 4) return bn == 64 ? launch_split_as<4, 64, F32>(a, dev, s) : launch_split_as<4, 128, F32>(a, dev, s);
    return bn == 64 ? launch_split_as<2, 64, F32>(a, dev, s) : launch_split_as<2, 128, F32>(a, dev, s);
}

template <bool BF16, int MT, int NT>
cudaError_t launch_few_as(const LinearArgs& a, int sms, cudaStream_t s)
{
    const int rows = a.gated ? 16 : 16 * MT;
    const unsigned grid = (unsigned)((a.N + rows - 1) / rows);
    // two blocks of 8 warps per SM, or one of 16 where there is no second block.  Measured (us,
    // 8 / 16 warps): 8 x 8192 -> 2048 10.7 / 9.1, 8 x 2048 -> 2048 4.4 / 4.1, 8 x 2048 -> 3000
    // 4.5 / 7.0, 8 x 2048 -> 4096 5.0 / 7.4.
    if (grid > (unsigned)sms) return lin_launch(linear_few_kernel<BF16, MT, NT, 8>, grid, 256, 0, 0, s, a);
    return lin_launch(linear_few_kernel<BF16, MT, NT, 16>, grid, 512, 0, 0, s, a);
}

// At most 8 tokens, or 16 when not gated.  Two blocks of w rows per warp (MT = 2): gated, or
// where one block each would take a second wave and two do not.  Measured (us, MT = 1 / 2), 8
// tokens: 2048 -> 4736 5.2 / 5.6, 2048 -> 5000 6.9 / 6.3, 7168 -> 6144 19.8 / 16.6, 2048 -> 8192
// 8.9 / 7.2, 2048 -> 9472 9.3 / 7.7; over more waves 7168 -> 12288 31.2 / 33.1, 4096 -> 32768
// 43.7 / 45.7, 2048 -> 16384 13.9 / 13.5.
cudaError_t launch_few(const LinearArgs& a, int sms, cudaStream_t s)
{
    const bool bf16 = a.type == MOE_DT_BF16;
    if (a.T > 8) return bf16 ? launch_few_as<true, 1, 2>(a, sms, s) : launch_few_as<false, 1, 2>(a, sms, s);
    if (a.gated || (a.N > 32LL * sms && a.N <= 64LL * sms))
        return bf16 ? launch_few_as<true, 2, 1>(a, sms, s) : launch_few_as<false, 2, 1>(a, sms, s);
    return bf16 ? launch_few_as<true, 1, 1>(a, sms, s) : launch_few_as<false, 1, 1>(a, sms, s);
}

// How to share out k when the 128 x 128 tiles leave SMs idle.  The model, in ns: a k block
// costs 160 (whole tiles), 200 (split, 128 columns) or 130 (64 columns: half the bytes) and
// the exchange of partial sums 800 and its bytes at 21 per ns, the rate measured for
// distributed shared memory.  `cap` is how many CTAs run at once: a cluster of 8 (4, 2)
// finds room 15 (33, 74) times.  Against the measured order: 128 x 2048 -> 2048: <4, 64>
// 7.9 us, <2, 64> 8.6, <4, 128> 10.3, whole tiles 11.1; 17 x 7168 -> 256: <8, 128> 8.3,
// <4, 64> 8.7, <4, 128> 12.2; 512 x 2048 -> 2048: whole tiles 11.5, <2, 128> 13.4.
struct SplitChoice {
    int S, bn;
};
SplitChoice choose_split(int T, long long wrows, int nk, int sms)
{
    static const struct {
        int S, bn, cap;
    } opt[] = {{1, 128, 148}, {2, 128, 148}, {4, 128, 132}, {8, 128, 120}, {2, 64, 148}, {4, 64, 132}};
    SplitChoice best = {1, 128};
    double least = 1e30;
    const int rows = T >= LG_BM ? LG_BM : (T + 31) / 32 * 32;
    for (const auto& o : opt) {
        if (o.S > nk) continue;
        const long long tiles = (long long)((T + LG_BM - 1) / LG_BM) * ((wrows + o.bn - 1) / o.bn);
        const long long cap = (long long)o.cap * sms / 148 > o.S ? (long long)o.cap * sms / 148 : o.S;
        const double waves = (double)((tiles * o.S + cap - 1) / cap);
        const double kb = o.S == 1 ? 160.0 : (o.bn == 64 ? 130.0 : 200.0);
        const double exchange = o.S == 1 ? 0.0 : 800.0 + rows * o.bn * 4.0 * (o.S - 1) / o.S / 21.0;
        const double cost = waves * ((nk + o.S - 1) / o.S * kb + exchange);
        if (cost < least) {
            least = cost;
            best = {o.S, o.bn};
        }
    }
    return best;
}

// What MOE_LINEAR_TILE may name, and what MoeLinearKernel answers.
enum LinKind { LIN_NONE, LIN_FEW, LIN_NARROW, LIN_PAIRN, LIN_WIDE, LIN_PAIR, LIN_SPLIT };
struct LinChoice {
    LinKind kind;
    int S, bn;  // LIN_SPLIT only
    const char* name;
};
const LinChoice LIN_CHOICES[] = {
    {LIN_FEW, 0, 0, "few"},          {LIN_NARROW, 0, 0, "narrow"},    {LIN_PAIRN, 0, 0, "pairn"},
    {LIN_WIDE, 0, 0, "wide"},        {LIN_PAIR, 0, 0, "pair"},        {LIN_SPLIT, 2, 128, "split2"},
    {LIN_SPLIT, 4, 128, "split4"},   {LIN_SPLIT, 8, 128, "split8"},   {LIN_SPLIT, 2, 64, "split2n"},
    {LIN_SPLIT, 4, 64, "split4n"},
};

LinChoice lin_choice(LinKind kind, int S = 0, int bn = 0)
{
    for (const LinChoice& c : LIN_CHOICES)
        if (c.kind == kind && c.S == S && c.bn == bn) return c;
    return {LIN_NONE, 0, 0, nullptr};
}

// The kernel that MOE_LINEAR_TILE asks for; `bad` when it names none.
struct LinForced {
    const LinChoice* choice;
    bool bad;
};
const LinForced& lin_forced()
{
    static const LinForced f = [] {
        const char* v = getenv("MOE_LINEAR_TILE");
        if (!v || !*v) return LinForced{nullptr, false};
        for (const LinChoice& c : LIN_CHOICES)
            if (!strcmp(c.name, v)) return LinForced{&c, false};
        return LinForced{nullptr, true};
    }();
    return f;
}

LinChoice choose_linear(int T, int K, int N, bool f32, bool gated, int sms)
{
    const long long wrows = (long long)N * (gated ? 2 : 1);
    const int nk = (K + LG_BK - 1) / LG_BK;
    const long long mt = (T + LG_BM - 1) / LG_BM, nt128 = (wrows + 127) / 128;
    const LinForced& f = lin_forced();
    if (f.bad) return {LIN_NONE, 0, 0, nullptr};
    if (f.choice) {
        // where it can run: few up to 16 tokens, gated 8; pair, pairn and wide with a 16-bit
        // y; a split with as many k blocks as CTAs, or else the largest one that has them
        const LinChoice& c = *f.choice;
        if (c.kind == LIN_FEW && (T <= 8 || (T <= 16 && !gated))) return c;
        if (c.kind == LIN_NARROW) return c;
        if ((c.kind == LIN_PAIRN || c.kind == LIN_WIDE || c.kind == LIN_PAIR) && !f32) return c;
        if (c.kind == LIN_SPLIT) {
            int S = c.S;
            while (S > nk) S /= 2;
            if (S > 1) return lin_choice(LIN_SPLIT, S, c.bn);
        }
    }
    // Few tokens.  Measured (us, few / the best of the others): 8 x 2048 -> 2048 4.3 / 6.0,
    // 8 x 8192 -> 2048 9.1 / 13, gated 8 x 4096 -> 14336 40.0 / 40.6.  With two blocks of
    // tokens the registers hold less of w on its way: 16 x 2048 -> 2048 4.5 / 5.8,
    // 16 x 8192 -> 2048 9.7 / 10.9, but 16 x 4096 -> 16384 34 / 26.
    if (T <= 8 || (T <= 16 && !gated && N <= 16 * sms)) return lin_choice(LIN_FEW);
    // At most one wave of 128 x 128 tiles: those, or smaller ones with k split, whichever
    // the model says; else 256 x 256 over CTA pairs, or 128 x 256 where a pair's second half
    // would be empty.  Measured (us, pair / wide / narrow): 2048 x 2048 -> 2048 16.7 / 16.9 /
    // 19.1, gated 512 x 2048 -> 8192 28.7 / 31.8 / 36, gated 128 x 4096 -> 14336 53 / 43 / 47.
    // An fp32 y takes narrow tiles: their warps can hold its sums (see LG_SEGMENT).
    if (mt * nt128 > sms) return lin_choice(f32 ? LIN_NARROW : T > LG_BM ? LIN_PAIR : LIN_WIDE);
    const SplitChoice c = choose_split(T, wrows, nk, sms);
    if (c.S > 1) return lin_choice(LIN_SPLIT, c.S, c.bn);
    // Whole tiles of one wave: 256 x 128 over pairs need 24 KB per CTA and k block where 128 x
    // 128 need 32, and what SMs take in from L2 bounds these (us): 1024 x 8192 -> 2048 30.2 /
    // 34.8, 512 x 2048 -> 2048 10.8 / 11.7; with few k blocks the set-up of a pair costs more:
    // 512 x 512 -> 4096 7.3 / 6.7.
    return lin_choice(!f32 && T > LG_BM && nk >= 16 ? LIN_PAIRN : LIN_NARROW);
}

}  // namespace

const char* linear_kernel_name(int T, int K, int N, bool f32, bool gated)
{
    int dev = 0;
    cudaGetDevice(&dev);
    return choose_linear(T, K, N, f32, gated, lin_sm_count(dev)).name;
}

cudaError_t launch_clear_word(int* word, cudaStream_t s) { return lin_launch(clear_word_kernel, 1, 1, 0, 0, s, word); }

bool linear_waits(const LinearArgs& a)
{
    int dev = 0;
    cudaGetDevice(&dev);
    return choose_linear(a.T, a.K, a.N, a.otype == MOE_DT_FLOAT, a.gated != 0, lin_sm_count(dev)).kind != LIN_FEW;
}

cudaError_t launch_linear(const LinearArgs& a, cudaStream_t s)
{
    int dev = 0;
    cudaGetDevice(&dev);
    const int sms = lin_sm_count(dev);
    const bool f32 = a.otype == MOE_DT_FLOAT;
    const LinChoice c = choose_linear(a.T, a.K, a.N, f32, a.gated != 0, sms);
    switch (c.kind) {
        case LIN_FEW: return launch_few(a, sms, s);
        case LIN_NARROW: return f32 ? launch_tiles<0, 128, true>(a, dev, s) : launch_tiles<0, 128>(a, dev, s);
        case LIN_PAIRN: return launch_tiles<1, 128>(a, dev, s);
        case LIN_WIDE: return launch_tiles<0, 256>(a, dev, s);
        case LIN_PAIR: return launch_tiles<1, 256>(a, dev, s);
        case LIN_SPLIT:
            return f32 ? launch_split<true>(a, c.S, c.bn, dev, s) : launch_split<false>(a, c.S, c.bn, dev, s);
        default: return cudaErrorInvalidValue;  // MOE_LINEAR_TILE names no kernel
    }
}

}  // namespace moe
