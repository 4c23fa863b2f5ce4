// attn_win.cu -- sliding-window attention forward on the 16-bit tensor cores, float32 in and out.
//
// No counterpart in DenseCore. Row i at t = i + offset sees the keys j <= t with t - j < window or
// j < sinks (common.cuh); the online softmax and its rules are those of attn_tc.cu.
//
// attn_tc.cu multiplies float32 operands as TF32 pairs, three products each; here they are pairs of fp16,
// x = hi + lo to 22 bits rounded to nearest, three products each (hi lo + lo hi + hi hi), at twice the
// rate: a block of 64 keys costs 24 products of 128 x 64 x 16 and 12 of 128 x 128 x 16 at head dim 128,
// 1540 cycles at the nominal rate against 3070.
//
// fp16's range is met by powers of two, one for every row of q and every 64 rows of a head of k and v,
// which bring the largest value to [2^14, 2^15); what they stand for is a factor of the row's and block's
// scores, and of the block's P V where it is added up. Below 2^-17 of its tile's largest value an element
// loses low bits (2^-40 of that value at most), so a single huge key or value, seen or hidden, would cost
// the other 63 of its tile theirs: with a hidden key of 1e10 times the others' size the rows that do not
// see it came out 3e-3 wrong. P, scaled to at most 2^15, keeps 2^-36 of the running maximum's weight, which
// a value far above the others' would show too. So the packing marks a tile as wide when a row's or a
// column's largest value is below 2^-14 of the tile's (rows of v: 2^-8), and a call in which a query tile
// meets a wide tile, or tiles of v more than 2^8 apart, is left to attn_tc.cu, whose TF32 has float32's
// range.
//
// Three launches:
//   pack   one pass over k and v (HBM-bound): a block takes 64 rows of a head, finds their power of two
//          and whether it is wide, and writes hi and lo to contiguous scratch, padded to D columns. Keys
//          are split once, not by every query tile that reads them, so the attention kernel has no
//          converting warps.
//   attend one CTA per 128 query rows of a head. Warp 8 loads K and V blocks (hi and lo) into rings of
//          three; warp 9 issues S_j = Q K_j^T into one of two TMEM buffers, Q in TMEM; warp 10 O_j = P_j
//          V_j with P from TMEM into one of two buffers; warps 0-7 split their rows of Q into TMEM, run
//          the softmax, two threads a row, and fold O_j into float32 registers, by twos (packed
//          float32).
//   tc     attn_tc.cu's kernel, one CTA per SM, which returns at once unless the call is left to it.
// Measured with 16 heads of 16383 tokens, head dim 128, a window of 2048 (us): pack 119, attend 752, tc 7,
// 868 in all against attn_tc.cu's 1427; its error against 64 bits is 4e-7 of the norm against 5.8e-7. What
// bounds attend now is no pipe: the tensor pipe is active 56 % of the cycles, issue slots are 38 % busy; the
// chain S, softmax, P of a block is longer than its products. Four threads a row took 825, and two groups of
// warps on alternate blocks, a thread a row, 869.
// Every mbarrier wait is bounded, as in attn_tc.cu.
#include <cuda.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>

#include "common.cuh"
#include "kernels.h"
#include "sm100.cuh"
#include "tma_host.h"
#include "trace.h"

namespace dc {
namespace {

using namespace sm100;

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr unsigned FULL = 0xffffffffu;
constexpr int TILE_ROWS = 64;  // rows that share a power of two
constexpr float P_SHIFT = 11.0f;  // log2 of P's scale
constexpr float GROWTH = 4.0f;    // the running maximum moves when it grows by more than this (log2)
constexpr float WIDE = 0x1p-14f, WIDE_V = 0x1p-8f;
constexpr unsigned WIDE_TILES = 8;         // log2
constexpr float EMPTY_TILE = 1.5f;  // the factor of a tile without a finite value but zero

// ------------------------------------------------------------------------------- pack ----
struct PackOperand {
    const float *x;
    int64_t xs[4];
    int64_t heads, rows, n;  // n: columns of x (the rest up to D is zero)
    int64_t tiles;           // per head
    __half *hi, *lo;         // (B * heads, rows, D)
    float *factor;           // (B * heads, tiles): what a scaled value of 1 stands for
    uint8_t *wide;           // (B * heads, tiles, 4): a part of the tile is wide
    int vec;
};
struct PackArgs {
    PackOperand op[2];  // keys, values
    int64_t first;      // first block of the values
    int *left;          // set to zero
};

__device__ __forceinline__ float finite_abs(float x) {
    const float a = fabsf(x);
    return a <= 3.402823466e38f ? a : 0.0f;
}

constexpr int D = 128;  // columns of the packed copies; head dims up to it are padded with zeros

constexpr int PACK_THREADS = 512, PACK_WARPS = PACK_THREADS / 32;

__global__ void __launch_bounds__(PACK_THREADS, 3) window_pack_kernel(const PackArgs a) {
    constexpr int PER = TILE_ROWS * D / 4 / PACK_THREADS, LANES = D / 4;  // float4 per thread; lanes per row
    __shared__ __align__(16) float s_col[PACK_WARPS][D];
    __shared__ float s_max[PACK_WARPS], s_low[PACK_WARPS];
    griddep_launch_dependents();
    if (blockIdx.x == 0 && threadIdx.x == 0) *a.left = 0;
    const int which = (int64_t)blockIdx.x >= a.first;
    const PackOperand &o = a.op[which];
    const int64_t idx = blockIdx.x - (which ? a.first : 0), bh = idx / o.tiles, tile = idx - bh * o.tiles;
    const int64_t b = bh / o.heads, h = bh - b * o.heads, row0 = tile * TILE_ROWS;
    const float *base = o.x + b * o.xs[0] + h * o.xs[1];
    float4 v[PER], col = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    float top = 0.0f, low = INFINITY;  // low: the smallest row maximum but zero; a warp holds one row per step
    static_assert(LANES == 32, "one row per warp and step");
#pragma unroll
    for (int i = 0; i < PER; i++) {
        const int at = i * PACK_THREADS + (int)threadIdx.x, c = at % LANES * 4;
        const int64_t row = row0 + at / LANES;
        v[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (row < o.rows) {
            const float *p = base + row * o.xs[2];
            if (o.vec && c + 4 <= o.n) {
                v[i] = *reinterpret_cast<const float4 *>(p + c);
            } else {
                if (c < o.n) v[i].x = p[c * o.xs[3]];
                if (c + 1 < o.n) v[i].y = p[(c + 1) * o.xs[3]];
                if (c + 2 < o.n) v[i].z = p[(c + 2) * o.xs[3]];
                if (c + 3 < o.n) v[i].w = p[(c + 3) * o.xs[3]];
            }
        }
        const float4 m = make_float4(finite_abs(v[i].x), finite_abs(v[i].y), finite_abs(v[i].z), finite_abs(v[i].w));
        col = make_float4(fmaxf(col.x, m.x), fmaxf(col.y, m.y), fmaxf(col.z, m.z), fmaxf(col.w, m.w));
        // (Nonnegative floats are ordered as their bits.)
        const float r = __uint_as_float(__reduce_max_sync(FULL, __float_as_uint(fmaxf(fmaxf(m.x, m.y), fmaxf(m.z, m.w)))));
        top = fmaxf(top, r);
        if (r > 0.0f) low = fminf(low, r);
    }
    if ((threadIdx.x & 31) == 0) s_max[threadIdx.x >> 5] = top, s_low[threadIdx.x >> 5] = low;
    *reinterpret_cast<float4 *>(&s_col[threadIdx.x >> 5][threadIdx.x % LANES * 4]) = col;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < PACK_WARPS; w++) top = fmaxf(top, s_max[w]);
    // Four warps look at 32 columns and four warps' rows each, without another barrier.
    if (threadIdx.x < D) {
        float c = 0.0f;
#pragma unroll
        for (int w = 0; w < PACK_WARPS; w++) c = fmaxf(c, s_col[w][threadIdx.x]);
        const bool wide = (c > 0.0f && c < top * WIDE) || s_low[threadIdx.x % PACK_WARPS] < top * (which ? WIDE_V : WIDE) ||
                          (top > 0.0f && top < 0x1p-100f);
        const int any = __any_sync(FULL, wide);
        if ((threadIdx.x & 31) == 0) o.wide[(bh * o.tiles + tile) * 4 + threadIdx.x / 32] = (uint8_t)any;
    }
    int e = 0;  // the largest value is in [2^(e-1), 2^e)
    if (top > 0.0f) frexpf(top, &e);
    e = max(e, -100);
    const float up = ldexpf(1.0f, 15 - e);
    if (threadIdx.x == 0) o.factor[bh * o.tiles + tile] = top > 0.0f ? ldexpf(1.0f, e - 15) : EMPTY_TILE;
#pragma unroll
    for (int i = 0; i < PER; i++) {
        const int at = i * PACK_THREADS + (int)threadIdx.x, c = at % LANES * 4;
        const int64_t row = row0 + at / LANES;
        if (row >= o.rows) continue;
        const float x[4] = {v[i].x * up, v[i].y * up, v[i].z * up, v[i].w * up};
        __half2 hi[2], lo[2];
#pragma unroll
        for (int j = 0; j < 2; j++) {
            hi[j] = __floats2half2_rn(x[2 * j], x[2 * j + 1]);
            const float2 f = __half22float2(hi[j]);
            lo[j] = __floats2half2_rn(x[2 * j] - f.x, x[2 * j + 1] - f.y);
        }
        const int64_t out = (bh * o.rows + row) * D + c;
        *reinterpret_cast<uint2 *>(o.hi + out) = make_uint2(*reinterpret_cast<uint32_t *>(&hi[0]), *reinterpret_cast<uint32_t *>(&hi[1]));
        *reinterpret_cast<uint2 *>(o.lo + out) = make_uint2(*reinterpret_cast<uint32_t *>(&lo[0]), *reinterpret_cast<uint32_t *>(&lo[1]));
    }
}

// ----------------------------------------------------------------------------- attend ----

// Instruction descriptor of kind::f16 with fp16 operands and fp32 accumulation (bit layout as
// sm100::idesc_tf32, operand format 0).
__host__ __device__ constexpr uint32_t idesc_f16(int M, int N, int b_mn_major) {
    return (1u << 4) | (uint32_t(b_mn_major) << 16) | (uint32_t(N >> 3) << 17) | (uint32_t(M >> 4) << 24);
}

// D (+)= A B, A in TMEM (fp16, two K elements a column), B in shared memory, K = 16. A whole converged
// warp calls it; one elected lane issues.
__device__ __forceinline__ void mma_f16_ts_w(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred e, p;\n\t"
        "elect.sync _|e, 0xffffffff;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
        "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}

struct WinCfg {
    static constexpr int BM = 128, BN = 64, KST = 3, VST = 3;
    static constexpr int CHUNKS = D / 64;            // 128-byte column chunks of an fp16 row
    static constexpr int PARTS = 2;                          // threads of a row
    static constexpr int HB = BN / PARTS, HD = D / PARTS;    // their S and output columns
    static constexpr uint32_t KV_CHUNK = BN * 128, KV_HALF = CHUNKS * KV_CHUNK;  // hi or lo
    static constexpr uint32_t KV_STAGE = 2 * KV_HALF;
    static constexpr uint32_t OFF_K = 0, OFF_V = KST * KV_STAGE;
    static constexpr uint32_t OFF_XMAX = OFF_V + VST * KV_STAGE;         // float [2][PARTS][BM]
    static constexpr uint32_t OFF_XSUM = OFF_XMAX + 2 * PARTS * BM * 4;  // float [PARTS][BM]
    static constexpr uint32_t OFF_BAR = OFF_XSUM + PARTS * BM * 4;
    static constexpr int Q_READY = 0, QX = 1, K_FULL = 2, K_EMPTY = K_FULL + KST, V_FULL = K_EMPTY + KST, V_EMPTY = V_FULL + VST,
                         S_FULL = V_EMPTY + VST, P_FULL = S_FULL + 2, PV_DONE = P_FULL + 2, OB_FREE = PV_DONE + 2, XCH = OB_FREE + 2,
                         XSUM = XCH + 8, DRAIN = XSUM + 1, DRAIN_PV = DRAIN + 1, NBAR = DRAIN_PV + 1;
    static constexpr uint32_t OFF_MISC = OFF_BAR + NBAR * 8;
    static constexpr uint32_t SMEM = OFF_MISC + 16 + 1024;  // + slack for 1024-byte alignment
    // TMEM: Q hi | Q lo | 2 x S, overwritten by P hi | P lo | 2 x O_j.
    static constexpr uint32_t COL_QHI = 0, COL_QLO = D / 2, COL_S = D, COL_OB = D + 2 * BN, TMEM_COLS = 512;
    static_assert(COL_OB + 2 * D <= TMEM_COLS, "tensor memory budget");
    static_assert(SMEM <= 232448, "shared memory budget");
    static constexpr int SOFTMAX = 128 * PARTS, W_PROD = 4 * PARTS, W_MMA = W_PROD + 1, W_PV = W_PROD + 2, THREADS = SOFTMAX + 96;
    static constexpr uint32_t IDESC_S = idesc_f16(128, BN, 0), IDESC_O = idesc_f16(128, D, 1);
    __host__ __device__ static constexpr uint32_t col_s(int b) { return COL_S + (uint32_t)b * BN; }
    __host__ __device__ static constexpr uint32_t col_ob(int i) { return COL_OB + (uint32_t)(i & 1) * D; }
};

using C = WinCfg;

struct WinArgs {
    AttnProblem p;
    int num_q_tiles;
    int64_t kv_tiles;      // 64-row tiles per head
    const float *kf, *vf;  // their factors
    const uint32_t *kw, *vw;  // nonzero: a wide tile
    int *left;             // set when the call is left to attn_tc.cu
    int q_vec;             // q's rows are 16-byte aligned with unit inner stride
    float scale_log2;
    int *err;
};

__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
__device__ __forceinline__ float max32(const float (&v)[32]) {
    float t[11];
#pragma unroll
    for (int i = 0; i < 10; i++) t[i] = max3(v[3 * i], v[3 * i + 1], v[3 * i + 2]);
    t[10] = fmaxf(v[30], v[31]);
    return max3(max3(max3(t[0], t[1], t[2]), t[9], t[10]), max3(t[3], t[4], t[5]), max3(t[6], t[7], t[8]));
}
// Two sums (products) in one instruction, each rounded as alone.
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(reinterpret_cast<uint64_t &>(r)) : "l"(reinterpret_cast<uint64_t &>(a)), "l"(reinterpret_cast<uint64_t &>(b)));
    return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;"
        : "=l"(reinterpret_cast<uint64_t &>(r))
        : "l"(reinterpret_cast<uint64_t &>(a)), "l"(reinterpret_cast<uint64_t &>(b)), "l"(reinterpret_cast<uint64_t &>(c)));
    return r;
}
// (x, y) as fp16 pairs: hi rounded to nearest, lo what is left.
__device__ __forceinline__ void split2(float2 x, uint32_t &hi, uint32_t &lo) {
    const __half2 h = __floats2half2_rn(x.x, x.y);
    const float2 f = __half22float2(h);
    const float2 d = fma2(f, make_float2(-1.0f, -1.0f), x);
    const __half2 g = __floats2half2_rn(d.x, d.y);
    hi = *reinterpret_cast<const uint32_t *>(&h);
    lo = *reinterpret_cast<const uint32_t *>(&g);
}

// tm*: (D, rows, heads, 2 * B) over the packed copies, lo at batch B + b; boxes of 64 columns.
template <bool MASKED>
__global__ void __maxnreg__(168)
    window_attend_kernel(const __grid_constant__ CUtensorMap tmk, const __grid_constant__ CUtensorMap tmv, const WinArgs a) {
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_addr(smem_raw);
    const uint32_t sb = (raw + 1023u) & ~1023u;
    uint8_t *sg = smem_raw + (sb - raw);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const AttnProblem &p = a.p;
    const int qt = a.num_q_tiles - 1 - (int)blockIdx.x;
    const int64_t h = blockIdx.y, b = blockIdx.z, hk = h / p.group;
    const int64_t q0 = (int64_t)qt * C::BM;
    const WindowSpan span = window_span<C::BN>(p, q0, C::BM);
    const int nblk = span.n;
    auto bar = [&](int i) { return sb + C::OFF_BAR + 8u * (uint32_t)i; };
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(sg + C::OFF_MISC);
    volatile int *abort = reinterpret_cast<volatile int *>(sg + C::OFF_MISC + 4);
    int *err = a.err;

    if (threadIdx.x == 0) {
        mbar_init(bar(C::Q_READY), C::SOFTMAX);
        mbar_init(bar(C::QX), C::SOFTMAX);
        for (int s = 0; s < C::KST; s++) {
            mbar_init(bar(C::K_FULL + s), 1);
            mbar_init(bar(C::K_EMPTY + s), 1);
        }
        for (int s = 0; s < C::VST; s++) {
            mbar_init(bar(C::V_FULL + s), 1);
            mbar_init(bar(C::V_EMPTY + s), 1);
        }
        for (int s = 0; s < 2; s++) {
            mbar_init(bar(C::S_FULL + s), 1);
            mbar_init(bar(C::P_FULL + s), C::SOFTMAX);
            mbar_init(bar(C::PV_DONE + s), 1);
            mbar_init(bar(C::OB_FREE + s), C::SOFTMAX);
        }
        for (int s = 0; s < 8; s++) mbar_init(bar(C::XCH + s), 64);
        mbar_init(bar(C::XSUM), C::SOFTMAX);
        mbar_init(bar(C::DRAIN), 1);
        mbar_init(bar(C::DRAIN_PV), 1);
        *abort = 0;
        fence_mbar_init();
    }
    if (warp == C::W_MMA) {
        tmem_alloc(smem_addr(tmem_slot), C::TMEM_COLS);
        tmem_relinquish();
    }
    if (warp == C::W_PROD && lane == 0) {
        prefetch_tmap(&tmk);
        prefetch_tmap(&tmv);
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    const int64_t kv_head = (b * p.Hkv + hk) * a.kv_tiles;

    if (warp == C::W_PROD) {
        // ------------------------------------------------------------ TMA producer ----
        griddep_wait();  // the packed copies and their factors are read only from here on
        if (lane == 0) {
            int k_issued = -1, v_issued = -1;
            const int lo_b = (int)(p.B + b);
            auto load = [&](const CUtensorMap *tm, uint32_t dst, uint32_t full, int key) {
                mbar_expect_tx(full, C::KV_STAGE);
                for (int c = 0; c < C::CHUNKS; c++) {
                    tma_load_4d(tm, dst + c * C::KV_CHUNK, full, 64 * c, key, (int)hk, (int)b);
                    tma_load_4d(tm, dst + C::KV_HALF + c * C::KV_CHUNK, full, 64 * c, key, (int)hk, lo_b);
                }
            };
            for (int j = 0; j < nblk; j++) {
                const int ks = j % C::KST, vs = j % C::VST, key = span.block(j) * C::BN;
                if (j >= C::KST && !mbar_wait(bar(C::K_EMPTY + ks), ((j / C::KST) - 1) & 1, abort, err)) break;
                load(&tmk, sb + C::OFF_K + ks * C::KV_STAGE, bar(C::K_FULL + ks), key);
                k_issued = j;
                if (j >= C::VST && !mbar_wait(bar(C::V_EMPTY + vs), ((j / C::VST) - 1) & 1, abort, err)) break;
                load(&tmv, sb + C::OFF_V + vs * C::KV_STAGE, bar(C::V_FULL + vs), key);
                v_issued = j;
            }
            if (*abort) {
                // Let the copies already in flight land before the CTA's memory goes away.
                volatile int never = 0;
                for (int j = max(0, k_issued - C::KST + 1); j <= k_issued; j++)
                    mbar_wait(bar(C::K_FULL + j % C::KST), (j / C::KST) & 1, &never, nullptr);
                for (int j = max(0, v_issued - C::VST + 1); j <= v_issued; j++)
                    mbar_wait(bar(C::V_FULL + j % C::VST), (j / C::VST) & 1, &never, nullptr);
            }
        }
        __syncwarp();
        // While the last blocks are computed: are the tiles too wide, or v's too far apart?
        int wide = 0;
        unsigned low = 255u, high = 0u;  // exponents of v's factors
        for (int j = lane; j < nblk; j += 32) {
            const int64_t t = kv_head + span.block(j);
            const float vf = a.vf[t];
            wide |= (a.kw[t] | a.vw[t]) != 0;
            if (vf != EMPTY_TILE) {
                const unsigned e = (__float_as_uint(vf) >> 23) & 255u;
                low = min(low, e);
                high = max(high, e);
            }
        }
        wide = __any_sync(FULL, wide);
        low = __reduce_min_sync(FULL, low);
        high = __reduce_max_sync(FULL, high);
        if (lane == 0 && (wide || (low < high && high - low > WIDE_TILES))) atomicOr(a.left, 1);
    } else if (warp == C::W_MMA) {
        // -------------------------------------------------------- MMA issuer: S = Q K^T ----
        const uint64_t kdesc0 = sdesc_sw128(sb + C::OFF_K, 16, 1024);
        const uint32_t q_hi = tmem + C::COL_QHI, q_lo = tmem + C::COL_QLO;
        bool ok = mbar_wait_warp(bar(C::Q_READY), 0, abort, err);
        tc_fence_after();
        for (int j = 0; ok && j < nblk; j++) {
            const int bb = j & 1, ks = j % C::KST;
            // S buffer bb held P_{j-2}, read by PV_{j-2}.
            if (j >= 2 && !mbar_wait_warp(bar(C::PV_DONE + bb), ((j - 2) >> 1) & 1, abort, err)) break;
            if (!mbar_wait_warp(bar(C::K_FULL + ks), (j / C::KST) & 1, abort, err)) break;
            tc_fence_after();
            const uint64_t hi = kdesc0 + ((ks * C::KV_STAGE) >> 4), lo = hi + (C::KV_HALF >> 4);
            const uint32_t d_s = tmem + C::col_s(bb);
#pragma unroll
            for (int kk = 0; kk < D / 16; kk++) {  // the cross terms first, then the main products
                const uint32_t off = ((kk >> 2) * C::KV_CHUNK + (kk & 3) * 32) >> 4;
                mma_f16_ts_w(d_s, q_hi + kk * 8, lo + off, C::IDESC_S, kk > 0 ? 1u : 0u);
                mma_f16_ts_w(d_s, q_lo + kk * 8, hi + off, C::IDESC_S, 1u);
            }
#pragma unroll
            for (int kk = 0; kk < D / 16; kk++) {
                const uint32_t off = ((kk >> 2) * C::KV_CHUNK + (kk & 3) * 32) >> 4;
                mma_f16_ts_w(d_s, q_hi + kk * 8, hi + off, C::IDESC_S, 1u);
            }
            tc_commit_w(bar(C::S_FULL + bb));
            tc_commit_w(bar(C::K_EMPTY + ks));
        }
        // Every MMA this warp issued completes before TMEM is released.
        tc_commit_w(bar(C::DRAIN));
        volatile int never = 0;
        mbar_wait_warp(bar(C::DRAIN), 0, &never, nullptr);
    } else if (warp == C::W_PV) {
        // ----------------------------------------------------- MMA issuer: O_j = P_j V_j ----
        // V is MN-major: 128-byte rows of 64 columns, 8 keys (1024 bytes) a swizzle atom, 64-column chunks
        // KV_CHUNK apart.
        const uint64_t vdesc0 = sdesc_sw128(sb + C::OFF_V, C::KV_CHUNK, 1024);
        for (int i = 0; i < nblk; i++) {
            const int bi = i & 1, vs = i % C::VST;
            if (!mbar_wait_warp(bar(C::P_FULL + bi), (i >> 1) & 1, abort, err)) break;
            if (!mbar_wait_warp(bar(C::V_FULL + vs), (i / C::VST) & 1, abort, err)) break;
            if (i >= 2 && !mbar_wait_warp(bar(C::OB_FREE + bi), ((i - 2) >> 1) & 1, abort, err)) break;
            tc_fence_after();
            const uint64_t hi = vdesc0 + ((vs * C::KV_STAGE) >> 4), lo = hi + (C::KV_HALF >> 4);
            const uint32_t d_o = tmem + C::col_ob(i), p_hi = tmem + C::col_s(bi), p_lo = p_hi + C::BN / 2;
#pragma unroll
            for (int kk = 0; kk < C::BN / 16; kk++) {
                const uint32_t off = (kk * 2048) >> 4;
                mma_f16_ts_w(d_o, p_hi + kk * 8, lo + off, C::IDESC_O, kk > 0 ? 1u : 0u);
                mma_f16_ts_w(d_o, p_lo + kk * 8, hi + off, C::IDESC_O, 1u);
            }
#pragma unroll
            for (int kk = 0; kk < C::BN / 16; kk++)
                mma_f16_ts_w(d_o, p_hi + kk * 8, hi + ((kk * 2048) >> 4), C::IDESC_O, 1u);
            tc_commit_w(bar(C::PV_DONE + bi));
            tc_commit_w(bar(C::V_EMPTY + vs));
        }
        tc_commit_w(bar(C::DRAIN_PV));
        volatile int never = 0;
        mbar_wait_warp(bar(C::DRAIN_PV), 0, &never, nullptr);
    } else if (warp < C::W_PROD) {
        // ------------------------------------------------------------------ softmax ----
        const int row = threadIdx.x & 127, part = threadIdx.x >> 7;
        const int64_t qrow = q0 + row;
        const bool row_ok = qrow < p.L;
        const uint32_t tl = tmem + ((uint32_t)((warp & 3) * 32) << 16);
        float *xmax = reinterpret_cast<float *>(sg + C::OFF_XMAX);  // [2][PARTS][BM]
        float *xsum = reinterpret_cast<float *>(sg + C::OFF_XSUM);  // [PARTS][BM]
        // The maximum of the row's PARTS values, left in slot `at` by each of its threads; past the wait
        // the other's earlier TMEM loads are done too.
        auto row_max = [&](int at) {
            const float *x = xmax + at * C::PARTS * C::BM + row;
            return fmaxf(x[0], x[C::BM]);
        };
        // This thread's HD columns of its row of Q, by the row's power of two, into TMEM.
        bool ok = true;
        float qf = 0.0f;
        {
            float x[C::HD], top = 0.0f;
            const float *src = p.q + b * p.qs[0] + h * p.qs[1] + qrow * p.qs[2];
            const int col0 = part * C::HD;
#pragma unroll
            for (int c = 0; c < C::HD; c += 4) {
                if (row_ok && a.q_vec && col0 + c + 4 <= p.E) {
                    const float4 v = *reinterpret_cast<const float4 *>(src + col0 + c);
                    x[c] = v.x, x[c + 1] = v.y, x[c + 2] = v.z, x[c + 3] = v.w;
                } else {
#pragma unroll
                    for (int i = 0; i < 4; i++) x[c + i] = row_ok && col0 + c + i < p.E ? src[(col0 + c + i) * p.qs[3]] : 0.0f;
                }
            }
#pragma unroll
            for (int c = 0; c < C::HD; c++) top = fmaxf(top, finite_abs(x[c]));
            xmax[part * C::BM + row] = top;
            mbar_arrive(bar(C::QX));
            ok = mbar_wait_warp(bar(C::QX), 0, abort, err);
            int e = 0;
            top = row_max(0);
            if (top > 0.0f) frexpf(top, &e);
            e = max(e, -100);
            const float up = ldexpf(1.0f, 15 - e);
            qf = ldexpf(1.0f, e - 15) * a.scale_log2;
            if (ok) {
#pragma unroll
                for (int c = 0; c < C::HD; c += 32) {
                    uint32_t hi[16], lo[16];
#pragma unroll
                    for (int i = 0; i < 16; i++) split2(make_float2(x[c + 2 * i] * up, x[c + 2 * i + 1] * up), hi[i], lo[i]);
                    tmem_st16(tl + C::COL_QHI + col0 / 2 + c / 2, hi);
                    tmem_st16(tl + C::COL_QLO + col0 / 2 + c / 2, lo);
                }
                tmem_wait_st();
                tc_fence_before();
                mbar_arrive(bar(C::Q_READY));
            }
        }
        griddep_wait();  // the factors are the packing's
        const int xch = C::XCH + 2 * (warp & 3);  // of the two warps that hold this row
        float m = -INFINITY, l = 0.0f, vf_prev = 0.0f;
        float2 o[C::HD / 2];
#pragma unroll
        for (int x = 0; x < C::HD / 2; x++) o[x] = make_float2(0.0f, 0.0f);
        for (int j = 0; ok && j < nblk; j++) {
            const int bb = j & 1, kb = span.block(j);
            const int64_t k0 = (int64_t)kb * C::BN + part * C::HB;
            const float kf = a.kf[kv_head + kb], vf = a.vf[kv_head + kb];
            const bool edge = MASKED || !window_interior(p, q0, C::BM, k0, C::HB);
            uint32_t vbits = 0xFFFFFFFFu;
            if (edge) vbits = row_ok ? window_key_bits(p, qrow, k0) : 0u;
            // The user mask's values, loaded before the wait for S so that the wait hides their latency.
            float mk[MASKED ? C::HB : 1];
            if constexpr (MASKED) {
                    mask_run<C::HB>(p, b, h, qrow, k0, p.ms[3], vbits, mk);
                vbits = mask_visible(mk, vbits);
            }
            if (!mbar_wait_warp(bar(C::S_FULL + bb), (j >> 1) & 1, abort, err)) {
                ok = false;
                break;
            }
            tc_fence_after();
            float s[C::HB];
            {
                uint32_t r[C::HB];
                tmem_ld32(tl + C::col_s(bb) + part * C::HB, r);
                tmem_wait_ld();
#pragma unroll
                for (int x = 0; x < C::HB; x++) s[x] = __uint_as_float(r[x]);
            }
            // Interior blocks keep the raw scores and fold the scale into the exponent's FFMA; edge blocks
            // scale, mask and fill first.
            const float f = qf * kf;
            const bool rawp = !edge && f > 0.0f;
            float smul = rawp ? f : 1.0f;
            if (!rawp) {
#pragma unroll
                for (int c = 0; c < C::HB; c++) {
                    float x = s[c] * f;
                    if (MASKED) x += mk[MASKED ? c : 0] * LOG2E;
                    s[c] = ((vbits >> c) & 1u) ? x : -INFINITY;
                }
            }
            // The row max, shared with the row's other thread; past this both have read their S, and P may
            // overwrite any of its columns.
            xmax[(bb * C::PARTS + part) * C::BM + row] = max32(s) * smul;
            tc_fence_before();
            mbar_arrive(bar(xch + bb));
            if (!mbar_wait_warp(bar(xch + bb), (j >> 1) & 1, abort, err)) {
                ok = false;
                break;
            }
            tc_fence_after();
            const float m_new = fmaxf(m, row_max(bb));
            float corr = 1.0f;
            if (m_new - m > GROWTH) {  // (both -inf: NaN, no growth)
                corr = ex2_approx(m - m_new);
                m = m_new;
            }
            // The FFMA does not round s smul, the maximum is rounded: past 2^20 a difference of up to half an
            // ulp counts (past 2^24 it takes P out of fp16's range), so the scores are rounded too.
            if (smul != 1.0f && fabsf(m) > 0x1p20f) {
#pragma unroll
                for (int c = 0; c < C::HB; c++) s[c] *= smul;
                smul = 1.0f;
            }
            // (A row that has seen no key keeps the maximum -inf; its scores are all -inf, its weights 0.)
            const float shift = m == -INFINITY ? 0.0f : P_SHIFT - m;
            const float2 mul2v = make_float2(smul, smul), base = make_float2(shift, shift);
            float2 sum = make_float2(0.0f, 0.0f);
            uint32_t phi[C::HB / 2], plo[C::HB / 2];
#pragma unroll
            for (int c = 0; c < C::HB; c += 2) {
                const float2 x = fma2(make_float2(s[c], s[c + 1]), mul2v, base);
                const float2 pc = make_float2(ex2_approx(x.x), ex2_approx(x.y));
                sum = add2(sum, pc);
                split2(pc, phi[c / 2], plo[c / 2]);
            }
            tmem_st16(tl + C::col_s(bb) + part * (C::HB / 2), phi);
            tmem_st16(tl + C::col_s(bb) + C::BN / 2 + part * (C::HB / 2), plo);
            l = fmaf(l, corr, sum.x + sum.y);
            tmem_wait_st();
            tc_fence_before();
            mbar_arrive(bar(C::P_FULL + bb));
            // Fold the previous block: o = (o + O_{j-1} vf_{j-1}) * corr.
            if (j >= 1) {
                if (!mbar_wait_warp(bar(C::PV_DONE + ((j - 1) & 1)), ((j - 1) >> 1) & 1, abort, err)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                const bool scaled = __any_sync(FULL, corr != 1.0f);
                uint32_t r[C::HD / 32][32];
#pragma unroll
                for (int c = 0; c < C::HD / 32; c++) tmem_ld32(tl + C::col_ob(j - 1) + part * C::HD + c * 32, r[c]);
                tmem_wait_ld();
                tc_fence_before();
                mbar_arrive(bar(C::OB_FREE + ((j - 1) & 1)));
#pragma unroll
                for (int x = 0; x < C::HD / 2; x++)
                    o[x] = fma2(make_float2(__uint_as_float(r[x / 16][x % 16 * 2]), __uint_as_float(r[x / 16][x % 16 * 2 + 1])), make_float2(vf_prev, vf_prev), o[x]);
                if (scaled) {
#pragma unroll
                    for (int x = 0; x < C::HD / 2; x++) o[x] = make_float2(o[x].x * corr, o[x].y * corr);
                }
            }
            vf_prev = vf;
        }
        if (ok) {
            ok = mbar_wait_warp(bar(C::PV_DONE + ((nblk - 1) & 1)), ((nblk - 1) >> 1) & 1, abort, err);
            tc_fence_after();
        }
        const bool read_o = __all_sync(FULL, ok);
        const bool aborted = __any_sync(FULL, *abort != 0);
        if (read_o) {
            uint32_t r[C::HD / 32][32];
#pragma unroll
            for (int c = 0; c < C::HD / 32; c++) tmem_ld32(tl + C::col_ob(nblk - 1) + part * C::HD + c * 32, r[c]);
            tmem_wait_ld();
#pragma unroll
            for (int x = 0; x < C::HD / 2; x++)
                o[x] = fma2(make_float2(__uint_as_float(r[x / 16][x % 16 * 2]), __uint_as_float(r[x / 16][x % 16 * 2 + 1])), make_float2(vf_prev, vf_prev), o[x]);
        }
        // The row sum: the two threads' parts, in their order.
        xsum[part * C::BM + row] = l;
        mbar_arrive(bar(C::XSUM));
        const bool have_sum = mbar_wait_warp(bar(C::XSUM), 0, abort, err);
        l = xsum[row] + xsum[C::BM + row];
        if (!aborted && have_sum && read_o && row_ok) {
            // (l and o are both 2^P_SHIFT of what they stand for.)
            const float lfin = l == 0.0f ? 1.0f : l, inv = 1.0f / lfin;
            const int cols = (int)min((int64_t)C::HD, p.Ev - part * C::HD);
            float *orow = p.out + b * p.os[0] + h * p.os[1] + qrow * p.os[2] + (int64_t)part * C::HD * p.os[3];
            if (p.os[3] == 1 && (reinterpret_cast<uintptr_t>(orow) & 15u) == 0 && cols % 4 == 0) {
#pragma unroll
                for (int x = 0; x < C::HD; x += 4)
                    if (x < cols)
                        *reinterpret_cast<float4 *>(orow + x) = make_float4(o[x / 2].x * inv, o[x / 2].y * inv, o[x / 2 + 1].x * inv, o[x / 2 + 1].y * inv);
            } else {
#pragma unroll
                for (int x = 0; x < C::HD; x++)
                    if (x < cols) orow[x * p.os[3]] = (x & 1 ? o[x / 2].y : o[x / 2].x) * inv;
            }
            if (part == 0)
                p.lse[b * p.ls[0] + h * p.ls[1] + qrow * p.ls[2]] = m == -INFINITY ? 0.0f : (m - P_SHIFT) * LN2 + logf(lfin);
        }
    }

    tc_fence_before();
    __syncthreads();
    if (warp == C::W_MMA) {
        tc_fence_after();
        tmem_dealloc(tmem, C::TMEM_COLS);
    }
}

// A 4-D fp16 map over (D, rows, heads, 2 * B): hi, then lo; boxes of 64 columns by box_rows rows.
int make_tmap16(CUtensorMap *m, const __half *base, int64_t D, int64_t rows, int64_t heads, int64_t batch2, int box_rows) {
    const int64_t st[3] = {heads * rows * D, rows * D, D};
    return make_tmap_16bit(m, base, D, rows, heads, batch2, st, box_rows);
}

struct Scratch {
    void *ptr = nullptr;
    cudaStream_t stream = nullptr;
    ~Scratch() { pool_free(ptr, stream); }
};

bool rows_vec(const float *ptr, const int64_t *st) {
    return st[3] == 1 && st[0] % 4 == 0 && st[1] % 4 == 0 && st[2] % 4 == 0 && (reinterpret_cast<uintptr_t>(ptr) & 15u) == 0;
}

}  // namespace

bool window_forward_pick(const AttnProblem &p) {
    if (!p.window || p.S == 0 || max(p.E, p.Ev) <= 64 || !tc_forward_supported(p) || p.H > 65535 || p.B > 65535) return false;
    if (2 * p.B * p.Hkv * ((p.S + TILE_ROWS - 1) / TILE_ROWS) >= (1ll << 31)) return false;
    if (p.B * p.H * ((p.L + C::BM - 1) / C::BM) >= (1ll << 31)) return false;
    // Packing costs a pass over the S keys of a key head, attending saves time per query row and key it
    // sees. At 16 heads of 16383 tokens, head dim 128, against attn_tc.cu (us): 868 : 1427 with a window of
    // 2048, 533 : 538 of 512, 428 : 285 of 128. Those lines meet where the mean row sees 192 keys and 384
    // more per key row that is packed for it, which also holds for groups of heads (32 on 8, 4096 tokens:
    // window 512 193 : 245, 256 162 : 166), masks (8 heads, 2048 tokens: whole window 93 : 133, 512 46 :
    // 50), head dim 96 (16 heads, 4096 tokens: window 1024 157 : 188) and batches (8 x 512 tokens, whole
    // window, 32 heads on 8: 160 : 155; 1024 tokens 367 : 481). Heads of 64 gain nothing at any window (16
    // heads, 16384 tokens, window 2048: 661 : 653, 256: 253 : 195): there the softmax, not the products,
    // bounds both.
    // (These are times of calls without a wide tile. A call with one, seen by any query tile, is done over
    // whole: the 16 x 16383 one took 875 us, 2440 with one row of v in the first tile of each head scaled by 2^-9,
    // which every query tile sees among its first tokens, and 2540 with such a row in one head; attn_tc.cu alone
    // takes 1427.)
    const double most = (double)min(p.window, p.S), L = (double)p.L, first = (double)max(p.offset, (int64_t)0) + 1.0;
    // The mean over the rows of min(position, most), positions rising from `first`.
    const double ramp = min(max(most - first, 0.0), L), mean = most - (most > first ? ramp * (most - first - 0.5 * ramp) / L : 0.0);
    return mean * L * (double)p.H >= 192.0 * L * (double)p.H + 384.0 * (double)p.S * (double)p.Hkv;
}

int window_forward(const AttnProblem &p, cudaStream_t stream) {
    const int64_t kt = (p.S + TILE_ROWS - 1) / TILE_ROWS, nk = p.B * p.Hkv * p.S * D, fk = p.B * p.Hkv * kt;
    Scratch ws;
    ws.stream = stream;
    int st = pool_alloc(&ws.ptr, sizeof(__half) * (size_t)(4 * nk) + sizeof(float) * (size_t)(4 * fk + 1), stream);
    if (st) return tc_forward(p, DC_PREC_3XTF32, stream);  // no room for the copies: the kernel that needs none
    __half *k16 = static_cast<__half *>(ws.ptr), *v16 = k16 + 2 * nk;
    float *kf = reinterpret_cast<float *>(v16 + 2 * nk), *vf = kf + fk;
    uint8_t *kw = reinterpret_cast<uint8_t *>(vf + fk), *vw = kw + 4 * fk;
    int *left = reinterpret_cast<int *>(vw + 4 * fk);
    PackArgs pa{};
    pa.left = left;
    const int64_t per = p.B * p.Hkv * kt, blocks = 2 * per;
    pa.first = per;
    for (int i = 0; i < 2; i++) {
        PackOperand &o = pa.op[i];
        o.x = i ? p.v : p.k;
        for (int d = 0; d < 4; d++) o.xs[d] = i ? p.vs[d] : p.ks[d];
        o.heads = p.Hkv;
        o.rows = p.S;
        o.n = i ? p.Ev : p.E;
        o.tiles = kt;
        o.hi = i ? v16 : k16;
        o.lo = o.hi + nk;
        o.factor = i ? vf : kf;
        o.wide = i ? vw : kw;
        o.vec = rows_vec(o.x, o.xs);
    }
    {
        KernelTrace tr("window_pack", stream);
        window_pack_kernel<<<(unsigned)blocks, PACK_THREADS, 0, stream>>>(pa);
        if ((st = check_launch("window_pack"))) return st;
    }
    CUtensorMap tk, tv;
    st = make_tmap16(&tk, k16, D, p.S, p.Hkv, 2 * p.B, C::BN);
    if (!st) st = make_tmap16(&tv, v16, D, p.S, p.Hkv, 2 * p.B, C::BN);
    if (st) return st;
    WinArgs a;
    a.p = p;
    a.num_q_tiles = (int)((p.L + C::BM - 1) / C::BM);
    a.q_vec = rows_vec(p.q, p.qs);
    a.kv_tiles = kt;
    a.kf = kf;
    a.vf = vf;
    a.kw = reinterpret_cast<const uint32_t *>(kw);
    a.vw = reinterpret_cast<const uint32_t *>(vw);
    a.left = left;
    a.scale_log2 = p.scale * LOG2E;
    a.err = device_error_word();
    if (!a.err) return fail(DC_ERR_CUDA, "device error word is unavailable");
    auto kernel = p.mask_kind != MASK_NONE ? window_attend_kernel<true> : window_attend_kernel<false>;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)C::SMEM);
    if (e != cudaSuccess) return cuda_fail(e, "window_attend smem attribute");
    {
        KernelTrace tr("window_attend", stream);
        e = launch_dependent(kernel, dim3((unsigned)a.num_q_tiles, (unsigned)p.H, (unsigned)p.B), dim3(C::THREADS), C::SMEM, stream, tk, tv, a);
        if (e != cudaSuccess) return cuda_fail(e, "window_attend");
    }
    return tc_forward_if(p, left, stream);
}

}  // namespace dc
