// cache4.cu -- a paged key/value cache held in 4 bits: filling it, reading it back, and the
// attention of one token per sequence over it.
//
// No counterpart in DenseCore. Format, for each token and key/value head, per group of 32 channels
// x (key and value alike):
//   low    min(x) rounded down to bfloat16
//   scale  (max(x) - low) / 15 rounded up to bfloat16
//   code   (x - low) / scale rounded to nearest even, 0..15 (0 where scale is 0)
// in 32-bit arithmetic; the group stands for low + scale * code. low and scale are rounded outward,
// so no value is clipped, and bfloat16 has the range of every input type. A group with an infinity
// or a NaN stands for NaN. 20 bytes per 32 values: 5 bits a value, against 32 in the fp32 cache.
// A row of D channels is stored as halfwords of four codes, halfword r * D/32 + g holding channels
// 32 g + 4 r .. + 3 in ascending nibbles (r = 0..7): the order in which both tensor-core products of
// the attention kernel want them, so that a lane's codes are one wide load.
//
// Attention. Bound: HBM, 2 * 20/32 D bytes per key and head, and close behind it the integer work
// of unpacking: so both products run on the tensor cores with the codes as they are, and the scales
// are applied to their results (keys) or to the weights before (values):
//   s_j    = sum_g scale_jg (q_g . c_jg) + mid_jg sum(q_g)
//   out_c  = sum_j (p_j scale_jg) c_jc + sum_j p_j mid_jg
// with c = code - 8 and mid = low + 8 scale: centred, so that the two parts cancel little. c is exact
// in 16 bits, and a normal number there: fed as fp16 subnormals (code * 2^-24, one instruction a pair
// less) the same products came out 10 times less exact, the tensor core aligning its terms by the
// exponents as written. q is scaled by a power of two and split into two fp16 parts (22
// bits below the head's largest channel), p * scale into bfloat16 parts (three for float32 queries:
// 24 bits; two for 16-bit queries), a part being a row or column of the product: one m16n8k16
// product takes 16 keys, 4 heads and both parts. mma.sync, not tcgen05: at one query row per head the
// products fill an eighth of even these tiles, their time is far from the bound, and their operands
// come straight from registers (4-bit codes would have to be expanded into shared memory first).
// A warp works alone: blocks of 16 keys (never across a page) with the next block's loads in flight
// and the page after that looked up, its own running maximum, which moves only when it grows by more
// than 2^8 (sum, lows and accumulators share it), joined with the other warps' at the end.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>

#include <algorithm>

#include "common.cuh"
#include "kernels.h"
#include "split_rows.cuh"
#include "trace.h"

namespace dc {
namespace {

constexpr unsigned ALL = 0xffffffffu;
constexpr float LOG2E = 1.4426950408889634f;
constexpr int BAD_TABLE = 3;  // dc_device_status: a length, position or page id out of range
constexpr int GROUP = 32;
constexpr int WARPS = 4;

__device__ __forceinline__ float bf16_low(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf16_high(uint32_t w) { return __uint_as_float(w & 0xFFFF0000u); }
// low + 8 scale of a group's word.
__device__ __forceinline__ float mid(uint32_t w) { return fmaf(8.0f, bf16_low(w), bf16_high(w)); }

// ------------------------------------------------------------------ fill and read back ----

template <typename T>
__device__ __forceinline__ void load4(const T *p, int64_t inner, bool vec, float (&f)[4]) {
    if constexpr (sizeof(T) == 4) {
        if (vec) {
            const float4 v = *reinterpret_cast<const float4 *>(p);
            f[0] = v.x, f[1] = v.y, f[2] = v.z, f[3] = v.w;
            return;
        }
#pragma unroll
        for (int i = 0; i < 4; i++) f[i] = p[i * inner];
    } else {
        T e[4];
        if (vec) {
            *reinterpret_cast<uint2 *>(e) = *reinterpret_cast<const uint2 *>(p);
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++) e[i] = p[i * inner];
        }
#pragma unroll
        for (int i = 0; i < 4; i++) f[i] = (float)e[i];
    }
}

// Row of `slot` of `page` in the codes and scales.
__device__ __forceinline__ int64_t cache_row(const Cache4 &c, int64_t page, int which, int head, int slot) {
    return (((page * 2 + which) * c.Hkv + head) * c.page_size + slot);
}

// The row of position pos of sequence b, or -1 (and the device status) where the table has none.
__device__ __forceinline__ int64_t row_of(const Cache4Args &a, int64_t b, int64_t pos, int which, int head) {
    if (pos >= 0 && pos < a.P * a.c.page_size) {
        const uint32_t entry = (uint32_t)pos / (uint32_t)a.c.page_size, slot = (uint32_t)pos - entry * (uint32_t)a.c.page_size;
        const int64_t page = a.table[b * a.ts[0] + entry * a.ts[1]];
        if (page >= 0 && page < a.c.pages) return cache_row(a.c, page, which, head, (int)slot);
    }
    atomicExch(a.err, BAD_TABLE);
    return -1;
}

// Filling and reading back are bound by HBM. A block takes a run of tokens of one (sequence, head) of
// the keys or the values (grid: token runs, 2 Hkv, B); a thread four channels of ROWS tokens, whose
// loads are issued together; eight neighbours make a group of 32.
constexpr int ROWS = 4;

// rint(d / scale) of the correctly rounded quotient, by a product with the reciprocal where that
// cannot round the other way (the product is off by less than 1e-5 for quotients up to 15).
__device__ __forceinline__ float code_of(float d, float scale, float inv) {
    const float q = d * inv;
    float c = rintf(q);
    if (!(fabsf(q - c) < 0.4999f)) c = rintf(__fdiv_rn(d, scale));
    return fminf(fmaxf(c, 0.0f), 15.0f);
}

template <typename T>
__global__ void __launch_bounds__(256) cache4_append_kernel(const Cache4Args a, bool vec) {
    const int which = blockIdx.y & 1, head = blockIdx.y >> 1, lanes = a.c.D / 4, ng = a.c.D / GROUP;
    const int64_t b = blockIdx.z;
    const int quad = threadIdx.x & (lanes - 1), g = quad / 8, r = quad % 8, pass = 256 / lanes;
    const int64_t t0 = (int64_t)blockIdx.x * (pass * ROWS) + threadIdx.x / lanes, start = a.starts[b * a.starts_stride];
    const int64_t last = min(a.T, a.ends ? a.ends[b * a.ends_stride] - start : a.T);  // tokens from here on stay out
    const T *src = static_cast<const T *>(a.x[which]) + b * a.xs[which][0] + head * a.xs[which][1] + (int64_t)(4 * quad) * a.xs[which][3];
    float x[ROWS][4];
#pragma unroll
    for (int i = 0; i < ROWS; i++) {
        const int64_t t = t0 + i * pass;
        if (t < last) {
            load4(src + t * a.xs[which][2], a.xs[which][3], vec, x[i]);
        } else {
#pragma unroll
            for (int e = 0; e < 4; e++) x[i][e] = 0.0f;
        }
    }
#pragma unroll
    for (int i = 0; i < ROWS; i++) {
        const int64_t t = t0 + i * pass;
        float mn = fminf(fminf(x[i][0], x[i][1]), fminf(x[i][2], x[i][3]));
        float mx = fmaxf(fmaxf(x[i][0], x[i][1]), fmaxf(x[i][2], x[i][3]));
        bool finite = true;
#pragma unroll
        for (int e = 0; e < 4; e++) finite = finite && fabsf(x[i][e]) <= 3.402823466e38f;
        if (!finite) mx = INFINITY;
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) {
            mn = fminf(mn, __shfl_xor_sync(ALL, mn, o));
            mx = fmaxf(mx, __shfl_xor_sync(ALL, mx, o));
        }
        if (t >= last) continue;
        // low: bits below bfloat16 cut, one step further down for a negative value that had some.
        uint32_t lb = __float_as_uint(mn);
        if ((lb >> 31) && (lb & 0xFFFFu)) lb += 0x10000u;
        lb &= 0xFFFF0000u;
        const float low = __uint_as_float(lb);
        const float width = __fdiv_rn(__fsub_rn(mx, low), 15.0f);
        uint32_t sb = (__float_as_uint(width) + 0xFFFFu) & 0xFFFF0000u;  // up to bfloat16 (width >= 0)
        uint32_t codes = 0;
        if (!(fabsf(low) <= 3.402823466e38f) || !(width <= 3.3e38f)) {
            lb = sb = 0x7FC00000u;  // NaN
        } else if (sb) {
            const float scale = __uint_as_float(sb);
            const float inv = scale > 1e-37f && scale < 1e37f ? __frcp_rn(scale) : NAN;  // NaN: divide
#pragma unroll
            for (int e = 0; e < 4; e++) codes |= (uint32_t)code_of(__fsub_rn(x[i][e], low), scale, inv) << (4 * e);
        }
        const int64_t at = row_of(a, b, start + t, which, head);
        if (at < 0) continue;
        reinterpret_cast<uint16_t *>(a.c.codes + at * (a.c.D / 2))[r * ng + g] = (uint16_t)codes;
        if (r == 0) a.c.scales[at * ng + g] = (sb >> 16) | lb;
    }
}

// Token t of sequence b from the cache, in float32; zeros from the sequence's length on.
__global__ void __launch_bounds__(256) cache4_read_kernel(const Cache4Args a, bool vec) {
    const int which = blockIdx.y & 1, head = blockIdx.y >> 1, lanes = a.c.D / 4, ng = a.c.D / GROUP;
    const int64_t b = blockIdx.z;
    const int quad = threadIdx.x & (lanes - 1), g = quad / 8, r = quad % 8, pass = 256 / lanes;
    const int64_t t0 = (int64_t)blockIdx.x * (pass * ROWS) + threadIdx.x / lanes, len = a.lens[b * a.lens_stride];
    uint32_t codes[ROWS], sl[ROWS];
#pragma unroll
    for (int i = 0; i < ROWS; i++) {
        const int64_t t = t0 + i * pass;
        codes[i] = sl[i] = 0u;  // a zero
        const int64_t at = t < a.T && t < len ? row_of(a, b, t, which, head) : -1;
        if (at >= 0) {
            codes[i] = reinterpret_cast<const uint16_t *>(a.c.codes + at * (a.c.D / 2))[r * ng + g];
            sl[i] = a.c.scales[at * ng + g];
        }
    }
#pragma unroll
    for (int i = 0; i < ROWS; i++) {
        const int64_t t = t0 + i * pass;
        if (t >= a.T) continue;
        const float scale = bf16_low(sl[i]), low = bf16_high(sl[i]);
        const float4 y = make_float4(fmaf(scale, (float)(codes[i] & 15u), low), fmaf(scale, (float)((codes[i] >> 4) & 15u), low),
                                     fmaf(scale, (float)((codes[i] >> 8) & 15u), low), fmaf(scale, (float)(codes[i] >> 12), low));
        float *dst = a.y[which] + b * a.ys[which][0] + head * a.ys[which][1] + t * a.ys[which][2] + (int64_t)(4 * quad) * a.ys[which][3];
        if (vec) {
            *reinterpret_cast<float4 *>(dst) = y;
        } else {
            const int64_t s = a.ys[which][3];
            dst[0] = y.x, dst[s] = y.y, dst[2 * s] = y.z, dst[3 * s] = y.w;
        }
    }
}

// --------------------------------------------------------------------------- attention ----

__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_bf16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// (a, b) rounded to bfloat16, a in the low half.
__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
    return r;
}
// Pair i of codes, less 8, as fp16 and as bfloat16.
__device__ __forceinline__ uint32_t codes_f16(uint32_t y, int i) {
    const uint32_t z = ((y >> (4 * i)) & 0x000F000Fu) | 0x64006400u;  // 1024 + code
    uint32_t r;
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(z), "r"(0x64086408u));
    return r;
}
__device__ __forceinline__ uint32_t codes_bf16(uint32_t y, int i) {
    const uint32_t z = ((y >> (4 * i)) & 0x000F000Fu) | 0x43004300u;  // 128 + code
    uint32_t r;
    asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(z), "r"(0x43084308u));
    return r;
}

template <int N>
__device__ __forceinline__ void load_words(const void *p, uint32_t *w) {
    if constexpr (N == 1) {
        asm volatile("ld.global.nc.L1::no_allocate.b32 %0, [%1];" : "=r"(w[0]) : "l"(p));
    } else if constexpr (N == 2) {
        asm volatile("ld.global.nc.L1::no_allocate.v2.b32 {%0,%1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "l"(p));
    } else {
#pragma unroll
        for (int i = 0; i < N; i += 4)
            asm volatile("ld.global.nc.L1::no_allocate.v4.b32 {%0,%1,%2,%3}, [%4];"
                         : "=r"(w[i]), "=r"(w[i + 1]), "=r"(w[i + 2]), "=r"(w[i + 3])
                         : "l"(reinterpret_cast<const uint32_t *>(p) + i));
    }
}

// A block of 16 keys as a lane holds it (lane = 4 r + t): the codes of keys r and r + 8 (its
// quarter of each group) with their scales, and those of values t, t + 8, t + 4, t + 12 (its eighth
// of each group) with the scales of values r and r + 8.
template <int NG>
struct Block {
    uint32_t k[2][NG], ks[2][NG], v[4][NG / 2], vs[2][NG];
};

template <int D, int PARTS, int NT>
struct AttnCfg {
    static constexpr int NG = D / GROUP, HC = 4 * NT;  // groups; query heads per CTA
    static constexpr int ROWS = HC * PARTS;            // rows of the second product in use
    static_assert(ROWS <= 16, "the parts of the weights fill one product's rows");
    static constexpr int ROW_BYTES = 48;               // 16 weights of a row, padded against bank conflicts
    // Shared memory: q fragments | the warps' weight tiles; after the loop the accumulators.
    static constexpr int Q_BYTES = NT * NG * 32 * 16, W_BYTES = NG * 16 * ROW_BYTES;
    static constexpr int LOOP_BYTES = Q_BYTES + WARPS * W_BYTES;
    static constexpr int ACC_BYTES = WARPS * ROWS * D * 4;
    static constexpr int SMEM = LOOP_BYTES > ACC_BYTES ? LOOP_BYTES : ACC_BYTES;
};

__device__ __forceinline__ float load_q(const Cache4Args &a, int64_t at) {
    if (a.dtype == DC_F32) return static_cast<const float *>(a.x[0])[at];
    if (a.dtype == DC_F16) return __half2float(static_cast<const __half *>(a.x[0])[at]);
    return __bfloat162float(static_cast<const __nv_bfloat16 *>(a.x[0])[at]);
}

template <int D, int PARTS, int NT>
__global__ void __launch_bounds__(WARPS * 32, D == 256 ? 2 : 3) cache4_attention_kernel(const Cache4Args a, const SplitRows rows) {
    using C = AttnCfg<D, PARTS, NT>;
    constexpr int NG = C::NG, HC = C::HC;
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ float s_qsum[HC][NG], s_exp[HC], s_m[WARPS][HC], s_l[WARPS][HC], s_low[WARPS][HC][NG];
    griddep_launch_dependents();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, t = lane & 3;
    const int group = (int)(a.H / a.c.Hkv), chunks = (group + HC - 1) / HC;
    const int64_t b = blockIdx.z;
    const int hk = blockIdx.y / chunks;
    const int64_t h0 = (int64_t)hk * group + (blockIdx.y % chunks) * HC;
    const int nh = min(HC, group - (int)(blockIdx.y % chunks) * HC);

    // The sequence's visible keys: [0, sinks) and [lo, len), in blocks of 16.
    const int64_t capacity = a.P * a.c.page_size;
    int64_t len = a.lens[b * a.lens_stride];
    if (len < 0 || len > capacity) {
        if (threadIdx.x == 0) atomicExch(a.err, BAD_TABLE);
        len = len < 0 ? 0 : capacity;
    }
    const int64_t lo = a.window ? max((int64_t)0, len - a.window) : 0, sinks = min(a.sinks, lo);
    const int first = (int)(lo / 16), sink_blocks = min((int)((sinks + 15) / 16), first);
    const int total = len == 0 ? 0 : sink_blocks + (int)((len + 15) / 16) - first;
    const int per = (total + rows.splits - 1) / rows.splits, v0 = blockIdx.x * per, v1 = min(total, v0 + per);
    const int page16 = a.c.page_size / 16;
    auto block_of = [&](int v) { return v < sink_blocks ? v : first + v - sink_blocks; };
    // Page ids are read a block ahead of the page; -1 where the table's entry is out of range.
    auto page_id = [&](int v) -> int {
        if (v >= v1) return -1;
        const int id = a.table[b * a.ts[0] + (int64_t)(block_of(v) / page16) * a.ts[1]];
        return id;
    };
    const int64_t half_page = (int64_t)a.c.Hkv * a.c.page_size;  // rows from a page's keys to its values
    auto load_block = [&](int v, int id, Block<NG> &x) -> bool {
        if ((unsigned)id >= (unsigned)min(a.c.pages, (int64_t)0x7fffffff)) {
            atomicExch(a.err, BAD_TABLE);
            return false;
        }
        const int64_t krow = ((int64_t)id * 2 * a.c.Hkv + hk) * a.c.page_size + (block_of(v) % page16) * 16, vrow = krow + half_page;
        const uint8_t *kc = a.c.codes + krow * (D / 2), *vc = a.c.codes + vrow * (D / 2);
#pragma unroll
        for (int i = 0; i < 2; i++) {
            load_words<NG>(kc + (r + 8 * i) * (D / 2) + t * 4 * NG, x.k[i]);
            load_words<NG>(a.c.scales + (krow + r + 8 * i) * NG, x.ks[i]);
            load_words<NG>(a.c.scales + (vrow + r + 8 * i) * NG, x.vs[i]);
        }
#pragma unroll
        for (int i = 0; i < 4; i++) load_words<NG / 2>(vc + (t + 4 * ((i >> 1) + 2 * (i & 1))) * (D / 2) + r * 2 * NG, x.v[i]);
        return true;
    };
    Block<NG> cur;
    bool cur_ok = false;
    int v = v0 + warp;
    int next_id = page_id(v + WARPS);
    if (v < v1) cur_ok = load_block(v, page_id(v), cur);

    // q: per head a power of two that brings its largest channel below 1, the sums of its groups,
    // and the two fp16 parts in the order of the products' B fragments.
    for (int h = warp; h < HC; h += WARPS) {
        float x[NG], top = 0.0f;
#pragma unroll
        for (int g = 0; g < NG; g++) {
            x[g] = h < nh ? load_q(a, b * a.xs[0][0] + (h0 + h) * a.xs[0][1] + (int64_t)(32 * g + lane) * a.xs[0][3]) : 0.0f;
            top = fmaxf(top, fabsf(x[g]));
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(ALL, top, o));
        int e = 0;
        if (top > 0.0f && top <= 3.402823466e38f) frexpf(top, &e);
#pragma unroll
        for (int g = 0; g < NG; g++) {
            float s = x[g];
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(ALL, s, o);
            if (lane == 0) s_qsum[h][g] = s * (a.scale * LOG2E);
            // Channel 32 g + lane = 4 r' + i of a group: k-pair member r' & 1 of lane t' = r' / 2, pair i.
            const float y = ldexpf(x[g], -e);
            const __half hi = __float2half_rn(y), lo16 = __float2half_rn(y - __half2float(hi));
            const int rr = lane >> 2, i = lane & 3;
#pragma unroll
            for (int part = 0; part < 2; part++) {
                const int col = (h & 3) * 2 + part;
                __half *frag = reinterpret_cast<__half *>(smem + (((h >> 2) * NG + g) * 32 + col * 4 + (rr >> 1)) * 16);
                frag[i * 2 + (rr & 1)] = part ? lo16 : hi;
            }
        }
        if (lane == 0) s_exp[h] = ldexpf(a.scale * LOG2E, e);
    }
    __syncthreads();

    float mul[NT], qsum[NT][NG], m[NT], l[NT], low[NT][NG];
    float acc[4 * NG][4];
#pragma unroll
    for (int n = 0; n < NT; n++) {
        mul[n] = s_exp[n * 4 + t];
        m[n] = -INFINITY;
        l[n] = 0.0f;
#pragma unroll
        for (int g = 0; g < NG; g++) {
            qsum[n][g] = s_qsum[n * 4 + t][g];
            low[n][g] = 0.0f;
        }
    }
#pragma unroll
    for (int i = 0; i < 4 * NG; i++)
#pragma unroll
        for (int c = 0; c < 4; c++) acc[i][c] = 0.0f;
    uint8_t *wt = smem + C::Q_BYTES + warp * C::W_BYTES;
    const uint32_t wt_addr = (uint32_t)__cvta_generic_to_shared(wt) + (lane & 15) * C::ROW_BYTES + (lane >> 4) * 16;

    for (; v < v1; v += WARPS) {
        Block<NG> nxt;
        bool nxt_ok = false;
        if (v + WARPS < v1) nxt_ok = load_block(v + WARPS, next_id, nxt);
        next_id = page_id(v + 2 * WARPS);
        const int64_t j0 = (int64_t)block_of(v) * 16 + r, j1 = j0 + 8;
        const bool ok0 = cur_ok && j0 < len && (j0 >= lo || j0 < sinks), ok1 = cur_ok && j1 < len && (j1 >= lo || j1 < sinks);
        // Scores of keys r and r + 8 for head t of each tile.
        float s0[NT], s1[NT];
#pragma unroll
        for (int n = 0; n < NT; n++) s0[n] = s1[n] = 0.0f;
        float b0[NT], b1[NT];
#pragma unroll
        for (int n = 0; n < NT; n++) b0[n] = b1[n] = 0.0f;
#pragma unroll
        for (int g = 0; g < NG; g++) {
            const uint32_t sel = (g & 1) ? 0x7632u : 0x5410u;
            const uint32_t y0 = __byte_perm(cur.k[0][g / 2], cur.k[0][NG / 2 + g / 2], sel);
            const uint32_t y1 = __byte_perm(cur.k[1][g / 2], cur.k[1][NG / 2 + g / 2], sel);
            const uint32_t a0[4] = {codes_f16(y0, 0), codes_f16(y1, 0), codes_f16(y0, 1), codes_f16(y1, 1)};
            const uint32_t a1[4] = {codes_f16(y0, 2), codes_f16(y1, 2), codes_f16(y0, 3), codes_f16(y1, 3)};
#pragma unroll
            for (int n = 0; n < NT; n++) {
                const uint4 q = *reinterpret_cast<const uint4 *>(smem + ((n * NG + g) * 32 + lane) * 16);
                float c[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                mma_f16(c, a0, q.x, q.y);
                mma_f16(c, a1, q.z, q.w);
                s0[n] = fmaf(bf16_low(cur.ks[0][g]), c[0] + c[1], s0[n]);
                s1[n] = fmaf(bf16_low(cur.ks[1][g]), c[2] + c[3], s1[n]);
                b0[n] = fmaf(mid(cur.ks[0][g]), qsum[n][g], b0[n]);
                b1[n] = fmaf(mid(cur.ks[1][g]), qsum[n][g], b1[n]);
            }
        }
        float corr[NT];
        bool moved = false;
#pragma unroll
        for (int n = 0; n < NT; n++) {
            s0[n] = ok0 ? fmaf(s0[n], mul[n], b0[n]) : -INFINITY;
            s1[n] = ok1 ? fmaf(s1[n], mul[n], b1[n]) : -INFINITY;
            float top = fmaxf(s0[n], s1[n]);
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) top = fmaxf(top, __shfl_xor_sync(ALL, top, o));
            corr[n] = 1.0f;
            if (top > m[n] + 8.0f || (m[n] == -INFINITY && top > m[n])) {
                corr[n] = exp2_fast(m[n] - top);
                m[n] = top;
                moved = true;
            }
        }
        if (__any_sync(ALL, moved)) {
#pragma unroll
            for (int n = 0; n < NT; n++) {
                l[n] *= corr[n];
#pragma unroll
                for (int g = 0; g < NG; g++) low[n][g] *= corr[n];
            }
            float f[2];
#pragma unroll
            for (int i = 0; i < 2; i++) {  // the factors of accumulator rows r and r + 8
                const int h = min((r + 8 * i) / PARTS, HC - 1);
                f[i] = __shfl_sync(ALL, corr[0], h & 3);
                if constexpr (NT == 2) {
                    const float other = __shfl_sync(ALL, corr[NT - 1], h & 3);
                    if (h >= 4) f[i] = other;
                }
            }
#pragma unroll
            for (int i = 0; i < 4 * NG; i++) {
                acc[i][0] *= f[0];
                acc[i][1] *= f[0];
                acc[i][2] *= f[1];
                acc[i][3] *= f[1];
            }
        }
        // Weights times the values' scales, in bfloat16 parts, to the warp's tile: row head * PARTS
        // + part, slots 2 r and 2 r + 1 for keys r and r + 8.
        __syncwarp();
#pragma unroll
        for (int n = 0; n < NT; n++) {
            // No key yet: every score is -inf (weight 0) or a NaN.
            const bool none = m[n] == -INFINITY;
            const float p0 = none ? (s0[n] != s0[n] ? s0[n] : 0.0f) : exp2_fast(s0[n] - m[n]);
            const float p1 = none ? (s1[n] != s1[n] ? s1[n] : 0.0f) : exp2_fast(s1[n] - m[n]);
            l[n] += p0 + p1;
#pragma unroll
            for (int g = 0; g < NG; g++) {
                // A place behind the sequence's end may hold anything.
                const uint32_t z0 = ok0 ? cur.vs[0][g] : 0u, z1 = ok1 ? cur.vs[1][g] : 0u;
                low[n][g] = fmaf(p0, mid(z0), fmaf(p1, mid(z1), low[n][g]));
                float w0 = p0 * bf16_low(z0), w1 = p1 * bf16_low(z1);
#pragma unroll
                for (int part = 0; part < PARTS; part++) {
                    const uint32_t w = pack_bf16(w0, w1);
                    *reinterpret_cast<uint32_t *>(wt + (g * 16 + (n * 4 + t) * PARTS + part) * C::ROW_BYTES + 4 * r) = w;
                    w0 -= bf16_low(w);
                    w1 -= bf16_high(w);
                }
            }
        }
        __syncwarp();
#pragma unroll
        for (int g = 0; g < NG; g++) {
            uint32_t w[4];
            ldmatrix4(w, wt_addr + g * 16 * C::ROW_BYTES);
            const uint32_t sel = (g & 1) ? 0x7632u : 0x5410u;
            const uint32_t y0 = __byte_perm(cur.v[0][g / 2], cur.v[1][g / 2], sel);
            const uint32_t y1 = __byte_perm(cur.v[2][g / 2], cur.v[3][g / 2], sel);
#pragma unroll
            for (int i = 0; i < 4; i++) mma_bf16(acc[g * 4 + i], w, codes_bf16(y0, i), codes_bf16(y1, i));
        }
        cur = nxt;
        cur_ok = nxt_ok;
    }

    // Join the warps.
#pragma unroll
    for (int n = 0; n < NT; n++) {
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) {
            l[n] += __shfl_xor_sync(ALL, l[n], o);
#pragma unroll
            for (int g = 0; g < NG; g++) low[n][g] += __shfl_xor_sync(ALL, low[n][g], o);
        }
        if (r == 0) {
            s_m[warp][n * 4 + t] = m[n];
            s_l[warp][n * 4 + t] = l[n];
#pragma unroll
            for (int g = 0; g < NG; g++) s_low[warp][n * 4 + t][g] = low[n][g];
        }
    }
    __syncthreads();
    float *sacc = reinterpret_cast<float *>(smem) + warp * C::ROWS * D;
#pragma unroll
    for (int i = 0; i < 4 * NG; i++)
#pragma unroll
        for (int c = 0; c < 4; c++) {
            const int row = r + 8 * (c >> 1), ch = (i / 4) * 32 + (2 * t + (c & 1)) * 4 + (i & 3);
            if (row < C::ROWS) sacc[row * D + ch] = acc[i][c];
        }
    __syncthreads();
    for (int i = threadIdx.x; i < nh * D; i += WARPS * 32) {
        const int h = i / D, d = i % D;
        float top = -INFINITY, sum = 0.0f, o = 0.0f;
#pragma unroll
        for (int w = 0; w < WARPS; w++) top = fmaxf(top, s_m[w][h]);
#pragma unroll
        for (int w = 0; w < WARPS; w++) {
            const float f = s_m[w][h] == -INFINITY ? 1.0f : exp2f(s_m[w][h] - top);
            float x = s_low[w][h][d / 32];
#pragma unroll
            for (int part = 0; part < PARTS; part++)
                x += reinterpret_cast<const float *>(smem)[(w * C::ROWS + h * PARTS + part) * D + d];
            sum = fmaf(s_l[w][h], f, sum);
            o = fmaf(x, f, o);
        }
        split_store(rows, b * a.H + h0 + h, blockIdx.x, d, top, sum, o);
    }
}

template <int D, int PARTS, int NT>
int launch_attention(const Cache4Args &a, const SplitRows &rows, cudaStream_t stream) {
    using C = AttnCfg<D, PARTS, NT>;
    auto kernel = cache4_attention_kernel<D, PARTS, NT>;
    if (C::SMEM > 40 * 1024) {  // with the static arrays, past the 48 KB that need no attribute
        cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
        if (e != cudaSuccess) return cuda_fail(e, "cache4_attention smem attribute");
    }
    const int64_t group = a.H / a.c.Hkv, chunks = (group + C::HC - 1) / C::HC;
    KernelTrace tr("cache4_attention", stream);
    kernel<<<dim3((unsigned)rows.splits, (unsigned)(a.c.Hkv * chunks), (unsigned)a.B), WARPS * 32, C::SMEM, stream>>>(a, rows);
    return check_launch("cache4_attention");
}

// Heads of one key/value head that a CTA takes: 4, or 8 where the parts of 8 heads' weights fit the
// product's 16 rows.
int heads_per_cta(int64_t group, int dtype) { return dtype != DC_F32 && group > 4 ? 8 : 4; }

template <int D>
int launch_dim(const Cache4Args &a, const SplitRows &rows, cudaStream_t stream) {
    if (a.dtype == DC_F32) return launch_attention<D, 3, 1>(a, rows, stream);
    return heads_per_cta(a.H / a.c.Hkv, a.dtype) == 8 ? launch_attention<D, 2, 2>(a, rows, stream)
                                                      : launch_attention<D, 2, 1>(a, rows, stream);
}

// Whether runs of four channels of a (B, H, T, D) view start on 4-element boundaries.
bool vec4(const void *ptr, const int64_t *st, int size) {
    return st[3] == 1 && st[0] % 4 == 0 && st[1] % 4 == 0 && st[2] % 4 == 0 && (reinterpret_cast<uintptr_t>(ptr) & (4 * size - 1)) == 0;
}

}  // namespace

// Grid of the fill and read kernels.
dim3 token_grid(const Cache4Args &a) {
    const int64_t run = 256 / (a.c.D / 4) * ROWS;
    return dim3((unsigned)((a.T + run - 1) / run), (unsigned)(2 * a.c.Hkv), (unsigned)a.B);
}

int cache4_append(const Cache4Args &a, cudaStream_t stream) {
    const int size = a.dtype == DC_F32 ? 4 : 2;
    const bool vec = vec4(a.x[0], a.xs[0], size) && vec4(a.x[1], a.xs[1], size);
    KernelTrace tr("cache4_append", stream);
    if (a.dtype == DC_F32) cache4_append_kernel<float><<<token_grid(a), 256, 0, stream>>>(a, vec);
    else if (a.dtype == DC_F16) cache4_append_kernel<__half><<<token_grid(a), 256, 0, stream>>>(a, vec);
    else cache4_append_kernel<__nv_bfloat16><<<token_grid(a), 256, 0, stream>>>(a, vec);
    return check_launch("cache4_append");
}

int cache4_read(const Cache4Args &a, cudaStream_t stream) {
    const bool vec = vec4(a.y[0], a.ys[0], 4) && vec4(a.y[1], a.ys[1], 4);
    KernelTrace tr("cache4_read", stream);
    cache4_read_kernel<<<token_grid(a), 256, 0, stream>>>(a, vec);
    return check_launch("cache4_read");
}

// Splits of each row: three CTAs of 4 warps on every SM twice over, at least one block a warp.
int cache4_splits(int64_t B, int64_t H, int64_t Hkv, int64_t capacity, int64_t window, int64_t sinks, int dtype) {
    const int64_t group = H / Hkv, per = heads_per_cta(group, dtype), chunks = (group + per - 1) / per;
    const int64_t ctas = std::max<int64_t>(1, B * Hkv * chunks);
    const int64_t keys = window ? std::min(capacity, std::min(window, capacity) + std::min(sinks, capacity)) : capacity;
    const int64_t fill = (int64_t)device_sm_count() * 6 / ctas, most = (keys + 16 * WARPS - 1) / (16 * WARPS);
    return (int)std::max<int64_t>(1, std::min<int64_t>(128, std::min(fill, most)));
}

int cache4_attention(const Cache4Args &a, const SplitRows &rows, cudaStream_t stream) {
    int st;
    if (a.c.D == 64) st = launch_dim<64>(a, rows, stream);
    else if (a.c.D == 128) st = launch_dim<128>(a, rows, stream);
    else st = launch_dim<256>(a, rows, stream);
    return st ? st : split_combine(rows, stream);
}

}  // namespace dc
