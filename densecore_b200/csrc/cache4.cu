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
// Sixteen tokens of a head lie together, 20 D bytes: the keys' codes (8 D bytes) and scales (16 rows of
// D / 32 words, scale | low << 16), then the values'; so a warp fetches them with one bulk copy. The
// codes are halfwords of four channels, 32 g + 4 r .. + 3 in ascending nibbles (r = 0..7), placed so
// that the words of a lane's wide load are pairs as the attention kernel's products take them: for the
// keys r and r + 1 of a token, for the values tokens s and s + 8 (code_at).
//
// Attention. Bound: HBM, 2 * 20/32 D bytes per key and head, and close behind it the integer work
// of unpacking: so both products run on the tensor cores with the codes as they are, and the scales
// are applied to their results (keys) or to the weights before (values):
//   s_j    = sum_g scale_jg (q_g . c_jg) + mid_jg sum(q_g)
//   out_c  = sum_j (p_j scale_jg) c_jc + sum_j p_j mid_jg
// with c = code - 8 and mid = low + 8 scale: centred, so that the two parts cancel little. The small
// operand is scaled by a power of two and split into parts that a product takes as rows or columns:
//   weights  p * scale into bfloat16 parts (three for float32 queries: 24 bits; two for 16-bit ones)
//   q        one head per CTA: as a 28-bit integer in four signed digits to the base 128, multiplied
//            with the codes as bytes (m16n8k32, exact sums; half the unpacking of 16-bit codes);
//            several: two fp16 parts (22 bits below the head's largest channel), so that a group's
//            product gives a lane both parts of one head (m16n8k16)
// Codes are exact in every one of these types. (As fp16 subnormals, code * 2^-24, they come without a
// subtraction, but the sums came out 10 times less exact: the tensor core aligns its terms by the
// exponents as written.) mma.sync, not tcgen05: at one query row per head the products fill an eighth of
// even these tiles, their time is far from the bound, and their operands come straight from registers
// (4-bit codes would have to be expanded into shared memory first).
// A warp works alone on blocks of 16 keys (never across a page), which bulk copies bring into a ring of
// its own in shared memory a few blocks ahead; its own running maximum, which moves only when it grows
// by more than 2^8 (sum, mids and accumulators share it), is joined with the other warps' at the end.
// (With the blocks fetched into registers one ahead the warps waited on loads 2.2 cycles per issue.)
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>

#include <algorithm>

#include "common.cuh"
#include "kernels.h"
#include "sm100.cuh"
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

// Two sums (fused products) in one instruction, each rounded as alone.
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(reinterpret_cast<uint64_t &>(r)) : "l"(reinterpret_cast<uint64_t &>(a)), "l"(reinterpret_cast<uint64_t &>(b)));
    return r;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(reinterpret_cast<uint64_t &>(r)) : "l"(reinterpret_cast<uint64_t &>(a)), "l"(reinterpret_cast<uint64_t &>(b)));
    return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;"
        : "=l"(reinterpret_cast<uint64_t &>(r))
        : "l"(reinterpret_cast<uint64_t &>(a)), "l"(reinterpret_cast<uint64_t &>(b)), "l"(reinterpret_cast<uint64_t &>(c)));
    return r;
}
__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }
// (x & mask) | bits in one instruction (the compiler made two of it).
__device__ __forceinline__ uint32_t and_or(uint32_t x, uint32_t mask, uint32_t bits) {
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(x), "r"(mask), "r"(bits));
    return r;
}

// Eight channels as the pairs (x_e, x_{e + 4}).
template <typename T>
__device__ __forceinline__ void load8(const T *p, int64_t inner, bool vec, float2 (&f)[4]) {
    T e[8];
    if (vec) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; i++) reinterpret_cast<uint4 *>(e)[i] = reinterpret_cast<const uint4 *>(p)[i];
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) e[i] = p[i * inner];
    }
#pragma unroll
    for (int i = 0; i < 4; i++) f[i] = make_float2((float)e[i], (float)e[i + 4]);
}

// Bytes of a block of 16 tokens of a head, keys and values.
__host__ __device__ constexpr int block_bytes(int D) { return 20 * D; }

// Where halfword (group g, r) of token `slot` (0..15) lies among a block's codes of keys or values: the
// token's part and the halfword's, in bytes.
__device__ __forceinline__ int slot_at(int which, int slot, int ng) {
    return which ? (slot / 4 % 2 * 32 + slot % 4) * 4 * ng + slot / 8 * 2 : slot * 16 * ng;
}
__device__ __forceinline__ int code_at(int which, int r, int g, int ng) {
    return which ? 4 * (4 * r * ng + g) : 4 * (r / 2 * ng + g) + r % 2 * 2;
}

// Position pos of sequence b, keys or values: the token's part of the codes, and from there the way to its
// scales in bytes; null (and the device status) where the table has no page for it.
struct Place {
    uint8_t *codes;
    int scales;
};
__device__ __forceinline__ Place place_of(const Cache4Args &a, int64_t b, int64_t pos, int which, int head) {
    if (pos >= 0 && pos < a.P * a.c.page_size) {
        const uint32_t entry = (uint32_t)pos / (uint32_t)a.c.page_size, slot = (uint32_t)pos - entry * (uint32_t)a.c.page_size;
        const int64_t page = a.table[b * a.ts[0] + entry * a.ts[1]];
        if (page >= 0 && page < a.c.pages) {
            const int ng = a.c.D / GROUP, at = slot_at(which, (int)(slot % 16), ng);
            uint8_t *half = a.c.data + ((page * a.c.Hkv + head) * (a.c.page_size / 16) + slot / 16) * block_bytes(a.c.D) + which * 10 * a.c.D;
            return {half + at, 8 * a.c.D + (int)(slot % 16) * 4 * ng - at};
        }
    }
    atomicExch(a.err, BAD_TABLE);
    return {nullptr, 0};
}

// Filling and reading back are bound by instructions (issue slots 70 and 77 % busy, HBM below 30 %). Grid:
// token runs, 2 Hkv (keys or values of a head), B. Appending, a thread takes eight channels of APPEND_ROWS
// tokens, whose loads are issued together, four neighbours make a group of 32, and a warp finds its tokens'
// places (a division by the page size, a look into the table) by itself. Reading, a thread takes four
// channels, so that a warp's stores are contiguous (eight: 24 -> 28 us), and the block finds the places.
// 8 sequences of 700 to 1500 tokens, 8 heads of 128: append 28.5 us, read 22.5 us. (Appending with four
// channels a thread: 37; two rows 32, eight 41.)
constexpr int FILL_WARPS = 8, APPEND_ROWS = 4, READ_ROWS = 4;

// Appending: the places of a warp's tokens, those from `last` on null.
__device__ __forceinline__ void warp_places(const Cache4Args &a, int64_t b, int64_t pos0, int64_t t0, int64_t last, int run, int which, int head,
                                            Place *places) {
    const int lane = threadIdx.x & 31;
    if (lane < run) places[lane] = t0 + lane < last ? place_of(a, b, pos0 + t0 + lane, which, head) : Place{nullptr, 0};
    __syncwarp();
}

// Reading: the places of the block's tokens t0 .. (at most 64), those from `last` on null.
__device__ __forceinline__ void block_places(const Cache4Args &a, int64_t b, int64_t pos0, int64_t t0, int64_t last, int run, int which,
                                             int head, Place *places) {
    if ((int)threadIdx.x < run) {
        const int64_t t = t0 + threadIdx.x;
        places[threadIdx.x] = t < last ? place_of(a, b, pos0 + t, which, head) : Place{nullptr, 0};
    }
    __syncthreads();
}

__device__ __forceinline__ float max_nan(float a, float b) {  // NaN if either is
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float rcp_fast(float x) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// x / 15, correctly rounded, then up to bfloat16 (x >= 0), as bits. The product with 1/15 is off by less
// than two units in the last place, which matters only where those cross a bfloat16: there, and where it
// is not a normal number, the division is done.
__device__ __forceinline__ uint32_t fifteenth_up(float x) {
    uint32_t w = __float_as_uint(x * (1.0f / 15.0f));
    if (((w + 4u) & 0xFFFFu) <= 8u || w < 0x01000000u || w > 0x7E000000u) w = __float_as_uint(__fdiv_rn(x, 15.0f));
    return (w + 0xFFFFu) & 0xFFFF0000u;
}

// The codes of eight values d = x - low (pairs e, e + 4), as a word: the correctly rounded d / scale to the
// nearest whole number (ties to even), by a product with the reciprocal (off by less than 3e-6 for
// quotients up to 15) where that cannot round the other way.
__device__ __forceinline__ uint32_t codes_of(const float2 (&d)[4], float scale) {
    constexpr float MAGIC = 12582912.0f;  // 1.5 * 2^23: sums with it are rounded to whole numbers
    const bool fast = scale > 1e-37f && scale < 1e37f;
    const float2 inv = both(fast ? rcp_fast(scale) : 0.0f);
    float2 n[4];
    float2 r[4];
    float off = fast ? 0.0f : 1.0f;
#pragma unroll
    for (int e = 0; e < 4; e++) {
        const float2 q = mul2(d[e], inv);
        n[e] = add2(add2(q, both(MAGIC)), both(-MAGIC));
        r[e] = fma2(n[e], both(-1.0f), q);
        off = fmaxf(off, fmaxf(fabsf(r[e].x), fabsf(r[e].y)));
    }
    if (off >= 0.49999f) {
#pragma unroll
        for (int e = 0; e < 4; e++) {
            if (!fast || fabsf(r[e].x) >= 0.49999f) n[e].x = __fdiv_rn(d[e].x, scale) + MAGIC - MAGIC;
            if (!fast || fabsf(r[e].y) >= 0.49999f) n[e].y = __fdiv_rn(d[e].y, scale) + MAGIC - MAGIC;
        }
    }
    // n_0 + 16 n_1 + 256 n_2 + 4096 n_3, exactly, then 2^23 more: the sum's low 16 bits.
    const float2 w = add2(fma2(n[3], both(4096.0f), fma2(n[2], both(256.0f), fma2(n[1], both(16.0f), n[0]))), both(8388608.0f));
    return __byte_perm(__float_as_uint(w.x), __float_as_uint(w.y), 0x5410);
}

template <typename T>
__global__ void __launch_bounds__(FILL_WARPS * 32, 4) cache4_append_kernel(const Cache4Args a, bool vec) {
    constexpr int ROWS = APPEND_ROWS;
    __shared__ Place places_of[FILL_WARPS][32 / (64 / 8) * ROWS];
    const int which = blockIdx.y & 1, head = blockIdx.y >> 1, ng = a.c.D / GROUP;
    const int64_t b = blockIdx.z, start = a.starts[b * a.starts_stride];
    const int64_t last = min(a.T, a.ends ? a.ends[b * a.ends_stride] - start : a.T);  // tokens from here on stay out
    // Lanes of a row, rows a pass of the warp; this lane's row and first quad of channels.
    const int lane = threadIdx.x & 31, lanes = a.c.D / 8, per = 32 / lanes, sub = lane / lanes, quad = 2 * (lane & (lanes - 1)), g = quad / 8, r = quad % 8;
    const int64_t t0 = ((int64_t)blockIdx.x * FILL_WARPS + threadIdx.x / 32) * (per * ROWS);
    if (t0 >= last) return;
    const int code = code_at(which, r, g, ng);
    Place *places = places_of[threadIdx.x / 32];
    const T *src = static_cast<const T *>(a.x[which]) + b * a.xs[which][0] + head * a.xs[which][1] + (int64_t)(4 * quad) * a.xs[which][3];
    src += (t0 + sub) * a.xs[which][2];
    const int64_t step = per * a.xs[which][2];
    const int here = (int)min(last - t0, (int64_t)(per * ROWS));  // the warp's tokens
    float2 x[ROWS][4];
#pragma unroll
    for (int i = 0; i < ROWS; i++) {
        if (sub + i * per < here) {
            load8(src + i * step, a.xs[which][3], vec, x[i]);
        } else {
#pragma unroll
            for (int e = 0; e < 4; e++) x[i][e] = both(0.0f);
        }
    }
    warp_places(a, b, start, t0, last, per * ROWS, which, head, places);
#pragma unroll
    for (int i = 0; i < ROWS; i++) {
        float mn = fminf(x[i][0].x, x[i][0].y), mx = max_nan(x[i][0].x, x[i][0].y);
#pragma unroll
        for (int e = 1; e < 4; e++) {
            mn = fminf(mn, fminf(x[i][e].x, x[i][e].y));
            mx = max_nan(mx, max_nan(x[i][e].x, x[i][e].y));
        }
#pragma unroll
        for (int o = 2; o > 0; o >>= 1) {
            mn = fminf(mn, __shfl_xor_sync(ALL, mn, o));
            mx = max_nan(mx, __shfl_xor_sync(ALL, mx, o));
        }
        const Place at = places[sub + i * per];
        if (!at.codes) continue;
        // low: bits below bfloat16 cut, one step further down for a negative value that had some.
        uint32_t lb = __float_as_uint(mn);
        if ((lb >> 31) && (lb & 0xFFFFu)) lb += 0x10000u;
        lb &= 0xFFFF0000u;
        const float low = __uint_as_float(lb), width = __fsub_rn(mx, low);
        uint32_t sb = 0, codes = 0;
        if (!(width <= 3.402823466e38f)) {  // an infinity or a NaN among the values, or their range overflows
            lb = sb = 0x7FC00000u;  // NaN
        } else if (width > 0.0f) {
            sb = fifteenth_up(width);
            float2 d[4];
#pragma unroll
            for (int e = 0; e < 4; e++) d[e] = add2(x[i][e], both(-low));
            codes = codes_of(d, __uint_as_float(sb));
        }
        uint8_t *to = at.codes + code;
        if (which) {
            *reinterpret_cast<uint16_t *>(to) = (uint16_t)codes;
            *reinterpret_cast<uint16_t *>(to + 16 * ng) = (uint16_t)(codes >> 16);
        } else {  // halfwords r and r + 1 side by side
            *reinterpret_cast<uint32_t *>(to) = codes;
        }
        if (r == 0) *reinterpret_cast<uint32_t *>(at.codes + at.scales + 4 * g) = (sb >> 16) | lb;
    }
}

// Token t of sequence b from the cache, in float32; zeros from the sequence's length on.
__global__ void __launch_bounds__(256) cache4_read_kernel(const Cache4Args a, bool vec) {
    constexpr int ROWS = READ_ROWS;
    __shared__ Place places[256 / 16 * ROWS];
    const int which = blockIdx.y & 1, head = blockIdx.y >> 1, lanes = a.c.D / 4, ng = a.c.D / GROUP;
    const int64_t b = blockIdx.z;
    const int quad = threadIdx.x & (lanes - 1), g = quad / 8, r = quad % 8, pass = 256 / lanes, row0 = threadIdx.x / lanes;
    const int64_t t0 = (int64_t)blockIdx.x * (pass * ROWS), len = a.lens[b * a.lens_stride];
    block_places(a, b, 0, t0, min(a.T, len), pass * ROWS, which, head, places);
    const int code = code_at(which, r, g, ng);
    uint32_t codes[ROWS], sl[ROWS];
#pragma unroll
    for (int i = 0; i < ROWS; i++) {
        const Place at = places[row0 + i * pass];
        codes[i] = sl[i] = 0u;  // a zero
        if (at.codes) {
            codes[i] = *reinterpret_cast<const uint16_t *>(at.codes + code);
            sl[i] = *reinterpret_cast<const uint32_t *>(at.codes + at.scales + 4 * g);
        }
    }
    float *dst = a.y[which] + b * a.ys[which][0] + head * a.ys[which][1] + (t0 + row0) * a.ys[which][2] + (int64_t)(4 * quad) * a.ys[which][3];
    const int64_t step = pass * a.ys[which][2];
    const int here = (int)min(a.T - t0, (int64_t)(pass * ROWS));  // the block's tokens
#pragma unroll
    for (int i = 0; i < ROWS; i++) {
        if (row0 + i * pass >= here) continue;
        const float2 scale = both(bf16_low(sl[i])), low = both(bf16_high(sl[i]));
        float2 y[2];
#pragma unroll
        for (int e = 0; e < 2; e++) {
            // 2^23 + 16^n code, less 2^23, over 16^n: the code, exactly, without shifts or the conversion unit.
            const float2 n = e ? make_float2(0x1p-8f, 0x1p-12f) : make_float2(1.0f, 0x1p-4f);
            const float2 c = make_float2(__uint_as_float(and_or(codes[i], 15u << (8 * e), 0x4B000000u)),
                                         __uint_as_float(and_or(codes[i], 15u << (8 * e + 4), 0x4B000000u)));
            y[e] = fma2(scale, fma2(c, n, make_float2(-8388608.0f * n.x, -8388608.0f * n.y)), low);
        }
        float *row = dst + i * step;
        if (vec) {
            *reinterpret_cast<float4 *>(row) = make_float4(y[0].x, y[0].y, y[1].x, y[1].y);
        } else {
            const int64_t st = a.ys[which][3];
            row[0] = y[0].x, row[st] = y[0].y, row[2 * st] = y[1].x, row[3 * st] = y[1].y;
        }
    }
    // Tokens past the table have no place; a length out of range is told whether or not they are read. (One
    // thread of a sequence looks, at the end: there it takes 0.2 us of the kernel's 22, before the loads 0.5 to 1.5.)
    if ((blockIdx.x | blockIdx.y | threadIdx.x) == 0) {
        const int64_t n = a.lens[b * a.lens_stride];
        if (n < 0 || n > a.P * a.c.page_size) atomicExch(a.err, BAD_TABLE);
    }
}

// --------------------------------------------------------------------------- attention ----

// d = a b + c. (d may be c.)
__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, const float (&c)[4]) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}
__device__ __forceinline__ void mma_bf16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_u8s8(int (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, const int (&c)[4]) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
                 : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "r"(c[0]), "r"(c[1]), "r"(c[2]), "r"(c[3]));
}
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// (a, b) rounded to bfloat16, a in the low half.
__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
    return r;
}
// The four pairs of codes of y, less 8, as fp16: pairs 0 and 2 as they are, 1 and 3 times 16 (their
// bits lie four higher in the mantissa, which saves a shift; q is divided by 16 there).
__device__ __forceinline__ void codes_f16(uint32_t y, uint32_t (&c)[4]) {
    const uint32_t z = y >> 8;
    const uint32_t w[4] = {and_or(y, 0x000F000Fu, 0x64006400u), and_or(y, 0x00F000F0u, 0x64006400u),  // 1024 + code, 1024 + 16 code
                           and_or(z, 0x000F000Fu, 0x64006400u), and_or(z, 0x00F000F0u, 0x64006400u)};
#pragma unroll
    for (int i = 0; i < 4; i++) asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(c[i]) : "r"(w[i]), "r"((i & 1) ? 0x64806480u : 0x64086408u));
}
// Pair i of codes, less 8, as bfloat16.
__device__ __forceinline__ uint32_t codes_bf16(uint32_t y, int i) {
    const uint32_t z = and_or(y >> (4 * i), 0x000F000Fu, 0x43004300u);  // 128 + code
    uint32_t r;
    asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(z), "r"(0x43084308u));
    return r;
}

// N words from shared memory, on a boundary of their size (at most 16 bytes at a time).
template <int N>
__device__ __forceinline__ void read_words(const uint8_t *p, uint32_t *w) {
    if constexpr (N == 1) {
        w[0] = *reinterpret_cast<const uint32_t *>(p);
    } else if constexpr (N == 2) {
        const uint2 x = *reinterpret_cast<const uint2 *>(p);
        w[0] = x.x, w[1] = x.y;
    } else {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const uint4 x = *reinterpret_cast<const uint4 *>(p + 4 * i);
            w[i] = x.x, w[i + 1] = x.y, w[i + 2] = x.z, w[i + 3] = x.w;
        }
    }
}

// A contiguous copy from global to shared memory, completing on the mbarrier (16-byte multiples).
__device__ __forceinline__ void bulk_copy(uint32_t dst, const void *src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src),
                 "r"(bytes), "r"(bar)
                 : "memory");
}

// HEADS query heads of one key/value head per CTA: 1, 4 or 8.
//   4, 8  head t (and t + 4) of a lane; a group's product is a head's two parts per column pair, and the
//         lane applies every group's scales for its heads;
//   1     the column pairs are the groups instead: lane t gets group t's dots and applies that group's
//         scales alone, keys and values, and the groups are added up by two shuffles. (With the
//         columns left to absent heads a block of 16 keys took 722 instructions.)
template <int D, int PARTS, int HEADS>
struct AttnCfg {
    static constexpr int NG = D / GROUP;
    static constexpr bool ONE = HEADS == 1;
    static constexpr int NT = ONE ? 1 : HEADS / 4;              // heads of a lane
    static constexpr int NS = ONE ? (NG + 3) / 4 : NG;          // groups of a lane
    // The values' product: channels x keys times keys x columns, a column being a part of a head's weights.
    // A lane's columns 2 t, 2 t + 1 of tile n are its own heads': parts 0, 1 of head 4 n + t (two parts), or
    // parts 2 n, 2 n + 1 of head t (three); of one head simply parts 0, 1, ...
    static constexpr int COLS = ONE ? 8 : (PARTS == 2 ? 2 * HEADS : 16), NC = COLS / 8;
    static_assert(ONE || PARTS == 2 || HEADS == 4, "three parts: four heads");
    __host__ __device__ static constexpr int column(int head, int part) {
        return ONE ? part : (PARTS == 2 ? head / 4 * 8 + head % 4 * 2 + part : part / 2 * 8 + head * 2 + part % 2);
    }
    // A group's tile of weights: COLS rows of 16 keys in bfloat16, padded against bank conflicts.
    static constexpr int W_GROUP = COLS * 32 + 32;
    // Blocks a warp takes at a time (their chains overlap, and waiting, masks and maxima are paid once), and
    // how many such sets its ring holds.
    static constexpr int KB = D == 256 ? 1 : 2, STAGES = D == 64 ? 3 : 2;
    // Shared memory: the warps' rings | q fragments | the warps' weight tiles; after the loop the
    // accumulators.
    static constexpr int BLOCK = block_bytes(D), STAGE = KB * BLOCK, RING = STAGES * STAGE;
    static constexpr int Q_BYTES = NT * NG * 32 * 16, W_BYTES = KB * NG * W_GROUP;
    static constexpr int OFF_Q = WARPS * RING, OFF_W = OFF_Q + Q_BYTES, LOOP_BYTES = OFF_W + WARPS * W_BYTES;
    static constexpr int ACC_COLS = ONE ? PARTS : COLS, ACC_BYTES = WARPS * ACC_COLS * D * 4;
    static constexpr int SMEM = LOOP_BYTES > ACC_BYTES ? LOOP_BYTES : ACC_BYTES;
};

__device__ __forceinline__ float load_q(const Cache4Args &a, int64_t at) {
    if (a.dtype == DC_F32) return static_cast<const float *>(a.x[0])[at];
    if (a.dtype == DC_F16) return __half2float(static_cast<const __half *>(a.x[0])[at]);
    return __bfloat162float(static_cast<const __nv_bfloat16 *>(a.x[0])[at]);
}

template <int D, int PARTS, int HEADS>
__global__ void __launch_bounds__(WARPS * 32, D == 256 ? 2 : (HEADS == 8 ? 3 : 4))
    cache4_attention_kernel(const Cache4Args a, const SplitRows rows) {
    using C = AttnCfg<D, PARTS, HEADS>;
    constexpr int NG = C::NG, NT = C::NT, NS = C::NS, KB = C::KB;
    constexpr bool ONE = C::ONE;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ uint64_t s_full[WARPS][C::STAGES];
    __shared__ int s_abort;
    __shared__ int s_digits[NG][4];  // one head: the sums of each group's digits
    __shared__ float s_qsum[HEADS][NG], s_exp[HEADS], s_m[WARPS][HEADS], s_l[WARPS][HEADS], s_low[WARPS][HEADS][NG];
    griddep_launch_dependents();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, t = lane & 3;
    const int group = (int)(a.H / a.c.Hkv), chunks = (group + HEADS - 1) / HEADS;
    const int64_t b = blockIdx.z;
    const int hk = blockIdx.y / chunks;
    const int64_t h0 = (int64_t)hk * group + (blockIdx.y % chunks) * HEADS;
    const int nh = min(HEADS, group - (int)(blockIdx.y % chunks) * HEADS);

    // The sequence's visible keys: [0, sinks) and [lo, len), in blocks of 16.
    const int64_t capacity = a.P * a.c.page_size;
    int64_t len64 = a.lens[b * a.lens_stride];
    if (len64 < 0 || len64 > capacity) {
        if (threadIdx.x == 0) atomicExch(a.err, BAD_TABLE);
        len64 = len64 < 0 ? 0 : capacity;
    }
    const int len = (int)len64;
    const int lo = a.window ? (int)max((int64_t)0, len64 - a.window) : 0, sinks = (int)min(a.sinks, (int64_t)lo);
    const int first = lo / 16, sink_blocks = min((sinks + 15) / 16, first);
    const int total = len == 0 ? 0 : sink_blocks + (len + 15) / 16 - first;
    const int per = (total + rows.splits - 1) / rows.splits, v0 = blockIdx.x * per, v1 = min(total, v0 + per);
    const uint32_t page16 = (uint32_t)a.c.page_size / 16;
    auto block_of = [&](int v) { return v < sink_blocks ? v : first + v - sink_blocks; };
    // The warp's sets of KB blocks: from v0 + warp * KB on, every WARPS-th. The pool's block numbers of its
    // next 32 blocks, one to a lane, and of the 32 after those: the division by the page size and the
    // table's latency are paid once in 32 blocks. BAD: the table's entry is out of range; ABSENT: no block.
    constexpr int BAD = -1, ABSENT = -2;
    const int32_t *table = a.table + b * a.ts[0];
    auto numbers = [&](int set) -> int {  // of the 32 / KB sets from number `set` on
        const int v = v0 + (warp + (set + lane / KB) * WARPS) * KB + lane % KB;
        if (v >= v1) return ABSENT;
        const uint32_t at = (uint32_t)block_of(v), entry = at / page16;
        const int id = table[entry * a.ts[1]];
        return (uint32_t)id < (uint32_t)a.c.pages ? (int)(((uint32_t)id * (uint32_t)a.c.Hkv + hk) * page16 + (at - entry * page16)) : BAD;
    };
    // This warp's ring. A block whose page id is out of range is not copied: its keys are left out
    // (stage_ok: KB bits a stage).
    const uint32_t ring = (uint32_t)__cvta_generic_to_shared(smem) + warp * C::RING;
    const uint32_t full = (uint32_t)__cvta_generic_to_shared(&s_full[warp][0]);
    volatile int *abort = &s_abort;
    uint32_t stage_ok = 0;
    int v = v0 + warp * KB, fetched = 0;
    int numbers_now = numbers(0), numbers_next = numbers(32 / KB);
    auto fetch = [&](int stage) {  // the warp's set number `fetched`
        int number[KB], there = 0;
#pragma unroll
        for (int e = 0; e < KB; e++) {
            number[e] = __shfl_sync(ALL, numbers_now, (fetched * KB + e) & 31);
            there += number[e] >= 0;
            const int bit = stage * KB + e;
            stage_ok = (stage_ok & ~(1u << bit)) | ((uint32_t)(number[e] >= 0) << bit);
        }
        if ((++fetched * KB & 31) == 0) {
            numbers_now = numbers_next;
            numbers_next = numbers(fetched + 32 / KB);
        }
        if (lane == 0) {
            if (there) sm100::mbar_expect_tx(full + 8 * stage, there * C::BLOCK);
            else sm100::mbar_arrive(full + 8 * stage);
#pragma unroll
            for (int e = 0; e < KB; e++) {
                if (number[e] >= 0)
                    bulk_copy(ring + stage * C::STAGE + e * C::BLOCK, a.c.data + (int64_t)number[e] * C::BLOCK, C::BLOCK, full + 8 * stage);
                else if (number[e] == BAD)
                    atomicExch(a.err, BAD_TABLE);
            }
        }
    };
    if (lane == 0) {
        for (int i = 0; i < C::STAGES; i++) sm100::mbar_init(full + 8 * i, 1);
        sm100::fence_mbar_init();
    }
    if (threadIdx.x == 0) s_abort = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < C::STAGES; i++)
        if (v + i * WARPS * KB < v1) fetch(i);

    // q: per head a power of two that brings its largest channel below 1, the sums of its groups,
    // and the two fp16 parts in the order of the products' B fragments.
    if constexpr (ONE) {  // the other groups' columns of a group's fragment are zero
        for (int i = threadIdx.x; i < C::Q_BYTES / 16; i += WARPS * 32) reinterpret_cast<uint4 *>(smem + C::OFF_Q)[i] = make_uint4(0, 0, 0, 0);
        __syncthreads();
    }
    for (int h = warp; h < HEADS; h += WARPS) {
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
        bool finite = true;
#pragma unroll
        for (int g = 0; g < NG; g++) {
            float s = x[g];
            finite = finite && fabsf(s) <= 3.402823466e38f;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(ALL, s, o);
            if (lane == 0) s_qsum[h][g] = s * (a.scale * LOG2E);
            if constexpr (ONE) {
                // Channel 32 g + lane = 8 t' + 2 j + high: byte j of lane t', low or high nibbles.
                int y = __float2int_rn(ldexpf(x[g], 27 - e));
#pragma unroll
                for (int digit = 0; digit < 4; digit++) {  // lowest first
                    const int d = digit == 3 ? y : ((y + 64) & 127) - 64;
                    y = (y - d) >> 7;
                    // columns 2 (g & 3), + 1: of the high pair (digits 3, 2) or the low pair (1, 0)
                    const int col = (g & 3) * 2 + 1 - (digit & 1), pair = digit >= 2 ? 0 : 1;
                    int8_t *frag = reinterpret_cast<int8_t *>(smem + C::OFF_Q + (g * 32 + col * 4 + (lane >> 3)) * 16);
                    frag[pair * 8 + (lane & 1) * 4 + ((lane >> 1) & 3)] = (int8_t)d;
                    const int sum = __reduce_add_sync(ALL, d);
                    if (lane == 0) s_digits[g][3 - digit] = sum;
                }
            } else {
                // Channel 32 g + lane = 4 r' + i of a group: k-pair member r' & 1 of lane t' = r' / 2, pair i.
                const int rr = lane >> 2, i = lane & 3;
                const float y = ldexpf(x[g], (i & 1) ? 10 - e : 14 - e);  // far above the subnormals, low part too
                const __half hi = __float2half_rn(y), lo16 = __float2half_rn(y - __half2float(hi));
#pragma unroll
                for (int part = 0; part < 2; part++) {
                    const int col = (h & 3) * 2 + part;
                    __half *frag = reinterpret_cast<__half *>(smem + C::OFF_Q + (((h >> 2) * NG + g) * 32 + col * 4 + (rr >> 1)) * 16);
                    frag[i * 2 + (rr & 1)] = part ? lo16 : hi;
                }
            }
        }
        // (An infinity or a NaN does not survive the digits: it goes into the factor.)
        finite = __all_sync(ALL, finite);
        if (lane == 0) s_exp[h] = finite ? ldexpf(a.scale * LOG2E, ONE ? e - 27 : e - 14) : NAN;
    }
    __syncthreads();

    // Heads n * 4 + t (one head: head 0), groups g (one head: t + 4 g) of this lane.
    // m: the running maximum; base: what the weights are relative to (m, or 0 before there is one).
    float mul[NT], qsum[NT][NS], m[NT], base[NT], l[NT], low[NT][NS];
    float acc[2 * NG][C::NC][4];  // channels 32 g + 4 r + 2 j (and + 1) of tile 2 g + j
#pragma unroll
    for (int n = 0; n < NT; n++) {
        mul[n] = s_exp[ONE ? 0 : n * 4 + t];
        m[n] = -INFINITY;
        base[n] = l[n] = 0.0f;
#pragma unroll
        for (int g = 0; g < NS; g++) {
            const int own = ONE ? t + 4 * g : g;
            qsum[n][g] = own < NG ? s_qsum[ONE ? 0 : n * 4 + t][own] : 0.0f;
            low[n][g] = 0.0f;
        }
    }
    // One head: -8 times the sums of digits 3, 2 (and 1, 0), which turns codes into code - 8.
    int centre_hi[ONE ? NS : 1][4], centre_lo[ONE ? NS : 1][4];
    if constexpr (ONE) {
#pragma unroll
        for (int g = 0; g < NS; g++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                centre_hi[g][i] = t + 4 * g < NG ? -8 * s_digits[t + 4 * g][i & 1] : 0;
                centre_lo[g][i] = t + 4 * g < NG ? -8 * s_digits[t + 4 * g][2 + (i & 1)] : 0;
            }
    }
#pragma unroll
    for (int i = 0; i < 2 * NG; i++)
#pragma unroll
        for (int n = 0; n < C::NC; n++)
#pragma unroll
            for (int c = 0; c < 4; c++) acc[i][n][c] = 0.0f;
    // The warp's weight tiles. Keys r and r + 8 (slots 2 r, 2 r + 1 of the product) are stored at place
    // r % 4, half r / 4, so that a lane's four slots 2 t, 2 t + 1, 2 t + 8, 2 t + 9 are eight bytes.
    uint8_t *wt = smem + C::OFF_W + warp * C::W_BYTES;
    const uint32_t wt_put = (r & 3) * 8 + (r >> 2) * 4, wt_get = r * 32 + t * 8;

    // This lane's places in a block: codes of keys r and r + 8 (its quarter of each group), of values
    // (t, t + 8) and (t + 4, t + 12) (its eighth of each group), and of both the scales of places r and
    // r + 8.
    const uint8_t *blk = smem + warp * C::RING;
    const uint32_t koff = r * (D / 2) + t * 4 * NG, voff = 10 * D + lane * 4 * NG;
    const uint32_t soff = 8 * D + (r * NG + (ONE ? (NG < 4 ? t % NG : t) : 0)) * 4;
    int stage = 0;
    uint32_t parity = 0;
    for (; v < v1; v += WARPS * KB) {
        if (!sm100::mbar_wait_warp(full + 8 * stage, parity, abort, a.err)) break;
        const uint8_t *cur = blk + stage * C::STAGE;
        // Which of keys r and r + 8 of each block are seen; all of them in most sets.
        bool ok0[KB], ok1[KB], edge = false;
#pragma unroll
        for (int e = 0; e < KB; e++) {
            const int k0 = block_of(v + e) * 16;
            ok0[e] = ok1[e] = true;
            edge = edge || !((stage_ok >> (stage * KB + e)) & 1u) || k0 + 16 > len || (k0 < lo && k0 + 16 > sinks);
        }
        if (edge) {
#pragma unroll
            for (int e = 0; e < KB; e++) {
                const bool there = (stage_ok >> (stage * KB + e)) & 1u;
                const int j0 = block_of(v + e) * 16 + r, j1 = j0 + 8;
                ok0[e] = there && j0 < len && (j0 >= lo || j0 < sinks);
                ok1[e] = there && j1 < len && (j1 >= lo || j1 < sinks);
            }
        }
        // Scores of keys r and r + 8.
        float s0[KB][NT], s1[KB][NT];
#pragma unroll
        for (int e = 0; e < KB; e++) {
            const uint8_t *at = cur + e * C::BLOCK;
            uint32_t kc[2][NG], ks[2][NS];
#pragma unroll
            for (int i = 0; i < 2; i++) {
                read_words<NG>(at + koff + 8 * i * (D / 2), kc[i]);
                if constexpr (ONE) {
#pragma unroll
                    for (int j = 0; j < NS; j++) read_words<1>(at + soff + 8 * i * NG * 4 + 16 * j, &ks[i][j]);
                } else {
                    read_words<NG>(at + soff + 8 * i * NG * 4, ks[i]);
                }
            }
            if constexpr (ONE) {
                int hi[NS][4], lw[NS][4];  // digits 3, 2 and 1, 0 of keys r, r + 8
#pragma unroll
                for (int g = 0; g < NG; g++) {
                    const uint32_t y[4] = {kc[0][g] & 0x0F0F0F0Fu, kc[1][g] & 0x0F0F0F0Fu, (kc[0][g] >> 4) & 0x0F0F0F0Fu,
                                           (kc[1][g] >> 4) & 0x0F0F0F0Fu};
                    const uint4 q = *reinterpret_cast<const uint4 *>(smem + C::OFF_Q + (g * 32 + lane) * 16);
                    mma_u8s8(hi[g / 4], y, q.x, q.y, g % 4 ? hi[g / 4] : centre_hi[g / 4]);
                    mma_u8s8(lw[g / 4], y, q.z, q.w, g % 4 ? lw[g / 4] : centre_lo[g / 4]);
                }
                float x0 = 0.0f, x1 = 0.0f;
#pragma unroll
                for (int i = 0; i < NS; i++) {
                    // Each pair of digits is below 2^23: exact in 32 bits, their sum rounded once.
                    const float d0 = fmaf((float)(hi[i][0] * 128 + hi[i][1]), 16384.0f, (float)(lw[i][0] * 128 + lw[i][1]));
                    const float d1 = fmaf((float)(hi[i][2] * 128 + hi[i][3]), 16384.0f, (float)(lw[i][2] * 128 + lw[i][3]));
                    x0 = fmaf(bf16_low(ks[0][i]) * mul[0], d0, fmaf(mid(ks[0][i]), qsum[0][i], x0));
                    x1 = fmaf(bf16_low(ks[1][i]) * mul[0], d1, fmaf(mid(ks[1][i]), qsum[0][i], x1));
                }
                if (NG < 4 && t >= NG) x0 = x1 = 0.0f;  // head dim 64: two groups for four lanes
#pragma unroll
                for (int o = 1; o < 4; o <<= 1) {
                    x0 += __shfl_xor_sync(ALL, x0, o);
                    x1 += __shfl_xor_sync(ALL, x1, o);
                }
                s0[e][0] = x0;
                s1[e][0] = x1;
            } else {
                float b0[NT], b1[NT];
#pragma unroll
                for (int n = 0; n < NT; n++) s0[e][n] = s1[e][n] = b0[n] = b1[n] = 0.0f;
#pragma unroll
                for (int g = 0; g < NG; g++) {
                    uint32_t y0[4], y1[4];
                    codes_f16(kc[0][g], y0);
                    codes_f16(kc[1][g], y1);
                    const uint32_t a0[4] = {y0[0], y1[0], y0[1], y1[1]}, a1[4] = {y0[2], y1[2], y0[3], y1[3]};
                    const float sc0 = bf16_low(ks[0][g]), sc1 = bf16_low(ks[1][g]), mid0 = mid(ks[0][g]), mid1 = mid(ks[1][g]);
#pragma unroll
                    for (int n = 0; n < NT; n++) {
                        const uint4 q = *reinterpret_cast<const uint4 *>(smem + C::OFF_Q + ((n * NG + g) * 32 + lane) * 16);
                        const float zero[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                        float c[4];
                        mma_f16(c, a0, q.x, q.y, zero);
                        mma_f16(c, a1, q.z, q.w, c);
                        s0[e][n] = fmaf(sc0, c[0] + c[1], s0[e][n]);
                        s1[e][n] = fmaf(sc1, c[2] + c[3], s1[e][n]);
                        b0[n] = fmaf(mid0, qsum[n][g], b0[n]);
                        b1[n] = fmaf(mid1, qsum[n][g], b1[n]);
                    }
                }
#pragma unroll
                for (int n = 0; n < NT; n++) {
                    s0[e][n] = fmaf(s0[e][n], mul[n], b0[n]);
                    s1[e][n] = fmaf(s1[e][n], mul[n], b1[n]);
                }
            }
        }
        if (edge) {
#pragma unroll
            for (int e = 0; e < KB; e++)
#pragma unroll
                for (int n = 0; n < NT; n++) {
                    s0[e][n] = ok0[e] ? s0[e][n] : -INFINITY;
                    s1[e][n] = ok1[e] ? s1[e][n] : -INFINITY;
                }
        }
        float corr[NT];
        bool moved = false;
#pragma unroll
        for (int n = 0; n < NT; n++) {
            float top = fmaxf(s0[0][n], s1[0][n]);
            if (KB == 2) top = fmaxf(top, fmaxf(s0[KB - 1][n], s1[KB - 1][n]));
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) top = fmaxf(top, __shfl_xor_sync(ALL, top, o));
            corr[n] = 1.0f;
            if (top > m[n] + 8.0f || (m[n] == -INFINITY && top > m[n])) {
                corr[n] = exp2_fast(m[n] - top);
                m[n] = base[n] = top;
                moved = true;
            }
        }
        if (__any_sync(ALL, moved)) {
#pragma unroll
            for (int n = 0; n < NT; n++) {
                l[n] *= corr[n];
#pragma unroll
                for (int g = 0; g < NS; g++) low[n][g] *= corr[n];
            }
            // (A lane's columns are its own heads'.)
#pragma unroll
            for (int i = 0; i < 2 * NG; i++)
#pragma unroll
                for (int n = 0; n < C::NC; n++)
#pragma unroll
                    for (int c = 0; c < 4; c++) acc[i][n][c] *= corr[NT == 2 ? n : 0];
        }
        // Weights times the values' scales, in bfloat16 parts, to the warp's tiles.
        __syncwarp();
#pragma unroll
        for (int e = 0; e < KB; e++) {
            uint32_t vs[2][NS];
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const uint8_t *at = cur + e * C::BLOCK + 10 * D + soff + 8 * i * NG * 4;
                if constexpr (ONE) {
#pragma unroll
                    for (int j = 0; j < NS; j++) read_words<1>(at + 16 * j, &vs[i][j]);
                } else {
                    read_words<NG>(at, vs[i]);
                }
            }
            if (edge) {  // a place behind the sequence's end may hold anything
#pragma unroll
                for (int g = 0; g < NS; g++) {
                    if (!ok0[e]) vs[0][g] = 0u;
                    if (!ok1[e]) vs[1][g] = 0u;
                }
            }
#pragma unroll
            for (int n = 0; n < NT; n++) {
                const float p0 = exp2_fast(s0[e][n] - base[n]), p1 = exp2_fast(s1[e][n] - base[n]);
                l[n] += p0 + p1;
#pragma unroll
                for (int g = 0; g < NS; g++) {
                    const uint32_t z0 = vs[0][g], z1 = vs[1][g];
                    low[n][g] = fmaf(p0, mid(z0), fmaf(p1, mid(z1), low[n][g]));
                    float w0 = p0 * bf16_low(z0), w1 = p1 * bf16_low(z1);
                    const int own = ONE ? t + 4 * g : g;
                    if (own < NG) {
#pragma unroll
                        for (int part = 0; part < PARTS; part++) {
                            const uint32_t w = pack_bf16(w0, w1);
                            *reinterpret_cast<uint32_t *>(wt + (e * NG + own) * C::W_GROUP + C::column(ONE ? 0 : n * 4 + t, part) * 32 + wt_put) = w;
                            w0 -= bf16_low(w);
                            w1 -= bf16_high(w);
                        }
                    }
                }
            }
        }
        __syncwarp();
#pragma unroll
        for (int e = 0; e < KB; e++) {
            uint32_t vc[2][NG];
#pragma unroll
            for (int i = 0; i < 2; i++) read_words<NG>(cur + e * C::BLOCK + voff + i * 32 * 4 * NG, vc[i]);
            if (e == KB - 1) {
                // Every lane holds its part of the blocks: the stage takes the set STAGES further on.
                __syncwarp();
                if (v + C::STAGES * WARPS * KB < v1) fetch(stage);
                if (++stage == C::STAGES) stage = 0, parity ^= 1u;
            }
#pragma unroll
            for (int g = 0; g < NG; g++) {
                // (Columns without a part are read as they come: what they give is never looked at.)
                uint2 w[C::NC];
#pragma unroll
                for (int n = 0; n < C::NC; n++) w[n] = *reinterpret_cast<const uint2 *>(wt + (e * NG + g) * C::W_GROUP + n * 256 + wt_get);
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    const uint32_t y[4] = {codes_bf16(vc[0][g], 2 * j), codes_bf16(vc[0][g], 2 * j + 1), codes_bf16(vc[1][g], 2 * j),
                                           codes_bf16(vc[1][g], 2 * j + 1)};
#pragma unroll
                    for (int n = 0; n < C::NC; n++) mma_bf16(acc[2 * g + j][n], y, w[n].x, w[n].y);
                }
            }
        }
    }
    if (v < v1) {
        // A wait ran out: let this warp's copies land before the block's memory goes away. (fetch at v
        // has refilled the stages of the blocks before v: those of v .. v + STAGES - 1 may be in flight.)
        volatile int never = 0;
        for (int i = 0; i < C::STAGES && v + i * WARPS * KB < v1; i++) {
            sm100::mbar_wait_warp(full + 8 * stage, parity, &never, nullptr);
            if (++stage == C::STAGES) stage = 0, parity ^= 1u;
        }
    }

    // Join the warps.
#pragma unroll
    for (int n = 0; n < NT; n++) {
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) {
            l[n] += __shfl_xor_sync(ALL, l[n], o);
#pragma unroll
            for (int g = 0; g < NS; g++) low[n][g] += __shfl_xor_sync(ALL, low[n][g], o);
        }
        if (r == 0) {
            const int h = ONE ? 0 : n * 4 + t;
            s_m[warp][h] = m[n];
            s_l[warp][h] = l[n];
#pragma unroll
            for (int g = 0; g < NS; g++) {
                const int own = ONE ? t + 4 * g : g;
                if (own < NG) s_low[warp][h][own] = low[n][g];
            }
        }
    }
    __syncthreads();
    if (*abort) return;  // the row is left unwritten; the device status tells
    float *sacc = reinterpret_cast<float *>(smem) + warp * C::ACC_COLS * D;
#pragma unroll
    for (int i = 0; i < 2 * NG; i++)
#pragma unroll
        for (int n = 0; n < C::NC; n++)
#pragma unroll
            for (int c = 0; c < 4; c++) {
                const int col = n * 8 + 2 * t + (c & 1), ch = (i / 2) * 32 + 4 * r + 2 * (i & 1) + (c >> 1);
                if (col < C::ACC_COLS) sacc[col * D + ch] = acc[i][n][c];
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
                x += reinterpret_cast<const float *>(smem)[(w * C::ACC_COLS + C::column(h, part)) * D + d];
            sum = fmaf(s_l[w][h], f, sum);
            o = fmaf(x, f, o);
        }
        split_store(rows, b * a.H + h0 + h, blockIdx.x, d, top, sum, o);
    }
}

template <int D, int PARTS, int HEADS>
int launch_attention(const Cache4Args &a, const SplitRows &rows, cudaStream_t stream) {
    using C = AttnCfg<D, PARTS, HEADS>;
    auto kernel = cache4_attention_kernel<D, PARTS, HEADS>;
    if (C::SMEM > 40 * 1024) {  // with the static arrays, past the 48 KB that need no attribute
        cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
        if (e != cudaSuccess) return cuda_fail(e, "cache4_attention smem attribute");
    }
    const int64_t group = a.H / a.c.Hkv, chunks = (group + HEADS - 1) / HEADS;
    KernelTrace tr("cache4_attention", stream);
    kernel<<<dim3((unsigned)rows.splits, (unsigned)(a.c.Hkv * chunks), (unsigned)a.B), WARPS * 32, C::SMEM, stream>>>(a, rows);
    return check_launch("cache4_attention");
}

// Heads of one key/value head that a CTA takes: a single one has its own kernel; otherwise 4, or 8 where
// the weights take two parts (16-bit queries: two tiles of columns, as three parts of four heads).
int heads_per_cta(int64_t group, int dtype) {
    return group == 1 ? 1 : (dtype != DC_F32 && group > 4 ? 8 : 4);
}

template <int D>
int launch_dim(const Cache4Args &a, const SplitRows &rows, cudaStream_t stream) {
    const int heads = heads_per_cta(a.H / a.c.Hkv, a.dtype);
    if (a.dtype == DC_F32) return heads == 1 ? launch_attention<D, 3, 1>(a, rows, stream) : launch_attention<D, 3, 4>(a, rows, stream);
    if (heads == 1) return launch_attention<D, 2, 1>(a, rows, stream);
    return heads == 8 ? launch_attention<D, 2, 8>(a, rows, stream) : launch_attention<D, 2, 4>(a, rows, stream);
}

// Whether the rows of a (B, H, T, D) view start on 16-byte boundaries.
bool rows16(const void *ptr, const int64_t *st, int size) {
    return st[3] == 1 && st[0] * size % 16 == 0 && st[1] * size % 16 == 0 && st[2] * size % 16 == 0 && (reinterpret_cast<uintptr_t>(ptr) & 15u) == 0;
}

}  // namespace

// Grid of the fill and read kernels, whose blocks take `run` tokens of a row of keys or values.
dim3 token_grid(const Cache4Args &a, int64_t run) { return dim3((unsigned)((a.T + run - 1) / run), (unsigned)(2 * a.c.Hkv), (unsigned)a.B); }

int cache4_append(const Cache4Args &a, cudaStream_t stream) {
    const int size = a.dtype == DC_F32 ? 4 : 2;
    const bool vec = rows16(a.x[0], a.xs[0], size) && rows16(a.x[1], a.xs[1], size);
    const dim3 grid = token_grid(a, FILL_WARPS * 32 / (a.c.D / 8) * APPEND_ROWS);
    KernelTrace tr("cache4_append", stream);
    if (a.dtype == DC_F32) cache4_append_kernel<float><<<grid, FILL_WARPS * 32, 0, stream>>>(a, vec);
    else if (a.dtype == DC_F16) cache4_append_kernel<__half><<<grid, FILL_WARPS * 32, 0, stream>>>(a, vec);
    else cache4_append_kernel<__nv_bfloat16><<<grid, FILL_WARPS * 32, 0, stream>>>(a, vec);
    return check_launch("cache4_append");
}

int cache4_read(const Cache4Args &a, cudaStream_t stream) {
    const bool vec = rows16(a.y[0], a.ys[0], 4) && rows16(a.y[1], a.ys[1], 4);
    KernelTrace tr("cache4_read", stream);
    cache4_read_kernel<<<token_grid(a, 256 / (a.c.D / 4) * READ_ROWS), 256, 0, stream>>>(a, vec);
    return check_launch("cache4_read");
}

// Splits of each row: enough CTAs to fill every SM's four places six times over, so that sequences of
// different lengths even out, with at least 8 blocks a warp then; below that, down to one set of two
// blocks a warp, as many as fill the places once.
int cache4_splits(int64_t B, int64_t H, int64_t Hkv, int64_t capacity, int64_t window, int64_t sinks, int dtype) {
    const int64_t group = H / Hkv, per = heads_per_cta(group, dtype), chunks = (group + per - 1) / per;
    const int64_t ctas = std::max<int64_t>(1, B * Hkv * chunks);
    const int64_t keys = window ? std::min(capacity, std::min(window, capacity) + std::min(sinks, capacity)) : capacity;
    const int64_t places = (int64_t)device_sm_count() * 4, most = (keys + 32 * WARPS - 1) / (32 * WARPS);
    const int64_t once = std::min(places / ctas, most), even = std::min((6 * places + ctas - 1) / ctas, most / 4);
    return (int)std::max<int64_t>(1, std::min<int64_t>(128, std::max(once, even)));
}

int cache4_attention(const Cache4Args &a, const SplitRows &rows, cudaStream_t stream) {
    int st;
    if (a.c.D == 64) st = launch_dim<64>(a, rows, stream);
    else if (a.c.D == 128) st = launch_dim<128>(a, rows, stream);
    else st = launch_dim<256>(a, rows, stream);
    return st ? st : split_combine(rows, stream);
}

}  // namespace dc
