// rotary.cu -- rotary positions of queries and keys, alone or behind a norm of each head.
//
// No counterpart in DenseCore (its nanoGPT path adds learned positions to the embeddings); these
// stand in front of its attention call (python/densecore/functional.py:276). With x one head's row
// of D channels at position t, f_i the frequencies and A the amplitude:
//
//   rotation   (a, b) -> (a cos - b sin, b cos + a sin) A, angle t f_i, for the pairs of the first
//              `rot` channels: (x_i, x_{i + rot/2}) or, interleaved, (x_2i, x_2i+1); the other
//              channels pass through
//   norm       n = x r, r = 1 / sqrt(mean(x^2) + eps), y = R(n w) over the whole head
//   backward   u = R^T g (the rotation by -angle); gw = sum over rows of u n; gn = u w;
//              gx = r (gn - n mean(gn n)), with r recomputed from x
//
// Bound: HBM. Each element is read once and written once (the backward of the norm reads x and g),
// and some seven instructions an element are below what the loads allow, as long as the angles cost
// little beside them:
//   * a row is held by D / 8 lanes, two pieces of four channels each: a lane owns both members of its
//     four pairs, so the rotation needs no exchange and the norm one butterfly over the row's lanes.
//     (Pieces of 16 bytes in the 16-bit types, eight channels, cost twice the registers and spilled:
//     the norm of 40 heads of 8188 tokens took 101 us against the 26 of its bytes.)
//   * a warp takes one token and a run of its heads, queries then keys. The run's sines and cosines
//     are computed once, two or four to a lane, and handed out through shared memory. The angle is
//     reduced to a fraction of a turn in 64 bits (position 10^6 in 32 bits would already be 0.06 rad
//     off), its sine and cosine taken in 32. No table: nothing bounds the positions, and nothing
//     else is read;
//   * runs are cut short (down to one row a lane group) when a call has too few tokens to fill the
//     GPU, as in a decode step;
//   * the weight gradients are summed in fixed order: per lane over its rows, then over the warps
//     of a block, then over the blocks by a second kernel. No atomics.
// Sums, angles and products are held in 32 bits (or 64), and each output is rounded once.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "common.cuh"
#include "kernels.h"
#include "trace.h"

namespace dc {
namespace {

constexpr int WPB = 8;  // warps per block
constexpr unsigned ALL = 0xffffffffu;
constexpr int MAX_BWD_BLOCKS = 296;  // blocks of the norm's backward: 2 of 8 warps on each of 148 SMs
constexpr int MAX_PAIRS = 128;

constexpr int ROTATE = ROTARY_ROTATE, NORM = ROTARY_NORM, NORM_BWD = ROTARY_NORM_BWD;

template <typename T>
__device__ __forceinline__ T from_f(float x);
template <>
__device__ __forceinline__ float from_f<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half from_f<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// One piece of a row, V elements as loaded: kept as words until they are used (as separate 16-bit
// elements they took a register each, and the loads in flight spilled).
template <typename T, int V>
struct Piece {
    static constexpr int WORDS = V == 1 ? 1 : V * (int)sizeof(T) / 4;
    uint32_t w[WORDS];

    // The piece at p, zeros where it is not `there`. (Predicated: as branches the loads of a row cost more
    // instructions than its arithmetic.)
    __device__ __forceinline__ void load(const T *p, bool there) {
        if constexpr (V == 1) {
            w[0] = 0u;
            if (there) {
                if constexpr (sizeof(T) == 4) w[0] = __float_as_uint(*p);
                else w[0] = *reinterpret_cast<const uint16_t *>(p);
            }
        } else if constexpr (WORDS == 4) {
            asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %5, 0;\n\tmov.b32 %0, 0;\n\tmov.b32 %1, 0;\n\tmov.b32 %2, 0;\n\tmov.b32 %3, 0;\n\t"
                         "@p ld.global.v4.b32 {%0, %1, %2, %3}, [%4];\n\t}"
                         : "=&r"(w[0]), "=&r"(w[1]), "=&r"(w[2]), "=&r"(w[3])
                         : "l"(p), "r"((int)there)
                         : "memory");
        } else {
            asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %3, 0;\n\tmov.b32 %0, 0;\n\tmov.b32 %1, 0;\n\t@p ld.global.v2.b32 {%0, %1}, [%2];\n\t}"
                         : "=&r"(w[0]), "=&r"(w[1])
                         : "l"(p), "r"((int)there)
                         : "memory");
        }
    }
    __device__ __forceinline__ float at(int i) const {
        if constexpr (sizeof(T) == 4) return __uint_as_float(w[i]);
        else if constexpr (std::is_same<T, __half>::value) return __half2float(__ushort_as_half((unsigned short)(w[i / 2] >> (16 * (i & 1)))));
        else return __uint_as_float((i & 1) ? (w[i / 2] & 0xFFFF0000u) : (w[i / 2] << 16));
    }
    // Values of a unit (this piece, then `next`) by twos.
    __device__ __forceinline__ float2 two(const Piece &next, int i) const {
        if constexpr (V == 1) return make_float2(at(0), next.at(0));
        const Piece &p = i < 2 ? *this : next;
        return make_float2(p.at(2 * (i & 1)), p.at(2 * (i & 1) + 1));
    }
};

template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    if constexpr (std::is_same<T, __half>::value) {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t *>(&h);
    } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
}

template <typename T>
__device__ __forceinline__ void store4(T *p, float2 a, float2 b, bool there) {
    if constexpr (sizeof(T) == 4)
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %5, 0;\n\t@p st.global.v4.f32 [%0], {%1, %2, %3, %4};\n\t}" ::"l"(p), "f"(a.x), "f"(a.y),
                     "f"(b.x), "f"(b.y), "r"((int)there)
                     : "memory");
    else
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %3, 0;\n\t@p st.global.v2.b32 [%0], {%1, %2};\n\t}" ::"l"(p), "r"(pack2<T>(a.x, a.y)),
                     "r"(pack2<T>(b.x, b.y)), "r"((int)there)
                     : "memory");
}

// The sum over a row's lanes (1 << k of them; unrolled and predicated, not a loop over k).
__device__ __forceinline__ float row_sum(float s, int lpr) {
#pragma unroll
    for (int m = 16; m > 0; m >>= 1) {
        const float other = __shfl_xor_sync(ALL, s, m);
        if (m < lpr) s += other;
    }
    return s;
}

// Two products (and sums) in one instruction, each rounded as alone.
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

__device__ __forceinline__ float weight_at(const RotaryOperand &o, int at) {
    if (!o.w) return 1.0f;
    const int64_t i = at * o.ws;
    if (o.w_dtype == DC_F32) return static_cast<const float *>(o.w)[i];
    if (o.w_dtype == DC_F16) return __half2float(static_cast<const __half *>(o.w)[i]);
    return __bfloat162float(static_cast<const __nv_bfloat16 *>(o.w)[i]);
}

// Rows in flight per lane group: their loads are issued together.
template <int MODE, int UPL>
constexpr int rows_ahead() {
    return UPL > 1 ? 1 : (MODE == NORM_BWD ? 2 : 4);
}

// UPL units (two pieces of V elements: V pairs, or 2 V channels that pass through) per lane; a row
// takes 1 << lpr_log lanes. An item is a token and a run of heads_per_item of its rows, the query
// heads first, then the keys'.
template <typename T, int V, int UPL, int MODE, bool INTER>
__global__ void __launch_bounds__(WPB * 32, MODE == NORM_BWD ? 2 : 3) rotary_kernel(const RotaryArgs a) {
    constexpr int R = rows_ahead<MODE, UPL>();
    constexpr int NW = MODE == ROTATE ? 1 : UPL, NG = MODE == NORM_BWD ? UPL : 1;
    __shared__ __align__(16) float s_cos[WPB][MAX_PAIRS], s_sin[WPB][MAX_PAIRS];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int lpr = 1 << a.lpr_log, sub = lane >> a.lpr_log, rpw = 32 >> a.lpr_log, ul = lane & (lpr - 1);
    const int nrot = INTER ? a.rot / (2 * V) : a.rot / 2 / V, nunit = a.D / (2 * V);

    // This lane's units: offsets of the two pieces.
    int e0[UPL], e1[UPL];
    bool has[UPL], turns[UPL];
#pragma unroll
    for (int u = 0; u < UPL; u++) {
        const int unit = ul + u * lpr;
        has[u] = unit < nunit;
        turns[u] = unit < nrot;
        if (INTER) {
            e0[u] = unit * 2 * V;
            e1[u] = e0[u] + V;
        } else if (turns[u]) {
            e0[u] = unit * V;
            e1[u] = a.rot / 2 + unit * V;
        } else {
            e0[u] = a.rot + (unit - nrot) * 2 * V;
            e1[u] = e0[u] + V;
        }
    }
    const bool all_turn = a.rot == a.D;  // no channel passes through
    float2 gw[2][NG][V];
    if constexpr (MODE == NORM_BWD) {
#pragma unroll
        for (int k = 0; k < 2; k++)
#pragma unroll
            for (int u = 0; u < UPL; u++)
#pragma unroll
                for (int i = 0; i < V; i++) gw[k][u][i] = make_float2(0.0f, 0.0f);
    }
    // The weights, in 32 bits, for every item of the block.
    __shared__ __align__(16) float s_w[2][MODE == ROTATE ? 4 : 2 * MAX_PAIRS];
    if constexpr (MODE != ROTATE) {
        for (int i = threadIdx.x; i < 2 * a.D; i += WPB * 32) {
            const int k = i >= a.D;
            s_w[k][i - k * a.D] = weight_at(a.op[k], i - k * a.D);
        }
        __syncthreads();
    }
    const int64_t items = a.B * a.L * a.chunks;
    for (int64_t item = (int64_t)blockIdx.x * WPB + warp; item < items; item += (int64_t)gridDim.x * WPB) {
        int64_t token, b;
        int chunk;
        if (items < (1ll << 31)) {  // 32-bit divisions
            const uint32_t t32 = (uint32_t)item / (uint32_t)a.chunks, b32 = t32 / (uint32_t)a.L;
            token = t32, b = b32;
            chunk = (int)((uint32_t)item - t32 * (uint32_t)a.chunks);
        } else {
            token = item / a.chunks, b = token / a.L;
            chunk = (int)(item - token * a.chunks);
        }
        const int64_t l = token - b * a.L, at = b * a.ps[0] + l * a.ps[1];
        const double t = a.pos64 ? (double)static_cast<const int64_t *>(a.positions)[at]
                                 : (double)static_cast<const int32_t *>(a.positions)[at];
        __syncwarp();
        for (int i = lane; i < a.rot / 2; i += 32) {
            double turn = t * (a.freq[i * a.freq_stride] * 0.15915494309189535);
            turn -= rint(turn);
            float sn, cs;
            sincospif(2.0f * (float)turn, &sn, &cs);
            s_cos[warp][i] = cs * a.amplitude;
            s_sin[warp][i] = (a.inverse ? -sn : sn) * a.amplitude;
        }
        __syncwarp();
        float cs[UPL][V], sn[UPL][V];
#pragma unroll
        for (int u = 0; u < UPL; u++)
#pragma unroll
            for (int i = 0; i < V; i++) {
                const int pair = (ul + u * lpr) * V + i;
                cs[u][i] = turns[u] ? s_cos[warp][pair] : 1.0f;
                sn[u][i] = turns[u] ? s_sin[warp][pair] : 0.0f;
            }
        // Rows h0 .. h1 - 1 of operand K. Values go in twos (P to a unit): (0, 1), (2, 3) of each piece, or, with
        // single elements, the unit's two.
        constexpr int P = V;
        auto rows = [&](auto operand, int h0, int h1) {
            constexpr int K = decltype(operand)::value;
            if (h0 >= h1) return;
            const RotaryOperand &o = a.op[K];
            float2 w[NW][P];
            if constexpr (MODE != ROTATE) {
#pragma unroll
                for (int u = 0; u < UPL; u++)
#pragma unroll
                    for (int i = 0; i < P; i++) {
                        w[u][i] = make_float2(0.0f, 0.0f);
                        if (has[u]) w[u][i] = V == 1 ? make_float2(s_w[K][e0[u]], s_w[K][e1[u]])
                                                     : *reinterpret_cast<const float2 *>(&s_w[K][(i < 2 ? e0[u] : e1[u]) + 2 * (i & 1)]);
                    }
            }
            // This lane's first row, and from one of its rows to the next; its pieces within a row.
            const T *xr = static_cast<const T *>(o.x) + b * o.xs[0] + l * o.xs[2] + (h0 + sub) * o.xs[1];
            const T *gr = MODE == NORM_BWD ? static_cast<const T *>(o.g) + b * o.gs[0] + l * o.gs[2] + (h0 + sub) * o.gs[1] : nullptr;
            T *yr = static_cast<T *>(o.y) + b * o.ys[0] + l * o.ys[2] + (h0 + sub) * o.ys[1];
            const int64_t x_step = rpw * o.xs[1], g_step = rpw * o.gs[1], y_step = rpw * o.ys[1];
            const int64_t xi = V == 1 ? o.xs[3] : 1, gi = V == 1 ? o.gs[3] : 1, yi = V == 1 ? o.ys[3] : 1;
            for (int hb = h0; hb < h1; hb += rpw * R) {
                // (Rows past the run and lanes past the row hold zeros.)
                Piece<T, V> x[R][UPL][2], g[MODE == NORM_BWD ? R : 1][UPL][2];
#pragma unroll
                for (int r = 0; r < R; r++) {
                    const bool live = hb + r * rpw + sub < h1;
#pragma unroll
                    for (int u = 0; u < UPL; u++) {
                        x[r][u][0].load(xr + e0[u] * xi, live && has[u]);
                        x[r][u][1].load(xr + e1[u] * xi, live && has[u]);
                        if constexpr (MODE == NORM_BWD) {
                            g[r][u][0].load(gr + e0[u] * gi, live && has[u]);
                            g[r][u][1].load(gr + e1[u] * gi, live && has[u]);
                        }
                    }
                    xr += x_step;
                    if (MODE == NORM_BWD) gr += g_step;
                }
#pragma unroll
                for (int r = 0; r < R; r++) {
                    const bool live = hb + r * rpw + sub < h1;
                    float2 f[UPL][P], v[NG][P];
                    float2 ss = make_float2(0.0f, 0.0f);
#pragma unroll
                    for (int u = 0; u < UPL; u++)
#pragma unroll
                        for (int i = 0; i < P; i++) {
                            f[u][i] = x[r][u][0].two(x[r][u][1], i);
                            if constexpr (MODE != ROTATE) ss = fma2(f[u][i], f[u][i], ss);
                            if constexpr (MODE == NORM_BWD) v[u][i] = g[r][u][0].two(g[r][u][1], i);
                        }
                    float2 rinv = make_float2(1.0f, 1.0f);
                    if constexpr (MODE != ROTATE) {
                        const float sum = row_sum(ss.x + ss.y, lpr);
                        rinv.x = rinv.y = live ? rsqrtf(fmaf(sum, a.inv_D, a.eps)) : 0.0f;
                    }
                    if constexpr (MODE == NORM) {
#pragma unroll
                        for (int u = 0; u < UPL; u++)
#pragma unroll
                            for (int i = 0; i < P; i++) f[u][i] = mul2(mul2(f[u][i], rinv), w[u][i]);
                    }
                    // The rotation: of the row, or (backward) transposed, of the gradient. Channels that
                    // pass through are left alone, not multiplied by 1: an infinity beside them would
                    // come back as NaN.
#pragma unroll
                    for (int u = 0; u < UPL; u++) {
                        float2 *z = MODE == NORM_BWD ? v[MODE == NORM_BWD ? u : 0] : f[u];
                        if (all_turn || turns[u]) {
                            if constexpr (V == 1 || INTER) {  // a pair in each two
#pragma unroll
                                for (int i = 0; i < P; i++)
                                    z[i] = make_float2(fmaf(z[i].x, cs[u][i], -z[i].y * sn[u][i]), fmaf(z[i].y, cs[u][i], z[i].x * sn[u][i]));
                            } else {  // the first and second members of two pairs in z[i] and z[2 + i]
#pragma unroll
                                for (int i = 0; i < 2; i++) {
                                    const float2 c = make_float2(cs[u][2 * i], cs[u][2 * i + 1]), s = make_float2(sn[u][2 * i], sn[u][2 * i + 1]);
                                    const float2 ns = make_float2(-s.x, -s.y), za = z[i], zb = z[(2 + i) % P];
                                    z[i] = fma2(za, c, mul2(zb, ns));
                                    z[(2 + i) % P] = fma2(zb, c, mul2(za, s));
                                }
                            }
                        }
                    }
                    if constexpr (MODE == NORM_BWD) {
                        float2 dots = make_float2(0.0f, 0.0f);
#pragma unroll
                        for (int u = 0; u < UPL; u++)
#pragma unroll
                            for (int i = 0; i < P; i++) {
                                f[u][i] = mul2(f[u][i], rinv);
                                gw[K][u][i] = fma2(v[u][i], f[u][i], gw[K][u][i]);
                                v[u][i] = mul2(v[u][i], w[u][i]);
                                dots = fma2(v[u][i], f[u][i], dots);
                            }
                        const float dot = row_sum(dots.x + dots.y, lpr) * -a.inv_D;
#pragma unroll
                        for (int u = 0; u < UPL; u++)
#pragma unroll
                            for (int i = 0; i < P; i++) f[u][i] = mul2(rinv, fma2(f[u][i], make_float2(dot, dot), v[u][i]));
                    }
#pragma unroll
                    for (int u = 0; u < UPL; u++) {
                        const bool there = live && has[u];
                        if constexpr (V == 1) {
                            if (there) {
                                yr[e0[u] * yi] = from_f<T>(f[u][0].x);
                                yr[e1[u] * yi] = from_f<T>(f[u][0].y);
                            }
                        } else {
                            store4(yr + e0[u], f[u][0], f[u][1 % P], there);
                            store4(yr + e1[u], f[u][2 % P], f[u][3 % P], there);
                        }
                    }
                    yr += y_step;
                }
            }
        };
        const int r0 = chunk * a.heads_per_item, r1 = r0 + a.heads_per_item, hq = a.op[0].H;
        rows(std::integral_constant<int, 0>{}, r0, min(r1, hq));
        rows(std::integral_constant<int, 1>{}, max(r0 - hq, 0), min(r1 - hq, a.op[1].H));
    }
    if constexpr (MODE == NORM_BWD) {
        // This block's part of the weight gradients: over the warp's lane groups, then its warps.
        __shared__ float part[WPB][2 * MAX_PAIRS];
#pragma unroll
        for (int k = 0; k < 2; k++) {
            __syncthreads();
#pragma unroll
            for (int u = 0; u < UPL; u++)
#pragma unroll
                for (int i = 0; i < 2 * V; i++) {
                    float s = i & 1 ? gw[k][u][i / 2].y : gw[k][u][i / 2].x;
                    for (int m = lpr; m < 32; m <<= 1) s += __shfl_xor_sync(ALL, s, m);
                    if (has[u] && sub == 0) part[warp][(i < V ? e0[u] : e1[u]) + i % V] = s;
                }
            __syncthreads();
            for (int d = threadIdx.x; d < a.D; d += WPB * 32) {
                float s = 0.0f;
#pragma unroll
                for (int x = 0; x < WPB; x++) s += part[x][d];
                a.wpart[((int64_t)k * gridDim.x + blockIdx.x) * a.D + d] = s;
            }
        }
    }
}

// gw[d] = sum over the blocks' parts, 32 columns a block, in a fixed order.
__global__ void __launch_bounds__(1024) weight_grad_kernel(const RotaryArgs a, int blocks) {
    __shared__ float sums[32][33];
    griddep_wait();
    const RotaryOperand &o = a.op[blockIdx.y];
    const int d = blockIdx.x * 32 + threadIdx.x;
    const float *part = a.wpart + (int64_t)blockIdx.y * blocks * a.D;
    float s = 0.0f;
    if (d < a.D)
        for (int i = threadIdx.y; i < blocks; i += 32) s += part[(int64_t)i * a.D + d];
    sums[threadIdx.y][threadIdx.x] = s;
    __syncthreads();
    if (threadIdx.y == 0 && d < a.D && o.gw) {
        s = 0.0f;
#pragma unroll
        for (int y = 0; y < 32; y++) s += sums[y][threadIdx.x];
        const int64_t i = d * o.gws;
        if (o.gw_dtype == DC_F32) static_cast<float *>(o.gw)[i] = s;
        else if (o.gw_dtype == DC_F16) static_cast<__half *>(o.gw)[i] = __float2half_rn(s);
        else static_cast<__nv_bfloat16 *>(o.gw)[i] = __float2bfloat16_rn(s);
    }
}

// Whether every row of the tensor can be read in pieces of four elements.
bool vec_rows(const void *ptr, const int64_t *st, int size) {
    return (reinterpret_cast<uintptr_t>(ptr) & (4 * size - 1)) == 0 && st[3] == 1 && st[0] % 4 == 0 && st[1] % 4 == 0 && st[2] % 4 == 0;
}

template <typename T, int V, int UPL, int MODE>
int launch(RotaryArgs &a, bool interleaved, const char *name, cudaStream_t stream) {
    const int units = a.D / (2 * V), lanes = (units + UPL - 1) / UPL;
    a.lpr_log = 0;
    while ((1 << a.lpr_log) < lanes) a.lpr_log++;
    const int rpw = 32 >> a.lpr_log, sms = device_sm_count(), heads = a.op[0].H + a.op[1].H;
    const int64_t tokens = a.B * a.L;
    // A run of all of a token's rows, or as much of it as still gives every SM 32 warps.
    int chunks = 1;
    while (heads > rpw * chunks && tokens * chunks < 32ll * sms) chunks++;
    a.heads_per_item = heads ? ((heads + chunks - 1) / chunks + rpw - 1) / rpw * rpw : rpw;
    a.chunks = heads ? (heads + a.heads_per_item - 1) / a.heads_per_item : 0;
    int64_t blocks = (tokens * a.chunks + WPB - 1) / WPB;
    if (MODE == NORM_BWD) blocks = std::min<int64_t>(blocks, MAX_BWD_BLOCKS);
    if (blocks >= (1ll << 31)) return fail(DC_ERR_UNSUPPORTED, "rotary: more than 2^31 blocks of rows");
    const unsigned grid = (unsigned)blocks;
    if (grid > 0) {
        KernelTrace tr(name, stream);
        if (interleaved) rotary_kernel<T, V, UPL, MODE, true><<<grid, WPB * 32, 0, stream>>>(a);
        else rotary_kernel<T, V, UPL, MODE, false><<<grid, WPB * 32, 0, stream>>>(a);
        const int st = check_launch(name);
        if (st) return st;
    }
    if (MODE == NORM_BWD && (a.op[0].gw || a.op[1].gw)) {
        KernelTrace tr("qk_norm_weight_grad", stream);
        const cudaError_t e = launch_dependent(weight_grad_kernel, dim3((unsigned)((a.D + 31) / 32), 2), dim3(32, 32), 0, stream, a, (int)grid);
        if (e != cudaSuccess) return cuda_fail(e, "qk_norm_weight_grad");
    }
    return DC_OK;
}

template <typename T, int MODE>
int dispatch(RotaryArgs &a, bool interleaved, const char *name, cudaStream_t stream) {
    constexpr int V = 4, S = (int)sizeof(T);
    // Pieces of four where the pairs, the passing channels and every row come in whole ones; otherwise
    // single elements at any stride.
    bool vec = a.rot % (2 * V) == 0 && a.D % (2 * V) == 0;
    for (int i = 0; i < 2 && vec; i++) {
        const RotaryOperand &o = a.op[i];
        if (!o.x) continue;
        vec = vec_rows(o.x, o.xs, S) && vec_rows(o.y, o.ys, S) && (MODE != NORM_BWD || vec_rows(o.g, o.gs, S));
    }
    return vec ? launch<T, V, 1, MODE>(a, interleaved, name, stream) : launch<T, 1, 4, MODE>(a, interleaved, name, stream);
}

template <int MODE>
int by_type(RotaryArgs &a, int dtype, bool interleaved, const char *name, cudaStream_t stream) {
    if (dtype == DC_F32) return dispatch<float, MODE>(a, interleaved, name, stream);
    if (dtype == DC_F16) return dispatch<__half, MODE>(a, interleaved, name, stream);
    return dispatch<__nv_bfloat16, MODE>(a, interleaved, name, stream);
}

}  // namespace

size_t rotary_bwd_workspace_bytes(int64_t D) { return (size_t)2 * MAX_BWD_BLOCKS * D * sizeof(float); }

int rotary_launch(RotaryArgs &a, int dtype, bool interleaved, int mode, cudaStream_t stream) {
    if (mode == ROTATE) return by_type<ROTATE>(a, dtype, interleaved, "rotary", stream);
    if (mode == NORM) return by_type<NORM>(a, dtype, interleaved, "qk_norm_rotary", stream);
    return by_type<NORM_BWD>(a, dtype, interleaved, "qk_norm_rotary_bwd", stream);
}

}  // namespace dc
