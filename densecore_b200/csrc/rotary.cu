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
// and about ten instructions an element are far below what the loads allow, so the design is about
// wide loads and about not paying for the angles:
//   * a row is held by D / (2 V) lanes (V = 16 bytes of elements): a lane owns both members of its
//     V pairs, so the rotation needs no exchange and the norm one butterfly over the row's lanes;
//   * a warp takes one token and a run of its heads, and computes each lane's V sines and cosines
//     once for the run. The angle is reduced to a fraction of a turn in 64 bits (position 10^6 in
//     32 bits would already be 0.06 rad off), its sine and cosine taken in 32. No table: nothing
//     bounds the positions, and nothing else is read;
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

#include "common.cuh"
#include "kernels.h"
#include "trace.h"

namespace dc {
namespace {

constexpr int WPB = 8;  // warps per block
constexpr unsigned ALL = 0xffffffffu;
constexpr int BWD_BLOCKS = 592;  // blocks of the norm's backward: 4 of 8 warps on each of 148 SMs

constexpr int ROTATE = ROTARY_ROTATE, NORM = ROTARY_NORM, NORM_BWD = ROTARY_NORM_BWD;

template <typename T>
__device__ __forceinline__ float to_f(T x);
template <>
__device__ __forceinline__ float to_f<float>(float x) { return x; }
template <>
__device__ __forceinline__ float to_f<__half>(__half x) { return __half2float(x); }
template <>
__device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }

template <typename T>
__device__ __forceinline__ T from_f(float x);
template <>
__device__ __forceinline__ float from_f<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half from_f<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// One piece of a row: V elements as loaded.
template <typename T, int V>
struct Piece {
    T e[V];
};

// V == 1 reads at any element stride; wider pieces are 16 bytes on a 16-byte boundary.
template <typename T, int V>
__device__ __forceinline__ Piece<T, V> load(const T *row, int at, int64_t inner) {
    Piece<T, V> p;
    if constexpr (V == 1) {
        p.e[0] = row[at * inner];
    } else {
        static_assert(V * sizeof(T) == 16, "a piece is 16 bytes");
        *reinterpret_cast<uint4 *>(p.e) = *reinterpret_cast<const uint4 *>(row + at);
    }
    return p;
}

template <typename T, int V>
__device__ __forceinline__ void store(T *row, int at, int64_t inner, const float *f) {
    Piece<T, V> p;
#pragma unroll
    for (int i = 0; i < V; i++) p.e[i] = from_f<T>(f[i]);
    if constexpr (V == 1) row[at * inner] = p.e[0];
    else *reinterpret_cast<uint4 *>(row + at) = *reinterpret_cast<const uint4 *>(p.e);
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
// takes 1 << lpr_log lanes. Blocks below a.blocks_q work on the queries, the others on the keys.
template <typename T, int V, int UPL, int MODE, bool INTER>
__global__ void __launch_bounds__(WPB * 32, MODE == NORM_BWD ? 2 : 3) rotary_kernel(const RotaryArgs a) {
    constexpr int R = rows_ahead<MODE, UPL>();
    const bool key = (int)blockIdx.x >= a.blocks_q;
    const RotaryOperand &o = a.op[key];
    const int blk = (int)blockIdx.x - (key ? a.blocks_q : 0), nblk = key ? (int)gridDim.x - a.blocks_q : a.blocks_q;
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
    float w[MODE == ROTATE ? 1 : UPL][2 * V], gw[MODE == NORM_BWD ? UPL : 1][2 * V];
    if constexpr (MODE != ROTATE) {
#pragma unroll
        for (int u = 0; u < UPL; u++)
#pragma unroll
            for (int i = 0; i < 2 * V; i++) {
                w[u][i] = has[u] ? weight_at(o, (i < V ? e0[u] : e1[u]) + i % V) : 0.0f;
                if constexpr (MODE == NORM_BWD) gw[u][i] = 0.0f;
            }
    }
    const int64_t items = a.B * a.L * o.chunks;
    for (int64_t item = (int64_t)blk * WPB + warp; item < items; item += (int64_t)nblk * WPB) {
        const int64_t token = item / o.chunks, b = token / a.L, l = token - b * a.L;
        const int h0 = (int)(item - token * o.chunks) * o.heads_per_item, h1 = min(o.H, h0 + o.heads_per_item);
        const int64_t at = b * a.ps[0] + l * a.ps[1];
        const double t = a.pos64 ? (double)static_cast<const int64_t *>(a.positions)[at]
                                 : (double)static_cast<const int32_t *>(a.positions)[at];
        float cs[UPL][V], sn[UPL][V];
#pragma unroll
        for (int u = 0; u < UPL; u++)
#pragma unroll
            for (int i = 0; i < V; i++) {
                cs[u][i] = 1.0f;
                sn[u][i] = 0.0f;
                if (has[u] && turns[u]) {
                    double turn = t * a.freq[((ul + u * lpr) * V + i) * a.freq_stride] * 0.15915494309189535;
                    turn -= rint(turn);
                    sincospif(2.0f * (float)turn, &sn[u][i], &cs[u][i]);
                    cs[u][i] *= a.amplitude;
                    sn[u][i] *= a.amplitude;
                    if (a.inverse) sn[u][i] = -sn[u][i];
                }
            }
        const T *xb = static_cast<const T *>(o.x) + b * o.xs[0] + l * o.xs[2];
        const T *gb = MODE == NORM_BWD ? static_cast<const T *>(o.g) + b * o.gs[0] + l * o.gs[2] : nullptr;
        T *yb = static_cast<T *>(o.y) + b * o.ys[0] + l * o.ys[2];
        for (int hb = h0; hb < h1; hb += rpw * R) {
            Piece<T, V> x[R][UPL][2], g[MODE == NORM_BWD ? R : 1][UPL][2];
#pragma unroll
            for (int r = 0; r < R; r++) {
                const int h = hb + r * rpw + sub;
#pragma unroll
                for (int u = 0; u < UPL; u++)
                    if (h < h1 && has[u]) {
                        const T *row = xb + h * o.xs[1];
                        x[r][u][0] = load<T, V>(row, e0[u], o.xs[3]);
                        x[r][u][1] = load<T, V>(row, e1[u], o.xs[3]);
                        if constexpr (MODE == NORM_BWD) {
                            const T *gr = gb + h * o.gs[1];
                            g[r][u][0] = load<T, V>(gr, e0[u], o.gs[3]);
                            g[r][u][1] = load<T, V>(gr, e1[u], o.gs[3]);
                        }
                    }
            }
#pragma unroll
            for (int r = 0; r < R; r++) {
                const int h = hb + r * rpw + sub;
                const bool live = h < h1;
                float f[UPL][2 * V], v[MODE == NORM_BWD ? UPL : 1][2 * V];
                float ss = 0.0f;
#pragma unroll
                for (int u = 0; u < UPL; u++)
#pragma unroll
                    for (int i = 0; i < 2 * V; i++) {
                        const bool in = live && has[u];
                        f[u][i] = in ? to_f(x[r][u][i / V].e[i % V]) : 0.0f;
                        if constexpr (MODE != ROTATE) ss = fmaf(f[u][i], f[u][i], ss);
                        if constexpr (MODE == NORM_BWD) v[u][i] = in ? to_f(g[r][u][i / V].e[i % V]) : 0.0f;
                    }
                float rinv = 1.0f;
                if constexpr (MODE != ROTATE) {
                    for (int s = lpr >> 1; s > 0; s >>= 1) ss += __shfl_xor_sync(ALL, ss, s);
                    rinv = 1.0f / sqrtf(ss * a.inv_D + a.eps);
                }
                if constexpr (MODE == NORM) {
#pragma unroll
                    for (int u = 0; u < UPL; u++)
#pragma unroll
                        for (int i = 0; i < 2 * V; i++) f[u][i] = f[u][i] * rinv * w[u][i];
                }
                // The rotation: of the row, or (backward) transposed, of the gradient.
#pragma unroll
                for (int u = 0; u < UPL; u++) {
                    float *z = MODE == NORM_BWD ? v[MODE == NORM_BWD ? u : 0] : f[u];
                    if (turns[u]) {
#pragma unroll
                        for (int i = 0; i < V; i++) {
                            const int ia = INTER ? 2 * i : i, ib = INTER ? 2 * i + 1 : V + i;
                            const float za = z[ia], zb = z[ib];
                            z[ia] = fmaf(za, cs[u][i], -zb * sn[u][i]);
                            z[ib] = fmaf(zb, cs[u][i], za * sn[u][i]);
                        }
                    }
                }
                if constexpr (MODE == NORM_BWD) {
                    float dot = 0.0f;
#pragma unroll
                    for (int u = 0; u < UPL; u++)
#pragma unroll
                        for (int i = 0; i < 2 * V; i++) {
                            const float n = f[u][i] * rinv;
                            gw[u][i] = fmaf(v[u][i], n, gw[u][i]);
                            f[u][i] = n;
                            v[u][i] *= w[u][i];
                            dot = fmaf(v[u][i], n, dot);
                        }
                    for (int s = lpr >> 1; s > 0; s >>= 1) dot += __shfl_xor_sync(ALL, dot, s);
                    dot *= a.inv_D;
#pragma unroll
                    for (int u = 0; u < UPL; u++)
#pragma unroll
                        for (int i = 0; i < 2 * V; i++) f[u][i] = rinv * fmaf(-f[u][i], dot, v[u][i]);
                }
                if (live) {
                    T *row = yb + h * o.ys[1];
#pragma unroll
                    for (int u = 0; u < UPL; u++)
                        if (has[u]) {
                            store<T, V>(row, e0[u], o.ys[3], f[u]);
                            store<T, V>(row, e1[u], o.ys[3], f[u] + V);
                        }
                }
            }
        }
    }
    if constexpr (MODE == NORM_BWD) {
        // This block's part of the weight gradient: over the warp's lane groups, then its warps.
        __shared__ float part[WPB][256];
#pragma unroll
        for (int u = 0; u < UPL; u++)
#pragma unroll
            for (int i = 0; i < 2 * V; i++) {
                float s = gw[u][i];
                for (int m = lpr; m < 32; m <<= 1) s += __shfl_xor_sync(ALL, s, m);
                if (has[u] && sub == 0) part[warp][(i < V ? e0[u] : e1[u]) + i % V] = s;
            }
        __syncthreads();
        for (int d = threadIdx.x; d < a.D; d += WPB * 32) {
            float s = 0.0f;
#pragma unroll
            for (int x = 0; x < WPB; x++) s += part[x][d];
            o.wpart[(int64_t)blk * a.D + d] = s;
        }
    }
}

// gw[d] = sum over the blocks' parts, 32 columns a block, in a fixed order.
__global__ void __launch_bounds__(1024) weight_grad_kernel(const RotaryArgs a, int blocks_k) {
    __shared__ float sums[32][33];
    const RotaryOperand &o = a.op[blockIdx.y];
    const int n = blockIdx.y ? blocks_k : a.blocks_q, d = blockIdx.x * 32 + threadIdx.x;
    float s = 0.0f;
    if (d < a.D)
        for (int i = threadIdx.y; i < n; i += 32) s += o.wpart[(int64_t)i * a.D + d];
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

// Whether every row of the tensor can be read in 16-byte pieces.
bool vec_rows(const void *ptr, const int64_t *st, int v, int64_t D) {
    return (reinterpret_cast<uintptr_t>(ptr) & 15u) == 0 && (st[3] == 1 || D == 1) && st[0] % v == 0 && st[1] % v == 0 &&
           st[2] % v == 0;
}

template <typename T, int V, int UPL, int MODE>
int launch(RotaryArgs &a, bool interleaved, const char *name, cudaStream_t stream) {
    const int units = (int)(a.D / (2 * V)), lanes = (units + UPL - 1) / UPL;
    a.lpr_log = 0;
    while ((1 << a.lpr_log) < lanes) a.lpr_log++;
    const int rpw = 32 >> a.lpr_log, sms = device_sm_count();
    // A run of heads per warp: as long as the call still gives every SM 16 warps, at most 8 rows a
    // lane group (the angles then cost an eighth of a row's work); short calls get one row each.
    int64_t blocks[2] = {0, 0};
    for (int i = 0; i < 2; i++) {
        RotaryOperand &o = a.op[i];
        if (!o.x || o.H == 0) continue;
        int run = 8;
        while (run > 1 && a.B * a.L * ((o.H + rpw * run - 1) / (rpw * run)) < 16ll * sms) run >>= 1;
        o.heads_per_item = rpw * run;
        o.chunks = (o.H + o.heads_per_item - 1) / o.heads_per_item;
        blocks[i] = (a.B * a.L * o.chunks + WPB - 1) / WPB;
    }
    if (MODE == NORM_BWD) {
        // At most BWD_BLOCKS blocks (their parts are summed by the second kernel), shared between
        // queries and keys by their work.
        const int64_t total = blocks[0] + blocks[1];
        if (total > BWD_BLOCKS) {
            const int64_t k = blocks[1] ? std::max<int64_t>(1, blocks[1] * BWD_BLOCKS / total) : 0;
            blocks[1] = std::min(blocks[1], k);
            blocks[0] = std::min(blocks[0], BWD_BLOCKS - blocks[1]);
        }
        a.op[1].wpart = a.op[0].wpart + blocks[0] * a.D;
    }
    if (blocks[0] + blocks[1] >= (1ll << 31)) return fail(DC_ERR_UNSUPPORTED, "rotary: more than 2^31 blocks of rows");
    a.blocks_q = (int)blocks[0];
    const unsigned grid = (unsigned)(blocks[0] + blocks[1]);
    if (grid > 0) {
        KernelTrace tr(name, stream);
        if (interleaved) rotary_kernel<T, V, UPL, MODE, true><<<grid, WPB * 32, 0, stream>>>(a);
        else rotary_kernel<T, V, UPL, MODE, false><<<grid, WPB * 32, 0, stream>>>(a);
        const int st = check_launch(name);
        if (st) return st;
    }
    if (MODE == NORM_BWD && (a.op[0].gw || a.op[1].gw)) {
        KernelTrace tr("qk_norm_weight_grad", stream);
        weight_grad_kernel<<<dim3((unsigned)((a.D + 31) / 32), 2), dim3(32, 32), 0, stream>>>(a, (int)blocks[1]);
        return check_launch("qk_norm_weight_grad");
    }
    return DC_OK;
}

template <typename T, int MODE>
int dispatch(RotaryArgs &a, bool interleaved, const char *name, cudaStream_t stream) {
    constexpr int V = 16 / sizeof(T);
    // 16-byte pieces where the pairs, the passing channels and every row come in whole ones;
    // otherwise single elements at any stride.
    bool vec = interleaved ? (a.rot % (2 * V) == 0 && a.D % (2 * V) == 0) : (a.rot % (2 * V) == 0 && (a.D - a.rot) % (2 * V) == 0);
    for (int i = 0; i < 2 && vec; i++) {
        const RotaryOperand &o = a.op[i];
        if (!o.x) continue;
        vec = vec_rows(o.x, o.xs, V, a.D) && vec_rows(o.y, o.ys, V, a.D) && (MODE != NORM_BWD || vec_rows(o.g, o.gs, V, a.D));
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

size_t rotary_bwd_workspace_bytes(int64_t D) { return (size_t)BWD_BLOCKS * D * sizeof(float); }

int rotary_launch(RotaryArgs &a, int dtype, bool interleaved, int mode, cudaStream_t stream) {
    if (mode == ROTATE) return by_type<ROTATE>(a, dtype, interleaved, "rotary", stream);
    if (mode == NORM) return by_type<NORM>(a, dtype, interleaved, "qk_norm_rotary", stream);
    return by_type<NORM_BWD>(a, dtype, interleaved, "qk_norm_rotary_bwd", stream);
}

}  // namespace dc
