// window_decode.cu -- one query row per sequence over a key/value cache through a sliding window.
//
// No counterpart in DenseCore (its q_len == 1 case, src/torch_attention.rs:157, sees every key).
// The row of sequence b stands at its last key t = len_b - 1 and sees the keys j <= t with
// t - j < window or j < sinks: at most window + sinks of them, wherever they lie in the cache.
//
// Bound: HBM, 8 D bytes per visible key of each key/value head and 4 D flops per query head: so
//   * the visible keys of a sequence are numbered 0 .. n - 1 (the sinks, then the window) and cut
//     into `splits` equal runs, one CTA each; nothing outside the window is read;
//   * a CTA serves up to four query heads of a key/value head at once, so grouped heads read the
//     cache once (8 heads: twice, the second time from L2);
//   * D / 8 lanes hold a key: two 128-bit loads each of K and V per lane, two keys ahead; every
//     lane group keeps its own running maximum and sum, joined once at the end.
// The partial results of a row's splits (maximum in base 2, sum, accumulators) are joined by
// split_combine, in the order of the splits; a single split writes its row itself.
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
constexpr int WARPS = 4;
constexpr int VEC = 8;  // channels per lane

__device__ __forceinline__ float4 ld_stream(const float *p) {
    float4 r;
    asm volatile("ld.global.nc.L1::no_allocate.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(r.x), "=f"(r.y), "=f"(r.z), "=f"(r.w)
                 : "l"(p));
    return r;
}

// Eight channels at p, of which the first n exist (a multiple of 4, perhaps none).
__device__ __forceinline__ void ld8(const float *p, int n, float (&f)[8]) {
    const float4 zero = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    const float4 a = n > 0 ? ld_stream(p) : zero, b = n > 4 ? ld_stream(p + 4) : zero;
    f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w;
    f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
}

// D: the head dim rounded up to 64, 128 or 256; the lanes past it hold zeros.
template <int D, int G>
__global__ void __launch_bounds__(WARPS * 32) window_decode_kernel(const AttnProblem p, const SplitRows rows) {
    constexpr int LPK = D / VEC, KPW = 32 / LPK, SLOTS = WARPS * KPW;  // lanes per key, keys per warp, per CTA
    constexpr int AHEAD = 2;                                           // keys in flight per lane group
    __shared__ float s_acc[SLOTS][G][D];
    __shared__ float s_m[SLOTS][G], s_l[SLOTS][G];
    griddep_launch_dependents();
    const int lane = threadIdx.x & 31, gl = lane % LPK;
    const int slot = (threadIdx.x >> 5) * KPW + lane / LPK;
    const int have = (int)p.E - gl * VEC;  // channels of this lane that exist
    const int chunks = (p.group + G - 1) / G;
    const int64_t b = blockIdx.z, hk = blockIdx.y / chunks;
    const int64_t h0 = hk * p.group + (int64_t)(blockIdx.y % chunks) * G;
    const int nh = (int)min((int64_t)G, (hk + 1) * p.group - h0);
    const int splits = rows.splits, split = blockIdx.x;

    int64_t len = p.S, t = p.offset;
    if (p.lens) {
        len = p.lens[b * p.lens_stride];
        len = len < 0 ? 0 : (len > p.S ? p.S : len);
        t = len - 1;
    }
    const int64_t end = min(len, t + 1);                            // keys [lo, end) and [0, sinks)
    const int64_t lo = max((int64_t)0, t - p.window + 1);
    const int64_t sinks = max((int64_t)0, min(p.sinks, min(lo, end)));
    const int64_t n = sinks + max((int64_t)0, end - lo), skip = lo - sinks;
    const int64_t per = (n + splits - 1) / splits, v0 = split * per, v1 = min(n, v0 + per);

    float q[G][VEC], acc[G][VEC], m[G], l[G];
#pragma unroll
    for (int g = 0; g < G; g++) {
        m[g] = -INFINITY;
        l[g] = 0.0f;
        const float *qr = p.q + b * p.qs[0] + (h0 + min(g, nh - 1)) * p.qs[1] + gl * VEC;
#pragma unroll
        for (int x = 0; x < VEC; x++) {
            q[g][x] = x < have ? qr[x] * (p.scale * LOG2E) : 0.0f;
            acc[g][x] = 0.0f;
        }
    }
    const float *kb = p.k + b * p.ks[0] + hk * p.ks[1] + gl * VEC;
    const float *vb = p.v + b * p.vs[0] + hk * p.vs[1] + gl * VEC;
    for (int64_t base = v0; base < v1; base += SLOTS * AHEAD) {
        float kk[AHEAD][VEC], vv[AHEAD][VEC];
        int64_t key[AHEAD];
        bool ok[AHEAD];
#pragma unroll
        for (int a = 0; a < AHEAD; a++) {
            const int64_t v = base + a * SLOTS + slot;
            ok[a] = v < v1;
            key[a] = v < sinks ? v : v + skip;
            if (ok[a]) {
                ld8(kb + key[a] * p.ks[2], have, kk[a]);
                ld8(vb + key[a] * p.vs[2], have, vv[a]);
            } else {
#pragma unroll
                for (int x = 0; x < VEC; x++) kk[a][x] = vv[a][x] = 0.0f;
            }
        }
#pragma unroll
        for (int a = 0; a < AHEAD; a++) {
            float s[G];
#pragma unroll
            for (int g = 0; g < G; g++) {
                s[g] = 0.0f;
#pragma unroll
                for (int x = 0; x < VEC; x++) s[g] = fmaf(q[g][x], kk[a][x], s[g]);
            }
#pragma unroll
            for (int o = LPK / 2; o > 0; o >>= 1)
#pragma unroll
                for (int g = 0; g < G; g++) s[g] += __shfl_xor_sync(ALL, s[g], o);
            if (!ok[a]) continue;
#pragma unroll
            for (int g = 0; g < G; g++) {
                if (p.mask_kind) {
                    const float mv = mask_value(p, b, h0 + min(g, nh - 1), 0, key[a]);
                    if (mv <= MASK_HIDES) continue;
                    s[g] += mv * LOG2E;
                }
                if (s[g] == -INFINITY) continue;
                if (s[g] > m[g]) {
                    const float c = exp2f(m[g] - s[g]);
                    l[g] *= c;
#pragma unroll
                    for (int x = 0; x < VEC; x++) acc[g][x] *= c;
                    m[g] = s[g];
                }
                const float w = exp2f(s[g] - m[g]);
                l[g] += w;
#pragma unroll
                for (int x = 0; x < VEC; x++) acc[g][x] = fmaf(w, vv[a][x], acc[g][x]);
            }
        }
    }
#pragma unroll
    for (int g = 0; g < G; g++) {
#pragma unroll
        for (int x = 0; x < VEC; x++) s_acc[slot][g][gl * VEC + x] = acc[g][x];
        if (gl == 0) {
            s_m[slot][g] = m[g];
            s_l[slot][g] = l[g];
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < nh * D; i += WARPS * 32) {
        const int g = i / D, d = i % D;
        if (d >= p.E) continue;
        float top = -INFINITY, sum = 0.0f, a = 0.0f;
#pragma unroll
        for (int s = 0; s < SLOTS; s++) top = fmaxf(top, s_m[s][g]);
#pragma unroll
        for (int s = 0; s < SLOTS; s++) {
            // A slot without a key adds its zeros (or the NaN of a NaN score).
            const float c = s_m[s][g] == -INFINITY ? 1.0f : exp2f(s_m[s][g] - top);
            sum = fmaf(s_l[s][g], c, sum);
            a = fmaf(s_acc[s][g][d], c, a);
        }
        split_store(rows, b * p.H + h0 + g, split, d, top, sum, a);
    }
}

// Joins a row's splits (at most MAX_SPLITS): a block per row, a thread per split for the factors, then
// each warp every fourth split's D channels, and the warps' sums in order.
constexpr int MAX_SPLITS = 128;

__global__ void __launch_bounds__(128) split_combine_kernel(const SplitRows r) {
    __shared__ float s_f[MAX_SPLITS], s_acc[4][256], s_top[4], s_sum[4];
    const int64_t row = blockIdx.x;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    griddep_wait();
    const int64_t stride = r.D + 2;
    const float *src = r.part + row * r.splits * stride;
    const bool mine = (int)threadIdx.x < r.splits;
    const float m = mine ? src[threadIdx.x * stride + r.D] : -INFINITY, l = mine ? src[threadIdx.x * stride + r.D + 1] : 0.0f;
    float top = m;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(ALL, top, o));
    if (lane == 0) s_top[warp] = top;
    __syncthreads();
    top = fmaxf(fmaxf(s_top[0], s_top[1]), fmaxf(s_top[2], s_top[3]));
    // A split without a key adds its zeros (or the NaN of a NaN score).
    const float f = m == -INFINITY ? 1.0f : exp2f(m - top);
    s_f[threadIdx.x] = f;
    float sum = l * f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(ALL, sum, o);
    if (lane == 0) s_sum[warp] = sum;
    __syncthreads();
    sum = (s_sum[0] + s_sum[1]) + (s_sum[2] + s_sum[3]);
    float acc[8] = {};
#pragma unroll 4
    for (int s = warp; s < r.splits; s += 4) {
        const float *part = src + s * stride;
        const float fs = s_f[s];
#pragma unroll
        for (int x = 0; x < 8; x++)
            if (lane + 32 * x < r.D) acc[x] = fmaf(part[lane + 32 * x], fs, acc[x]);
    }
#pragma unroll
    for (int x = 0; x < 8; x++)
        if (lane + 32 * x < r.D) s_acc[warp][lane + 32 * x] = acc[x];
    __syncthreads();
    for (int d = threadIdx.x; d < r.D; d += 128)
        split_finish(r, row, d, top, sum, (s_acc[0][d] + s_acc[1][d]) + (s_acc[2][d] + s_acc[3][d]));
}

bool aligned16(const void *ptr) { return (reinterpret_cast<uintptr_t>(ptr) & 15u) == 0; }

template <int D, int G>
int launch(const AttnProblem &p, const SplitRows &rows, cudaStream_t stream) {
    const int chunks = (p.group + G - 1) / G;
    KernelTrace tr("window_decode", stream);
    window_decode_kernel<D, G><<<dim3((unsigned)rows.splits, (unsigned)(p.Hkv * chunks), (unsigned)p.B), WARPS * 32, 0, stream>>>(p, rows);
    return check_launch("window_decode");
}

template <int D>
int launch_group(const AttnProblem &p, const SplitRows &rows, cudaStream_t stream) {
    if (p.group == 1) return launch<D, 1>(p, rows, stream);
    if (p.group == 2) return launch<D, 2>(p, rows, stream);
    return launch<D, 4>(p, rows, stream);
}

}  // namespace

size_t split_rows_bytes(int64_t rows, int splits, int64_t D) { return splits > 1 ? (size_t)rows * splits * (D + 2) * sizeof(float) : 0; }

int split_combine(const SplitRows &r, cudaStream_t stream) {
    if (r.splits <= 1 || r.rows == 0) return DC_OK;
    KernelTrace tr("split_combine", stream);
    const cudaError_t e = launch_dependent(split_combine_kernel, dim3((unsigned)r.rows), dim3(128), 0, stream, r);
    return e == cudaSuccess ? DC_OK : cuda_fail(e, "split_combine");
}

bool window_decode_supported(const AttnProblem &p) {
    if (p.L != 1 || p.window == 0 || p.E != p.Ev || p.E % 4 || p.E == 0 || p.E > 256) return false;
    if (p.qs[3] != 1 || p.ks[3] != 1 || p.vs[3] != 1) return false;
    for (int i = 0; i < 3; i++)
        if (p.ks[i] % 4 || p.vs[i] % 4) return false;
    const int64_t chunks = (p.group + 3) / 4;
    return aligned16(p.k) && aligned16(p.v) && p.Hkv * chunks <= 65535;
}

// Splits of each row: three CTAs of 4 warps on every SM twice over, at least 128 keys each, or once over
// with at least 32 keys each (two steps of the loop: one sequence's 1004 keys over 8 heads in 8 runs of
// 128 took 14 us, eight steps one after another).
int window_decode_splits(int64_t B, int64_t H, int64_t Hkv, int64_t S, int64_t window, int64_t sinks) {
    const int64_t group = H / Hkv, chunks = group <= 2 ? 1 : (group + 3) / 4;
    const int64_t ctas = std::max<int64_t>(1, B * Hkv * chunks), keys = std::min(S, std::min(window, S) + std::min(sinks, S));
    const int64_t sms = device_sm_count();
    const int64_t twice = std::min(6 * sms / ctas, (keys + 127) / 128), once = std::min(3 * sms / ctas, (keys + 31) / 32);
    return (int)std::max<int64_t>(1, std::min<int64_t>(MAX_SPLITS, std::max(twice, once)));
}

int window_decode(const AttnProblem &p, const SplitRows &rows, cudaStream_t stream) {
    const int st = p.E <= 64 ? launch_group<64>(p, rows, stream) : (p.E <= 128 ? launch_group<128>(p, rows, stream) : launch_group<256>(p, rows, stream));
    return st ? st : split_combine(rows, stream);
}

}  // namespace dc
