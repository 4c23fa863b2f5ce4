// capi_layer.cu -- the extern "C" entry points of the operators around attention: rotary positions,
// normed queries and keys, and the 4-bit key/value cache. Shapes, types and sizes are checked here,
// before any CUDA call; what lies in device memory (positions, lengths, page ids) is checked by the
// kernels.
#include <cuda_runtime.h>
#include <math.h>

#include <string>

#include "capi.h"
#include "common.cuh"
#include "kernels.h"

namespace dc {
namespace {

bool is_float(int dtype) { return dtype == DC_F32 || dtype == DC_F16 || dtype == DC_BF16; }

bool same_sizes(const dc_tensor_t *a, const dc_tensor_t *b) {
    if (a->ndim != b->ndim) return false;
    for (int i = 0; i < a->ndim; i++)
        if (a->sizes[i] != b->sizes[i]) return false;
    return true;
}

// Queries and keys (k null: none), positions and frequencies.
int fill_rotary(const char *what, const dc_tensor_t *q, const dc_tensor_t *k, const dc_tensor_t *positions,
                const dc_tensor_t *inv_freq, double amplitude, RotaryArgs &a) {
    const std::string name(what);
    if (!usable(q) || (k && !usable(k)) || !usable(positions) || !usable(inv_freq))
        return fail(DC_ERR_VALUE, name + ": queries, positions and frequencies are required, aligned to their types");
    if (q->ndim != 4 || !is_float(q->dtype)) return fail(DC_ERR_VALUE, name + " takes (B, H, L, D) float32, float16 or bfloat16 tensors");
    const int64_t B = q->sizes[0], L = q->sizes[2], D = q->sizes[3];
    if (k && (k->ndim != 4 || k->dtype != q->dtype || k->sizes[0] != B || k->sizes[2] != L || k->sizes[3] != D))
        return fail(DC_ERR_VALUE, name + ": keys " + shape_str(k) + " do not match queries " + shape_str(q) + " in batch, length, head dim or type");
    if (D < 2 || D % 2 || D > 256) return fail(DC_ERR_UNSUPPORTED, name + ": the head dim must be even and at most 256");
    if (q->sizes[1] > 65535 || (k && k->sizes[1] > 65535)) return fail(DC_ERR_UNSUPPORTED, name + ": more than 65535 heads");
    if (inv_freq->dtype != DC_F64 || inv_freq->ndim != 1 || 2 * inv_freq->sizes[0] > D)
        return fail(DC_ERR_VALUE, name + ": frequencies must be float64 (rotated channels / 2), at most half the head dim");
    if (positions->dtype != DC_I32 && positions->dtype != DC_I64) return fail(DC_ERR_VALUE, name + ": positions must be int32 or int64");
    const int pd = positions->ndim;
    if (!((pd == 1 && positions->sizes[0] == L) ||
          (pd == 2 && positions->sizes[1] == L && (positions->sizes[0] == B || positions->sizes[0] == 1))))
        return fail(DC_ERR_VALUE, name + ": positions " + shape_str(positions) + " must be (L) or (B, L)");
    a = RotaryArgs{};
    a.B = B;
    a.L = L;
    a.D = (int)D;
    a.rot = (int)(2 * inv_freq->sizes[0]);
    a.positions = positions->data;
    a.pos64 = positions->dtype == DC_I64;
    a.ps[0] = pd == 2 && positions->sizes[0] > 1 ? positions->strides[0] : 0;
    a.ps[1] = positions->strides[pd - 1];
    a.freq = static_cast<const double *>(inv_freq->data);
    a.freq_stride = inv_freq->strides[0];
    a.amplitude = (float)amplitude;
    a.inv_D = (float)(1.0 / (double)D);
    return DC_OK;
}

int fill_operand(const char *what, RotaryOperand &o, const dc_tensor_t *x, dc_tensor_t *y) {
    if (!usable(y) || y->dtype != x->dtype || !same_sizes(x, y) || overlaps(y))
        return fail(DC_ERR_VALUE, std::string(what) + ": outputs must have the inputs' shape and type");
    o.x = x->data;
    o.y = y->data;
    o.H = (int)x->sizes[1];
    copy_strides(x, o.xs, 4);
    copy_strides(y, o.ys, 4);
    return DC_OK;
}

int fill_weight(const char *what, const dc_tensor_t *w, int dtype, int64_t D) {
    if (w && (!usable(w) || w->ndim != 1 || w->sizes[0] != D || (w->dtype != DC_F32 && w->dtype != dtype)))
        return fail(DC_ERR_VALUE, std::string(what) + ": weights must be (head dim), float32 or of the inputs' type");
    return DC_OK;
}

// A cache's description.
int fill_cache(const dc_cache4_t *cache, Cache4 &c) {
    if (!cache || !cache->data) return fail(DC_ERR_VALUE, "cache: its memory is required");
    if (reinterpret_cast<uintptr_t>(cache->data) & 15u) return fail(DC_ERR_VALUE, "cache: its memory must be 16-byte aligned");
    if (cache->num_pages < 1 || cache->num_pages > 0x7fffffff || cache->kv_heads < 1 || cache->kv_heads > 32767)
        return fail(DC_ERR_VALUE, "cache: pages and heads must be at least 1, pages below 2^31, heads below 2^15");
    if (cache->head_dim != 64 && cache->head_dim != 128 && cache->head_dim != 256)
        return fail(DC_ERR_UNSUPPORTED, "cache: the head dim must be 64, 128 or 256");
    if (cache->page_size < 16 || cache->page_size % 16) return fail(DC_ERR_VALUE, "cache: the page size must be a multiple of 16");
    if (cache->num_pages * cache->kv_heads >= (1ll << 31) / (cache->page_size / 16))
        return fail(DC_ERR_UNSUPPORTED, "cache: 2^31 blocks of 16 tokens and more");
    c.data = static_cast<uint8_t *>(cache->data);
    c.pages = cache->num_pages;
    c.Hkv = cache->kv_heads;
    c.D = cache->head_dim;
    c.page_size = cache->page_size;
    return DC_OK;
}

int fill_table(const dc_tensor_t *table, Cache4Args &a) {
    if (!usable(table) || table->dtype != DC_I32 || table->ndim != 2) return fail(DC_ERR_VALUE, "cache: the page table must be int32 (B, pages)");
    a.B = table->sizes[0];
    a.P = table->sizes[1];
    if (a.B > 65535) return fail(DC_ERR_UNSUPPORTED, "cache: more than 65535 sequences in one call");
    if (a.P >= (1ll << 31) || a.P * a.c.page_size >= (1ll << 31)) return fail(DC_ERR_UNSUPPORTED, "cache: page tables of 2^31 positions and more");
    a.table = static_cast<const int32_t *>(table->data);
    a.ts[0] = table->strides[0];
    a.ts[1] = table->strides[1];
    return DC_OK;
}

int fill_counts(const dc_tensor_t *t, int64_t B, const char *what, const int32_t *&ptr, int64_t &stride) {
    if (!usable(t) || t->dtype != DC_I32 || t->ndim != 1 || t->sizes[0] != B)
        return fail(DC_ERR_VALUE, std::string("cache: ") + what + " must be int32 (B)");
    ptr = static_cast<const int32_t *>(t->data);
    stride = t->strides[0];
    return DC_OK;
}

int need_error_word(Cache4Args &a) {
    a.err = device_error_word();
    return a.err ? DC_OK : fail(DC_ERR_CUDA, "device error word is unavailable");
}

}  // namespace
}  // namespace dc

using namespace dc;

extern "C" {

int dc_rotary(const dc_tensor_t *q, const dc_tensor_t *k, const dc_tensor_t *positions, const dc_tensor_t *inv_freq,
              int interleaved, double amplitude, int inverse, dc_tensor_t *q_out, dc_tensor_t *k_out, void *stream) {
    RotaryArgs a;
    int st = fill_rotary("rotary", q, k, positions, inv_freq, amplitude, a);
    if (!st) st = fill_operand("rotary", a.op[0], q, q_out);
    if (!st && k) st = fill_operand("rotary", a.op[1], k, k_out);
    if (st) return st;
    a.inverse = inverse ? 1 : 0;
    if (a.B == 0 || a.L == 0) return DC_OK;
    if ((st = device_ok())) return st;
    return rotary_launch(a, q->dtype, interleaved != 0, ROTARY_ROTATE, static_cast<cudaStream_t>(stream));
}

int dc_qk_norm_rotary(const dc_tensor_t *q, const dc_tensor_t *k, const dc_tensor_t *q_weight, const dc_tensor_t *k_weight,
                      const dc_tensor_t *positions, const dc_tensor_t *inv_freq, double eps, int interleaved,
                      double amplitude, dc_tensor_t *q_out, dc_tensor_t *k_out, void *stream) {
    const char *what = "normed rotary";
    RotaryArgs a;
    int st = fill_rotary(what, q, k, positions, inv_freq, amplitude, a);
    if (!st) st = fill_operand(what, a.op[0], q, q_out);
    if (!st && k) st = fill_operand(what, a.op[1], k, k_out);
    const dc_tensor_t *ws[2] = {q_weight, k ? k_weight : nullptr};
    for (int i = 0; i < 2 && !st; i++) {
        if ((st = fill_weight(what, ws[i], q->dtype, a.D)) || !ws[i]) continue;
        a.op[i].w = ws[i]->data;
        a.op[i].w_dtype = ws[i]->dtype;
        a.op[i].ws = ws[i]->strides[0];
    }
    if (!st && !(eps >= 0.0)) st = fail(DC_ERR_VALUE, "normed rotary: eps must not be negative");
    if (st) return st;
    a.eps = (float)eps;
    if (a.B == 0 || a.L == 0) return DC_OK;
    if ((st = device_ok())) return st;
    return rotary_launch(a, q->dtype, interleaved != 0, ROTARY_NORM, static_cast<cudaStream_t>(stream));
}

size_t dc_qk_norm_rotary_bwd_workspace_size(int64_t head_dim) { return head_dim > 0 ? rotary_bwd_workspace_bytes(head_dim) : 0; }

int dc_qk_norm_rotary_bwd(const dc_tensor_t *q_grad, const dc_tensor_t *k_grad, const dc_tensor_t *q, const dc_tensor_t *k,
                          const dc_tensor_t *q_weight, const dc_tensor_t *k_weight, const dc_tensor_t *positions,
                          const dc_tensor_t *inv_freq, double eps, int interleaved, double amplitude, dc_tensor_t *q_out,
                          dc_tensor_t *k_out, dc_tensor_t *q_weight_grad, dc_tensor_t *k_weight_grad, void *workspace,
                          size_t workspace_bytes, void *stream) {
    const char *what = "normed rotary backward";
    RotaryArgs a;
    int st = fill_rotary(what, q, k, positions, inv_freq, amplitude, a);
    if (!st) st = fill_operand(what, a.op[0], q, q_out);
    if (!st && k) st = fill_operand(what, a.op[1], k, k_out);
    const dc_tensor_t *gs[2] = {q_grad, k_grad}, *xs[2] = {q, k}, *ws[2] = {q_weight, k_weight};
    dc_tensor_t *gws[2] = {q_weight_grad, k_weight_grad};
    for (int i = 0; i < 2 && !st && xs[i]; i++) {
        RotaryOperand &o = a.op[i];
        if (!usable(gs[i]) || gs[i]->dtype != q->dtype || !same_sizes(gs[i], xs[i])) {
            st = fail(DC_ERR_VALUE, "normed rotary backward: gradients must have the inputs' shape and type");
            break;
        }
        o.g = gs[i]->data;
        copy_strides(gs[i], o.gs, 4);
        if (!(st = fill_weight(what, ws[i], q->dtype, a.D)) && ws[i]) {
            o.w = ws[i]->data;
            o.w_dtype = ws[i]->dtype;
            o.ws = ws[i]->strides[0];
        }
        if (!st && !(st = fill_weight(what, gws[i], q->dtype, a.D)) && gws[i]) {
            if (overlaps(gws[i])) return fail(DC_ERR_VALUE, "normed rotary backward: weight gradients overlap");
            o.gw = gws[i]->data;
            o.gw_dtype = gws[i]->dtype;
            o.gws = gws[i]->strides[0];
        }
    }
    if (!st && !(eps >= 0.0)) st = fail(DC_ERR_VALUE, "normed rotary backward: eps must not be negative");
    if (st) return st;
    a.eps = (float)eps;
    a.inverse = 1;
    if ((st = device_ok())) return st;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    ScopedWorkspace scratch;
    if ((st = scratch.get(workspace, workspace_bytes, rotary_bwd_workspace_bytes(a.D), s, "normed rotary backward workspace"))) return st;
    a.wpart = static_cast<float *>(scratch.ptr);
    return rotary_launch(a, q->dtype, interleaved != 0, ROTARY_NORM_BWD, s);
}

int dc_cache4_append(const dc_cache4_t *cache, const dc_tensor_t *key, const dc_tensor_t *value, const dc_tensor_t *page_table,
                     const dc_tensor_t *start, const dc_tensor_t *end, void *stream) {
    Cache4Args a{};
    int st = fill_cache(cache, a.c);
    if (!st) st = fill_table(page_table, a);
    if (!st) st = fill_counts(start, a.B, "start positions", a.starts, a.starts_stride);
    if (!st && end) st = fill_counts(end, a.B, "end positions", a.ends, a.ends_stride);
    if (st) return st;
    if (!usable(key) || !usable(value) || key->ndim != 4 || !is_float(key->dtype) || value->dtype != key->dtype || !same_sizes(key, value) ||
        key->sizes[0] != a.B || key->sizes[1] != a.c.Hkv || key->sizes[3] != a.c.D)
        return fail(DC_ERR_VALUE, "cache append: keys and values must be (B, kv heads, T, head dim) of one float type");
    a.T = key->sizes[2];
    if (a.T >= (1ll << 31)) return fail(DC_ERR_UNSUPPORTED, "cache append: 2^31 tokens and more");
    a.dtype = key->dtype;
    a.x[0] = key->data;
    a.x[1] = value->data;
    copy_strides(key, a.xs[0], 4);
    copy_strides(value, a.xs[1], 4);
    if (a.B == 0 || a.T == 0) return DC_OK;
    if ((st = device_ok()) || (st = need_error_word(a))) return st;
    return cache4_append(a, static_cast<cudaStream_t>(stream));
}

int dc_cache4_read(const dc_cache4_t *cache, const dc_tensor_t *page_table, const dc_tensor_t *lengths, dc_tensor_t *key,
                   dc_tensor_t *value, void *stream) {
    Cache4Args a{};
    int st = fill_cache(cache, a.c);
    if (!st) st = fill_table(page_table, a);
    if (!st) st = fill_counts(lengths, a.B, "lengths", a.lens, a.lens_stride);
    if (st) return st;
    if (!usable(key) || !usable(value) || key->ndim != 4 || key->dtype != DC_F32 || value->dtype != DC_F32 || !same_sizes(key, value) ||
        key->sizes[0] != a.B || key->sizes[1] != a.c.Hkv || key->sizes[3] != a.c.D || overlaps(key) || overlaps(value))
        return fail(DC_ERR_VALUE, "cache read: keys and values must be float32 (B, kv heads, T, head dim)");
    a.T = key->sizes[2];
    if (a.T >= (1ll << 31)) return fail(DC_ERR_UNSUPPORTED, "cache read: 2^31 tokens and more");
    a.y[0] = static_cast<float *>(key->data);
    a.y[1] = static_cast<float *>(value->data);
    copy_strides(key, a.ys[0], 4);
    copy_strides(value, a.ys[1], 4);
    if (a.B == 0 || a.T == 0) return DC_OK;
    if ((st = device_ok()) || (st = need_error_word(a))) return st;
    return cache4_read(a, static_cast<cudaStream_t>(stream));
}

size_t dc_cache4_attention_workspace_size(int64_t batch, int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t capacity,
                                          int64_t window, int64_t sinks, int dtype) {
    if (batch <= 0 || kv_heads <= 0 || heads < kv_heads || capacity <= 0 || head_dim <= 0) return 0;
    return split_rows_bytes(batch * heads, cache4_splits(batch, heads, kv_heads, capacity, window, sinks, dtype), head_dim);
}

int dc_cache4_attention(const dc_cache4_t *cache, const dc_tensor_t *q, const dc_tensor_t *page_table, const dc_tensor_t *lengths,
                        int64_t window, int64_t sinks, int has_scale, double scale, dc_tensor_t *out, dc_tensor_t *lse,
                        void *workspace, size_t workspace_bytes, void *stream) {
    Cache4Args a{};
    int st = fill_cache(cache, a.c);
    if (!st) st = fill_table(page_table, a);
    if (!st) st = fill_counts(lengths, a.B, "lengths", a.lens, a.lens_stride);
    if (st) return st;
    if (!usable(q) || q->ndim != 4 || !is_float(q->dtype) || q->sizes[0] != a.B || q->sizes[2] != 1 || q->sizes[3] != a.c.D ||
        q->sizes[1] % a.c.Hkv)
        return fail(DC_ERR_VALUE, "cache attention: queries must be (B, H, 1, head dim), H a multiple of the cache's heads");
    if (!usable(out) || out->dtype != q->dtype || !same_sizes(out, q) || overlaps(out))
        return fail(DC_ERR_VALUE, "cache attention: the output must have the queries' shape and type");
    if (!usable(lse) || lse->dtype != DC_F32 || lse->ndim != 3 || lse->sizes[0] != a.B || lse->sizes[1] != q->sizes[1] || lse->sizes[2] != 1 ||
        overlaps(lse))
        return fail(DC_ERR_VALUE, "cache attention: the logsumexp must be float32 (B, H, 1)");
    if (window < 0 || sinks < 0) return fail(DC_ERR_VALUE, "cache attention: window and sinks must not be negative");
    a.H = q->sizes[1];
    if (a.H > 65535) return fail(DC_ERR_UNSUPPORTED, "cache attention: more than 65535 heads");
    a.x[0] = q->data;
    copy_strides(q, a.xs[0], 4);
    a.dtype = q->dtype;
    a.scale = has_scale ? (float)scale : (float)(1.0 / sqrt((double)a.c.D));
    a.window = window;
    a.sinks = sinks;
    if (a.B == 0 || a.H == 0) return DC_OK;
    if ((st = device_ok()) || (st = need_error_word(a))) return st;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    SplitRows rows{};
    rows.splits = cache4_splits(a.B, a.H, a.c.Hkv, a.P * a.c.page_size, window, sinks, a.dtype);
    rows.D = a.c.D;
    rows.out_dtype = q->dtype;
    rows.rows = a.B * a.H;
    rows.H = a.H;
    rows.out = out->data;
    rows.lse = static_cast<float *>(lse->data);
    copy_strides(out, rows.os, 4);
    copy_strides(lse, rows.ls, 3);
    ScopedWorkspace scratch;
    if ((st = scratch.get(workspace, workspace_bytes, split_rows_bytes(rows.rows, rows.splits, rows.D), s, "cache attention workspace")))
        return st;
    rows.part = static_cast<float *>(scratch.ptr);
    return cache4_attention(a, rows, s);
}

}  // extern "C"
