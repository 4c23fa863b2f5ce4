// kernels.h -- host-side launchers of the SDPA kernels (internal to the library).
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "common.cuh"

namespace dc {

struct MergeStrides {
    int64_t oas[4], las[3], ops[4], lps[3];
};

// CUDA-core kernels (attn_simt.cu): any head dim <= 256, any strides.
int simt_forward(const AttnProblem &p, cudaStream_t stream);
int bwd_delta(const AttnProblem &p, const AttnGrads &g, cudaStream_t stream);
int simt_backward(const AttnProblem &p, const AttnGrads &g, cudaStream_t stream);
int simt_probs(const AttnProblem &p, float *probs, const int64_t ps[4], int average,
               cudaStream_t stream);
int merge(float *oa, float *la, const float *op, const float *lp, int64_t B, int64_t H,
          int64_t L, int64_t Ev, const MergeStrides &st, cudaStream_t stream);

// Split-KV decode (decode.cu): q_len == 1, head dim 64 or 128, rows of 16-byte multiples.
bool decode_supported(const AttnProblem &p);
int decode_pick_splits(const AttnProblem &p);
size_t decode_workspace_bytes(int64_t B, int64_t H, int64_t Ev, int splits);
int decode_forward(const AttnProblem &p, int splits, void *workspace, cudaStream_t stream);

// Sliding-window forward on the 16-bit tensor cores (attn_win.cu): of what tc_forward takes, the calls with
// a head dim above 64 that see enough keys to pay for the packing.
bool window_forward_pick(const AttnProblem &p);
int window_forward(const AttnProblem &p, cudaStream_t stream);
// tc_forward (3xTF32, a window, a head dim above 64) if *when, in device memory, is not zero.
int tc_forward_if(const AttnProblem &p, const int *when, cudaStream_t stream);

// Rows whose keys are split over CTAs (window_decode.cu, cache4.cu): row (b, h) of out (B, H, 1, D)
// and lse (B, H, 1). With one split the CTA writes its row; otherwise the partial results go to
// `part` -- per row and split D accumulators, the maximum in base 2 and the sum, both relative to
// that maximum -- and split_combine joins them in order.
struct SplitRows {
    float *part;
    int splits, D, out_dtype;  // out: float32, float16 or bfloat16
    int64_t rows, H;
    void *out;
    float *lse;
    int64_t os[4], ls[3];
};
size_t split_rows_bytes(int64_t rows, int splits, int64_t D);
int split_combine(const SplitRows &r, cudaStream_t stream);

// One query row per sequence through a sliding window (window_decode.cu): head dims up to 256, rows on
// 16-byte boundaries.
bool window_decode_supported(const AttnProblem &p);
int window_decode_splits(int64_t B, int64_t H, int64_t Hkv, int64_t S, int64_t window, int64_t sinks);
int window_decode(const AttnProblem &p, const SplitRows &rows, cudaStream_t stream);

// Rotary positions (rotary.cu). op[0] is the queries, op[1] the keys (x null: none); per operand
// x, y and (norm backward) the upstream gradient g are (B, H, L, D) views of one type, w the norm's
// weight and gw its gradient (float32 or that type; either may be null).
struct RotaryOperand {
    const void *x, *g, *w;
    void *y, *gw;
    int64_t xs[4], gs[4], ys[4], ws, gws;
    int H, w_dtype, gw_dtype;
};
struct RotaryArgs {
    RotaryOperand op[2];
    int64_t B, L;
    int D, rot, lpr_log, heads_per_item, chunks;
    float *wpart;  // norm backward: the blocks' parts of the weight gradients, queries then keys
    const void *positions;
    int pos64;
    int64_t ps[2];  // (batch, token) strides of the positions
    const double *freq;
    int64_t freq_stride;
    float amplitude, eps, inv_D;
    int inverse;
};
enum RotaryMode { ROTARY_ROTATE = 0, ROTARY_NORM = 1, ROTARY_NORM_BWD = 2 };
size_t rotary_bwd_workspace_bytes(int64_t D);
int rotary_launch(RotaryArgs &a, int dtype, bool interleaved, int mode, cudaStream_t stream);

// The 4-bit key/value cache (cache4.cu).
struct Cache4 {
    uint8_t *data;  // (pages, Hkv, page_size / 16) blocks of 20 D bytes (cache4.cu)
    int64_t pages;
    int Hkv, D, page_size;
};
struct Cache4Args {
    Cache4 c;
    const int32_t *table, *lens, *starts, *ends;  // (B, P) page ids, (B) lengths / first / end positions
    int64_t ts[2], lens_stride, starts_stride, ends_stride;
    int64_t B, H, T, P;  // P: page table entries per sequence; T: tokens of an append or read
    const void *x[2];    // append: key, value; attention: x[0] the queries
    float *y[2];         // read: key, value
    int64_t xs[2][4], ys[2][4];
    int dtype;
    float scale;
    int64_t window, sinks;
    int *err;
};
int cache4_append(const Cache4Args &a, cudaStream_t stream);
int cache4_read(const Cache4Args &a, cudaStream_t stream);
int cache4_splits(int64_t B, int64_t H, int64_t Hkv, int64_t capacity, int64_t window, int64_t sinks, int dtype);
int cache4_attention(const Cache4Args &a, const SplitRows &rows, cudaStream_t stream);

// tcgen05 tensor-core kernels (attn_tc.cu, attn_tc_bwd.cu). Forward: head dim 64 or 128,
// E == Ev, unit-stride rows on 16-byte boundaries. Backward: E == Ev == 64, any strides (its
// pre-pass copies the operands into contiguous TF32 hi / lo buffers); it also writes delta.
bool tc_forward_supported(const AttnProblem &p);
int tc_forward(const AttnProblem &p, int precision, cudaStream_t stream);
bool tc_backward_supported(const AttnProblem &p, const AttnGrads &g);
int tc_backward(const AttnProblem &p, const AttnGrads &g, int precision, cudaStream_t stream);
// The tensor-core kernels' device error word (sm100::DeviceError); -1 if it cannot be read.
int device_error(int reset);
// Device address of that word (passed to the kernels), or nullptr.
int *device_error_word();

// Dropout keep masks (rng.cu): n bernoulli(keep_prob) draws of DenseCore's generator stream
// from the device state st_in (624 words, left, next) as packed bits; the advanced state goes
// to st_out (which may equal st_in). rng_skip: the same advance on host memory, no device.
int keep_bits(const uint32_t *st_in, uint32_t *st_out, int64_t n, double keep_prob, uint32_t *bits,
              cudaStream_t stream);
int rng_skip(const uint32_t *st_in, uint64_t outputs, uint32_t *st_out);

// SM count of the current device (cached per device; 148 if it cannot be read).
int device_sm_count();

// Side streams (streams.cu): the library's stream for `role` (0 = the backward's dQ kernel,
// 1 = ring attention's transfers) beside caller stream `caller` on the current device, and an
// event edge that makes `to` wait for the work enqueued on `from` so far.
int side_stream(cudaStream_t caller, int role, cudaStream_t *out);
int stream_edge(cudaStream_t from, cudaStream_t to);

// A fork of `side` from `caller` that is joined back exactly once: by join(), or, on an error
// path that returns early, by the destructor (which keeps the call's error message).
class StreamJoin {
   public:
    StreamJoin(cudaStream_t caller, cudaStream_t side) : caller_(caller), side_(side) {}
    ~StreamJoin();
    int join();
    StreamJoin(const StreamJoin &) = delete;
    StreamJoin &operator=(const StreamJoin &) = delete;

   private:
    cudaStream_t caller_, side_;
    bool joined_ = false;
};

// The library's stream-ordered scratch pool (pool.cu): memory for `bytes` on `stream`'s
// order of the current device, and its release on the same stream.
int pool_alloc(void **ptr, size_t bytes, cudaStream_t stream);
void pool_free(void *ptr, cudaStream_t stream);

}  // namespace dc
