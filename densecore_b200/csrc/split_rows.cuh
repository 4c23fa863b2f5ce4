// split_rows.cuh -- results of a query row whose keys were split over CTAs (SplitRows, kernels.h).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math.h>

#include "kernels.h"

namespace dc {

// Channel d of a finished row from its maximum (base 2), sum and accumulator, by the rules of the
// other kernels: a row without keys gives 0 and logsumexp 0.
__device__ __forceinline__ void split_finish(const SplitRows &r, int64_t row, int d, float top, float sum, float acc) {
    const int64_t b = row / r.H, h = row - b * r.H;
    const float l = sum == 0.0f ? 1.0f : sum, y = acc / l;
    const int64_t at = b * r.os[0] + h * r.os[1] + d * r.os[3];
    if (r.out_dtype == DC_F32) static_cast<float *>(r.out)[at] = y;
    else if (r.out_dtype == DC_F16) static_cast<__half *>(r.out)[at] = __float2half_rn(y);
    else static_cast<__nv_bfloat16 *>(r.out)[at] = __float2bfloat16_rn(y);
    if (d == 0) r.lse[b * r.ls[0] + h * r.ls[1]] = (top == -INFINITY ? 0.0f : top * 0.6931471805599453f) + logf(l);
}

// Channel d of a split's result: kept for split_combine, or the row itself when there is one split.
__device__ __forceinline__ void split_store(const SplitRows &r, int64_t row, int split, int d, float top, float sum, float acc) {
    if (r.splits == 1) {
        split_finish(r, row, d, top, sum, acc);
        return;
    }
    float *dst = r.part + (row * r.splits + split) * (int64_t)(r.D + 2);
    dst[d] = acc;
    if (d == 0) {
        dst[r.D] = top;
        dst[r.D + 1] = sum;
    }
}

}  // namespace dc
