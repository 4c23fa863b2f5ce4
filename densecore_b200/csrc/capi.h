// capi.h -- what the C entry points share (internal to the library).
#pragma once

#include <cuda_runtime.h>

#include <string>

#include "common.cuh"

namespace dc {

// "(2, 3)" of a tensor, for messages.
std::string shape_str(const dc_tensor_t *t);

// Whether a view can be followed: sizes not negative, memory where there are elements, on a boundary of
// their type (a kernel's access elsewhere would fault).
bool usable(const dc_tensor_t *t);

// Two writes to one place, or reads of another row's, would depend on order: outputs whose elements
// share memory (an expanded dim) are refused. (Without an element nothing is shared.)
bool overlaps(const dc_tensor_t *t);

// DC_OK when there is a CUDA device.
int device_ok();

inline void copy_strides(const dc_tensor_t *t, int64_t *dst, int n) {
    for (int i = 0; i < n; i++) dst[i] = t->strides[i];
}

// A caller's workspace, or stream-ordered memory that is released when the call returns.
struct ScopedWorkspace {
    void *ptr = nullptr;
    bool owned = false;
    cudaStream_t stream = nullptr;
    ~ScopedWorkspace() {
        if (owned && ptr) cudaFreeAsync(ptr, stream);
    }
    int get(void *given, size_t given_bytes, size_t need, cudaStream_t s, const char *what) {
        stream = s;
        if (need == 0) return DC_OK;
        if (given) {
            if (reinterpret_cast<uintptr_t>(given) & 3u) return fail(DC_ERR_VALUE, std::string(what) + ": must be 4-byte aligned");
            if (given_bytes < need)
                return fail(DC_ERR_VALUE, std::string(what) + ": workspace of " +
                                              std::to_string(given_bytes) + " bytes, " +
                                              std::to_string(need) + " needed");
            ptr = given;
            return DC_OK;
        }
        cudaError_t e = cudaMallocAsync(&ptr, need, s);
        if (e != cudaSuccess) return cuda_fail(e, what);
        owned = true;
        return DC_OK;
    }
};

}  // namespace dc
