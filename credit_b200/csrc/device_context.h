// What the translation units of the library other than launch.cu share of its host side: the
// current device's properties and status word, cached function attributes and occupancy, one way
// to launch a cluster kernel, and the checks every entry point makes of a shape. The functions
// return a credit_status and leave their text in credit_last_error().
#pragma once

#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include <initializer_list>

#include "../../include/credit_b200.h"
#include "error_state.h"

namespace credit {

struct DeviceContext {
    int device;
    int sm_count;
    int max_dynamic_smem;   // per block, opt-in
    int* status;            // device status word
};

int current_device_context(DeviceContext* out);

// Opt-in shared memory and clusters of 16 for `func` on `device`, once per pair.
int prepare_kernel(const DeviceContext& ctx, const void* func);

// Clusters of this shape that can be resident at once (cached).
int resident_clusters(const DeviceContext& ctx, const void* func, int cluster, int smem, int threads, int* out);

int launch_kernel(const void* func, int64_t grid, int threads, int cluster, int smem, void* stream, void** args);

// rows, cols and dtype within the range every entry point takes.
int check_matrix_shape(int64_t rows, int64_t cols, int dtype);

// The options of the entry points that only take a cluster size; *cluster receives it (0 = automatic).
int check_cluster_only(const credit_launch_opts* opts, int* cluster);

inline bool aligned_to(const void* p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

// All of them (a NULL is).
inline bool aligned_to(std::initializer_list<const void*> pointers, size_t bytes) {
    for (const void* p : pointers)
        if (!aligned_to(p, bytes)) return false;
    return true;
}

inline int element_bytes(int dtype) { return dtype == CREDIT_BF16 ? 2 : 4; }

// Nothing crosses the C boundary as an exception (the caches above allocate).
template <typename F>
int guarded(F&& body) {
    try {
        return body();
    } catch (...) {
        return report_error(CREDIT_ERR_CUDA, "out of host memory");
    }
}

}  // namespace credit
