// Host-side checks and the launch rule shared by the entry points that take rows of logits.
#pragma once

#include <cmath>

#include "device_context.h"
#include "launch_args.h"

namespace credit {

constexpr int64_t kMaxLogitCols = 1 << 22;

inline int check_logits(const void* logits, int64_t ld, int64_t rows, int64_t cols, float temperature, int dtype) {
    int rc = check_matrix_shape(rows, cols, dtype);
    if (rc != CREDIT_OK) return rc;
    if (cols > kMaxLogitCols)
        return report_error(CREDIT_ERR_UNSUPPORTED, "cols=%lld: rows of logits have at most %lld columns",
                            static_cast<long long>(cols), static_cast<long long>(kMaxLogitCols));
    if (ld < cols || ld > (1ll << 30))
        return report_error(CREDIT_ERR_INVALID_ARGUMENT, "row_stride=%lld must be in [cols, 2^30]", static_cast<long long>(ld));
    if (!(temperature > 0.0f) || !std::isfinite(temperature) || !std::isfinite(2.0f / temperature))
        return report_error(CREDIT_ERR_INVALID_ARGUMENT, "temperature must be positive and finite, and so must its inverse");
    if (rows != 0 && (logits == nullptr || !aligned_to(logits, element_bytes(dtype))))
        return report_error(CREDIT_ERR_INVALID_ARGUMENT, "logits must not be NULL and be aligned to their elements");
    return CREDIT_OK;
}

// The gradient matrix: a place of its own, the logits themselves, or other columns of the same buffer.
inline int check_gradient(const void* logits, int64_t ld, const void* dlogits, int64_t out_ld, int64_t rows, int64_t cols,
                          int dtype) {
    if (out_ld < cols || out_ld > (1ll << 30))
        return report_error(CREDIT_ERR_INVALID_ARGUMENT, "dlogits_row_stride=%lld must be in [cols, 2^30]",
                            static_cast<long long>(out_ld));
    if (rows == 0) return CREDIT_OK;
    const int size = element_bytes(dtype);
    if (dlogits == nullptr || !aligned_to(dlogits, size))
        return report_error(CREDIT_ERR_INVALID_ARGUMENT, "dlogits must not be NULL and be aligned to its elements");
    const uintptr_t in = reinterpret_cast<uintptr_t>(logits), out = reinterpret_cast<uintptr_t>(dlogits);
    if (in == out && (ld == out_ld || rows == 1)) return CREDIT_OK;
    const uintptr_t in_end = in + static_cast<uintptr_t>((rows - 1) * ld + cols) * size;
    const uintptr_t out_end = out + static_cast<uintptr_t>((rows - 1) * out_ld + cols) * size;
    if (in_end <= out || out_end <= in) return CREDIT_OK;
    const int64_t apart = static_cast<int64_t>(in < out ? out - in : in - out) / size % ld;
    if (ld == out_ld && apart >= cols && ld - apart >= cols) return CREDIT_OK;
    return report_error(CREDIT_ERR_INVALID_ARGUMENT, "dlogits must be the logits themselves (same stride) or not overlap them");
}

// Rows of both matrices start at the same place between two 16-byte boundaries.
inline bool same_phase(const void* logits, int64_t ld, const void* dlogits, int64_t out_ld, int64_t rows, int dtype) {
    const int size = element_bytes(dtype);
    const uintptr_t in = reinterpret_cast<uintptr_t>(logits), out = reinterpret_cast<uintptr_t>(dlogits);
    return (in - out) % 16 == 0 && (rows == 1 || (ld - out_ld) * size % 16 == 0);
}

// Chunks of a row that one CTA of an elementwise kernel takes: up to `most`, over which what a CTA does once is
// spread, as long as that leaves 16 CTAs an SM.
inline int chunks_per_piece(int64_t rows, int64_t cols, int chunk_elems, int most, int sm_count) {
    const int64_t all = (cols + chunk_elems - 1) / chunk_elems, each = rows * all / (16 * sm_count);
    return static_cast<int>(each < 1 ? 1 : (each > most ? most : each));
}

inline int row_slice(int64_t cols, int cluster) { return static_cast<int>(((cols + cluster - 1) / cluster + 63) / 64 * 64); }

// CTAs per row of the kernels that reduce a row: the largest cluster that leaves all of them resident at once (`ctas`)
// and slices of more than half of `chunk` columns, a bf16 chunk of the kernel for both types (so fp32 slices are a whole
// one of theirs at least). bf16, 131072 columns, 1 / 2 / 4 / 8 CTAs a row: token_logprobs with 100 rows
// 13.6 / 10.9 / 9.2 / 10.6 us, 300 rows 22.1 / 16.8 / 18.4 / 23.3, 400 rows 24.3 / 24.8 / 26.4 / 33.3; with
// alternatives 200 rows 23.4 / 20.9 / 26.4 / 34.5, 300 rows 27.7 / 31.0 / 36.0 / 49.7; distill_topk with 256 rows
// 27.6 / 20.8 / 19.3 / 21.7, 600 rows 41.0 / 42.3 / 42.0 / 49.1.
inline int row_split(int64_t rows, int64_t cols, int ctas, int chunk) {
    int cluster = 1;
    while (cluster < kMaxClusterSize && 2 * rows * cluster <= ctas && cols / cluster > chunk) cluster *= 2;
    return cluster;
}

}  // namespace credit
