// Log probabilities of given tokens with the row's entropy and top alternatives, and the gradient of
// the first two with respect to the logits. With z = x / temperature over a row of `cols` logits:
//   S = sum_j exp(z_j - z_max),  logprob = z_t - z_max - log S,  H = log S - sum_j p_j (z_j - z_max),
//   dlogits_j = (g (delta_jt - p_j) - gH p_j (log p_j + H)) / temperature.
// No reference kernel exists for these; the cluster split and the exchange of partial records through
// distributed shared memory are those of the softmax backward family
// (src/workloads/softmax_logits_backward.cu:410).
//
// Both directions are bound by HBM, the forward pass with the exponential unit at two thirds beside it: bf16 on one
// B200, 4096 x 131072 with entropy 161 us = 6.35 TB/s replayed from a graph, 189 us = 5.4 TB/s in a long loop over changing
// inputs (1024 threads an SM, 128 or 256 a row; a chunk of four vectors a thread with the next one in flight); with 20
// alternatives 198-207 us, with 64 224-234 (replayed); the gradient of 4096 x 65536 155 us = 6.7 TB/s (loop 158). Eight rows of
// 131072 with 20 alternatives take 10 us: latency of a selection in each CTA and one over the cluster.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cmath>

#include "device_context.h"
#include "top_keys.cuh"
#include "vocab_host.h"

namespace credit {
namespace {

constexpr int kThreads = 256;
constexpr int kUnroll = 4;
constexpr int64_t kLongRowBytes = 224 * 1024;   // a row that takes larger CTAs when it has alternatives

struct LogprobArgs {
    const void* logits;
    int64_t ld;
    const int64_t* targets;   // NULL: no token asked for
    float* logprob;
    float* stats;             // [rows, 2]
    float* entropy;
    float* top_logprob;       // [rows, top_k]
    int64_t* top_index;
    int top_k;
    int cols;
    int slice;                // columns per CTA of the cluster
    float inv_t;
    int* status;
};

// An ignored row, by the threads of one CTA.
template <bool ENTROPY, bool TOP>
__device__ __forceinline__ void write_ignored(const LogprobArgs& a, int64_t row) {
    const int tid = threadIdx.x;
    if (tid == 0) {
        a.logprob[row] = 0.0f;
        a.stats[2 * row] = a.stats[2 * row + 1] = 0.0f;
        if (ENTROPY) a.entropy[row] = 0.0f;
    }
    if (TOP && tid < a.top_k) {
        a.top_logprob[row * a.top_k + tid] = -CUDART_INF_F;
        a.top_index[row * a.top_k + tid] = -1;
    }
}

// The target's logit, by one thread; NaN when there is none to read.
template <typename T>
__device__ __forceinline__ float target_logit(const LogprobArgs& a, const T* x, int64_t target) {
    if (a.targets == nullptr) return CUDART_NAN_F;
    if (target < a.cols) return Vec<T>::load(x + target);
    atomicOr(a.status, kStatusBadIndex);
    return CUDART_NAN_F;
}

// A row's scalars from its record, by one thread; returns its log sum.
template <bool ENTROPY>
__device__ __forceinline__ float write_row(const LogprobArgs& a, int64_t row, const SoftmaxRecord& rec, int64_t target,
                                           float picked, float k2) {
    const bool broken = is_broken(rec.m), empty = rec.m == -CUDART_INF_F;
    const float log_sum = broken ? CUDART_NAN_F : (empty ? 0.0f : log_sum_of(rec, k2));
    a.stats[2 * row] = rec.m;
    a.stats[2 * row + 1] = log_sum;
    if (a.targets != nullptr)
        a.logprob[row] = empty && target < a.cols ? -CUDART_INF_F : (picked - rec.m) * a.inv_t - log_sum;
    if (ENTROPY) a.entropy[row] = broken ? CUDART_NAN_F : (empty ? 0.0f : logf(rec.s) - kLn2 * (rec.e / rec.s));
    return log_sum;
}

// The sorted alternatives in t.keys, by the threads of one CTA.
template <int THREADS>
__device__ __forceinline__ void write_top(const LogprobArgs& a, int64_t row, const TopBuffer<THREADS>& t, float row_max,
                                          float row_log_sum) {
    const int tid = threadIdx.x;
    if (tid >= a.top_k) return;
    const int64_t at = row * a.top_k + tid;
    const bool present = tid < t.fill;
    const uint64_t key = present ? t.keys[tid] : 0;
    a.top_logprob[at] = present ? (key_value(key) - row_max) * a.inv_t - row_log_sum : -CUDART_INF_F;
    a.top_index[at] = present ? key_column(key) : -1;
}

// ---------------------------------------------------------------------------
// forward: one cluster per row, the row read once
// ---------------------------------------------------------------------------
template <typename T, bool ENTROPY, bool TOP, int THREADS>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS) token_logprobs_kernel(const LogprobArgs a) {
    __shared__ SoftmaxRecord warp_records[THREADS / 32];
    __shared__ SoftmaxRecord records[kMaxClusterSize];   // rank 0: one per CTA
    __shared__ float row_max, row_log_sum;
    extern __shared__ __align__(16) unsigned char dynamic[];
    TopBuffer<THREADS>& t = *reinterpret_cast<TopBuffer<THREADS>*>(dynamic);

    const uint32_t rank = cluster_cta_rank(), nranks = cluster_cta_count();
    const int64_t row = blockIdx.x / nranks;
    const int tid = threadIdx.x;
    const T* x = static_cast<const T*>(a.logits) + row * a.ld;

    int64_t target = 0;
    if (a.targets != nullptr) {
        target = a.targets[row];
        if (target < 0) {   // ignored row: nothing is read (the whole cluster leaves here)
            if (rank == 0) write_ignored<ENTROPY, TOP>(a, row);
            return;
        }
    }
    const int start = static_cast<int>(rank) * a.slice;
    const RowSpan<T> span(x, start, max(0, min(a.slice, a.cols - start)));
    uint4 ahead[kUnroll];
    fetch_chunk<T, THREADS, kUnroll>(span, 0, ahead);
    const float edge = edge_element(span);
    cluster_arrive_release();   // "this CTA runs": its shared memory may be written from now on
    const float picked = rank == 0 && tid == 0 ? target_logit(a, x, target) : 0.0f;
    if (TOP && tid == 0) init_top_buffer(t);

    const float k2 = a.inv_t * kLog2e;
    SoftmaxRecord rec = empty_record();
    const int chunks = chunks_of<T, THREADS, kUnroll>(span);
    TopCollector<T, THREADS, kUnroll> collector(t, a.top_k, chunks);
    stream_chunks<T, THREADS, kUnroll>(span, ahead, [&](const uint4 (&v)[kUnroll], int it) {
        const float top = chunk_max<T>(v);
        if (TOP) collector.add(top, it);
        accumulate<T, kUnroll, ENTROPY>(v, top, k2, rec);
    });
    if (span.edges > 0) {
        const uint4 v[1] = {Vec<T>::single(edge)};
        accumulate<T, 1, ENTROPY>(v, edge, k2, rec);
    }
    const float thread_max = rec.m;
    rec = cta_record<THREADS>(rec, warp_records, k2);   // its barrier also lies behind the buffer's set-up
    if (TOP) {
        if (tid < span.edges) collector.add_edge(edge, span.start + span.edge_offset(tid));
        collector.finish(span, thread_max);
    }
    cluster_wait_acquire();
    if (nranks > 1) {
        // rank 0 gathers the records, and the lists behind its own buffer
        unsigned long long* gathered = reinterpret_cast<unsigned long long*>(&t + 1);
        if (rank != 0 && tid == 0) {
            const uint32_t to0 = map_to_rank(smem_u32(&records[rank]), 0);
            st_cluster_f32(to0, rec.m);
            st_cluster_f32(to0 + 4, rec.s);
            st_cluster_f32(to0 + 8, rec.e);
        }
        if (TOP && tid < a.top_k)
            st_cluster_u64(map_to_rank(smem_u32(&gathered[rank * a.top_k + tid]), 0), tid < t.fill ? t.keys[tid] : 0);
        cluster_sync_all();
        if (rank != 0) return;
        if constexpr (TOP && THREADS == kThreads) merge_lists(t, gathered, static_cast<int>(nranks), a.top_k);
        if (tid < 32) {
            if (tid == 0) records[0] = rec;
            __syncwarp();
            rec = warp_record<kMaxClusterSize>(tid < static_cast<int>(nranks) ? records[tid] : empty_record(), k2);
        }
    }

    if (tid == 0) {
        row_max = rec.m;
        row_log_sum = write_row<ENTROPY>(a, row, rec, target, picked, k2);
    }
    if (TOP) {
        __syncthreads();
        write_top(a, row, t, row_max, row_log_sum);
    }
}

// ---------------------------------------------------------------------------
// backward: elementwise with row scalars, the logits read once and the gradient written once
// ---------------------------------------------------------------------------
struct LogprobBwdArgs {
    const void* logits;
    int64_t ld;
    const int64_t* targets;
    const float* stats;
    const float* entropy;    // with dentropy
    const float* dlogprob;
    const float* dentropy;   // NULL: none
    void* dlogits;
    int64_t out_ld;
    int cols;
    int pieces;              // CTAs per row
    int chunks;              // of a piece
    float inv_t;
    int* status;
};

template <typename T, bool ENTROPY, bool VECTOR>
__global__ void __launch_bounds__(kThreads, 6) token_logprobs_bwd_kernel(const LogprobBwdArgs a) {
    const int64_t row = blockIdx.x / a.pieces;
    const int piece = static_cast<int>(blockIdx.x % a.pieces);
    const RowMap<T, kThreads, kUnroll, VECTOR> map(static_cast<const T*>(a.logits) + row * a.ld,
                                                   static_cast<T*>(a.dlogits) + row * a.out_ld, a.cols, piece, a.chunks);
    uint4 v[kUnroll];
    const int64_t target = a.targets[row];
    const float base = a.stats[2 * row], k2 = a.inv_t * kLog2e, log2_sum = a.stats[2 * row + 1] * kLog2e;
    // upstream gradients over the temperature, that of the entropy per unit of log2 p
    float g = a.dlogprob[row] * a.inv_t;
    const float gh = ENTROPY ? a.dentropy[row] * a.inv_t * kLn2 : 0.0f, h2 = ENTROPY ? a.entropy[row] * kLog2e : 0.0f;
    // an ignored row, or one without an unmasked logit: no gradient
    const bool zero = target < 0 || base == -CUDART_INF_F;
    if (!zero) map.first_chunk(v);
    if (target >= a.cols) {
        if (piece == 0 && threadIdx.x == 0) atomicOr(a.status, kStatusBadIndex);
        g = CUDART_NAN_F;
    }
    if (is_broken(base)) g = CUDART_NAN_F;   // NaN or +inf in the row: NaN throughout
    // the target's element is overwritten by the thread that writes the others around it: + g, with 1 - p taken
    // by expm1 so that nothing cancels when p is near 1
    const bool mine = !zero && target < a.cols && map.owns(static_cast<int>(target));
    const float at_target = mine ? Vec<T>::load(map.x + target) : 0.0f;
    const float2 minus = make_float2(-base, -base), scale = make_float2(k2, k2), shift = make_float2(-log2_sum, -log2_sum);
    const float2 gh_2 = make_float2(-gh, -gh), rest = make_float2(-fmaf(gh, h2, g), -fmaf(gh, h2, g));
    map.run(zero, v, [&](float2 z) {
        float2 d = __ffma2_rn(__fadd2_rn(z, minus), scale, shift);   // log2 p
        float2 weight = rest;
        if (ENTROPY) {
            d.x = fmaxf(d.x, -200.0f);   // p = 0 there, and 0 * -inf is kept out
            d.y = fmaxf(d.y, -200.0f);
            weight = __ffma2_rn(gh_2, d, rest);
        }
        return __fmul2_rn(make_float2(ex2_approx(d.x), ex2_approx(d.y)), weight);
    });
    if (mine) {
        const float d = fmaf(at_target - base, k2, -log2_sum), dc = fmaxf(d, -200.0f);
        const float entropy_part = ENTROPY ? -ex2_approx(dc) * gh * (dc + h2) : 0.0f;
        Vec<T>::store(map.out + target, fmaf(g, -expm1f(d * kLn2), entropy_part));
    }
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------
template <typename T, bool ENTROPY>
const void* forward_kernel(bool top, int threads) {
    if (threads == kThreads)
        return top ? reinterpret_cast<const void*>(&token_logprobs_kernel<T, ENTROPY, true, kThreads>)
                   : reinterpret_cast<const void*>(&token_logprobs_kernel<T, ENTROPY, false, kThreads>);
    return top ? reinterpret_cast<const void*>(&token_logprobs_kernel<T, ENTROPY, true, kThreads / 2>)
               : reinterpret_cast<const void*>(&token_logprobs_kernel<T, ENTROPY, false, kThreads / 2>);
}

template <typename T>
const void* forward_kernel(bool entropy, bool top, int threads) {
    return entropy ? forward_kernel<T, true>(top, threads) : forward_kernel<T, false>(top, threads);
}

template <typename T>
const void* backward_kernel(bool entropy, bool vector) {
    if (entropy)
        return vector ? reinterpret_cast<const void*>(&token_logprobs_bwd_kernel<T, true, true>)
                      : reinterpret_cast<const void*>(&token_logprobs_bwd_kernel<T, true, false>);
    return vector ? reinterpret_cast<const void*>(&token_logprobs_bwd_kernel<T, false, true>)
                  : reinterpret_cast<const void*>(&token_logprobs_bwd_kernel<T, false, false>);
}

int forward(const void* logits, int64_t ld, const int64_t* targets, float* logprob, float* stats, float* entropy,
            float* top_logprob, int64_t* top_index, int top_k, int64_t rows, int64_t cols, float temperature, int dtype,
            const credit_launch_opts* opts, void* stream) {
    int rc = check_logits(logits, ld, rows, cols, temperature, dtype);
    if (rc != CREDIT_OK) return rc;
    int cluster = 0;
    rc = check_cluster_only(opts, &cluster);
    if (rc != CREDIT_OK) return rc;
    if (top_k < 0 || top_k > kMaxTop)
        return report_error(CREDIT_ERR_INVALID_ARGUMENT, "top_k must be in [0, %d] (got %d)", kMaxTop, top_k);
    if (rows == 0) return CREDIT_OK;
    if (stats == nullptr || (targets == nullptr) != (logprob == nullptr))
        return report_error(CREDIT_ERR_INVALID_ARGUMENT, "stats must not be NULL, targets and logprob go together");
    if (targets == nullptr && top_k == 0 && entropy == nullptr)
        return report_error(CREDIT_ERR_INVALID_ARGUMENT, "nothing is asked for: targets, entropy and top_k are all absent");
    if (top_k > 0 && (top_logprob == nullptr || top_index == nullptr))
        return report_error(CREDIT_ERR_INVALID_ARGUMENT, "top_k = %d needs top_logprob and top_index", top_k);
    if (!aligned_to({targets, top_index}, sizeof(int64_t)) || !aligned_to({logprob, stats, entropy, top_logprob}, sizeof(float)))
        return report_error(CREDIT_ERR_INVALID_ARGUMENT, "every vector must be aligned to its elements");
    DeviceContext ctx;
    rc = current_device_context(&ctx);
    if (rc != CREDIT_OK) return rc;
    // four CTAs an SM fit, and a few rows more than that still gain; choosing alternatives takes them longer together
    if (cluster == 0) cluster = row_split(rows, cols, (top_k > 0 ? 30 : 41) * ctx.sm_count / 10, 8192);
    LogprobArgs a;
    a.logits = logits;
    a.ld = ld;
    a.targets = targets;
    a.logprob = logprob;
    a.stats = stats;
    a.entropy = entropy;
    a.top_logprob = top_logprob;
    a.top_index = top_index;
    a.top_k = top_k;
    a.cols = static_cast<int>(cols);
    a.slice = row_slice(cols, cluster);
    a.inv_t = 1.0f / temperature;
    a.status = ctx.status;
    const bool top = top_k > 0;
    // Half as many threads a row let twice as many rows overlap, whose reductions, selections and ends are then hidden,
    // once the rows fill the eight CTAs an SM that fit. 256 / 128 threads, us, one run of one build, inputs changing: bf16
    // 8192 x 2048 45.7 / 25.1, 8192 x 16384 68.3 / 52.7, 8192 x 32768 101.9 / 91.8; fewer rows: 300 x 131072 23.4 / 29.5,
    // 900 x 65536 26.8 / 26.7. Longer rows hide them anyway; without alternatives the two are within 6 % there, either way
    // (bf16 4096 x 131072 169 / 170, 2048 x 262144 177 / 181; fp32 2048 x 131072 160 / 155, 2400 x 61440 93 / 99). With them
    // the maxima of more threads bound a long row's alternatives closer. k = 20: bf16 8192 x 16384 137 / 95, 8192 x 32768
    // 174 / 132, 3000 x 98304 128 / 127, 2400 x 122880 127 / 130, 4096 x 131072 207 / 221; fp32 3000 x 49152 118 / 117, 2400 x
    // 61440 117 / 124. k = 64: bf16 8192 x 32768 223 / 192, 4096 x 131072 234 / 266; k = 128: 8192 x 32768 334 / 1033 (too few
    // maxima for so many).
    const bool half = !top || (top_k <= 32 && cols * element_bytes(dtype) < kLongRowBytes);
    const int threads = cluster == 1 && rows >= 8 * ctx.sm_count && half ? kThreads / 2 : kThreads;
    const void* func = dtype == CREDIT_BF16 ? forward_kernel<__nv_bfloat16>(entropy != nullptr, top, threads)
                                            : forward_kernel<float>(entropy != nullptr, top, threads);
    rc = prepare_kernel(ctx, func);
    if (rc != CREDIT_OK) return rc;
    void* args[] = {&a};
    // the candidates, and in a cluster the lists that rank 0 gathers
    const size_t buffer = threads == kThreads ? sizeof(TopBuffer<kThreads>) : sizeof(TopBuffer<kThreads / 2>);
    const size_t smem = top ? buffer + (cluster > 1 ? sizeof(uint64_t) * cluster * top_k : 0) : 0;
    return launch_kernel(func, rows * cluster, threads, cluster, static_cast<int>(smem), stream, args);
}

int backward(const void* logits, int64_t ld, const int64_t* targets, const float* stats, const float* entropy,
             const float* dlogprob, const float* dentropy, void* dlogits, int64_t out_ld, int64_t rows, int64_t cols,
             float temperature, int dtype, const credit_launch_opts* opts, void* stream) {
    int rc = check_logits(logits, ld, rows, cols, temperature, dtype);
    if (rc == CREDIT_OK) rc = check_gradient(logits, ld, dlogits, out_ld, rows, cols, dtype);
    int cluster = 0;
    if (rc == CREDIT_OK) rc = check_cluster_only(opts, &cluster);
    if (rc != CREDIT_OK) return rc;
    if (cluster > 1)
        return report_error(CREDIT_ERR_INVALID_ARGUMENT, "the gradient is elementwise: cluster_size must be 0 or 1");
    if (rows == 0) return CREDIT_OK;
    if (targets == nullptr || stats == nullptr || dlogprob == nullptr)
        return report_error(CREDIT_ERR_INVALID_ARGUMENT, "targets, stats and dlogprob must not be NULL");
    if (dentropy != nullptr && entropy == nullptr)
        return report_error(CREDIT_ERR_INVALID_ARGUMENT, "dentropy needs the entropy of the forward pass");
    if (!aligned_to(targets, sizeof(int64_t)) || !aligned_to({stats, entropy, dlogprob, dentropy}, sizeof(float)))
        return report_error(CREDIT_ERR_INVALID_ARGUMENT, "every vector must be aligned to its elements");
    DeviceContext ctx;
    rc = current_device_context(&ctx);
    if (rc != CREDIT_OK) return rc;
    LogprobBwdArgs a;
    a.logits = logits;
    a.ld = ld;
    a.targets = targets;
    a.stats = stats;
    a.entropy = entropy;
    a.dlogprob = dlogprob;
    a.dentropy = dentropy;
    a.dlogits = dlogits;
    a.out_ld = out_ld;
    a.cols = static_cast<int>(cols);
    a.inv_t = 1.0f / temperature;
    a.status = ctx.status;
    const bool vector = same_phase(logits, ld, dlogits, out_ld, rows, dtype);
    const int chunk = kThreads * kUnroll * (dtype == CREDIT_BF16 ? 8 : 4);
    a.chunks = chunks_per_piece(rows, cols, chunk, 2, ctx.sm_count);   // 1, 2, 4, 8: 156, 155, 163, 169 us at 4096 x 65536 bf16
    a.pieces = static_cast<int>((cols + static_cast<int64_t>(chunk) * a.chunks - 1) / (static_cast<int64_t>(chunk) * a.chunks));
    const void* func = dtype == CREDIT_BF16 ? backward_kernel<__nv_bfloat16>(dentropy != nullptr, vector)
                                            : backward_kernel<float>(dentropy != nullptr, vector);
    rc = prepare_kernel(ctx, func);
    if (rc != CREDIT_OK) return rc;
    void* args[] = {&a};
    return launch_kernel(func, rows * a.pieces, kThreads, 1, 0, stream, args);
}

}  // namespace
}  // namespace credit

extern "C" {

int credit_token_logprobs_forward(const void* logits, int64_t row_stride, const int64_t* targets, float* logprob,
                                  float* stats, float* entropy, float* top_logprob, int64_t* top_index, int top_k,
                                  int64_t rows, int64_t cols, float temperature, int dtype, const credit_launch_opts* opts,
                                  void* stream) {
    return credit::guarded([&] {
        return credit::forward(logits, row_stride, targets, logprob, stats, entropy, top_logprob, top_index, top_k, rows,
                               cols, temperature, dtype, opts, stream);
    });
}

int credit_token_logprobs_backward(const void* logits, int64_t row_stride, const int64_t* targets, const float* stats,
                                   const float* entropy, const float* dlogprob, const float* dentropy, void* dlogits,
                                   int64_t dlogits_row_stride, int64_t rows, int64_t cols, float temperature, int dtype,
                                   const credit_launch_opts* opts, void* stream) {
    return credit::guarded([&] {
        return credit::backward(logits, row_stride, targets, stats, entropy, dlogprob, dentropy, dlogits,
                                dlogits_row_stride, rows, cols, temperature, dtype, opts, stream);
    });
}

}  // extern "C"
