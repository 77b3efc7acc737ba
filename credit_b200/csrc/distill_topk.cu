// Distillation from a teacher's top logits: KL(teacher || student) per row, where the teacher is a
// list of up to 128 columns with log probabilities, and its gradient with respect to the student's
// logits. With z = logits / temperature, q = softmax(z), list entries k with column c_k:
//   without a tail  w_k = softmax(v)_k              (the teacher renormalised over its list)
//   with a tail     w_k = exp(v_k), w_r = 1 - sum w_k against q_r = sum of q outside the list
//   loss = sum_k w_k (log w_k - log q_{c_k}) [+ w_r (log w_r - log q_r)]
//   dlogits_j = g / temperature * (q_j - w_j)                      for j in the list
//             = g / temperature * exp(z_j - tail lse) (q_r - w_r)  outside it (q_j without a tail)
// The sum outside the list is accumulated as such (listed columns are marked in a bitmap and skipped),
// never as "all minus listed", so a student that has almost all of its mass in the list keeps q_r and
// its gradient to full precision; w_r is taken in 64 bits for the same reason.
// A renormalised list may lie anywhere (raw logits): its weights are taken from differences to its largest value.
// No reference kernel exists for this; the row pass is that of token_logprobs.cu and bound as it is: bf16 on one B200,
// 2048 x 131072 with a list of 64 98 us = 5.5 TB/s replayed from a graph, 109 us = 4.9 TB/s in a long loop over changing
// inputs; the gradient 179 us = 6.0 TB/s and 187 us. Shorter rows show what a row costs beside its logits (the list, its
// marks, one warp's finish): 8192 x 16384 88 us = 3.1 TB/s.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cmath>
#include <type_traits>

#include "device_context.h"
#include "vocab_host.h"
#include "vocab_rows.cuh"

namespace credit {
namespace {

constexpr int kThreads = 128;      // forward: eight CTAs an SM (four of 256 threads: 193 instead of 179 us at 4096 x 131072 bf16)
constexpr int kBwdThreads = 256;
constexpr int kUnroll = 4;
constexpr int kMaxList = 128;
constexpr int kPerLane = kMaxList / 32;
constexpr int kStats = 6;   // floats of saved state per row

struct DistillArgs {
    const void* logits;
    int64_t ld;
    const int64_t* index;    // [rows, top_k], negative = unused place
    const float* teacher;    // [rows, top_k]
    int top_k;
    float* loss;
    float* stats;            // [rows, 6]
    int cols;
    int slice;
    int map_words;           // of one slice
    float inv_t;
    int* status;
};

__device__ __forceinline__ double warp_sum_f64(double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

__device__ __forceinline__ float warp_max_nan(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = max_nan(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

// One row's list in shared memory.
struct TeacherList {
    int column[kMaxList];      // -1 = unused
    float value[kMaxList];
    float top;                 // largest value
    float base;
    double sum;                // of exp(value - base): 0 for a list without mass
    int bad;                   // some column lies outside the row
    int any;                   // some place is used
};

// One warp reads the list; the others see it behind a barrier that the caller places.
template <bool TAIL>
__device__ __forceinline__ void load_list(const DistillArgs& a, int64_t row, TeacherList& l) {
    const int lane = threadIdx.x & 31;
    float v[kPerLane];
    bool bad = false, any = false;
    float top = -CUDART_INF_F;
#pragma unroll
    for (int i = 0; i < kPerLane; ++i) {
        const int k = lane + 32 * i;
        int column = -1;
        v[i] = -CUDART_INF_F;
        if (k < a.top_k) {
            const int64_t c = a.index[row * a.top_k + k];
            if (c >= a.cols) {
                bad = true;
            } else if (c >= 0) {
                column = static_cast<int>(c);
                v[i] = a.teacher[row * a.top_k + k];
                any = true;
            }
        }
        l.column[k] = column;
        l.value[k] = v[i];
        top = max_nan(top, v[i]);
    }
    top = warp_max_nan(top);
    const float base = top == -CUDART_INF_F || (TAIL && fabsf(top) < 600.0f) ? 0.0f : top;   // 64 bits hold exp(+-600)
    double sum = 0.0;
#pragma unroll
    for (int i = 0; i < kPerLane; ++i) sum += exp(static_cast<double>(v[i]) - base);
    sum = warp_sum_f64(sum);
    bad = __any_sync(0xffffffffu, bad);
    any = __any_sync(0xffffffffu, any);
    if (lane == 0) {
        l.top = top;
        l.base = base;
        l.sum = sum;
        l.bad = bad;
        l.any = any;
    }
}

// What one thread holds of a row while it streams by, and how its listed columns are kept out of the sums: a map
// of the slice with a bit for each element of each vector, a thread's bits of one chunk in one word (bf16) or half
// word (fp32), and behind them a byte for each edge element.
template <typename T, bool TAIL>
struct DistillPass {
    static constexpr int E = Vec<T>::kElems;
    using Bits = std::conditional_t<E == 8, uint32_t, uint16_t>;
    const RowSpan<T>& span;
    uint32_t* map;
    float k2;
    SoftmaxRecord rec;

    __device__ __forceinline__ DistillPass(const RowSpan<T>& s, uint32_t* m, float k2_) : span(s), map(m), k2(k2_), rec(empty_record()) {}

    __device__ __forceinline__ int words() const {   // of vectors
        return chunks_of<T, kThreads, kUnroll>(span) * kThreads * static_cast<int>(sizeof(Bits)) / 4;
    }
    __device__ __forceinline__ bool holds(int column) const { return column >= span.start && column < span.start + span.local; }
    // true when the column was marked before
    __device__ __forceinline__ bool mark(int column) const {
        const int offset = column - span.start, e = offset - span.head;
        int word, bit;
        if (e >= 0 && e < span.nvec * E) {
            const int v = e / E, chunk = v / (kThreads * kUnroll), u = v / kThreads % kUnroll;
            const int place = chunk * kThreads + v % kThreads;   // of the thread's bits
            bit = u * E + e % E;
            word = E == 8 ? place : place >> 1;
            if (E == 4) bit += (place & 1) * 16;
        } else {
            const int i = offset < span.head ? offset : offset - span.nvec * E;
            word = words() + i / 4;
            bit = i % 4 * 8;
        }
        return atomicOr(&map[word], 1u << bit) >> bit & 1u;
    }

    template <int U>
    __device__ __forceinline__ void add(const uint4 (&v)[U]) {
        accumulate<T, U, false>(v, chunk_max<T, U>(v), k2, rec);
    }
    __device__ __forceinline__ void take(uint4 (&v)[kUnroll], int it) {
        if (TAIL) {
            const uint32_t word = reinterpret_cast<const Bits*>(map)[it * kThreads + threadIdx.x];
            if (word != 0) {
#pragma unroll
                for (int u = 0; u < kUnroll; ++u) {
                    float y[E];
                    Vec<T>::unpack(v[u], y);
#pragma unroll
                    for (int j = 0; j < E; ++j)
                        if (word >> (u * E + j) & 1u) y[j] = -CUDART_INF_F;
                    v[u] = Vec<T>::pack(y);
                }
            }
        }
        add(v);
    }
    __device__ __forceinline__ void take_edges(float edge) {
        if (span.edges == 0) return;
        const int i = threadIdx.x;
        const bool hidden = TAIL && i < span.edges && (map[words() + i / 4] >> (i % 4 * 8) & 1u) != 0;
        const uint4 v[1] = {Vec<T>::single(hidden ? -CUDART_INF_F : edge)};
        add(v);
    }
};

// 32-bit words of the map of a slice (whole 16 bytes).
inline int map_words(int slice, int vec_elems) {
    const int chunk = kThreads * kUnroll * vec_elems;
    return (slice + chunk - 1) / chunk * kThreads * vec_elems / 8 + 4;
}

__device__ __forceinline__ void write_no_teacher(const DistillArgs& a, int64_t row) {
    if (threadIdx.x == 0) a.loss[row] = 0.0f;
    if (threadIdx.x < kStats) a.stats[row * kStats + threadIdx.x] = threadIdx.x == 0 ? -CUDART_INF_F : 0.0f;   // no gradient
}

// A row's results, by warp 0: `rec` over the row's columns (with a tail: those outside the list), the student's
// logits at the list's entries (-inf for unused ones). Lane l holds entries l, l + 32, ...
template <bool TAIL>
__device__ __forceinline__ void finish_row(const DistillArgs& a, int64_t row, const TeacherList& list, const float* student,
                                           bool repeats, const SoftmaxRecord& rec, float k2) {
    const int lane = threadIdx.x;
    SoftmaxRecord all = rec;
    if (TAIL) {
        // the listed columns, each once: a repeated column counts where it appears first
        float y[kPerLane];
        float top = -CUDART_INF_F;
#pragma unroll
        for (int i = 0; i < kPerLane; ++i) {
            const int k = lane + 32 * i;
            y[i] = student[k];
            if (repeats)
                for (int j = 0; j < k; ++j)
                    if (list.column[j] == list.column[k]) y[i] = -CUDART_INF_F;
            top = max_nan(top, y[i]);
        }
        SoftmaxRecord mine = empty_record();
        mine.m = warp_max_nan(top);
        // relative to the base of this maximum, as the row's sums are
        const bool by_base = has_base(mine.m, k2);
#pragma unroll
        for (int i = 0; i < kPerLane; ++i)
            if (y[i] != -CUDART_INF_F)
                mine.s += ex2_approx(by_base ? fmaf(y[i], k2, -base_of(mine.m, k2)) : (y[i] - mine.m) * k2);
        mine.s = warp_sum(mine.s);
        all = merge_records(rec, mine, k2);
    }
    const bool broken = is_broken(all.m) || list.bad || isnan(list.sum);
    const bool empty = all.m == -CUDART_INF_F, no_tail = rec.m == -CUDART_INF_F;
    const float log_sum = empty ? 0.0f : log_sum_of(all, k2);
    const float tail_log_sum = no_tail ? 0.0f : log_sum_of(rec, k2);
    // the teacher: always a distribution. Without anything left outside the student's list, or with a
    // list of more than 1, it is renormalised over the list, by differences to the list's largest value: a
    // normaliser far from zero has too few bits for exp(value - normaliser).
    float top = 0.0f, shift = 0.0f, log_norm = 0.0f, rest = 0.0f;
    bool no_teacher = false;
    const double left = TAIL ? 1.0 - (list.base == 0.0f ? list.sum : list.sum * exp(static_cast<double>(list.base))) : 0.0;
    if (!TAIL || no_tail || left < 0.0) {
        no_teacher = list.sum == 0.0;   // all of it outside the list, and nothing is there
        if (!no_teacher) {
            const double log_mass = list.base + log(list.sum);
            top = list.top;
            shift = static_cast<float>(log_mass - top);
            log_norm = static_cast<float>(log_mass);
        }
    } else {
        rest = static_cast<float>(left);
    }
    double loss = 0.0;
#pragma unroll
    for (int i = 0; i < kPerLane; ++i) {
        const int k = lane + 32 * i;
        const float logw = (list.value[k] - top) - shift;
        const float w = expf(logw);
        if (list.column[k] >= 0 && w != 0.0f) {
            const float logq = empty ? -CUDART_INF_F : (student[k] - all.m) * a.inv_t - log_sum;
            loss += static_cast<double>(w) * (logw - logq);
        }
    }
    loss = warp_sum_f64(loss);
    if (lane == 0) {
        if (TAIL && rest > 0.0f) {
            const float log_rest_q = (rec.m - all.m) * a.inv_t + (tail_log_sum - log_sum);
            loss += static_cast<double>(rest) * (logf(rest) - log_rest_q);
        }
        if (list.bad) atomicOr(a.status, kStatusBadIndex);
        a.loss[row] = broken ? CUDART_NAN_F : static_cast<float>(loss);
        float* s = a.stats + row * kStats;
        s[0] = broken ? CUDART_NAN_F : (no_teacher ? -CUDART_INF_F : all.m);
        s[1] = log_sum;
        s[2] = TAIL ? rec.m : all.m;
        s[3] = TAIL ? tail_log_sum : log_sum;
        s[4] = log_norm;
        s[5] = rest;
    }
}

// ---------------------------------------------------------------------------
// forward: one cluster per row, the row read once
// ---------------------------------------------------------------------------
template <typename T, bool TAIL>
__global__ void __launch_bounds__(kThreads, 8) distill_topk_kernel(const DistillArgs a) {
    __shared__ SoftmaxRecord warp_records[kThreads / 32];
    __shared__ SoftmaxRecord records[kMaxClusterSize];   // rank 0: one per CTA; e = 1: a column repeats there
    __shared__ TeacherList list;
    __shared__ float student[kMaxList];
    extern __shared__ __align__(16) uint32_t map[];

    const uint32_t rank = cluster_cta_rank(), nranks = cluster_cta_count();
    const int64_t row = blockIdx.x / nranks;
    const int tid = threadIdx.x;
    const T* x = static_cast<const T*>(a.logits) + row * a.ld;
    const int start = static_cast<int>(rank) * a.slice;
    const RowSpan<T> span(x, start, max(0, min(a.slice, a.cols - start)));
    DistillPass<T, TAIL> pass(span, map, a.inv_t * kLog2e);
    uint4 ahead[kUnroll];
    fetch_chunk<T, kThreads, kUnroll>(span, 0, ahead);
    const float edge = edge_element(span);

    if (tid < 32) load_list<TAIL>(a, row, list);
    if (TAIL)
        for (int i = tid; i < a.map_words / 4; i += kThreads) reinterpret_cast<uint4*>(map)[i] = make_uint4(0, 0, 0, 0);
    __syncthreads();
    if (!list.bad && (TAIL ? !list.any : list.sum == 0.0)) {
        // no teacher in this row: nothing is read (the whole cluster leaves here)
        if (rank == 0) write_no_teacher(a, row);
        return;
    }
    cluster_arrive_release();
    bool repeats = false;
    if (tid < kMaxList) {
        const int column = tid < a.top_k ? list.column[tid] : -1;
        if (TAIL && pass.holds(column)) repeats = pass.mark(column);
        if (rank == 0) student[tid] = column >= 0 ? Vec<T>::load(x + column) : -CUDART_INF_F;
    }
    if (TAIL) repeats = __syncthreads_or(repeats);

    stream_chunks<T, kThreads, kUnroll>(span, ahead, [&](uint4 (&v)[kUnroll], int it) { pass.take(v, it); });
    pass.take_edges(edge);
    SoftmaxRecord rec = cta_record<kThreads>(pass.rec, warp_records, pass.k2);
    cluster_wait_acquire();
    if (nranks > 1) {
        if (rank != 0 && tid == 0) {
            const uint32_t to = map_to_rank(smem_u32(&records[rank]), 0);
            st_cluster_f32(to, rec.m);
            st_cluster_f32(to + 4, rec.s);
            st_cluster_f32(to + 8, repeats ? 1.0f : 0.0f);
        }
        cluster_sync_all();
        if (rank != 0) return;
    }
    if (tid >= 32) return;
    if (nranks > 1) {
        if (tid == 0) records[0] = rec;
        __syncwarp();
        if (tid < static_cast<int>(nranks)) {
            rec = records[tid];
            if (tid > 0 && rec.e != 0.0f) repeats = true;
            rec.e = 0.0f;
        } else {
            rec = empty_record();
        }
        repeats = __any_sync(0xffffffffu, repeats);
        rec = warp_record<kMaxClusterSize>(rec, pass.k2);
    }
    finish_row<TAIL>(a, row, list, student, repeats, rec, pass.k2);
}

// ---------------------------------------------------------------------------
// backward: elementwise with row scalars; a CTA writes the formula for unlisted columns over its piece of
// the row and then the listed columns that lie in it
// ---------------------------------------------------------------------------
struct DistillBwdArgs {
    const void* logits;
    int64_t ld;
    const int64_t* index;
    const float* teacher;
    int top_k;
    const float* stats;
    const float* dloss;
    void* dlogits;
    int64_t out_ld;
    int cols;
    int pieces;
    int chunks;
    float inv_t;
    int* status;
};

template <typename T, bool VECTOR>
__global__ void __launch_bounds__(kBwdThreads, 6) distill_topk_bwd_kernel(const DistillBwdArgs a) {
    __shared__ int column[kMaxList];
    const int64_t row = blockIdx.x / a.pieces;
    const int piece = static_cast<int>(blockIdx.x % a.pieces);
    const int tid = threadIdx.x;
    const RowMap<T, kBwdThreads, kUnroll, VECTOR> map(static_cast<const T*>(a.logits) + row * a.ld,
                                                   static_cast<T*>(a.dlogits) + row * a.out_ld, a.cols, piece, a.chunks);
    const float* s = a.stats + row * kStats;
    const float all_m = s[0], all_log = s[1], tail_m = s[2], tail_log = s[3], log_norm = s[4], rest = s[5];
    const float k2 = a.inv_t * kLog2e;
    float g = a.dloss[row] * a.inv_t;
    uint4 v[kUnroll];
    map.first_chunk(v);

    // this thread's list entry: its column, the student's logit there (before anything is written: the
    // gradient may take the logits' place) and whether the column lies in this CTA's piece
    const int64_t given = tid < a.top_k ? a.index[row * a.top_k + tid] : -1;
    const bool bad = given >= a.cols;
    const int c = given < 0 || bad ? -1 : static_cast<int>(given);
    const bool mine = c >= 0 && map.holds(c);
    const float listed = mine ? Vec<T>::load(map.x + c) : 0.0f;
    if (tid < kMaxList) column[tid] = c;
    // also the barrier between the loads above and the first write
    const bool any = __syncthreads_or(c >= 0), outside = __syncthreads_or(bad);

    // no teacher, or no unmasked logit: no gradient
    const bool zero = (!any && !outside) || all_m == -CUDART_INF_F;
    if (outside) {
        if (piece == 0 && tid == 0) atomicOr(a.status, kStatusBadIndex);
        g = CUDART_NAN_F;
    }
    if (is_broken(all_m)) g = CUDART_NAN_F;
    // outside the list: exp(z - tail lse) * (q_r - w_r); tail_m = -inf says that every such logit is masked
    const float factor = g * (ex2_approx((tail_m - all_m) * k2 + (tail_log - all_log) * kLog2e) - rest);
    const float base = tail_m == -CUDART_INF_F ? 0.0f : tail_m, log2_sum = tail_log * kLog2e;
    const float2 minus = make_float2(-base, -base), scale = make_float2(k2, k2), shift = make_float2(-log2_sum, -log2_sum),
                 by = make_float2(factor, factor);
    map.run(zero, v, [&](float2 z) {
        const float2 d = __ffma2_rn(__fadd2_rn(z, minus), scale, shift);
        return __fmul2_rn(make_float2(ex2_approx(d.x), ex2_approx(d.y)), by);
    });
    if (zero) return;
    __syncthreads();   // the piece is written; the listed columns follow
    if (mine) {
        // A renormalised list's log normaliser is saved in 32 bits. Where they resolve less than 2^-21 of a weight it is
        // taken again, from differences to the list's largest value.
        float base = log_norm, norm = 1.0f;
        if (fabsf(log_norm) >= 8.0f) {
            base = -CUDART_INF_F;
#pragma unroll 1
            for (int k = 0; k < a.top_k; ++k)
                if (column[k] >= 0) base = fmaxf(base, a.teacher[row * a.top_k + k]);
            float sum = 0.0f;
#pragma unroll 1
            for (int k = 0; k < a.top_k; ++k)
                if (column[k] >= 0) sum += expf(a.teacher[row * a.top_k + k] - base);
            norm = 1.0f / sum;
        }
        // a column that appears more than once: the first place writes for all, in list order
        float w = 0.0f;
        bool earlier = false;
        for (int k = 0; k < a.top_k; ++k) {
            if (column[k] == c) {
                earlier |= k < tid;
                w += expf(a.teacher[row * a.top_k + k] - base);
            }
        }
        const float q = ex2_approx(fmaf(listed - all_m, k2, -all_log * kLog2e));
        if (!earlier) Vec<T>::store(map.out + c, g * (q - w * norm));
    }
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------
int check_list(const int64_t* index, const float* teacher, int top_k, int64_t rows) {
    if (top_k < 1 || top_k > kMaxList)
        return report_error(CREDIT_ERR_INVALID_ARGUMENT, "top_k must be in [1, %d] (got %d)", kMaxList, top_k);
    if (rows != 0 && (index == nullptr || teacher == nullptr))
        return report_error(CREDIT_ERR_INVALID_ARGUMENT, "teacher_index and teacher_logprob must not be NULL");
    if (!aligned_to(index, sizeof(int64_t)) || !aligned_to(teacher, sizeof(float)))
        return report_error(CREDIT_ERR_INVALID_ARGUMENT, "teacher_index and teacher_logprob must be aligned to their elements");
    return CREDIT_OK;
}

int forward(const void* logits, int64_t ld, const int64_t* index, const float* teacher, int top_k, float* loss,
            float* stats, int64_t rows, int64_t cols, float temperature, int tail, int dtype,
            const credit_launch_opts* opts, void* stream) {
    int rc = check_logits(logits, ld, rows, cols, temperature, dtype);
    if (rc == CREDIT_OK) rc = check_list(index, teacher, top_k, rows);
    int cluster = 0;
    if (rc == CREDIT_OK) rc = check_cluster_only(opts, &cluster);
    if (rc != CREDIT_OK) return rc;
    if (rows == 0) return CREDIT_OK;
    if (loss == nullptr || stats == nullptr)
        return report_error(CREDIT_ERR_INVALID_ARGUMENT, "loss and stats must not be NULL");
    if (!aligned_to({loss, stats}, sizeof(float)))
        return report_error(CREDIT_ERR_INVALID_ARGUMENT, "loss and stats must be aligned to their elements");
    DeviceContext ctx;
    rc = current_device_context(&ctx);
    if (rc != CREDIT_OK) return rc;
    const bool asked = cluster != 0;
    if (!asked) cluster = row_split(rows, cols, 8 * ctx.sm_count, 4096);
    DistillArgs a;
    a.logits = logits;
    a.ld = ld;
    a.index = index;
    a.teacher = teacher;
    a.top_k = top_k;
    a.loss = loss;
    a.stats = stats;
    a.cols = static_cast<int>(cols);
    a.inv_t = 1.0f / temperature;
    a.status = ctx.status;
    void* args[] = {&a};
    a.slice = row_slice(cols, cluster);
    const int vec = dtype == CREDIT_BF16 ? 8 : 4;
    if (tail != 0) {   // the map of a slice: at most 128 KiB
        while (map_words(a.slice, vec) > 32 * 1024 + 4) {
            if (asked)
                return report_error(CREDIT_ERR_UNSUPPORTED, "cols=%lld: with a tail a row this wide needs a larger cluster than %d",
                                    static_cast<long long>(cols), cluster);
            cluster *= 2;
            a.slice = row_slice(cols, cluster);
        }
    }
    a.map_words = tail != 0 ? map_words(a.slice, vec) : 0;
    const void* func;
    if (dtype == CREDIT_BF16)
        func = tail ? reinterpret_cast<const void*>(&distill_topk_kernel<__nv_bfloat16, true>)
                    : reinterpret_cast<const void*>(&distill_topk_kernel<__nv_bfloat16, false>);
    else
        func = tail ? reinterpret_cast<const void*>(&distill_topk_kernel<float, true>)
                    : reinterpret_cast<const void*>(&distill_topk_kernel<float, false>);
    rc = prepare_kernel(ctx, func);
    if (rc != CREDIT_OK) return rc;
    return launch_kernel(func, rows * cluster, kThreads, cluster, a.map_words * 4, stream, args);
}

int backward(const void* logits, int64_t ld, const int64_t* index, const float* teacher, int top_k, const float* stats,
             const float* dloss, void* dlogits, int64_t out_ld, int64_t rows, int64_t cols, float temperature, int dtype,
             const credit_launch_opts* opts, void* stream) {
    int rc = check_logits(logits, ld, rows, cols, temperature, dtype);
    if (rc == CREDIT_OK) rc = check_gradient(logits, ld, dlogits, out_ld, rows, cols, dtype);
    if (rc == CREDIT_OK) rc = check_list(index, teacher, top_k, rows);
    int cluster = 0;
    if (rc == CREDIT_OK) rc = check_cluster_only(opts, &cluster);
    if (rc != CREDIT_OK) return rc;
    if (cluster > 1)
        return report_error(CREDIT_ERR_INVALID_ARGUMENT, "the gradient is elementwise: cluster_size must be 0 or 1");
    if (rows == 0) return CREDIT_OK;
    if (stats == nullptr || dloss == nullptr)
        return report_error(CREDIT_ERR_INVALID_ARGUMENT, "stats and dloss must not be NULL");
    if (!aligned_to({stats, dloss}, sizeof(float)))
        return report_error(CREDIT_ERR_INVALID_ARGUMENT, "stats and dloss must be aligned to their elements");
    DeviceContext ctx;
    rc = current_device_context(&ctx);
    if (rc != CREDIT_OK) return rc;
    DistillBwdArgs a;
    a.logits = logits;
    a.ld = ld;
    a.index = index;
    a.teacher = teacher;
    a.top_k = top_k;
    a.stats = stats;
    a.dloss = dloss;
    a.dlogits = dlogits;
    a.out_ld = out_ld;
    a.cols = static_cast<int>(cols);
    a.inv_t = 1.0f / temperature;
    a.status = ctx.status;
    const bool vector = same_phase(logits, ld, dlogits, out_ld, rows, dtype);
    const int chunk = kBwdThreads * kUnroll * (dtype == CREDIT_BF16 ? 8 : 4);
    a.chunks = chunks_per_piece(rows, cols, chunk, 4, ctx.sm_count);   // 1, 2, 4, 8: 239, 190, 175, 184 us at 2048 x 131072 bf16
    a.pieces = static_cast<int>((cols + static_cast<int64_t>(chunk) * a.chunks - 1) / (static_cast<int64_t>(chunk) * a.chunks));
    const void* func;
    if (dtype == CREDIT_BF16)
        func = vector ? reinterpret_cast<const void*>(&distill_topk_bwd_kernel<__nv_bfloat16, true>)
                      : reinterpret_cast<const void*>(&distill_topk_bwd_kernel<__nv_bfloat16, false>);
    else
        func = vector ? reinterpret_cast<const void*>(&distill_topk_bwd_kernel<float, true>)
                      : reinterpret_cast<const void*>(&distill_topk_bwd_kernel<float, false>);
    rc = prepare_kernel(ctx, func);
    if (rc != CREDIT_OK) return rc;
    void* args[] = {&a};
    return launch_kernel(func, rows * a.pieces, kBwdThreads, 1, 0, stream, args);
}

}  // namespace
}  // namespace credit

extern "C" {

int credit_distill_topk_forward(const void* logits, int64_t row_stride, const int64_t* teacher_index,
                                const float* teacher_logprob, int top_k, float* loss, float* stats, int64_t rows,
                                int64_t cols, float temperature, int tail, int dtype, const credit_launch_opts* opts,
                                void* stream) {
    return credit::guarded([&] {
        return credit::forward(logits, row_stride, teacher_index, teacher_logprob, top_k, loss, stats, rows, cols,
                               temperature, tail, dtype, opts, stream);
    });
}

int credit_distill_topk_backward(const void* logits, int64_t row_stride, const int64_t* teacher_index,
                                 const float* teacher_logprob, int top_k, const float* stats, const float* dloss,
                                 void* dlogits, int64_t dlogits_row_stride, int64_t rows, int64_t cols, float temperature,
                                 int dtype, const credit_launch_opts* opts, void* stream) {
    return credit::guarded([&] {
        return credit::backward(logits, row_stride, teacher_index, teacher_logprob, top_k, stats, dloss, dlogits,
                                dlogits_row_stride, rows, cols, temperature, dtype, opts, stream);
    });
}

}  // extern "C"
