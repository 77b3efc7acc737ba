// The norms after and before a block, fused with the block's gate and the scaled residual:
//   n  = o * r1,  r1 = rsqrt(mean(o^2) + eps)         (n = o without a post norm)
//   h' = alpha * h + n * c,  c = post_weight * gate   (either may be absent)
//   y  = h' * r2 * pre_weight,  r2 = rsqrt(mean(h'^2) + eps)
// and its gradient. With v = h' r2, t = dy * pre_weight, N columns:
//   D  = dh' + r2 (t - v mean(t v)),   dh = alpha * D
//   do = r1 (D c - n mean(D c n))      (D c without a post norm)
//   dpre_weight = sum_rows dy v;  with C = sum_rows D n:  dpost_weight = gate * C, dgate = post_weight * C
// No reference kernel exists for these; rows are split over a cluster and the partial sums meet in
// distributed shared memory as in cluster_bwd_staged_kernel (src/workloads/layernorm_backward.cu:376-438).
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cmath>
#include <type_traits>

#include "device_context.h"
#include "vocab_rows.cuh"

namespace credit {
namespace {

// A persistent cluster walks rows cluster, cluster + clusters, ... Its CTAs own fixed columns, 32 bytes' worth a
// thread, whose parameters (and, in the backward pass, sums over the rows) stay in registers. The rows come
// through a ring of shared-memory stages filled by bulk copies, so the next rows are on their way while one is
// reduced. A row step has one barrier. HBM bounds both directions (4 and 6 matrices move, some 10 and 26 flops an
// element): bf16 on one B200, forward 16384 x 8192 168 us = 6.4 TB/s replayed from a graph, 189 us = 5.7 TB/s in a long
// loop over changing inputs (without post norm and gate 190 us replayed); backward 16384 x 4096 136 us = 5.9 TB/s and
// 154 us = 5.2 TB/s, where three stages of four inputs are what fits. Unaligned rows are bound by their instructions, one
// element at a time: fp32 backward 2049 x 5003 66 us = 3.7 TB/s (loop 68), bf16 16384 x 5003 forward 242 us, backward 339.
constexpr int kMaxRing = 8;

template <typename T>
constexpr int kThreadElems = 32 / sizeof(T);   // a thread's columns

struct RingArgs {
    int rows;
    int cols;
    int slice;        // columns per CTA
    int slot_bytes;   // one input's slice in a stage
    int stages;
};

// How one input's slice of a row lies: it is copied into its slot in whole 16-byte pieces, at the place that has
// the same alignment, with what else those pieces hold. Only where a piece would reach over the matrix's first or
// last byte is it left out; the few elements of it are then patched in (the first and last row).
template <typename T>
struct SliceSource {
    const T* row;   // first element of the slice in this row
    int shift;      // its distance from a 16-byte boundary, in elements
    int head, body_end;   // elements [head, body_end) come with the copy
    uint32_t bytes;       // of the copy
    int from;             // its first element (-shift, or head)

    __device__ __forceinline__ SliceSource(const void* base, int64_t offset, int local, int64_t matrix) {
        constexpr int E = 16 / sizeof(T);
        row = static_cast<const T*>(base) + offset;
        shift = static_cast<int>((reinterpret_cast<uintptr_t>(row) & 15u) / sizeof(T));
        const int behind = (E - (shift + local) % E) % E;   // to the next boundary
        const bool first = offset >= shift, last = offset + local + behind <= matrix;
        head = first || shift == 0 ? 0 : min(E - shift, local);
        body_end = last ? local : max(head, local - (E - behind) % E);
        from = first ? -shift : head;
        const int to = last ? local + behind : body_end;
        bytes = body_end > head ? static_cast<uint32_t>(to - from) * sizeof(T) : 0;
        if (bytes == 0) body_end = head;
    }
    __device__ __forceinline__ bool complete(int local) const { return head == 0 && body_end == local; }
    // by all threads, when incomplete: the elements that the copy left out
    __device__ __forceinline__ void patch(unsigned char* slot, int local) const {
        T* at = reinterpret_cast<T*>(slot) + shift;
        for (int e = threadIdx.x; e < head; e += blockDim.x) at[e] = row[e];
        for (int e = body_end + threadIdx.x; e < local; e += blockDim.x) at[e] = row[e];
    }
};

// By one warp: the IN slices of a row into `stage` (a NULL input is left out), one bulk copy each: the
// same bytes in pieces of 4 KiB or 1 KiB cost 12 % or 50 % more time at 16384 x 8192 bf16.
template <typename T, int IN>
__device__ __forceinline__ void fill_stage(const void* const (&in)[IN], unsigned char* stage, uint64_t* full, int64_t offset,
                                           int local, int64_t matrix, int slot_bytes) {
    const int lane = threadIdx.x & 31, which = lane % IN;
    const void* mine = in[0];
#pragma unroll
    for (int i = 1; i < IN; ++i)
        if (which == i) mine = in[i];
    const SliceSource<T> s(mine, offset, local, matrix);
    const uint32_t bytes = mine != nullptr ? s.bytes : 0;
    const uint32_t total = __reduce_add_sync(0xffffffffu, lane < IN ? bytes : 0u);
    const uint32_t bar = smem_u32(full);
    if (lane == 0) mbar_arrive_expect_tx(bar, total);
    __syncwarp();
    if (lane < IN && bytes != 0)
        bulk_load(smem_u32(stage + which * slot_bytes) + (s.shift + s.from) * sizeof(T), s.row + s.from, bytes, bar);
}

// W consecutive columns of one input.
template <typename T, int W>
__device__ __forceinline__ void slot_elems(const T* at, float (&x)[W]) {
    if constexpr (W == 1) {
        x[0] = Vec<T>::load(at);
    } else {
        Vec<T>::unpack(*reinterpret_cast<const uint4*>(at), x);
    }
}

template <typename T, int W>
__device__ __forceinline__ void store_elems(T* p, const float (&x)[W]) {
    if constexpr (W == 1) {
        Vec<T>::store(p, x[0]);
    } else if constexpr (W * sizeof(T) == 32) {
        __stcs(reinterpret_cast<float4*>(p), make_float4(x[0], x[1], x[2], x[3]));
        __stcs(reinterpret_cast<float4*>(p) + 1, make_float4(x[4], x[5], x[6], x[7]));
    } else {
        __stcs(reinterpret_cast<uint4*>(p), Vec<T>::pack(x));
    }
}

template <int W>
__device__ __forceinline__ void load_params(const float* p, float (&x)[W]) {
    if constexpr (W == 1) {
        x[0] = __ldg(p);
    } else {
#pragma unroll
        for (int j = 0; j < W; j += 4) ldg_f32x4(p + j, x + j);
    }
}

// c = post_weight * gate of W columns.
template <int W>
__device__ __forceinline__ void load_channel_scale(const float* post_weight, const float* gate, int column, float (&c)[W]) {
#pragma unroll
    for (int j = 0; j < W; ++j) c[j] = 1.0f;
    if (post_weight != nullptr) load_params<W>(post_weight + column, c);
    if (gate != nullptr) {
        float g[W];
        load_params<W>(gate + column, g);
#pragma unroll
        for (int j = 0; j < W; ++j) c[j] *= g[j];
    }
}

// Sums of K = 2 or 4 partials over the CTA and the cluster, in every thread, added in a fixed order, in two
// halves: publish (one CTA barrier; in a cluster every CTA then sends its sums to every other, counted on the
// receiver's mbarrier) and collect. Two buffers: a step's publish may overtake a slow thread's collect of the step
// before, not of the one before that.
template <int K, int THREADS>
struct alignas(16) RowSums {
    float warp[2][THREADS / 32][K];
    float peer[2][kMaxClusterSize][K];
    uint64_t arrived[2];
};

template <int K>
struct SumsOf { using Packed = float4; };
template <>
struct SumsOf<2> { using Packed = float2; };

__device__ __forceinline__ void add_to(float2& a, const float2& b) { a.x += b.x; a.y += b.y; }
__device__ __forceinline__ void add_to(float4& a, const float4& b) { a.x += b.x; a.y += b.y; a.z += b.z; a.w += b.w; }

// Half the lanes go on with one of two values, the other half with the other.
__device__ __forceinline__ float fold(float a, float b, int distance) {
    const bool second = threadIdx.x & distance;
    return (second ? b : a) + __shfl_xor_sync(0xffffffffu, second ? a : b, distance);
}

template <int K, int THREADS>
__device__ __forceinline__ typename SumsOf<K>::Packed cta_sums(const RowSums<K, THREADS>& s, int buf) {
    typename SumsOf<K>::Packed t{};
#pragma unroll
    for (int w = 0; w < THREADS / 32; ++w) add_to(t, *reinterpret_cast<const typename SumsOf<K>::Packed*>(s.warp[buf][w]));
    return t;
}

template <int K, int THREADS>
__device__ __forceinline__ void publish_sums(const float (&v)[K], RowSums<K, THREADS>& s, int buf, uint32_t rank,
                                             uint32_t nranks) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    float t;
    if constexpr (K == 4) {
        t = fold(fold(v[0], v[2], 16), fold(v[1], v[3], 16), 8);
    } else {
        t = fold(v[0], v[1], 16);
        t += __shfl_xor_sync(0xffffffffu, t, 8);
    }
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
    if ((lane & (K == 4 ? 7 : 15)) == 0) s.warp[buf][warp][lane / (32 / K)] = t;
    __syncthreads();
    if (nranks > 1 && warp == 0) {
        const uint32_t bar = smem_u32(&s.arrived[buf]);
        if (lane == 0) mbar_arrive_expect_tx(bar, nranks * K * 4);
        const auto p = cta_sums<K, THREADS>(s, buf);
        if (lane < static_cast<int>(nranks)) {
            const uint32_t to = map_to_rank(smem_u32(s.peer[buf][rank]), lane), to_bar = map_to_rank(bar, lane);
            if constexpr (K == 4) {
                st_async_f32x4(to, p.x, p.y, p.z, p.w, to_bar);
            } else {
                st_async_f32x2(to, p.x, p.y, to_bar);
            }
        }
    }
}

template <int K, int THREADS>
__device__ __forceinline__ typename SumsOf<K>::Packed collect_sums(RowSums<K, THREADS>& s, int buf, uint32_t parity,
                                                                   uint32_t nranks, int* status) {
    if (nranks == 1) return cta_sums<K, THREADS>(s, buf);
    mbar_wait_bounded(smem_u32(&s.arrived[buf]), parity, status);
    typename SumsOf<K>::Packed t{};
    for (uint32_t r = 0; r < nranks; ++r) add_to(t, *reinterpret_cast<const typename SumsOf<K>::Packed*>(s.peer[buf][r]));
    return t;
}

// What both directions set up: this CTA's place, its ring and its barriers.
template <typename T, int IN>
struct RowWalk {
    const RingArgs& a;
    uint32_t rank, nranks;
    int cluster, clusters;
    int start, local;
    int steps;               // rows of this cluster
    int64_t matrix;          // elements
    unsigned char* ring;
    uint64_t* full;

    __device__ __forceinline__ RowWalk(const RingArgs& args, unsigned char* ring_, uint64_t* full_) : a(args), ring(ring_), full(full_) {
        rank = cluster_cta_rank();
        nranks = cluster_cta_count();
        cluster = static_cast<int>(blockIdx.x / nranks);
        clusters = static_cast<int>(gridDim.x / nranks);
        start = static_cast<int>(rank) * a.slice;
        local = max(0, min(a.slice, a.cols - start));
        steps = (a.rows - cluster + clusters - 1) / clusters;
        matrix = static_cast<int64_t>(a.rows) * a.cols;
    }
    __device__ __forceinline__ int64_t row(int step) const { return cluster + static_cast<int64_t>(step) * clusters; }
    __device__ __forceinline__ int64_t offset(int step) const { return row(step) * a.cols + start; }
    __device__ __forceinline__ unsigned char* stage(int i) const { return ring + i * (IN * a.slot_bytes); }
    __device__ __forceinline__ SliceSource<T> source(const void* in, int step) const { return {in, offset(step), local, matrix}; }
    // Waits for a row's stage; PATCH: rows may be unaligned. All threads. places[k]: the slice of input k.
    template <bool PATCH>
    __device__ __forceinline__ void wait(const void* const (&in)[IN], const RingCursor& at, int step, const T* (&places)[IN],
                                         int* status) const {
        mbar_wait_bounded(smem_u32(&full[at.stage]), at.parity, status);
#pragma unroll
        for (int k = 0; k < IN; ++k) places[k] = reinterpret_cast<const T*>(stage(at.stage) + k * a.slot_bytes);
        if (PATCH) {
#pragma unroll
            for (int k = 0; k < IN; ++k)
                places[k] += (static_cast<uint32_t>(reinterpret_cast<uintptr_t>(in[k])) + static_cast<uint32_t>(offset(step)) * sizeof(T)) %
                             16u / sizeof(T);
            // only a slice at the very start or end of the matrix can lack elements
            if (offset(step) < 16 || offset(step) + local + 16 > matrix) patch(in, at.stage, step);
        }
    }
    __device__ __forceinline__ void patch(const void* const (&in)[IN], int i, int step) const {
#pragma unroll
        for (int k = 0; k < IN; ++k)
            if (in[k] != nullptr) {
                const SliceSource<T> s = source(in[k], step);
                if (!s.complete(local)) s.patch(stage(i) + k * a.slot_bytes, local);
            }
        fence_proxy_async_smem();   // a later copy into this stage follows these stores
        __syncthreads();
    }
    // by warp 0
    __device__ __forceinline__ void fill(const void* const (&in)[IN], int i, int step) const {
        if (step < steps) fill_stage<T, IN>(in, stage(i), &full[i], offset(step), local, matrix, a.slot_bytes);
    }
    __device__ __forceinline__ void init(const void* const (&in)[IN], uint64_t (&arrived)[2]) const {
        if (threadIdx.x == 0) {
            for (int i = 0; i < a.stages; ++i) mbar_init(smem_u32(&full[i]), 1);
            mbar_init(smem_u32(&arrived[0]), 1);
            mbar_init(smem_u32(&arrived[1]), 1);
            fence_mbar_init();
        }
        __syncwarp();
        if (threadIdx.x < 32)
            for (int i = 0; i < a.stages; ++i) fill(in, i, i);
    }
};

struct NormFwdArgs {
    RingArgs ring;
    const void* block;
    const void* residual;
    const float* post_weight;
    const float* gate;
    const float* pre_weight;
    void* residual_out;
    void* y;
    float* post_rstd;
    float* pre_rstd;
    float alpha;
    float eps;
    int* status;
};

// ---------------------------------------------------------------------------
// forward: step i joins row i, squares row i + 1's block and writes row i - 1's y, so the two reductions that
// depend on each other share an exchange with those of the neighbouring rows (two exchanges a row: 195 us)
// ---------------------------------------------------------------------------
template <typename T, int W, int THREADS, bool POST>
__global__ void __launch_bounds__(THREADS, 512 / THREADS) residual_norm_kernel(const NormFwdArgs a) {
    constexpr int N = kThreadElems<T> / W, kStride = THREADS * W;
    __shared__ uint64_t full[kMaxRing];
    __shared__ RowSums<2, THREADS> sums;
    extern __shared__ __align__(128) unsigned char ring[];
    const RowWalk<T, 2> walk(a.ring, ring, full);
    const void* in[2] = {a.block, a.residual};
    walk.init(in, sums.arrived);
    const int local = walk.local, e0 = static_cast<int>(threadIdx.x) * W;
    float c[N][W], w[N][W];
#pragma unroll
    for (int u = 0; u < N; ++u) {
        const int e = e0 + u * kStride;
#pragma unroll
        for (int j = 0; j < W; ++j) c[u][j] = w[u][j] = 0.0f;
        if (e < local) {
            load_channel_scale<W>(a.post_weight, a.gate, walk.start + e, c[u]);
            load_params<W>(a.pre_weight + walk.start + e, w[u]);
        }
    }
    __syncthreads();
    if (walk.nranks > 1) cluster_sync_all();

    const float inv_n = 1.0f / static_cast<float>(a.ring.cols);
    RingCursor at{0, 0}, next{0, 0};
    // sum of squares of a step's block
    const T* ahead[2];
    auto squares = [&](int step) {
        float q = 0.0f;
        walk.template wait<W == 1>(in, next, step, ahead, a.status);
        if (POST) {
#pragma unroll
            for (int u = 0; u < N; ++u) {
                const int e = e0 + u * kStride;
                if (e < local) {
                    float o[W];
                    slot_elems<T, W>(ahead[0] + e, o);
#pragma unroll
                    for (int j = 0; j < W; ++j) q = fmaf(o[j], o[j], q);
                }
            }
        }
        next.advance(a.ring.stages);
        return q;
    };
    float before[N][W];   // the joined row of the step before
    auto write_y = [&](int step, float square_sum) {
        const float r2 = rsqrtf(fmaf(square_sum, inv_n, a.eps));
        T* y = static_cast<T*>(a.y) + walk.offset(step);
#pragma unroll
        for (int u = 0; u < N; ++u) {
            const int e = e0 + u * kStride;
#pragma unroll
            for (int j = 0; j < W; ++j) before[u][j] *= r2 * w[u][j];
            if (e < local) store_elems<T, W>(y + e, before[u]);
        }
        if (walk.rank == 0 && threadIdx.x == 0) a.pre_rstd[walk.row(step)] = r2;
    };
    {
        const float first[2] = {0.0f, squares(0)};
        publish_sums(first, sums, 0, walk.rank, walk.nranks);
    }
    for (int i = 0; i < walk.steps; ++i) {
        const float2 total = collect_sums(sums, i & 1, (i >> 1) & 1, walk.nranks, a.status);
        const float r1 = POST ? rsqrtf(fmaf(total.y, inv_n, a.eps)) : 1.0f;
        const int64_t offset = walk.offset(i);
        const T *block = ahead[0], *residual = ahead[1];
        T* out = static_cast<T*>(a.residual_out) + offset;
        float h[N][W], part[2] = {0.0f, 0.0f};
#pragma unroll
        for (int u = 0; u < N; ++u) {
            const int e = e0 + u * kStride;
            float o[W];
#pragma unroll
            for (int j = 0; j < W; ++j) o[j] = h[u][j] = 0.0f;
            if (e < local) {
                slot_elems<T, W>(block + e, o);
                slot_elems<T, W>(residual + e, h[u]);
            }
#pragma unroll
            for (int j = 0; j < W; ++j) {
                h[u][j] = fmaf(a.alpha, h[u][j], o[j] * r1 * c[u][j]);
                part[0] = fmaf(h[u][j], h[u][j], part[0]);
            }
            // stored rounded to the rows' type; y continues from the unrounded sum
            if (e < local) store_elems<T, W>(out + e, h[u]);
        }
        if (POST && walk.rank == 0 && threadIdx.x == 0) a.post_rstd[walk.row(i)] = r1;
        if (i + 1 < walk.steps) part[1] = squares(i + 1);
        publish_sums(part, sums, (i + 1) & 1, walk.rank, walk.nranks);
        if (threadIdx.x < 32) walk.fill(in, at.stage, i + a.ring.stages);   // everyone has read this stage
        at.advance(a.ring.stages);
        if (i > 0) write_y(i - 1, total.x);
#pragma unroll
        for (int u = 0; u < N; ++u)
#pragma unroll
            for (int j = 0; j < W; ++j) before[u][j] = h[u][j];
    }
    const float2 total = collect_sums(sums, walk.steps & 1, (walk.steps >> 1) & 1, walk.nranks, a.status);
    write_y(walk.steps - 1, total.x);
    if (walk.nranks > 1) cluster_sync_all();   // no CTA leaves while a peer may still send to it
}

// ---------------------------------------------------------------------------
// backward: a row's sums, one exchange, its gradients from the registers (taking the next row's sums in between
// leaves one stage in flight: 170 instead of 149 us)
// ---------------------------------------------------------------------------
struct NormBwdArgs {
    RingArgs ring;
    const void* dy;
    const void* dresidual_out;   // NULL: zero
    const void* block;
    const void* residual_out;
    const float* post_weight;
    const float* gate;
    const float* pre_weight;
    const float* post_rstd;
    const float* pre_rstd;
    void* dblock;
    void* dresidual;
    float* partials;             // [clusters][2][cols]: C, then dpre_weight
    float alpha;
    int* status;
};

// One exchange per row: with D = d + r2 (t - v m), m = mean(t v), the second mean is linear in m,
//   mean(D c n) = (sum c n d + r2 sum c n t - r2 m sum c n v) / N,
// so its three sums travel with sum t v.
template <typename T, int W, int THREADS, bool POST>
__global__ void __launch_bounds__(THREADS, 512 / THREADS) residual_norm_bwd_kernel(const NormBwdArgs a) {
    constexpr int N = kThreadElems<T> / W, kStride = THREADS * W;
    __shared__ uint64_t full[kMaxRing];
    __shared__ RowSums<4, THREADS> sums;
    extern __shared__ __align__(128) unsigned char ring[];
    const RowWalk<T, 4> walk(a.ring, ring, full);
    const void* in[4] = {a.dy, a.block, a.residual_out, a.dresidual_out};
    walk.init(in, sums.arrived);
    const int local = walk.local, e0 = static_cast<int>(threadIdx.x) * W;
    const bool has_d = a.dresidual_out != nullptr;
    float c[N][W], w[N][W], col_c[N][W], col_w[N][W];
#pragma unroll
    for (int u = 0; u < N; ++u) {
        const int e = e0 + u * kStride;
        if (W == 1 && sizeof(T) == 2 && u * kStride >= local) break;   // 374 -> 338 us at 16384 x 5003
#pragma unroll
        for (int j = 0; j < W; ++j) c[u][j] = w[u][j] = col_c[u][j] = col_w[u][j] = 0.0f;
        if (e < local) {
            load_channel_scale<W>(a.post_weight, a.gate, walk.start + e, c[u]);
            load_params<W>(a.pre_weight + walk.start + e, w[u]);
        }
    }
    // the rows' rstd: cold lines, fetched a step ahead of their first use
    float r1_next = POST ? a.post_rstd[walk.row(0)] : 1.0f, r2_next = a.pre_rstd[walk.row(0)];
    __syncthreads();
    if (walk.nranks > 1) cluster_sync_all();

    const float inv_n = 1.0f / static_cast<float>(a.ring.cols);
    RingCursor at{0, 0};
    // A row that fits the registers between the two passes leaves its stage free for the next one (149 -> 146 us);
    // unaligned bf16 rows, 16 single elements a thread, do not and are read twice.
    constexpr bool kKeep = W > 1 || sizeof(T) == 4;
    using Raw = std::conditional_t<(W > 1), uint4, T>;
    Raw kept[kKeep ? N : 1][4];
    const T* places[4];
    // W columns of the four inputs, as they are
    auto fetch = [&](int e, Raw (&raw)[4]) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            raw[k] = Raw{};
            if (k < 3 || has_d) raw[k] = *reinterpret_cast<const Raw*>(places[k] + e);
        }
    };
    auto widen = [&](const Raw& raw, float (&x)[W]) {
        if constexpr (W > 1) {
            Vec<T>::unpack(raw, x);
        } else {
            x[0] = Vec<T>::load(&raw);
        }
    };
    // a row's partial sums (with the rstd that *_next hold), and its part of dpre_weight
    auto reduce_row = [&](int step, float (&part)[4]) {
        walk.template wait<W == 1>(in, at, step, places, a.status);
#pragma unroll
        for (int k = 0; k < 4; ++k) part[k] = 0.0f;
#pragma unroll
        for (int u = 0; u < N; ++u) {
            const int e = e0 + u * kStride;
            if (W == 1 && sizeof(T) == 2 && u * kStride >= local) break;
            if (e < local) {
                Raw mine[4];
                fetch(e, mine);
                float dy[W], n[W], v[W], d[W];
                widen(mine[0], dy);
                widen(mine[1], n);
                widen(mine[2], v);
                widen(mine[3], d);
#pragma unroll
                for (int j = 0; j < W; ++j) {
                    v[j] *= r2_next;
                    const float t = dy[j] * w[u][j];
                    part[0] = fmaf(t, v[j], part[0]);
                    if (POST) {
                        const float cn = c[u][j] * (n[j] * r1_next);
                        part[1] = fmaf(cn, d[j], part[1]);
                        part[2] = fmaf(cn, t, part[2]);
                        part[3] = fmaf(cn, v[j], part[3]);
                    }
                    col_w[u][j] = fmaf(dy[j], v[j], col_w[u][j]);
                }
                if constexpr (kKeep) {
#pragma unroll
                    for (int k = 0; k < 4; ++k) kept[u][k] = mine[k];
                }
            }
        }
    };
    float part[4];
    int last = -1;   // stage of the row before
    for (int i = 0; i < walk.steps; ++i) {
        reduce_row(i, part);
        publish_sums(part, sums, i & 1, walk.rank, walk.nranks);
        if (kKeep) {   // the row is in registers
            if (threadIdx.x < 32) walk.fill(in, at.stage, i + a.ring.stages);
        } else if (threadIdx.x < 32 && last >= 0) {   // everyone is done with the row before
            walk.fill(in, last, i - 1 + a.ring.stages);
        }
        const float r1 = r1_next, r2 = r2_next;
        if (i + 1 < walk.steps) {
            if (POST) r1_next = a.post_rstd[walk.row(i + 1)];
            r2_next = a.pre_rstd[walk.row(i + 1)];
        }
        const float4 total = collect_sums(sums, i & 1, (i >> 1) & 1, walk.nranks, a.status);
        const float m1 = total.x * inv_n;
        const float m2 = POST ? (total.y + r2 * (total.z - m1 * total.w)) * inv_n : 0.0f;
        const int64_t offset = walk.offset(i);
#pragma unroll
        for (int u = 0; u < N; ++u) {
            const int e = e0 + u * kStride;
            if (W == 1 && sizeof(T) == 2 && u * kStride >= local) break;
            if (e < local) {
                Raw mine[4];
                if constexpr (kKeep) {
#pragma unroll
                    for (int k = 0; k < 4; ++k) mine[k] = kept[u][k];
                } else {
                    fetch(e, mine);
                }
                float dy[W], n[W], v[W], d[W];
                widen(mine[0], dy);
                widen(mine[1], n);
                widen(mine[2], v);
                widen(mine[3], d);
#pragma unroll
                for (int j = 0; j < W; ++j) {
                    n[j] *= r1;
                    d[j] = fmaf(r2, fmaf(-v[j] * r2, m1, dy[j] * w[u][j]), d[j]);
                    col_c[u][j] = fmaf(d[j], n[j], col_c[u][j]);
                    n[j] = POST ? r1 * fmaf(-n[j], m2, c[u][j] * d[j]) : c[u][j] * d[j];
                    d[j] *= a.alpha;
                }
                store_elems<T, W>(static_cast<T*>(a.dblock) + offset + e, n);
                store_elems<T, W>(static_cast<T*>(a.dresidual) + offset + e, d);
            }
        }
        last = at.stage;
        at.advance(a.ring.stages);
    }
    // the finishing kernel may be set up while these are written; it waits for this grid's end
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    float* sums_out = a.partials + static_cast<size_t>(walk.cluster) * 2 * a.ring.cols + walk.start;
#pragma unroll
    for (int u = 0; u < N; ++u) {
        const int e = e0 + u * kStride;
        if (W == 1 && sizeof(T) == 2 && u * kStride >= local) break;
        if (e < local) {
            store_elems<float, W>(sums_out + e, col_c[u]);
            store_elems<float, W>(sums_out + a.ring.cols + e, col_w[u]);
        }
    }
    if (walk.nranks > 1) cluster_sync_all();   // no CTA leaves while a peer may still send to it
}

// Adds the clusters' column sums in a fixed order: 32 columns a CTA, 32 strands of clusters.
constexpr int kFinishCols = 32, kFinishStrands = 32;
__global__ void __launch_bounds__(kFinishCols* kFinishStrands)
    residual_norm_finish_kernel(const float* partials, int clusters, int cols, const float* post_weight, const float* gate,
                                float* dpost_weight, float* dgate, float* dpre_weight) {
    __shared__ float strand[2][kFinishStrands][kFinishCols];
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int lane = threadIdx.x % kFinishCols, s = threadIdx.x / kFinishCols;
    const int c = blockIdx.x * kFinishCols + lane;
    float both[2] = {0.0f, 0.0f};
    if (c < cols)
#pragma unroll 4
        for (int i = s; i < clusters; i += kFinishStrands) {
            const float* p = partials + static_cast<size_t>(i) * 2 * cols + c;
            both[0] += p[0];
            both[1] += p[cols];
        }
    strand[0][s][lane] = both[0];
    strand[1][s][lane] = both[1];
    __syncthreads();
    if (s > 1 || c >= cols) return;
    float sum = 0.0f;   // C in strand 0's warp, dpre_weight in strand 1's
#pragma unroll
    for (int i = 0; i < kFinishStrands; ++i) sum += strand[s][i][lane];
    if (s == 1) {
        dpre_weight[c] = sum;
    } else {
        if (dpost_weight != nullptr) dpost_weight[c] = gate != nullptr ? sum * gate[c] : sum;
        if (dgate != nullptr) dgate[c] = post_weight != nullptr ? sum * post_weight[c] : sum;
    }
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------
// One compiled form: threads, with the kernels of both directions, [post norm].
struct Form {
    int threads;
    const void* forward[2];
    const void* backward[2];
};

template <typename T, int W, int THREADS>
Form make_form() {
    return {THREADS,
            {reinterpret_cast<const void*>(&residual_norm_kernel<T, W, THREADS, false>),
             reinterpret_cast<const void*>(&residual_norm_kernel<T, W, THREADS, true>)},
            {reinterpret_cast<const void*>(&residual_norm_bwd_kernel<T, W, THREADS, false>),
             reinterpret_cast<const void*>(&residual_norm_bwd_kernel<T, W, THREADS, true>)}};
}

constexpr int kForms = 4;
template <typename T>
const Form* forms(bool vector) {
    constexpr int E = Vec<T>::kElems;
    static const Form with_vectors[kForms] = {make_form<T, E, 64>(), make_form<T, E, 128>(), make_form<T, E, 256>(),
                                              make_form<T, E, 512>()};
    static const Form with_scalars[kForms] = {make_form<T, 1, 64>(), make_form<T, 1, 128>(), make_form<T, 1, 256>(),
                                              make_form<T, 1, 512>()};
    return vector ? with_vectors : with_scalars;
}

struct Plan {
    DeviceContext ctx;
    const void* func;
    int threads, cluster, clusters, smem;
    RingArgs ring;
};

int round_to(int64_t v, int m) { return static_cast<int>((v + m - 1) / m * m); }

// The shape's part of a plan, without a device: cluster size, slice and threads. A CTA holds 16 KiB of a row (32
// bytes for each of 512 threads), so that three stages of four inputs fit an SM; the automatic cluster is the
// smallest that holds the row.
int plan_shape(int64_t cols, int dtype, bool vector, int asked, Plan* p, const Form** form) {
    const int size = element_bytes(dtype), each = 32 / size;
    const int64_t most = 512 * each;
    int cluster = asked;
    if (cluster == 0)
        for (cluster = 1; cluster < kMaxClusterSize && (cols + cluster - 1) / cluster > most; cluster *= 2) {}
    const int64_t slice = cluster == 1 ? cols : round_to((cols + cluster - 1) / cluster, 64);
    if (slice > most)
        return report_error(CREDIT_ERR_UNSUPPORTED, "cols=%lld: a cluster of %d holds at most %lld columns of a row",
                            static_cast<long long>(cols), cluster, static_cast<long long>(most) * cluster);
    const Form* f = dtype == CREDIT_BF16 ? forms<__nv_bfloat16>(vector) : forms<float>(vector);
    while (static_cast<int64_t>(f->threads) * each < slice) ++f;
    *form = f;
    p->threads = f->threads;
    p->cluster = cluster;
    p->ring.cols = static_cast<int>(cols);
    p->ring.slice = static_cast<int>(slice);
    p->ring.slot_bytes = round_to(slice * size + 32, 128);
    return CREDIT_OK;
}

// The rest of it: ring depth and grid. An SM runs 512 threads' worth of CTAs (their registers fill it), which share
// its shared memory.
int plan_launch(int64_t rows, const void* func, int inputs, Plan* p) {
    int rc = current_device_context(&p->ctx);
    if (rc != CREDIT_OK) return rc;
    p->func = func;
    rc = prepare_kernel(p->ctx, func);
    if (rc != CREDIT_OK) return rc;
    const int per_sm = 512 / p->threads;
    const int stage = inputs * p->ring.slot_bytes;
    const int room = p->ctx.max_dynamic_smem - 4096;                      // of one CTA alone
    const int share = (p->ctx.max_dynamic_smem + 1024) / per_sm - 4096;   // 1 KiB of it is the system's
    int stages = share / stage;
    if (stages < 3) stages = room / stage < 3 ? room / stage : 3;   // 16 KiB slots: never fewer than three
    stages = stages > kMaxRing ? kMaxRing : stages;
    p->ring.stages = stages;
    p->ring.rows = static_cast<int>(rows);
    p->smem = stages * stage;
    int resident = 0;
    rc = resident_clusters(p->ctx, func, p->cluster, p->smem, p->threads, &resident);
    if (rc != CREDIT_OK) return rc;
    p->clusters = static_cast<int>(rows < resident ? rows : resident);
    return CREDIT_OK;
}

bool any_null(std::initializer_list<const void*> pointers) {
    for (const void* p : pointers)
        if (p == nullptr) return true;
    return false;
}

bool rows_of_vectors(int64_t cols, int dtype) { return cols * element_bytes(dtype) % 16 == 0; }

// The bulk copies round a matrix's address down to 16 bytes by whole elements.
int check_alignment(std::initializer_list<const void*> matrices, std::initializer_list<const void*> vectors, int dtype) {
    if (!aligned_to(matrices, element_bytes(dtype)) || !aligned_to(vectors, sizeof(float)))
        return report_error(CREDIT_ERR_INVALID_ARGUMENT, "matrices and fp32 vectors must be aligned to their elements");
    return CREDIT_OK;
}

int forward(const void* block, const void* residual, const float* post_weight, const float* gate, const float* pre_weight,
            void* residual_out, void* y, float* post_rstd, float* pre_rstd, int64_t rows, int64_t cols, float alpha,
            float eps, int dtype, const credit_launch_opts* opts, void* stream) {
    int rc = check_matrix_shape(rows, cols, dtype);
    int asked = 0;
    if (rc == CREDIT_OK) rc = check_cluster_only(opts, &asked);
    if (rc != CREDIT_OK) return rc;
    if (!std::isfinite(alpha) || !(eps > 0.0f) || !std::isfinite(eps))
        return report_error(CREDIT_ERR_INVALID_ARGUMENT, "residual_scale must be finite, eps positive and finite");
    const bool vector = rows_of_vectors(cols, dtype) &&
                        aligned_to({block, residual, post_weight, gate, pre_weight, residual_out, y}, 16);
    const Form* form = nullptr;
    Plan p;
    rc = plan_shape(cols, dtype, vector, asked, &p, &form);
    if (rc != CREDIT_OK || rows == 0) return rc;
    if (any_null({block, residual, pre_weight, residual_out, y, pre_rstd}))
        return report_error(CREDIT_ERR_INVALID_ARGUMENT, "block, residual, pre_weight, residual_out, y and pre_rstd must not be NULL");
    if ((post_weight == nullptr) != (post_rstd == nullptr))
        return report_error(CREDIT_ERR_INVALID_ARGUMENT, "post_weight and post_rstd go together");
    if (y == residual_out) return report_error(CREDIT_ERR_INVALID_ARGUMENT, "y and residual_out must differ");
    rc = check_alignment({block, residual, residual_out, y}, {post_weight, gate, pre_weight, post_rstd, pre_rstd}, dtype);
    if (rc != CREDIT_OK) return rc;
    rc = plan_launch(rows, form->forward[post_weight != nullptr], 2, &p);
    if (rc != CREDIT_OK) return rc;
    NormFwdArgs a;
    a.ring = p.ring;
    a.block = block;
    a.residual = residual;
    a.post_weight = post_weight;
    a.gate = gate;
    a.pre_weight = pre_weight;
    a.residual_out = residual_out;
    a.y = y;
    a.post_rstd = post_rstd;
    a.pre_rstd = pre_rstd;
    a.alpha = alpha;
    a.eps = eps;
    a.status = p.ctx.status;
    void* args[] = {&a};
    return launch_kernel(p.func, static_cast<int64_t>(p.clusters) * p.cluster, p.threads, p.cluster, p.smem, stream, args);
}

size_t partial_bytes(const Plan& p) { return static_cast<size_t>(p.clusters) * 2 * p.ring.cols * sizeof(float); }

int plan_backward(int64_t rows, int64_t cols, int dtype, bool vector, bool post, int asked, Plan* p) {
    const Form* form = nullptr;
    int rc = plan_shape(cols, dtype, vector, asked, p, &form);
    if (rc != CREDIT_OK) return rc;
    return plan_launch(rows, form->backward[post], 4, p);
}

int backward(const void* dy, const void* dresidual_out, const void* block, const void* residual_out,
             const float* post_weight, const float* gate, const float* pre_weight, const float* post_rstd,
             const float* pre_rstd, void* dblock, void* dresidual, float* dpost_weight, float* dgate, float* dpre_weight,
             int64_t rows, int64_t cols, float alpha, int dtype, const credit_launch_opts* opts, void* workspace,
             size_t workspace_bytes, void* stream) {
    int rc = check_matrix_shape(rows, cols, dtype);
    int asked = 0;
    if (rc == CREDIT_OK) rc = check_cluster_only(opts, &asked);
    if (rc != CREDIT_OK) return rc;
    if (!std::isfinite(alpha)) return report_error(CREDIT_ERR_INVALID_ARGUMENT, "residual_scale must be finite");
    if (dpre_weight == nullptr || (post_weight == nullptr) != (dpost_weight == nullptr) || (gate == nullptr) != (dgate == nullptr))
        return report_error(CREDIT_ERR_INVALID_ARGUMENT, "every weight that is given needs a place for its gradient, and no other");
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (rows == 0) {   // sums over no rows
        for (float* p : {dpost_weight, dgate, dpre_weight})
            if (p != nullptr && cudaMemsetAsync(p, 0, static_cast<size_t>(cols) * sizeof(float), s) != cudaSuccess)
                return report_error(CREDIT_ERR_CUDA, "cudaMemsetAsync: %s", cudaGetErrorString(cudaGetLastError()));
        return CREDIT_OK;
    }
    if (any_null({dy, block, residual_out, pre_weight, pre_rstd, dblock, dresidual}))
        return report_error(CREDIT_ERR_INVALID_ARGUMENT,
                            "dy, block, residual_out, pre_weight, pre_rstd, dblock and dresidual must not be NULL");
    if ((post_weight == nullptr) != (post_rstd == nullptr))
        return report_error(CREDIT_ERR_INVALID_ARGUMENT, "post_weight and post_rstd go together");
    if (dblock == dresidual) return report_error(CREDIT_ERR_INVALID_ARGUMENT, "dblock and dresidual must differ");
    rc = check_alignment({dy, dresidual_out, block, residual_out, dblock, dresidual},
                         {post_weight, gate, pre_weight, post_rstd, pre_rstd, dpost_weight, dgate, dpre_weight}, dtype);
    if (rc != CREDIT_OK) return rc;
    const bool vector = rows_of_vectors(cols, dtype) && aligned_to({dy, dresidual_out, block, residual_out, post_weight, gate,
                                                                    pre_weight, dblock, dresidual}, 16);
    Plan p;
    rc = plan_backward(rows, cols, dtype, vector, post_weight != nullptr, asked, &p);
    if (rc != CREDIT_OK) return rc;
    if (workspace == nullptr || !aligned_to(workspace, 16) || workspace_bytes < partial_bytes(p))
        return report_error(CREDIT_ERR_WORKSPACE, "the call needs a 16-byte aligned workspace of %zu bytes (got %zu)",
                            partial_bytes(p), workspace == nullptr ? static_cast<size_t>(0) : workspace_bytes);
    NormBwdArgs a;
    a.ring = p.ring;
    a.dy = dy;
    a.dresidual_out = dresidual_out;
    a.block = block;
    a.residual_out = residual_out;
    a.post_weight = post_weight;
    a.gate = gate;
    a.pre_weight = pre_weight;
    a.post_rstd = post_rstd;
    a.pre_rstd = pre_rstd;
    a.dblock = dblock;
    a.dresidual = dresidual;
    a.partials = static_cast<float*>(workspace);
    a.alpha = alpha;
    a.status = p.ctx.status;
    void* args[] = {&a};
    rc = launch_kernel(p.func, static_cast<int64_t>(p.clusters) * p.cluster, p.threads, p.cluster, p.smem, stream, args);
    if (rc != CREDIT_OK) return rc;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>((p.ring.cols + kFinishCols - 1) / kFinishCols));
    cfg.blockDim = dim3(kFinishCols * kFinishStrands);
    cfg.stream = s;
    cudaLaunchAttribute early{};
    early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &early;
    cfg.numAttrs = 1;
    const float* partials = a.partials;
    const cudaError_t err = cudaLaunchKernelEx(&cfg, residual_norm_finish_kernel, partials, p.clusters, p.ring.cols, post_weight,
                                               gate, dpost_weight, dgate, dpre_weight);
    if (err != cudaSuccess) return report_error(CREDIT_ERR_CUDA, "column sums: %s", cudaGetErrorString(err));
    return CREDIT_OK;
}

// The larger of the vector and scalar forms, with and without a post norm: a workspace of this size
// serves every call of the shape.
size_t backward_workspace(int64_t rows, int64_t cols, int dtype, const credit_launch_opts* opts) {
    int asked = 0;
    if (check_matrix_shape(rows, cols, dtype) != CREDIT_OK || check_cluster_only(opts, &asked) != CREDIT_OK) return 0;
    size_t most = 0;
    for (int form = 0; form < 4; ++form) {
        const bool vector = form & 1;
        if (vector && !rows_of_vectors(cols, dtype)) continue;
        Plan p;
        if (plan_backward(rows, cols, dtype, vector, (form & 2) != 0, asked, &p) == CREDIT_OK && partial_bytes(p) > most)
            most = partial_bytes(p);
    }
    return most;
}

}  // namespace
}  // namespace credit

extern "C" {

int credit_residual_norm_forward(const void* block, const void* residual, const float* post_weight, const float* gate,
                                 const float* pre_weight, void* residual_out, void* y, float* post_rstd, float* pre_rstd,
                                 int64_t rows, int64_t cols, float residual_scale, float eps, int dtype,
                                 const credit_launch_opts* opts, void* stream) {
    return credit::guarded([&] {
        return credit::forward(block, residual, post_weight, gate, pre_weight, residual_out, y, post_rstd, pre_rstd, rows,
                               cols, residual_scale, eps, dtype, opts, stream);
    });
}

size_t credit_residual_norm_backward_workspace_bytes(int64_t rows, int64_t cols, int dtype, const credit_launch_opts* opts) {
    size_t bytes = 0;
    credit::guarded([&] {
        bytes = credit::backward_workspace(rows, cols, dtype, opts);
        return 0;
    });
    return bytes;
}

int credit_residual_norm_backward(const void* dy, const void* dresidual_out, const void* block, const void* residual_out,
                                  const float* post_weight, const float* gate, const float* pre_weight,
                                  const float* post_rstd, const float* pre_rstd, void* dblock, void* dresidual,
                                  float* dpost_weight, float* dgate, float* dpre_weight, int64_t rows, int64_t cols,
                                  float residual_scale, int dtype, const credit_launch_opts* opts, void* workspace,
                                  size_t workspace_bytes, void* stream) {
    return credit::guarded([&] {
        return credit::backward(dy, dresidual_out, block, residual_out, post_weight, gate, pre_weight, post_rstd, pre_rstd,
                                dblock, dresidual, dpost_weight, dgate, dpre_weight, rows, cols, residual_scale, dtype,
                                opts, workspace, workspace_bytes, stream);
    });
}

}  // extern "C"
