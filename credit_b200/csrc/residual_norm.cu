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

#include "device_context.h"
#include "vocab_rows.cuh"

namespace credit {
namespace {

// A persistent cluster walks rows cluster, cluster + clusters, ... Its CTAs own fixed columns, 16 a thread, whose
// parameters (and, in the backward pass, sums over the rows) stay in registers. The rows come through a ring of
// shared-memory stages filled by bulk copies, so the next rows are on their way while one is reduced.
constexpr int kElems = 16;      // a thread's columns
constexpr int kMaxRing = 8;

struct RingArgs {
    int rows;
    int cols;
    int slice;        // columns per CTA
    int slot_bytes;   // one input's slice in a stage
    int stages;
};

// How one input's slice of a row lies: its aligned body is copied into the slot, at the place that has the
// same alignment; elements before and behind it are read from global memory.
template <typename T>
struct SliceSource {
    const T* row;   // first element of the slice in this row
    int shift;      // its distance from a 16-byte boundary, in elements
    int head, body_end;

    __device__ __forceinline__ SliceSource(const void* base, int64_t offset, int local) {
        constexpr int E = 16 / sizeof(T);
        row = static_cast<const T*>(base) + offset;
        shift = static_cast<int>((reinterpret_cast<uintptr_t>(row) & 15u) / sizeof(T));
        head = shift == 0 ? 0 : min(E - shift, local);
        body_end = head + (local - head) / E * E;
    }
    __device__ __forceinline__ uint32_t body_bytes() const { return static_cast<uint32_t>(body_end - head) * sizeof(T); }
    __device__ __forceinline__ float element(const unsigned char* slot, int e) const {
        return e >= head && e < body_end ? Vec<T>::load(reinterpret_cast<const T*>(slot) + shift + e) : Vec<T>::load(row + e);
    }
};

// By one thread: the IN slices of `row` into `stage` (a NULL input is left out).
template <typename T, int IN>
__device__ __forceinline__ void fill_stage(const void* const (&in)[IN], unsigned char* stage, uint64_t* full, int64_t offset,
                                           int local, int slot_bytes) {
    uint32_t total = 0;
    fence_proxy_async_smem();
#pragma unroll
    for (int i = 0; i < IN; ++i)
        if (in[i] != nullptr) total += SliceSource<T>(in[i], offset, local).body_bytes();
    const uint32_t bar = smem_u32(full);
    mbar_arrive_expect_tx(bar, total);
#pragma unroll
    for (int i = 0; i < IN; ++i) {
        if (in[i] == nullptr) continue;
        const SliceSource<T> s(in[i], offset, local);
        const uint32_t bytes = s.body_bytes();
        if (bytes != 0)
            bulk_load_chunked(smem_u32(stage + i * slot_bytes) + (s.shift + s.head) * sizeof(T), s.row + s.head, bytes, bar);
    }
}

// W consecutive columns of one input (zeros for an input that is absent).
template <typename T, int W>
__device__ __forceinline__ void slot_elems(const unsigned char* slot, const SliceSource<T>& s, int e, float (&x)[W]) {
    if constexpr (W == 1) {
        x[0] = s.element(slot, e);
    } else {
        Vec<T>::unpack(*reinterpret_cast<const uint4*>(slot + e * sizeof(T)), x);
    }
}

template <typename T, int W>
__device__ __forceinline__ void store_elems(T* p, const float (&x)[W]) {
    if constexpr (W == 1) {
        Vec<T>::store(p, x[0]);
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

// Sums of K = 1 or 4 partials over the CTA and the cluster, in every thread, added in a fixed order. One CTA
// barrier, and one cluster barrier when there is more than one CTA.
template <int K, int THREADS>
struct alignas(16) RowSums {
    float warp[THREADS / 32][K];
    float peer[kMaxClusterSize][K];
};

template <int THREADS>
__device__ __forceinline__ void row_sums(float (&v)[1], RowSums<1, THREADS>& s, uint32_t rank, uint32_t nranks) {
    constexpr int kWarps = THREADS / 32;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    v[0] = warp_sum(v[0]);
    if (lane == 0) s.warp[warp][0] = v[0];
    __syncthreads();
    v[0] = 0.0f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) v[0] += s.warp[w][0];
    if (nranks == 1) return;
    if (warp == 0 && lane < static_cast<int>(nranks))
        st_cluster_f32(map_to_rank(smem_u32(&s.peer[rank][0]), static_cast<uint32_t>(lane)), v[0]);
    cluster_sync_all();
    v[0] = 0.0f;
    for (uint32_t r = 0; r < nranks; ++r) v[0] += s.peer[r][0];
}

template <int THREADS>
__device__ __forceinline__ void row_sums(float (&v)[4], RowSums<4, THREADS>& s, uint32_t rank, uint32_t nranks) {
    constexpr int kWarps = THREADS / 32;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    // four sums over 32 lanes in six shuffles: each step halves what a lane still adds up
    const bool upper = lane & 16, odd = lane & 8;
    float a = upper ? v[2] : v[0], b = upper ? v[3] : v[1];
    a += __shfl_xor_sync(0xffffffffu, upper ? v[0] : v[2], 16);
    b += __shfl_xor_sync(0xffffffffu, upper ? v[1] : v[3], 16);
    float c = odd ? b : a;
    c += __shfl_xor_sync(0xffffffffu, odd ? a : b, 8);
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) c += __shfl_xor_sync(0xffffffffu, c, o);
    if ((lane & 7) == 0) s.warp[warp][lane >> 3] = c;
    __syncthreads();
    float4 t = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
        const float4 p = *reinterpret_cast<const float4*>(s.warp[w]);
        t.x += p.x; t.y += p.y; t.z += p.z; t.w += p.w;
    }
    if (nranks > 1) {
        if (warp == 0 && lane < static_cast<int>(nranks)) {
            const uint32_t to = map_to_rank(smem_u32(&s.peer[rank][0]), static_cast<uint32_t>(lane));
            st_cluster_f32(to, t.x);
            st_cluster_f32(to + 4, t.y);
            st_cluster_f32(to + 8, t.z);
            st_cluster_f32(to + 12, t.w);
        }
        cluster_sync_all();
        t = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (uint32_t r = 0; r < nranks; ++r) {
            const float4 p = *reinterpret_cast<const float4*>(s.peer[r]);
            t.x += p.x; t.y += p.y; t.z += p.z; t.w += p.w;
        }
    }
    v[0] = t.x; v[1] = t.y; v[2] = t.z; v[3] = t.w;
}

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
// forward
// ---------------------------------------------------------------------------
template <typename T, int W, int THREADS, bool POST>
__global__ void __launch_bounds__(THREADS, 512 / THREADS) residual_norm_kernel(const NormFwdArgs a) {
    constexpr int N = kElems / W, kStride = THREADS * W;
    __shared__ uint64_t full[kMaxRing];
    // two reductions a row, alternating rows: a slow thread may still read the last row's
    __shared__ RowSums<1, THREADS> sums[2][2];
    extern __shared__ __align__(128) unsigned char ring[];
    const uint32_t rank = cluster_cta_rank(), nranks = cluster_cta_count();
    const int cluster = static_cast<int>(blockIdx.x / nranks), clusters = static_cast<int>(gridDim.x / nranks);
    const int start = static_cast<int>(rank) * a.ring.slice;
    const int local = max(0, min(a.ring.slice, a.ring.cols - start));
    const int stage_bytes = 2 * a.ring.slot_bytes;
    const void* in[2] = {a.block, a.residual};
    if (threadIdx.x == 0) {
        for (int i = 0; i < a.ring.stages; ++i) mbar_init(smem_u32(&full[i]), 1);
        fence_mbar_init();
        for (int i = 0; i < a.ring.stages; ++i) {
            const int64_t row = cluster + static_cast<int64_t>(i) * clusters;
            if (row < a.ring.rows)
                fill_stage<T, 2>(in, ring + i * stage_bytes, &full[i], row * a.ring.cols + start, local, a.ring.slot_bytes);
        }
    }
    float c[N][W], w[N][W];
    const int e0 = static_cast<int>(threadIdx.x) * W;
#pragma unroll
    for (int u = 0; u < N; ++u) {
        const int e = e0 + u * kStride;
#pragma unroll
        for (int j = 0; j < W; ++j) c[u][j] = w[u][j] = 0.0f;
        if (e < local) {
            load_channel_scale<W>(a.post_weight, a.gate, start + e, c[u]);
            load_params<W>(a.pre_weight + start + e, w[u]);
        }
    }
    __syncthreads();
    if (nranks > 1) cluster_sync_all();

    const float inv_n = 1.0f / static_cast<float>(a.ring.cols);
    RingCursor at{0, 0};
    int turn = 0;
    for (int64_t row = cluster; row < a.ring.rows; row += clusters, turn ^= 1) {
        const int64_t offset = row * a.ring.cols + start;
        unsigned char* stage = ring + at.stage * stage_bytes;
        const SliceSource<T> os(a.block, offset, local), hs(a.residual, offset, local);
        mbar_wait_bounded(smem_u32(&full[at.stage]), at.parity, a.status);
        float o[N][W], h[N][W], q[1] = {0.0f};
#pragma unroll
        for (int u = 0; u < N; ++u) {
            const int e = e0 + u * kStride;
#pragma unroll
            for (int j = 0; j < W; ++j) o[u][j] = h[u][j] = 0.0f;
            if (e < local) {
                slot_elems<T, W>(stage, os, e, o[u]);
                slot_elems<T, W>(stage + a.ring.slot_bytes, hs, e, h[u]);
            }
#pragma unroll
            for (int j = 0; j < W; ++j) q[0] = fmaf(o[u][j], o[u][j], q[0]);
        }
        float r1 = 1.0f;
        if (POST) {
            row_sums(q, sums[turn][0], rank, nranks);
            r1 = rsqrtf(fmaf(q[0], inv_n, a.eps));
        }
        q[0] = 0.0f;
        T* out = static_cast<T*>(a.residual_out) + offset;
#pragma unroll
        for (int u = 0; u < N; ++u) {
            const int e = e0 + u * kStride;
#pragma unroll
            for (int j = 0; j < W; ++j) {
                h[u][j] = fmaf(a.alpha, h[u][j], o[u][j] * r1 * c[u][j]);
                q[0] = fmaf(h[u][j], h[u][j], q[0]);
            }
            // stored rounded to the rows' type; y continues from the unrounded sum
            if (e < local) store_elems<T, W>(out + e, h[u]);
        }
        row_sums(q, sums[turn][1], rank, nranks);
        // every thread has read this stage: refill it
        const int64_t ahead = row + static_cast<int64_t>(a.ring.stages) * clusters;
        if (threadIdx.x == 0 && ahead < a.ring.rows)
            fill_stage<T, 2>(in, stage, &full[at.stage], ahead * a.ring.cols + start, local, a.ring.slot_bytes);
        at.advance(a.ring.stages);
        const float r2 = rsqrtf(fmaf(q[0], inv_n, a.eps));
        T* y = static_cast<T*>(a.y) + offset;
#pragma unroll
        for (int u = 0; u < N; ++u) {
            const int e = e0 + u * kStride;
#pragma unroll
            for (int j = 0; j < W; ++j) h[u][j] *= r2 * w[u][j];
            if (e < local) store_elems<T, W>(y + e, h[u]);
        }
        if (rank == 0 && threadIdx.x == 0) {
            if (POST) a.post_rstd[row] = r1;
            a.pre_rstd[row] = r2;
        }
    }
    if (nranks > 1) cluster_sync_all();   // no CTA leaves while a peer may still write its sums
}

// ---------------------------------------------------------------------------
// backward
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
// so its three sums travel with sum t v. Both passes over a row read it from its stage.
template <typename T, int W, int THREADS, bool POST>
__global__ void __launch_bounds__(THREADS, 512 / THREADS) residual_norm_bwd_kernel(const NormBwdArgs a) {
    constexpr int N = kElems / W, kStride = THREADS * W;
    __shared__ uint64_t full[kMaxRing];
    __shared__ RowSums<4, THREADS> sums[2];   // alternating rows: a slow thread may still read the other
    extern __shared__ __align__(128) unsigned char ring[];
    const uint32_t rank = cluster_cta_rank(), nranks = cluster_cta_count();
    const int cluster = static_cast<int>(blockIdx.x / nranks), clusters = static_cast<int>(gridDim.x / nranks);
    const int start = static_cast<int>(rank) * a.ring.slice;
    const int local = max(0, min(a.ring.slice, a.ring.cols - start));
    const int slot = a.ring.slot_bytes, stage_bytes = 4 * slot;
    const void* in[4] = {a.dy, a.block, a.residual_out, a.dresidual_out};
    const bool has_d = a.dresidual_out != nullptr;
    auto fill = [&](int i, int64_t row) {
        fill_stage<T, 4>(in, ring + i * stage_bytes, &full[i], row * a.ring.cols + start, local, slot);
    };
    if (threadIdx.x == 0) {
        for (int i = 0; i < a.ring.stages; ++i) mbar_init(smem_u32(&full[i]), 1);
        fence_mbar_init();
        for (int i = 0; i < a.ring.stages; ++i) {
            const int64_t row = cluster + static_cast<int64_t>(i) * clusters;
            if (row < a.ring.rows) fill(i, row);
        }
    }
    float c[N][W], w[N][W], col_c[N][W], col_w[N][W];
    const int e0 = static_cast<int>(threadIdx.x) * W;
#pragma unroll
    for (int u = 0; u < N; ++u) {
        const int e = e0 + u * kStride;
#pragma unroll
        for (int j = 0; j < W; ++j) c[u][j] = w[u][j] = col_c[u][j] = col_w[u][j] = 0.0f;
        if (e < local) {
            load_channel_scale<W>(a.post_weight, a.gate, start + e, c[u]);
            load_params<W>(a.pre_weight + start + e, w[u]);
        }
    }
    __syncthreads();
    if (nranks > 1) cluster_sync_all();

    const float inv_n = 1.0f / static_cast<float>(a.ring.cols);
    RingCursor at{0, 0};
    int turn = 0, last = -1;   // the stage of the row before
    float r1_next = POST && cluster < a.ring.rows ? a.post_rstd[cluster] : 1.0f;
    float r2_next = cluster < a.ring.rows ? a.pre_rstd[cluster] : 1.0f;
    for (int64_t row = cluster; row < a.ring.rows; row += clusters, turn ^= 1) {
        const int64_t offset = row * a.ring.cols + start;
        const unsigned char* stage = ring + at.stage * stage_bytes;
        const SliceSource<T> ys(a.dy, offset, local), os(a.block, offset, local), hs(a.residual_out, offset, local),
            ds(has_d ? a.dresidual_out : a.dy, offset, local);
        const float r1 = r1_next, r2 = r2_next;
        if (row + clusters < a.ring.rows) {   // a cold line each: a row ahead
            if (POST) r1_next = a.post_rstd[row + clusters];
            r2_next = a.pre_rstd[row + clusters];
        }
        mbar_wait_bounded(smem_u32(&full[at.stage]), at.parity, a.status);
        float part[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int u = 0; u < N; ++u) {
            const int e = e0 + u * kStride;
            if (e < local) {
                float dy[W], n[W], v[W], d[W];
                slot_elems<T, W>(stage, ys, e, dy);
                slot_elems<T, W>(stage + slot, os, e, n);
                slot_elems<T, W>(stage + 2 * slot, hs, e, v);
#pragma unroll
                for (int j = 0; j < W; ++j) d[j] = 0.0f;
                if (POST && has_d) slot_elems<T, W>(stage + 3 * slot, ds, e, d);
#pragma unroll
                for (int j = 0; j < W; ++j) {
                    v[j] *= r2;
                    const float t = dy[j] * w[u][j];
                    part[0] = fmaf(t, v[j], part[0]);
                    if (POST) {
                        const float cn = c[u][j] * (n[j] * r1);
                        part[1] = fmaf(cn, d[j], part[1]);
                        part[2] = fmaf(cn, t, part[2]);
                        part[3] = fmaf(cn, v[j], part[3]);
                    }
                    col_w[u][j] = fmaf(dy[j], v[j], col_w[u][j]);
                }
            }
        }
        row_sums(part, sums[turn], rank, nranks);
        // every thread is done with the row before: refill its stage
        if (threadIdx.x == 0 && last >= 0) {
            const int64_t ahead = row + static_cast<int64_t>(a.ring.stages - 1) * clusters;
            if (ahead < a.ring.rows) fill(last, ahead);
        }
        const float m1 = part[0] * inv_n;
        const float m2 = POST ? (part[1] + r2 * (part[2] - m1 * part[3])) * inv_n : 0.0f;
#pragma unroll
        for (int u = 0; u < N; ++u) {
            const int e = e0 + u * kStride;
            if (e < local) {
                float dy[W], n[W], v[W], d[W];
                slot_elems<T, W>(stage, ys, e, dy);
                slot_elems<T, W>(stage + slot, os, e, n);
                slot_elems<T, W>(stage + 2 * slot, hs, e, v);
#pragma unroll
                for (int j = 0; j < W; ++j) d[j] = 0.0f;
                if (has_d) slot_elems<T, W>(stage + 3 * slot, ds, e, d);
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
        if (a.ring.stages == 1) {   // nothing to hide behind: refill at once
            __syncthreads();
            if (threadIdx.x == 0 && row + clusters < a.ring.rows) fill(0, row + clusters);
        } else {
            last = at.stage;
        }
        at.advance(a.ring.stages);
    }
    float* mine = a.partials + static_cast<size_t>(cluster) * 2 * a.ring.cols + start;
#pragma unroll
    for (int u = 0; u < N; ++u) {
        const int e = e0 + u * kStride;
        if (e < local) {
#pragma unroll
            for (int j = 0; j < W; ++j) {
                mine[e + j] = col_c[u][j];
                mine[a.ring.cols + e + j] = col_w[u][j];
            }
        }
    }
    if (nranks > 1) cluster_sync_all();   // no CTA leaves while a peer may still write its sums
}

// Adds the clusters' column sums in a fixed order: 32 columns a CTA, 32 strands of clusters.
constexpr int kFinishCols = 32, kFinishStrands = 32;
__global__ void __launch_bounds__(kFinishCols* kFinishStrands)
    residual_norm_finish_kernel(const float* partials, int clusters, int cols, const float* post_weight, const float* gate,
                                float* dpost_weight, float* dgate, float* dpre_weight) {
    __shared__ float strand[2][kFinishStrands][kFinishCols];
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
    if (s != 0 || c >= cols) return;
    both[0] = both[1] = 0.0f;
    for (int i = 0; i < kFinishStrands; ++i) {
        both[0] += strand[0][i][lane];
        both[1] += strand[1][i][lane];
    }
    dpre_weight[c] = both[1];
    if (dpost_weight != nullptr) dpost_weight[c] = gate != nullptr ? both[0] * gate[c] : both[0];
    if (dgate != nullptr) dgate[c] = post_weight != nullptr ? both[0] * post_weight[c] : both[0];
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

// The shape's part of a plan, without a device: cluster size, slice and threads. A CTA holds 8192 columns (16
// for each of 512 threads). The automatic cluster is the smallest whose slices do, and whose stages are at most
// 72 KiB, so that three fit an SM.
int plan_shape(int64_t cols, int dtype, bool vector, int inputs, int asked, Plan* p, const Form** form) {
    const int size = dtype == CREDIT_BF16 ? 2 : 4;
    const int64_t most = 512 * kElems;
    int cluster = asked;
    if (cluster == 0) {
        for (cluster = 1; cluster < kMaxClusterSize; cluster *= 2) {
            const int64_t slice = (cols + cluster - 1) / cluster;
            if (slice <= most && slice * size * inputs <= 72 * 1024) break;
        }
    }
    const int64_t slice = cluster == 1 ? cols : round_to((cols + cluster - 1) / cluster, 64);
    if (slice > most)
        return report_error(CREDIT_ERR_UNSUPPORTED, "cols=%lld: a cluster of %d holds at most %lld columns of a row",
                            static_cast<long long>(cols), cluster, static_cast<long long>(most) * cluster);
    const Form* f = dtype == CREDIT_BF16 ? forms<__nv_bfloat16>(vector) : forms<float>(vector);
    while (static_cast<int64_t>(f->threads) * kElems < slice) ++f;
    *form = f;
    p->threads = f->threads;
    p->cluster = cluster;
    p->ring.cols = static_cast<int>(cols);
    p->ring.slice = static_cast<int>(slice);
    p->ring.slot_bytes = round_to(slice * size + 16, 128);
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
    if (stages < 2) stages = room / stage < 2 ? 1 : 2;
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

bool all_aligned(std::initializer_list<const void*> pointers) {
    for (const void* p : pointers)
        if (!aligned_to(p, 16)) return false;
    return true;
}

bool any_null(std::initializer_list<const void*> pointers) {
    for (const void* p : pointers)
        if (p == nullptr) return true;
    return false;
}

bool rows_of_vectors(int64_t cols, int dtype) { return cols * (dtype == CREDIT_BF16 ? 2 : 4) % 16 == 0; }

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
                        all_aligned({block, residual, post_weight, gate, pre_weight, residual_out, y});
    const Form* form = nullptr;
    Plan p;
    rc = plan_shape(cols, dtype, vector, 2, asked, &p, &form);
    if (rc != CREDIT_OK || rows == 0) return rc;
    if (any_null({block, residual, pre_weight, residual_out, y, pre_rstd}))
        return report_error(CREDIT_ERR_INVALID_ARGUMENT, "block, residual, pre_weight, residual_out, y and pre_rstd must not be NULL");
    if ((post_weight == nullptr) != (post_rstd == nullptr))
        return report_error(CREDIT_ERR_INVALID_ARGUMENT, "post_weight and post_rstd go together");
    if (y == residual_out) return report_error(CREDIT_ERR_INVALID_ARGUMENT, "y and residual_out must differ");
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
    int rc = plan_shape(cols, dtype, vector, 4, asked, p, &form);
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
    const bool vector = rows_of_vectors(cols, dtype) && all_aligned({dy, dresidual_out, block, residual_out, post_weight,
                                                                     gate, pre_weight, dblock, dresidual});
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
    residual_norm_finish_kernel<<<(p.ring.cols + kFinishCols - 1) / kFinishCols, kFinishCols * kFinishStrands, 0, s>>>(
        a.partials, p.clusters, p.ring.cols, post_weight, gate, dpost_weight, dgate, dpre_weight);
    const cudaError_t err = cudaGetLastError();
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
