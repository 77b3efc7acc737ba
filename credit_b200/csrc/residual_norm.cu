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

struct NormFwdArgs {
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
    int cols;
    int slice;
};

// W elements (a 16-byte vector, or one) of a row or of an fp32 parameter vector.
template <typename T, int W>
__device__ __forceinline__ void load_elems(const T* p, float (&x)[W]) {
    if constexpr (W == 1) {
        x[0] = Vec<T>::load(p);
    } else {
        Vec<T>::unpack(load_stream(reinterpret_cast<const uint4*>(p)), x);
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

// Sums of K partials over the CTA and the cluster, in every thread, added in a fixed order. One CTA
// barrier, and one cluster barrier when there is more than one CTA.
template <int K, int THREADS>
struct RowSums {
    float warp[K][THREADS / 32];
    float peer[K][kMaxClusterSize];
};

template <int K, int THREADS>
__device__ __forceinline__ void row_sums(float (&v)[K], RowSums<K, THREADS>& s, uint32_t rank, uint32_t nranks) {
    constexpr int kWarps = THREADS / 32;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] = warp_sum(v[k]);
    if (lane == 0) {
#pragma unroll
        for (int k = 0; k < K; ++k) s.warp[k][warp] = v[k];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; ++k) {
        float t = 0.0f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) t += s.warp[k][w];
        v[k] = t;
    }
    if (nranks == 1) return;
    if (warp == 0 && lane < static_cast<int>(nranks)) {
#pragma unroll
        for (int k = 0; k < K; ++k)
            st_cluster_f32(map_to_rank(smem_u32(&s.peer[k][rank]), static_cast<uint32_t>(lane)), v[k]);
    }
    cluster_sync_all();
#pragma unroll
    for (int k = 0; k < K; ++k) {
        float t = 0.0f;
        for (uint32_t r = 0; r < nranks; ++r) t += s.peer[k][r];
        v[k] = t;
    }
}

// ---------------------------------------------------------------------------
// forward: a cluster per row, the row in registers between its two reductions
// ---------------------------------------------------------------------------
template <typename T, int W, int N, int THREADS, bool POST>
__global__ void __launch_bounds__(THREADS) residual_norm_kernel(const NormFwdArgs a) {
    __shared__ RowSums<1, THREADS> sums[2];
    const uint32_t rank = cluster_cta_rank(), nranks = cluster_cta_count();
    if (nranks > 1) cluster_arrive_release();
    const int64_t row = blockIdx.x / nranks;
    const int start = static_cast<int>(rank) * a.slice;
    const int end = min(a.cols, start + a.slice);
    const int64_t offset = row * a.cols;
    const T* o = static_cast<const T*>(a.block) + offset;
    const T* h = static_cast<const T*>(a.residual) + offset;
    const int c0 = start + static_cast<int>(threadIdx.x) * W;
    constexpr int kStride = THREADS * W;

    float ov[N][W], hv[N][W];
#pragma unroll
    for (int u = 0; u < N; ++u) {
        const int c = c0 + u * kStride;
#pragma unroll
        for (int j = 0; j < W; ++j) ov[u][j] = hv[u][j] = 0.0f;
        if (c < end) {
            load_elems<T, W>(o + c, ov[u]);
            load_elems<T, W>(h + c, hv[u]);
        }
    }
    if (nranks > 1) cluster_wait_acquire();
    float r1 = 1.0f;
    if (POST) {
        float q[1] = {0.0f};
#pragma unroll
        for (int u = 0; u < N; ++u)
#pragma unroll
            for (int j = 0; j < W; ++j) q[0] = fmaf(ov[u][j], ov[u][j], q[0]);
        row_sums(q, sums[0], rank, nranks);
        r1 = rsqrtf(q[0] / static_cast<float>(a.cols) + a.eps);
    }
    float q[1] = {0.0f};
#pragma unroll
    for (int u = 0; u < N; ++u) {
        const int c = c0 + u * kStride;
        if (c < end) {
            float s[W];
            load_channel_scale<W>(a.post_weight, a.gate, c, s);
#pragma unroll
            for (int j = 0; j < W; ++j) {
                hv[u][j] = fmaf(a.alpha, hv[u][j], ov[u][j] * r1 * s[j]);
                q[0] = fmaf(hv[u][j], hv[u][j], q[0]);
            }
        }
    }
    // the sum is stored rounded to the rows' type; y continues from the unrounded one
    T* out = static_cast<T*>(a.residual_out) + offset;
#pragma unroll
    for (int u = 0; u < N; ++u) {
        const int c = c0 + u * kStride;
        if (c < end) store_elems<T, W>(out + c, hv[u]);
    }
    row_sums(q, sums[1], rank, nranks);
    const float r2 = rsqrtf(q[0] / static_cast<float>(a.cols) + a.eps);
    T* y = static_cast<T*>(a.y) + offset;
#pragma unroll
    for (int u = 0; u < N; ++u) {
        const int c = c0 + u * kStride;
        if (c < end) {
            float w[W];
            load_params<W>(a.pre_weight + c, w);
#pragma unroll
            for (int j = 0; j < W; ++j) w[j] *= hv[u][j] * r2;
            store_elems<T, W>(y + c, w);
        }
    }
    if (rank == 0 && threadIdx.x == 0) {
        if (POST) a.post_rstd[row] = r1;
        a.pre_rstd[row] = r2;
    }
}

// ---------------------------------------------------------------------------
// backward: clusters walk rows and keep their columns' sums over the rows in registers
// ---------------------------------------------------------------------------
struct NormBwdArgs {
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
    int rows;
    int cols;
    int slice;
};

// One exchange per row: with D = d + r2 (t - v m), m = mean(t v), the second mean is linear in m,
//   mean(D c n) = (sum c n d + r2 sum c n t - r2 m sum c n v) / N,
// so its three sums travel with sum t v.
template <typename T, int W, int N, int THREADS, bool POST>
__global__ void __launch_bounds__(THREADS) residual_norm_bwd_kernel(const NormBwdArgs a) {
    __shared__ RowSums<4, THREADS> sums[2];   // alternating rows: a slow thread may still read the other
    const uint32_t rank = cluster_cta_rank(), nranks = cluster_cta_count();
    const int cluster = static_cast<int>(blockIdx.x / nranks), clusters = static_cast<int>(gridDim.x / nranks);
    const int start = static_cast<int>(rank) * a.slice;
    const int end = min(a.cols, start + a.slice);
    const int c0 = start + static_cast<int>(threadIdx.x) * W;
    constexpr int kStride = THREADS * W;
    const float inv_n = 1.0f / static_cast<float>(a.cols);
    float col_c[N][W], col_w[N][W];
#pragma unroll
    for (int u = 0; u < N; ++u)
#pragma unroll
        for (int j = 0; j < W; ++j) col_c[u][j] = col_w[u][j] = 0.0f;
    if (nranks > 1) cluster_sync_all();

    int turn = 0;
    for (int64_t row = cluster; row < a.rows; row += clusters, turn ^= 1) {
        const int64_t offset = row * a.cols;
        const float r1 = POST ? a.post_rstd[row] : 1.0f, r2 = a.pre_rstd[row];
        float dyv[N][W], dv[N][W], nv[N][W], vv[N][W];
#pragma unroll
        for (int u = 0; u < N; ++u) {
            const int c = c0 + u * kStride;
#pragma unroll
            for (int j = 0; j < W; ++j) dyv[u][j] = dv[u][j] = nv[u][j] = vv[u][j] = 0.0f;
            if (c < end) {
                load_elems<T, W>(static_cast<const T*>(a.dy) + offset + c, dyv[u]);
                if (a.dresidual_out != nullptr) load_elems<T, W>(static_cast<const T*>(a.dresidual_out) + offset + c, dv[u]);
                load_elems<T, W>(static_cast<const T*>(a.block) + offset + c, nv[u]);
                load_elems<T, W>(static_cast<const T*>(a.residual_out) + offset + c, vv[u]);
            }
        }
        float part[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int u = 0; u < N; ++u) {
            const int c = c0 + u * kStride;
            if (c < end) {
                float s[W], w[W];
                load_channel_scale<W>(a.post_weight, a.gate, c, s);
                load_params<W>(a.pre_weight + c, w);
#pragma unroll
                for (int j = 0; j < W; ++j) {
                    nv[u][j] *= r1;
                    vv[u][j] *= r2;
                    const float t = dyv[u][j] * w[j];
                    part[0] = fmaf(t, vv[u][j], part[0]);
                    if (POST) {
                        const float cn = s[j] * nv[u][j];
                        part[1] = fmaf(cn, dv[u][j], part[1]);
                        part[2] = fmaf(cn, t, part[2]);
                        part[3] = fmaf(cn, vv[u][j], part[3]);
                    }
                    col_w[u][j] = fmaf(dyv[u][j], vv[u][j], col_w[u][j]);
                }
            }
        }
        row_sums(part, sums[turn], rank, nranks);
        const float m1 = part[0] * inv_n;
        const float m2 = POST ? (part[1] + r2 * (part[2] - m1 * part[3])) * inv_n : 0.0f;
#pragma unroll
        for (int u = 0; u < N; ++u) {
            const int c = c0 + u * kStride;
            if (c < end) {
                float s[W], w[W], dh[W], dblk[W];
                load_channel_scale<W>(a.post_weight, a.gate, c, s);
                load_params<W>(a.pre_weight + c, w);
#pragma unroll
                for (int j = 0; j < W; ++j) {
                    const float d = fmaf(r2, dyv[u][j] * w[j] - vv[u][j] * m1, dv[u][j]);
                    dh[j] = a.alpha * d;
                    dblk[j] = POST ? r1 * (s[j] * d - nv[u][j] * m2) : s[j] * d;
                    col_c[u][j] = fmaf(d, nv[u][j], col_c[u][j]);
                }
                store_elems<T, W>(static_cast<T*>(a.dblock) + offset + c, dblk);
                store_elems<T, W>(static_cast<T*>(a.dresidual) + offset + c, dh);
            }
        }
    }
    float* mine = a.partials + static_cast<size_t>(cluster) * 2 * a.cols;
#pragma unroll
    for (int u = 0; u < N; ++u) {
        const int c = c0 + u * kStride;
        if (c < end) {
#pragma unroll
            for (int j = 0; j < W; ++j) {
                mine[c + j] = col_c[u][j];
                mine[a.cols + c + j] = col_w[u][j];
            }
        }
    }
    if (nranks > 1) cluster_sync_all();   // no CTA leaves while a peer may still write its sums
}

// Adds the clusters' column sums in cluster order: 32 columns a CTA, 8 strands of clusters.
constexpr int kFinishCols = 32, kFinishStrands = 8;
__global__ void __launch_bounds__(kFinishCols* kFinishStrands)
    residual_norm_finish_kernel(const float* partials, int clusters, int cols, const float* post_weight, const float* gate,
                                float* dpost_weight, float* dgate, float* dpre_weight) {
    __shared__ float strand[2][kFinishStrands][kFinishCols];
    const int lane = threadIdx.x % kFinishCols, s = threadIdx.x / kFinishCols;
    const int c = blockIdx.x * kFinishCols + lane;
    float both[2] = {0.0f, 0.0f};
    if (c < cols)
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
// One compiled form: elements a thread takes at once, how many of those, threads.
struct Form {
    int width, count, threads;
    const void* forward[2];    // [post norm]
    const void* backward[2];
    int elems() const { return width * count * threads; }
};

template <typename T, int W, int N, int THREADS>
Form make_form() {
    return {W, N, THREADS,
            {reinterpret_cast<const void*>(&residual_norm_kernel<T, W, N, THREADS, false>),
             reinterpret_cast<const void*>(&residual_norm_kernel<T, W, N, THREADS, true>)},
            {reinterpret_cast<const void*>(&residual_norm_bwd_kernel<T, W, N, THREADS, false>),
             reinterpret_cast<const void*>(&residual_norm_bwd_kernel<T, W, N, THREADS, true>)}};
}

template <typename T>
const Form* forms(bool vector, int* count) {
    constexpr int E = Vec<T>::kElems;
    static const Form with_vectors[] = {make_form<T, E, 8 / E, 128>(), make_form<T, E, 8 / E, 256>(),
                                        make_form<T, E, 8 / E, 512>(), make_form<T, E, 16 / E, 512>()};
    static const Form with_scalars[] = {make_form<T, 1, 8, 128>(), make_form<T, 1, 8, 512>(), make_form<T, 1, 16, 512>()};
    *count = vector ? 4 : 3;
    return vector ? with_vectors : with_scalars;
}

// The smallest form that holds a slice, and the smallest cluster whose slices fit some form.
int choose_form(int64_t cols, int dtype, bool vector, int asked, const Form** form, int* cluster) {
    int n = 0;
    const Form* f = dtype == CREDIT_BF16 ? forms<__nv_bfloat16>(vector, &n) : forms<float>(vector, &n);
    const int most = f[n - 1].elems();
    int p = asked;
    if (p == 0)
        for (p = 1; p < kMaxClusterSize && (cols + p - 1) / p > most; p *= 2) {}
    const int64_t slice = ((cols + p - 1) / p + 63) / 64 * 64;
    if ((cols + p - 1) / p > most || slice > most)
        return report_error(CREDIT_ERR_UNSUPPORTED, "cols=%lld: a cluster of %d holds at most %lld columns of a row",
                            static_cast<long long>(cols), p, static_cast<long long>(most) * p);
    int i = 0;
    while (f[i].elems() < (p == 1 ? cols : slice)) ++i;
    *form = f + i;
    *cluster = p;
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
    int cluster = 0;
    rc = choose_form(cols, dtype, vector, asked, &form, &cluster);
    if (rc != CREDIT_OK || rows == 0) return rc;
    if (any_null({block, residual, pre_weight, residual_out, y, pre_rstd}))
        return report_error(CREDIT_ERR_INVALID_ARGUMENT, "block, residual, pre_weight, residual_out, y and pre_rstd must not be NULL");
    if ((post_weight == nullptr) != (post_rstd == nullptr))
        return report_error(CREDIT_ERR_INVALID_ARGUMENT, "post_weight and post_rstd go together");
    if (y == residual_out) return report_error(CREDIT_ERR_INVALID_ARGUMENT, "y and residual_out must differ");
    DeviceContext ctx;
    rc = current_device_context(&ctx);
    if (rc != CREDIT_OK) return rc;
    NormFwdArgs a;
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
    a.cols = static_cast<int>(cols);
    a.slice = cluster == 1 ? a.cols : static_cast<int>(((cols + cluster - 1) / cluster + 63) / 64 * 64);
    const void* func = form->forward[post_weight != nullptr];
    rc = prepare_kernel(ctx, func);
    if (rc != CREDIT_OK) return rc;
    void* args[] = {&a};
    return launch_kernel(func, rows * cluster, form->threads, cluster, 0, stream, args);
}

// Everything of a backward call that its workspace depends on.
struct BackwardPlan {
    DeviceContext ctx;
    const Form* form;
    const void* func;
    int cluster;
    int clusters;
    size_t workspace_bytes;
};

int plan_backward(int64_t rows, int64_t cols, int dtype, bool vector, bool post, int asked, BackwardPlan* p) {
    int rc = choose_form(cols, dtype, vector, asked, &p->form, &p->cluster);
    if (rc != CREDIT_OK) return rc;
    rc = current_device_context(&p->ctx);
    if (rc != CREDIT_OK) return rc;
    p->func = p->form->backward[post];
    rc = prepare_kernel(p->ctx, p->func);
    if (rc != CREDIT_OK) return rc;
    int resident = 0;
    rc = resident_clusters(p->ctx, p->func, p->cluster, 0, p->form->threads, &resident);
    if (rc != CREDIT_OK) return rc;
    p->clusters = static_cast<int>(rows < resident ? rows : resident);
    p->workspace_bytes = static_cast<size_t>(p->clusters) * 2 * cols * sizeof(float);
    return CREDIT_OK;
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
    BackwardPlan p;
    rc = plan_backward(rows, cols, dtype, vector, post_weight != nullptr, asked, &p);
    if (rc != CREDIT_OK) return rc;
    if (workspace == nullptr || !aligned_to(workspace, 16) || workspace_bytes < p.workspace_bytes)
        return report_error(CREDIT_ERR_WORKSPACE, "the call needs a 16-byte aligned workspace of %zu bytes (got %zu)",
                            p.workspace_bytes, workspace == nullptr ? static_cast<size_t>(0) : workspace_bytes);
    NormBwdArgs a;
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
    a.rows = static_cast<int>(rows);
    a.cols = static_cast<int>(cols);
    a.slice = p.cluster == 1 ? a.cols : static_cast<int>(((cols + p.cluster - 1) / p.cluster + 63) / 64 * 64);
    void* args[] = {&a};
    rc = launch_kernel(p.func, static_cast<int64_t>(p.clusters) * p.cluster, p.form->threads, p.cluster, 0, stream, args);
    if (rc != CREDIT_OK) return rc;
    residual_norm_finish_kernel<<<(a.cols + kFinishCols - 1) / kFinishCols, kFinishCols * kFinishStrands, 0, s>>>(
        a.partials, p.clusters, a.cols, post_weight, gate, dpost_weight, dgate, dpre_weight);
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
        BackwardPlan p;
        if (plan_backward(rows, cols, dtype, vector, (form & 2) != 0, asked, &p) == CREDIT_OK && p.workspace_bytes > most)
            most = p.workspace_bytes;
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
