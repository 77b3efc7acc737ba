// Building blocks of the kernels that read a row of logits once (token_logprobs.cu,
// distill_topk.cu): the 16-byte-vector view of a row slice of any alignment, the chunked streaming
// loop, and the softmax record of one pass,
//     m = max x,  s = sum exp(k (x - m)),  e = sum exp(k (x - m)) * k (x - m),   k = 1 / temperature,
// in 32 bits. Differences x - m are taken before the scaling, so rows far from zero (and rows whose
// every logit is the type's lowest value) lose nothing; the exponential is ex2.approx (relative
// error 2^-22) of the difference in base-2 units, and so is e.
//
// -inf is a masked logit: it adds nothing (differences are clamped at -200, where ex2 gives 0, before
// they are multiplied by that 0). A NaN makes m NaN (max.NaN), +inf makes it +inf; both are turned
// into NaN results when the row is finished.
#pragma once

#include <math_constants.h>

#include "cluster_primitives.cuh"

namespace credit {

constexpr float kLn2 = 0.6931471805599453f;
constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

__device__ __forceinline__ float ex2_approx(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// 16 bytes that nobody reads again soon.
__device__ __forceinline__ uint4 load_stream(const uint4* p) {
    uint4 v;
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "l"(p)
                 : "memory");
    return v;
}

// ---------------------------------------------------------------------------
// 16-byte vectors
// ---------------------------------------------------------------------------
template <typename T>
struct Vec;

template <>
struct Vec<float> {
    static constexpr int kElems = 4;
    static constexpr uint32_t kMaskedWord = 0xff800000u;   // -inf
    __device__ __forceinline__ static void unpack(const uint4& v, float (&x)[4]) {
        x[0] = __uint_as_float(v.x); x[1] = __uint_as_float(v.y);
        x[2] = __uint_as_float(v.z); x[3] = __uint_as_float(v.w);
    }
    __device__ __forceinline__ static uint4 pack(const float (&x)[4]) {
        return make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
    }
    __device__ __forceinline__ static float max(const uint4& v) {
        float x[4];
        unpack(v, x);
        return max_nan(max_nan(x[0], x[1]), max_nan(x[2], x[3]));
    }
    __device__ __forceinline__ static uint4 single(float x) {
        return make_uint4(__float_as_uint(x), kMaskedWord, kMaskedWord, kMaskedWord);
    }
    __device__ __forceinline__ static float load(const float* p) { return *p; }
    __device__ __forceinline__ static void store(float* p, float x) { *p = x; }
};

template <>
struct Vec<__nv_bfloat16> {
    static constexpr int kElems = 8;
    static constexpr uint32_t kMaskedWord = 0xff80ff80u;
    __device__ __forceinline__ static void unpack(const uint4& v, float (&x)[8]) {
        RowVec<__nv_bfloat16>::unpack(v, x);
    }
    __device__ __forceinline__ static uint4 pack(const float (&x)[8]) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
            w[i] = *reinterpret_cast<const uint32_t*>(&h);
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
    __device__ __forceinline__ static uint32_t max2(uint32_t a, uint32_t b) {
        uint32_t r;
        asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
        return r;
    }
    __device__ __forceinline__ static float max(const uint4& v) {
        const uint32_t m = max2(max2(v.x, v.y), max2(v.z, v.w));
        return max_nan(__uint_as_float(m << 16), __uint_as_float(m & 0xffff0000u));
    }
    __device__ __forceinline__ static uint4 single(float x) {
        return make_uint4((kMaskedWord & 0xffff0000u) | (__float_as_uint(x) >> 16), kMaskedWord, kMaskedWord,
                          kMaskedWord);
    }
    __device__ __forceinline__ static float load(const __nv_bfloat16* p) { return __bfloat162float(*p); }
    __device__ __forceinline__ static void store(__nv_bfloat16* p, float x) { *p = __float2bfloat16_rn(x); }
};

template <typename T>
__device__ __forceinline__ uint4 masked_vec() {
    return make_uint4(Vec<T>::kMaskedWord, Vec<T>::kMaskedWord, Vec<T>::kMaskedWord, Vec<T>::kMaskedWord);
}

// ---------------------------------------------------------------------------
// a slice [start, start + local) of one row: up to kElems - 1 elements before the first 16-byte
// boundary, whole vectors, up to kElems - 1 elements behind the last one
// ---------------------------------------------------------------------------
template <typename T>
struct RowSpan {
    const T* first;     // element `start` of the row
    int start;          // its column
    int local;          // elements
    int head;           // elements before the vectors
    int nvec;
    int edges;          // head + elements behind the vectors

    __device__ __forceinline__ RowSpan(const T* row, int start_, int local_) : first(row + start_), start(start_), local(local_) {
        constexpr int E = Vec<T>::kElems;
        const int off = static_cast<int>((reinterpret_cast<uintptr_t>(first) & 15u) / sizeof(T));
        head = off == 0 ? 0 : E - off;
        if (head > local) head = local;
        nvec = (local - head) / E;
        edges = local - nvec * E;
    }
    __device__ __forceinline__ const uint4* vectors() const { return reinterpret_cast<const uint4*>(first + head); }
    // offset inside the slice of edge element i, and column of a vector's first element
    __device__ __forceinline__ int edge_offset(int i) const { return i < head ? i : nvec * Vec<T>::kElems + i; }
    __device__ __forceinline__ int vector_column(int v) const { return start + head + v * Vec<T>::kElems; }
};

// Calls f(v, first_vec, it) for chunks of U vectors a thread (vector first_vec + u * THREADS is v[u];
// places past the end hold -inf) and once more with it = number of chunks for the edge elements,
// if there are any, as f's `edge` call: v[0] holds edge element threadIdx.x alone. Every thread of
// the CTA makes the same calls, so f may synchronise. The next chunk is in flight while f runs.
template <typename T, int THREADS, int U, typename F, typename G>
__device__ __forceinline__ void stream_slice(const RowSpan<T>& s, F&& f, G&& edge) {
    constexpr int kPerChunk = THREADS * U;
    const int chunks = (s.nvec + kPerChunk - 1) / kPerChunk;
    const uint4* base = s.vectors();
    uint4 next[U];
    auto fetch = [&](int it) {
        const int i0 = it * kPerChunk + static_cast<int>(threadIdx.x);
        if ((it + 1) * kPerChunk <= s.nvec) {
#pragma unroll
            for (int u = 0; u < U; ++u) next[u] = load_stream(base + i0 + u * THREADS);
        } else {
#pragma unroll
            for (int u = 0; u < U; ++u)
                next[u] = i0 + u * THREADS < s.nvec ? load_stream(base + i0 + u * THREADS) : masked_vec<T>();
        }
    };
    float lone = -CUDART_INF_F;
    if (static_cast<int>(threadIdx.x) < s.edges) lone = Vec<T>::load(s.first + s.edge_offset(threadIdx.x));
    if (chunks > 0) fetch(0);
    for (int it = 0; it < chunks; ++it) {
        uint4 v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) v[u] = next[u];
        if (it + 1 < chunks) fetch(it + 1);
        f(v, it * kPerChunk + static_cast<int>(threadIdx.x), it);
    }
    if (s.edges > 0) {
        uint4 v[1] = {Vec<T>::single(lone)};
        edge(v);
    }
}

// ---------------------------------------------------------------------------
// the softmax record
// ---------------------------------------------------------------------------
struct SoftmaxRecord {
    float m;   // maximum logit
    float s;   // sum of ex2(k2 (x - m)), k2 = log2(e) / temperature
    float e;   // sum of the same times k2 (x - m)
};

__device__ __forceinline__ SoftmaxRecord empty_record() { return {-CUDART_INF_F, 0.0f, 0.0f}; }

// Moves a record to a maximum that is at least its own.
__device__ __forceinline__ void raise_maximum(SoftmaxRecord& a, float m, float k2) {
    const float d = fmaxf((a.m - m) * k2, -200.0f);   // -200 too for a.m = m = -inf (s = e = 0 there)
    const float r = a.m == m ? 1.0f : ex2_approx(d);
    a.e = a.m == m ? a.e : (a.e + a.s * d) * r;
    a.s *= r;
    a.m = m;
}

__device__ __forceinline__ SoftmaxRecord merge_records(SoftmaxRecord a, SoftmaxRecord b, float k2) {
    const float m = max_nan(a.m, b.m);
    raise_maximum(a, m, k2);
    raise_maximum(b, m, k2);
    return {m, a.s + b.s, a.e + b.e};
}

// Adds U vectors whose maximum is `top`. The rescaling is rare: a thread's maximum settles after a
// few chunks.
template <typename T, int U, bool ENTROPY>
__device__ __forceinline__ void accumulate(const uint4 (&v)[U], float top, float k2, SoftmaxRecord& a) {
    constexpr int E = Vec<T>::kElems;
    if (!(top <= a.m)) raise_maximum(a, max_nan(a.m, top), k2);   // a NaN stays
    const float base = a.m == -CUDART_INF_F ? 0.0f : a.m;   // nothing but masked logits yet: ex2(-inf) = 0
    const float2 minus = make_float2(-base, -base), scale = make_float2(k2, k2);
    float2 s[2] = {{0.0f, 0.0f}, {0.0f, 0.0f}}, e[2] = {{0.0f, 0.0f}, {0.0f, 0.0f}};
#pragma unroll
    for (int u = 0; u < U; ++u) {
        float x[E];
        Vec<T>::unpack(v[u], x);
#pragma unroll
        for (int j = 0; j < E; j += 2) {
            float2 d = __fmul2_rn(__fadd2_rn(make_float2(x[j], x[j + 1]), minus), scale);
            if (ENTROPY) {
                d.x = fmaxf(d.x, -200.0f);
                d.y = fmaxf(d.y, -200.0f);
            }
            const float2 p = make_float2(ex2_approx(d.x), ex2_approx(d.y));
            const int w = (j / 2) & 1;
            s[w] = __fadd2_rn(s[w], p);
            if (ENTROPY) e[w] = __ffma2_rn(p, d, e[w]);
        }
    }
    a.s += (s[0].x + s[0].y) + (s[1].x + s[1].y);
    if (ENTROPY) a.e += (e[0].x + e[0].y) + (e[1].x + e[1].y);
}

template <typename T, int U>
__device__ __forceinline__ float chunk_max(const uint4 (&v)[U], float (&part)[U]) {
    float top = -CUDART_INF_F;
#pragma unroll
    for (int u = 0; u < U; ++u) {
        part[u] = Vec<T>::max(v[u]);
        top = max_nan(top, part[u]);
    }
    return top;
}

// The CTA's record, in every thread of warp 0 (the other warps get their own warp's). `slots` holds one
// record per warp. One barrier.
template <int THREADS>
__device__ __forceinline__ SoftmaxRecord cta_record(SoftmaxRecord a, SoftmaxRecord* slots, float k2) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        SoftmaxRecord b;
        b.m = __shfl_xor_sync(0xffffffffu, a.m, o);
        b.s = __shfl_xor_sync(0xffffffffu, a.s, o);
        b.e = __shfl_xor_sync(0xffffffffu, a.e, o);
        a = merge_records(a, b, k2);
    }
    if (lane == 0) slots[warp] = a;
    __syncthreads();
    if (warp == 0) {
        a = slots[0];
        for (int w = 1; w < THREADS / 32; ++w) a = merge_records(a, slots[w], k2);
    }
    return a;
}

// A row whose maximum is NaN or +inf has no distribution.
__device__ __forceinline__ bool is_broken(float m) { return !(m < CUDART_INF_F); }

}  // namespace credit
