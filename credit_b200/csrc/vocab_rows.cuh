// Building blocks of the kernels that read a row of logits once (token_logprobs.cu,
// distill_topk.cu): the 16-byte-vector view of a row slice of any alignment, the chunked streaming
// loop, and the softmax record of one pass.
//
// With k2 = log2(e) / temperature and a base b = m k2 rounded to fp32, m the maximum so far,
//     s = sum 2^(x k2 - b),   e = sum 2^(x k2 - b) (x k2 - b)        in 32 bits.
// x k2 - b is one fused multiply-add: exact products, so rows far from zero lose nothing; what the rounding
// of b shifts (at most half an ulp of b) is known and taken out again when the row is finished:
//     log sum exp((x - m) / T) = ln s - ln2 (m k2 - b),   entropy = ln s - ln2 e / s.
// The exponential is ex2.approx (relative error 2^-22).
//
// A base of 2^24 or more no longer resolves 1 (a row whose mask of finite values leaves nothing, a temperature near
// zero): such records, and those of temperatures that would bring kDeepLogit near or out of range, take the same sums
// from differences x - m instead (bf16 4096 x 65536 of -1e9 only: 109 us, of ordinary rows 91).
//
// -inf is a masked logit: 2^-inf adds nothing, and where it would meet e it is replaced by -1e30. A NaN makes m NaN
// (max.NaN), +inf makes it +inf; both are turned into NaN results when the row is finished.
#pragma once

#include <math_constants.h>

#include "cluster_primitives.cuh"

namespace credit {

constexpr float kLn2 = 0.6931471805599453f;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kDeepLogit = -1e30f;    // stands for -inf where a product with 0 follows
constexpr float kMostBase = 16777216.0f;

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

// Monotone image of a float: unsigned order is the order of the values, -0 equal to +0, NaN above +inf.
__device__ __forceinline__ uint32_t ordered_image(float x) {
    const uint32_t b = __float_as_uint(x + 0.0f);   // -0 + 0 = +0
    if (x != x) return 0xffffffffu;
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

__device__ __forceinline__ float image_value(uint32_t k) {
    return __uint_as_float((k & 0x80000000u) ? (k ^ 0x80000000u) : ~k);
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
    // -inf (and anything below kDeepLogit) raised to kDeepLogit
    __device__ __forceinline__ static uint4 deep(const uint4& v) {
        float x[4];
        unpack(v, x);
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = fmaxf(x[i], kDeepLogit);
        return pack(x);
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
    __device__ __forceinline__ static uint4 deep(const uint4& v) {
        constexpr uint32_t kDeepWord = 0xf149f149u;   // -0.995e30 twice
        uint4 r;
        asm("max.bf16x2 %0, %1, %2;" : "=r"(r.x) : "r"(v.x), "r"(kDeepWord));
        asm("max.bf16x2 %0, %1, %2;" : "=r"(r.y) : "r"(v.y), "r"(kDeepWord));
        asm("max.bf16x2 %0, %1, %2;" : "=r"(r.z) : "r"(v.z), "r"(kDeepWord));
        asm("max.bf16x2 %0, %1, %2;" : "=r"(r.w) : "r"(v.w), "r"(kDeepWord));
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

template <typename T, int THREADS, int U>
__device__ __forceinline__ int chunks_of(const RowSpan<T>& s) {
    return (s.nvec + THREADS * U - 1) / (THREADS * U);
}

// A row in chunks of U vectors a thread: v[u] of chunk `it` is vector (it * U + u) * THREADS + threadIdx.x, places
// past the end hold -inf. stream_chunks calls f(v, it) for every chunk, with the next one in flight; the first one
// is fetched by the caller, before it sets anything else up.
template <typename T, int THREADS, int U>
__device__ __forceinline__ void fetch_chunk(const RowSpan<T>& s, int it, uint4 (&v)[U]) {
    const uint4* base = s.vectors();
    const int i0 = it * THREADS * U + static_cast<int>(threadIdx.x);
    if ((it + 1) * THREADS * U <= s.nvec) {
#pragma unroll
        for (int u = 0; u < U; ++u) v[u] = load_stream(base + i0 + u * THREADS);
    } else {
#pragma unroll
        for (int u = 0; u < U; ++u)
            v[u] = i0 + u * THREADS < s.nvec ? load_stream(base + i0 + u * THREADS) : masked_vec<T>();
    }
}

template <typename T, int THREADS, int U, typename F>
__device__ __forceinline__ void stream_chunks(const RowSpan<T>& s, uint4 (&a)[U], F&& f) {
    const int chunks = chunks_of<T, THREADS, U>(s);
    uint4 b[U];
#pragma unroll 1
    for (int it = 0; it < chunks; it += 2) {
        if (it + 1 < chunks) fetch_chunk<T, THREADS, U>(s, it + 1, b);
        f(a, it);
        if (it + 1 >= chunks) break;
        if (it + 2 < chunks) fetch_chunk<T, THREADS, U>(s, it + 2, a);
        f(b, it + 1);
    }
}

// Edge element threadIdx.x of the slice (load it early, before the chunks), -inf when there is none.
template <typename T>
__device__ __forceinline__ float edge_element(const RowSpan<T>& s) {
    const int i = static_cast<int>(threadIdx.x);
    return i < s.edges ? Vec<T>::load(s.first + s.edge_offset(i)) : -CUDART_INF_F;
}

// Elementwise over chunks [piece * chunks, (piece + 1) * chunks) of a row (and its edges, in piece 0):
// out = f(x) for pairs of elements, or zeros. out may be x. VECTOR: both start at the same place between two
// 16-byte boundaries. Element c belongs to the thread that owns(c) names.
template <typename T, int THREADS, int U, bool VECTOR>
struct RowMap {
    const T* x;
    T* out;
    RowSpan<T> span;
    int cols, piece, chunks;

    __device__ __forceinline__ RowMap(const T* x_, T* out_, int cols_, int piece_, int chunks_)
        : x(x_), out(out_), span(x_, 0, cols_), cols(cols_), piece(piece_), chunks(chunks_) {}

    static constexpr int kVecs = THREADS * U;
    __device__ __forceinline__ int piece_elems() const { return chunks * kVecs * Vec<T>::kElems; }

    // whether column c is this thread's
    __device__ __forceinline__ bool owns(int c) const {
        constexpr int E = Vec<T>::kElems;
        if (!VECTOR) return c / piece_elems() == piece && c % THREADS == static_cast<int>(threadIdx.x);
        const int v = c - span.head;
        if (v < 0 || v >= span.nvec * E)
            return piece == 0 && (c < span.head ? c : c - span.nvec * E) == static_cast<int>(threadIdx.x);
        return v / piece_elems() == piece && v / E % THREADS == static_cast<int>(threadIdx.x);
    }
    // whether it is this CTA's
    __device__ __forceinline__ bool holds(int c) const {
        if (!VECTOR) return c / piece_elems() == piece;
        const int v = c - span.head;
        if (v < 0 || v >= span.nvec * Vec<T>::kElems) return piece == 0;
        return v / piece_elems() == piece;
    }

    // The piece's first chunk, on its way while the caller sets up; `run` takes it.
    __device__ __forceinline__ void first_chunk(uint4 (&v)[U]) const {
        if (VECTOR) fetch_chunk<T, THREADS, U>(span, piece * chunks, v);
    }

    template <typename F>
    __device__ __forceinline__ void run(bool zero, uint4 (&v)[U], F&& f) const {
        constexpr int E = Vec<T>::kElems;
        if (!VECTOR) {
            const int first = piece * piece_elems(), last = min(cols, first + piece_elems());
            for (int i = first + static_cast<int>(threadIdx.x); i < last; i += THREADS)
                Vec<T>::store(out + i, zero ? 0.0f : f(make_float2(Vec<T>::load(x + i), 0.0f)).x);
            return;
        }
        uint4* out_vec = reinterpret_cast<uint4*>(out + span.head);
        if (piece == 0 && static_cast<int>(threadIdx.x) < span.edges) {
            const int i = span.edge_offset(threadIdx.x);
            Vec<T>::store(out + i, zero ? 0.0f : f(make_float2(Vec<T>::load(x + i), 0.0f)).x);
        }
        const int from = piece * chunks, to = min(from + chunks, chunks_of<T, THREADS, U>(span));
        if (zero) {
            for (int i = from * kVecs + static_cast<int>(threadIdx.x); i < min(to * kVecs, span.nvec); i += THREADS)
                __stcs(out_vec + i, make_uint4(0, 0, 0, 0));
            return;
        }
        for (int it = from; it < to; ++it) {
            if (it > from) fetch_chunk<T, THREADS, U>(span, it, v);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                float y[E];
                Vec<T>::unpack(v[u], y);
#pragma unroll
                for (int j = 0; j < E; j += 2) {
                    const float2 r = f(make_float2(y[j], y[j + 1]));
                    y[j] = r.x;
                    y[j + 1] = r.y;
                }
                const int i = it * kVecs + static_cast<int>(threadIdx.x) + u * THREADS;
                if (i < span.nvec) __stcs(out_vec + i, Vec<T>::pack(y));
            }
        }
    }
};

// ---------------------------------------------------------------------------
// the softmax record
// ---------------------------------------------------------------------------
struct SoftmaxRecord {
    float m;   // maximum logit
    float s, e;
};

__device__ __forceinline__ SoftmaxRecord empty_record() { return {-CUDART_INF_F, 0.0f, 0.0f}; }

__device__ __forceinline__ float base_of(float m, float k2) { return __fmul_rn(m, k2); }

// kDeepLogit k2 lies between -1e38 and -1e10 then: finite, and far below every base.
__device__ __forceinline__ bool has_base(float m, float k2) {
    return fabsf(base_of(m, k2)) < kMostBase && k2 > 1e-20f && k2 < 1e8f;
}

// By how much m k2 exceeds what a record of this maximum is taken against.
__device__ __forceinline__ float base_shift(float m, float k2) {
    return has_base(m, k2) ? fmaf(m, k2, -base_of(m, k2)) : 0.0f;
}

// Moves a record to a maximum that is at least its own.
__device__ __forceinline__ void raise_maximum(SoftmaxRecord& a, float m, float k2) {
    if (a.m == m) return;
    float d = has_base(a.m, k2) && has_base(m, k2) ? __fsub_rn(base_of(a.m, k2), base_of(m, k2))
                                                   : (a.m - m) * k2 + (base_shift(m, k2) - base_shift(a.m, k2));
    d = fmaxf(d, -200.0f);   // 2^-200 is 0 here; also for a.m = -inf, where s = e = 0
    const float r = ex2_approx(d);
    a.e = (a.e + a.s * d) * r;
    a.s *= r;
    a.m = m;
}

__device__ __forceinline__ SoftmaxRecord merge_records(SoftmaxRecord a, SoftmaxRecord b, float k2) {
    const float m = max_nan(a.m, b.m);
    raise_maximum(a, m, k2);
    raise_maximum(b, m, k2);
    return {m, a.s + b.s, a.e + b.e};
}

// ln of the sum relative to the maximum.
__device__ __forceinline__ float log_sum_of(const SoftmaxRecord& a, float k2) {
    return logf(a.s) - kLn2 * base_shift(a.m, k2);
}

// Adds U vectors whose maximum is `top`. The rescaling is rare: a thread's maximum settles after a
// few chunks.
template <typename T, int U, bool ENTROPY>
__device__ __forceinline__ void accumulate(const uint4 (&v)[U], float top, float k2, SoftmaxRecord& a) {
    constexpr int E = Vec<T>::kElems;
    if (!(top <= a.m)) raise_maximum(a, max_nan(a.m, top), k2);   // a NaN stays
    if (!has_base(a.m, k2)) {
        if (a.m == -CUDART_INF_F) return;   // nothing but masked logits yet
#pragma unroll 1
        for (int u = 0; u < U; ++u) {
            float x[E];
            uint4 w = v[0];
#pragma unroll
            for (int i = 1; i < U; ++i)
                if (i == u) w = v[i];
            Vec<T>::unpack(w, x);
#pragma unroll
            for (int j = 0; j < E; ++j) {
                const float d = fmaxf((x[j] - a.m) * k2, -200.0f), p = ex2_approx(d);
                a.s += p;
                a.e = fmaf(p, d, a.e);
            }
        }
        return;
    }
    const float base = -base_of(a.m, k2);
    const float2 minus = make_float2(base, base), scale = make_float2(k2, k2);
    float2 s[2] = {{0.0f, 0.0f}, {0.0f, 0.0f}}, e[2] = {{0.0f, 0.0f}, {0.0f, 0.0f}};
#pragma unroll
    for (int u = 0; u < U; ++u) {
        float x[E];
        Vec<T>::unpack(ENTROPY ? Vec<T>::deep(v[u]) : v[u], x);
#pragma unroll
        for (int j = 0; j < E; j += 2) {
            const float2 d = __ffma2_rn(make_float2(x[j], x[j + 1]), scale, minus);
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
__device__ __forceinline__ float chunk_max(const uint4 (&v)[U]) {
    float top = Vec<T>::max(v[0]);
#pragma unroll
    for (int u = 1; u < U; ++u) top = max_nan(top, Vec<T>::max(v[u]));
    return top;
}

// Records of the first COUNT lanes (a power of two; the others must hold empty ones) in every lane: one maximum
// over the warp, one rescaling, plain sums.
template <int COUNT>
__device__ __forceinline__ SoftmaxRecord warp_record(SoftmaxRecord a, float k2) {
    const float m = image_value(__reduce_max_sync(0xffffffffu, ordered_image(a.m)));
    raise_maximum(a, m, k2);
#pragma unroll
    for (int o = COUNT / 2; o > 0; o >>= 1) {
        a.s += __shfl_xor_sync(0xffffffffu, a.s, o);
        a.e += __shfl_xor_sync(0xffffffffu, a.e, o);
    }
    a.s = __shfl_sync(0xffffffffu, a.s, 0);
    a.e = __shfl_sync(0xffffffffu, a.e, 0);
    return a;
}

// The CTA's record, in every lane of warp 0 (the other warps get their own warp's). `slots` holds one
// record per warp. One barrier.
template <int THREADS>
__device__ __forceinline__ SoftmaxRecord cta_record(SoftmaxRecord a, SoftmaxRecord* slots, float k2) {
    constexpr int kWarps = THREADS / 32;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    a = warp_record<32>(a, k2);
    if (lane == 0) slots[warp] = a;
    __syncthreads();
    if (warp == 0) a = warp_record<kWarps>(lane < kWarps ? slots[lane] : empty_record(), k2);
    return a;
}

// A row whose maximum is NaN or +inf has no distribution.
__device__ __forceinline__ bool is_broken(float m) { return !(m < CUDART_INF_F); }

}  // namespace credit
