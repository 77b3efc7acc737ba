// The k largest of a row slice that is read once: vectors that may hold one of them are noted in shared
// memory as they stream by (their number, nothing more: a note costs a dozen instructions, a key of an
// element several times that), a threshold (always the key of a real element that k elements reach) keeps
// the rest out. Between intervals of chunks the noted vectors are read again, a thread each, and the keys
// of their elements compete.
//
// Order. An element is the 64-bit key (monotone image of its value, complement of its column): larger
// keys first is "value descending, column ascending", all keys of a row differ, so the chosen set
// does not depend on the order in which threads append. NaN ranks above +inf, -0 equals +0, -inf is
// never an element (its image lies under kLowestKey).
//
// The threshold starts from the threads' first-chunk maxima: every warp takes its ceil(k / 8)-th largest,
// and the smallest of the eight has k elements that reach it. On rows in no particular order it lets about
// 50 (k = 20) to 250 (k = 128) elements of a chunk through. It is tightened to the k-th largest candidate
// after chunks 1, 4, 16, 64, ...; each later interval then notes about 3k vectors, so 1024 notes hold every
// k up to 128. A row that brings more (sorted ascending, say) overflows; its slice is then searched by
// the digit-by-digit selection straight from global memory, at most 8 more reads of it.
#pragma once

#include "vocab_rows.cuh"

namespace credit {

constexpr int kMaxTop = 128;
constexpr int kTopThreads = 256;
constexpr int kTopCapacity = 2048;
constexpr int kTopNotes = 1024;
constexpr uint64_t kLowestKey = 0x0080000000000000ull;   // the image of -FLT_MAX, any column

__device__ __forceinline__ uint64_t element_key(float x, int column) {
    return (static_cast<uint64_t>(ordered_image(x)) << 32) | (0xffffffffu - static_cast<uint32_t>(column));
}

__device__ __forceinline__ float key_value(uint64_t key) { return image_value(static_cast<uint32_t>(key >> 32)); }
__device__ __forceinline__ int key_column(uint64_t key) { return static_cast<int>(0xffffffffu - static_cast<uint32_t>(key)); }

struct TopBuffer {
    unsigned long long keys[kTopCapacity];
    unsigned int hist[256];
    unsigned long long lowest;   // smallest kept key
    unsigned long long floor[kTopThreads / 32];   // first threshold of each warp
    unsigned int differ[2];      // bits in which the keys differ (high, low word); zero between calls
    int notes[kTopNotes];        // vectors of the slice
    int noted;                   // (may exceed the places, like count)
    int count;                   // candidates appended
    int fill, digit, above, here;
};

// By one thread, before the first barrier.
__device__ __forceinline__ void init_top_buffer(TopBuffer& t) {
    t.count = t.noted = 0;
    t.differ[0] = t.differ[1] = 0;
}

// Warp 0: the digit in which the need-th largest lies, how many lie above it and in it.
__device__ __forceinline__ void find_digit(TopBuffer& t, int need) {
    const int lane = threadIdx.x & 31;
    int part[8], sum = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        part[j] = static_cast<int>(t.hist[255 - 8 * lane - j]);
        sum += part[j];
    }
    int upto = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += v;
    }
    int before = upto - sum;
    if (before < need && upto >= need) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            if (before < need && before + part[j] >= need) {
                t.digit = 255 - 8 * lane - j;
                t.above = before;
                t.here = part[j];
            }
            before += part[j];
        }
    }
}

// Keeps the k largest of keys[0, n), n <= kTopCapacity (fewer when fewer are non-zero: zeros are
// empty places), and returns the smallest of them (0 when there are fewer than k). All threads call
// it behind a barrier; it ends with one, the number kept in t.fill.
__device__ __forceinline__ uint64_t keep_largest(TopBuffer& t, int n, int k) {
    constexpr int kPer = kTopCapacity / kTopThreads;
    const int tid = threadIdx.x;
    uint64_t mine[kPer];
    const uint64_t some = t.keys[0];
    uint64_t diff = 0;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
        const int i = tid + j * kTopThreads;
        mine[j] = i < n ? t.keys[i] : some;
        diff |= mine[j] ^ some;
        if (i >= n) mine[j] = 0;
    }
    const uint32_t hi = __reduce_or_sync(0xffffffffu, static_cast<uint32_t>(diff >> 32));
    const uint32_t lo = __reduce_or_sync(0xffffffffu, static_cast<uint32_t>(diff));
    if ((tid & 31) == 0) {
        if (hi != 0) atomicOr(&t.differ[0], hi);
        if (lo != 0) atomicOr(&t.differ[1], lo);
    }
    __syncthreads();
    diff = (static_cast<uint64_t>(t.differ[0]) << 32) | t.differ[1];
    uint64_t threshold = some;
    if (diff != 0 && n > k) {
        int bits = 64 - __clzll(static_cast<long long>(diff));   // undecided low bits
        uint64_t mask = bits == 64 ? 0 : ~0ull << bits;
        threshold = some & mask;
        int need = k;
        while (bits > 0) {
            const int shift = bits > 8 ? bits - 8 : 0;
            const uint32_t digits = (1u << (bits - shift)) - 1u;
            t.hist[tid] = 0;
            __syncthreads();
#pragma unroll
            for (int j = 0; j < kPer; ++j)
                if (tid + j * kTopThreads < n && ((mine[j] ^ threshold) & mask) == 0)
                    atomicAdd(&t.hist[static_cast<uint32_t>(mine[j] >> shift) & digits], 1u);
            __syncthreads();
            if (tid < 32) find_digit(t, need);
            __syncthreads();
            threshold |= static_cast<uint64_t>(t.digit) << shift;
            mask |= static_cast<uint64_t>(digits) << shift;
            need -= t.above;
            bits = shift;
            if (t.here == need) break;
        }
    } else if (n <= k) {
        threshold = 0;
    }
    if (tid == 0) {
        t.fill = 0;
        t.lowest = ~0ull;
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
        if (mine[j] != 0 && mine[j] >= threshold) {
            t.keys[atomicAdd(&t.fill, 1)] = mine[j];
            atomicMin(&t.lowest, static_cast<unsigned long long>(mine[j]));
        }
    }
    if (tid == 0) t.differ[0] = t.differ[1] = 0;
    __syncthreads();
    return t.fill < k ? 0 : t.lowest;
}

// The same, sorted descending: with one key a thread at most, every key counts the larger ones, which is
// its place; more go through the digits first. Returns the k-th (0 when there are fewer).
__device__ __noinline__ uint64_t rank_largest(TopBuffer& t, int n, int k) {
    const int tid = threadIdx.x;
    if (n > kTopThreads) {
        keep_largest(t, n, k);
        n = t.fill;
        __syncthreads();
    }
    const uint64_t mine = tid < n ? t.keys[tid] : 0;
    int place = 0;
    if (mine != 0) {
        int i = 0;
#pragma unroll 1
        for (; i + 4 <= n; i += 4) {
            const ulonglong2 p = *reinterpret_cast<const ulonglong2*>(&t.keys[i]);
            const ulonglong2 q = *reinterpret_cast<const ulonglong2*>(&t.keys[i + 2]);
            place += (p.x > mine) + (p.y > mine) + (q.x > mine) + (q.y > mine);
        }
#pragma unroll 1
        for (; i < n; ++i) place += t.keys[i] > mine;
    }
    const int kept = __syncthreads_count(mine != 0);
    if (mine != 0 && place < k) t.keys[place] = mine;
    if (tid == 0) t.fill = min(kept, k);
    __syncthreads();
    return kept >= k ? t.keys[k - 1] : 0;
}

// The slow path: the same selection straight from the slice in global memory. Leaves at most k keys
// in keys[0, fill) and ends with a barrier.
template <typename T>
__device__ __noinline__ void select_from_slice(const T* first, int start, int local, int k, TopBuffer& t) {
    const int tid = threadIdx.x;
    uint64_t threshold = 0, mask = 0;
    int need = k;
    for (int shift = 56; shift >= 0; shift -= 8) {
        t.hist[tid] = 0;
        if (tid == 0) t.digit = -1;
        __syncthreads();
        for (int base = 0; base < local; base += kTopThreads) {
            int digit = -1;
            if (base + tid < local) {
                const uint64_t key = element_key(Vec<T>::load(first + base + tid), start + base + tid);
                if (key >= kLowestKey && ((key ^ threshold) & mask) == 0) digit = static_cast<int>(key >> shift) & 255;
            }
            int same;   // rows of one value: one addition a warp
            __match_all_sync(0xffffffffu, digit, &same);
            if (same) {
                if (digit >= 0 && (tid & 31) == 0) atomicAdd(&t.hist[digit], 32u);
            } else if (digit >= 0) {
                atomicAdd(&t.hist[digit], 1u);
            }
        }
        __syncthreads();
        if (tid < 32) find_digit(t, need);
        __syncthreads();
        const int digit = t.digit;
        if (digit < 0) break;   // (first digit only) fewer than k elements: all of them
        threshold |= static_cast<uint64_t>(digit) << shift;
        mask |= 255ull << shift;
        need -= t.above;
        const int here = t.here;
        __syncthreads();
        if (here == need) break;
    }
    if (threshold < kLowestKey) threshold = kLowestKey;
    if (tid == 0) t.fill = 0;
    __syncthreads();
    for (int c = tid; c < local; c += kTopThreads) {
        const uint64_t key = element_key(Vec<T>::load(first + c), start + c);
        if (key >= threshold) {
            const int at = atomicAdd(&t.fill, 1);
            if (at < kTopCapacity) t.keys[at] = key;
        }
    }
    __syncthreads();
}

// One CTA's candidates while its slice streams by.
template <typename T>
struct TopCollector {
    TopBuffer& t;
    const int k;
    uint64_t key;    // threshold
    float value;     // its value (+inf when that is NaN, which then lets NaN and +inf through)
    bool overflow;

    __device__ __forceinline__ TopCollector(TopBuffer& t_, int k_) : t(t_), k(k_), key(kLowestKey), overflow(false) {
        set_threshold(kLowestKey);
    }

    __device__ __forceinline__ void set_threshold(uint64_t to) {
        if (to > key) key = to;
        value = key_value(key);
        if (value != value) value = CUDART_INF_F;
    }

    // The first chunk: see the top of the file. `column` is that of the thread's first vector.
    template <int U>
    __device__ __forceinline__ void first_threshold(const uint4 (&v)[U], const float (&part)[U], float top, int column,
                                                    int stride) {
        uint32_t hi = 0, lo = 0;   // this thread's largest element
        if (!(top < value)) {
            const bool nan = top != top;
            int at = 0;
#pragma unroll
            for (int u = U - 1; u >= 0; --u)
                if (nan ? part[u] != part[u] : part[u] == top) at = u;
            float x[Vec<T>::kElems];
            Vec<T>::unpack(pick(v, at), x);
            int j = 0;
#pragma unroll
            for (int i = Vec<T>::kElems - 1; i >= 0; --i)
                if (nan ? x[i] != x[i] : x[i] == top) j = i;
            hi = ordered_image(top);
            lo = 0xffffffffu - static_cast<uint32_t>(column + at * stride + j);
        }
        const int lane = threadIdx.x & 31;
        bool taken = false;
        uint32_t m = 0;
#pragma unroll 1
        for (int i = 0; i < (k + 7) / 8; ++i) {
            m = __reduce_max_sync(0xffffffffu, taken ? 0u : hi);
            const unsigned int same = __ballot_sync(0xffffffffu, !taken && hi == m);
            taken |= lane == __ffs(same) - 1;
        }
        const uint32_t low = __reduce_min_sync(0xffffffffu, taken && hi == m ? lo : 0xffffffffu);
        if (lane == 0) t.floor[threadIdx.x >> 5] = (static_cast<uint64_t>(m) << 32) | low;
        __syncthreads();
        uint64_t least = t.floor[0];
#pragma unroll
        for (int w = 1; w < kTopThreads / 32; ++w) least = t.floor[w] < least ? t.floor[w] : least;
        set_threshold(least);
    }

    __device__ __forceinline__ void offer(float x, int column) {
        if (x < value) return;
        const uint64_t c = element_key(x, column);
        if (c < key) return;
        const int at = atomicAdd(&t.count, 1);
        if (at < kTopCapacity) t.keys[at] = c;
    }

    // v[at] without an indexed register file
    template <int U>
    __device__ __forceinline__ static uint4 pick(const uint4 (&v)[U], int at) {
        uint4 r = v[0];
#pragma unroll
        for (int u = 1; u < U; ++u)
            if (at == u) r = v[u];
        return r;
    }

    // Notes the vectors of a chunk that reach the threshold; among equals of its value only those that start at
    // its column or before it.
    template <int U>
    __device__ __forceinline__ void note_chunk(const float (&part)[U], float top, int first, int column, int stride) {
        if (top < value) return;
        const uint32_t last = 0xffffffffu - static_cast<uint32_t>(key);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (!(part[u] <= value) || (part[u] == value && static_cast<uint32_t>(column + u * stride) <= last)) {
                const int at = atomicAdd(&t.noted, 1);
                if (at < kTopNotes) t.notes[at] = first + u * kTopThreads;
            }
        }
    }

    // The elements of the noted vectors become candidates. All threads; ends with a barrier.
    __device__ __forceinline__ void expand(const RowSpan<T>& span) {
        __syncthreads();
        const int n = t.noted;
        __syncthreads();   // everyone has read it
        if (n > kTopNotes) overflow = true;
        if (threadIdx.x == 0) t.noted = 0;
        if (!overflow) {
#pragma unroll 1
            for (int i = threadIdx.x; i < n; i += kTopThreads) {
                const int v = t.notes[i], column = span.vector_column(v);
                float x[Vec<T>::kElems];
                Vec<T>::unpack(span.vectors()[v], x);
#pragma unroll
                for (int j = 0; j < Vec<T>::kElems; ++j) offer(x[j], column + j);
            }
        }
        __syncthreads();
        if (t.count > kTopCapacity) overflow = true;
    }

    // Between intervals of chunks: keep the k largest so far.
    __device__ __forceinline__ void tighten(const RowSpan<T>& span) {
        expand(span);
        const int n = t.count;
        if (n > k && !overflow) {
            set_threshold(rank_largest(t, n, k));
            if (threadIdx.x == 0) t.count = t.fill;
        }
        __syncthreads();
    }

    // The k largest of the slice in keys[0, fill), sorted, behind a barrier.
    __device__ __forceinline__ void finish(const RowSpan<T>& span) {
        expand(span);
        int n = t.count;
        if (overflow) {
            select_from_slice(span.first, span.start, span.local, k, t);
            n = t.fill;
            __syncthreads();
        }
        rank_largest(t, n, k);
    }
};

// Rank 0: the k largest of `lists` sorted lists of k keys (zeros at their ends) into t.keys[0, fill), sorted. Of
// every list the first ceil(k / lists) entries are k together, so nothing below the smallest of those can
// be among the k largest. All threads, behind a barrier.
__device__ __forceinline__ void merge_lists(TopBuffer& t, const unsigned long long* gathered, int lists, int k) {
    const int share = (k + lists - 1) / lists - 1;
    uint64_t floor = ~0ull;
    for (int r = 0; r < lists; ++r) floor = min(floor, static_cast<uint64_t>(gathered[r * k + share]));
    if (threadIdx.x == 0) t.count = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < lists * k; i += kTopThreads) {
        const uint64_t key = gathered[i];
        if (key != 0 && key >= floor) t.keys[atomicAdd(&t.count, 1)] = key;   // at most 16 * 128 of them
    }
    __syncthreads();
    const int n = t.count;
    rank_largest(t, n, k);
}
static_assert(kTopCapacity >= kMaxClusterSize * kMaxTop, "every gathered key may be a candidate");

}  // namespace credit
