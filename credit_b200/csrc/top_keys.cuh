// The k largest of a row slice that is read once. While it streams by, every thread stores the maximum of each
// group of its elements (32 bf16 or 16 fp32 a chunk; as many chunks a group as make at most 16 groups): one store
// and nothing else. At the end each of W warps takes its ceil(k / W)-th largest thread maximum; the smallest of the
// W has k elements that reach it, about 50 (k = 20) to 250 (k = 128) groups do in 8 warps, and those are read again:
// their elements that reach it compete by rank.
//
// Order. An element is the 64-bit key (monotone image of its value, complement of its column): larger
// keys first is "value descending, column ascending", all keys of a row differ, so the chosen set
// does not depend on the order in which threads append. NaN ranks above +inf, -0 equals +0, -inf is
// never an element (its image lies under kLowestKey).
//
// When more groups or elements reach the threshold than there are places, it is mostly one value that thousands of
// elements share: a constant row, or a finite mask that leaves some warp fewer tokens than its share. Then the
// elements above it compete, and those equal to it in the order of their columns until there are k: 592 x 131072 bf16
// rows of -1e9 with 8 tokens left, k = 20, 70 us a call (ordinary rows 40 us; by the digits below 2627 us). Only a
// slice with too many elements above it too is searched digit by digit straight from global memory, at most 9 more
// reads of it.
//
// What was measured before this form, 4096 rows of 131072 bf16, k = 20 (164 us without alternatives): a running
// threshold made exact after chunks 1, 4, 16 by all threads 270 us; kept by the warps without barriers 315 us: noting
// candidates costs a warp some 100 instructions in most chunks, whoever holds the threshold.
#pragma once

#include "vocab_rows.cuh"

namespace credit {

constexpr int kMaxTop = 128;
constexpr int kTopGroups = 16;   // a thread's
constexpr uint64_t kLowestKey = 0x0080000000000000ull;   // the image of -FLT_MAX, any column

__device__ __forceinline__ uint64_t element_key(float x, int column) {
    return (static_cast<uint64_t>(ordered_image(x)) << 32) | (0xffffffffu - static_cast<uint32_t>(column));
}

__device__ __forceinline__ float key_value(uint64_t key) { return image_value(static_cast<uint32_t>(key >> 32)); }
__device__ __forceinline__ int key_column(uint64_t key) { return static_cast<int>(0xffffffffu - static_cast<uint32_t>(key)); }

template <int THREADS>
struct TopBuffer {
    static constexpr int kPlaces = 8 * THREADS;
    unsigned long long keys[kPlaces];
    unsigned int hist[256];
    float group[kTopGroups][THREADS];   // maxima
    unsigned int floor[THREADS / 32];   // image of each warp's share of the threshold
    unsigned int differ[2];      // bits in which the keys differ (high, low word); zero between calls
    int noted[kPlaces];          // groups that reach the threshold
    int notes;                   // (may exceed the places, like count)
    int count;                   // candidates appended
    int fill, digit, above, here;
};

// By one thread, before the first barrier.
template <int THREADS>
__device__ __forceinline__ void init_top_buffer(TopBuffer<THREADS>& t) {
    t.count = t.notes = 0;
    t.differ[0] = t.differ[1] = 0;
}

// Warp 0: the digit in which the need-th largest lies, how many lie above it and in it.
template <int THREADS>
__device__ __forceinline__ void find_digit(TopBuffer<THREADS>& t, int need) {
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

// Keeps the k largest of keys[0, n), n <= kPlaces (fewer when fewer are non-zero: zeros are
// empty places). All threads call it behind a barrier; it ends with one, the number kept in t.fill.
template <int THREADS>
__device__ __forceinline__ void keep_largest(TopBuffer<THREADS>& t, int n, int k) {
    constexpr int kPer = TopBuffer<THREADS>::kPlaces / THREADS;
    const int tid = threadIdx.x;
    uint64_t mine[kPer];
    const uint64_t some = t.keys[0];
    uint64_t diff = 0;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
        const int i = tid + j * THREADS;
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
            for (int i = tid; i < 256; i += THREADS) t.hist[i] = 0;
            __syncthreads();
#pragma unroll
            for (int j = 0; j < kPer; ++j)
                if (tid + j * THREADS < n && ((mine[j] ^ threshold) & mask) == 0)
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
    if (tid == 0) t.fill = 0;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kPer; ++j)
        if (mine[j] != 0 && mine[j] >= threshold) t.keys[atomicAdd(&t.fill, 1)] = mine[j];
    if (tid == 0) t.differ[0] = t.differ[1] = 0;
    __syncthreads();
}

// The same, sorted descending: with one key a thread at most, the larger ones are counted for each, which is
// its place; more go through the digits first. The number kept is in t.fill.
template <int THREADS>
__device__ __noinline__ void rank_largest(TopBuffer<THREADS>& t, int n, int k) {
    const int tid = threadIdx.x;
    if (n > THREADS) {
        keep_largest(t, n, k);
        n = t.fill;
        __syncthreads();
    }
    // few keys: 4 or 2 neighbouring threads share one and count a part of the others each
    const int shift = n <= THREADS / 4 ? 2 : (n <= THREADS / 2 ? 1 : 0), share = 1 << shift;
    const int at = tid >> shift, part = tid & (share - 1);
    const uint64_t mine = at < n ? t.keys[at] : 0;
    int place = 0;
    if (mine != 0) {
        int i = part * 2;
#pragma unroll 2
        for (; i + 2 <= n; i += 2 * share) {
            const ulonglong2 p = *reinterpret_cast<const ulonglong2*>(&t.keys[i]);
            place += (p.x > mine) + (p.y > mine);
        }
        if (i < n) place += t.keys[i] > mine;
    }
    if (share > 1) place += __shfl_xor_sync(0xffffffffu, place, 1);
    if (share > 2) place += __shfl_xor_sync(0xffffffffu, place, 2);
    const int kept = __syncthreads_count(mine != 0 && part == 0);
    if (mine != 0 && part == 0 && place < k) t.keys[place] = mine;
    if (tid == 0) t.fill = min(kept, k);
    __syncthreads();
}

// The slow path: the same selection straight from the slice in global memory. Leaves at most k keys
// in keys[0, fill) and ends with a barrier.
template <typename T, int THREADS>
__device__ __noinline__ void select_from_slice(const T* first, int start, int local, int k, TopBuffer<THREADS>& t) {
    const int tid = threadIdx.x;
    uint64_t threshold = 0, mask = 0;
    int need = k;
    for (int shift = 56; shift >= 0; shift -= 8) {
        for (int i = tid; i < 256; i += THREADS) t.hist[i] = 0;
        if (tid == 0) t.digit = -1;
        __syncthreads();
        for (int base = 0; base < local; base += THREADS) {
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
    for (int c = tid; c < local; c += THREADS) {
        const uint64_t key = element_key(Vec<T>::load(first + c), start + c);
        if (key >= threshold) {
            const int at = atomicAdd(&t.fill, 1);
            if (at < TopBuffer<THREADS>::kPlaces) t.keys[at] = key;
        }
    }
    __syncthreads();
}

// The middle path: the elements above the bound `least` (an image), and when they are fewer than k the first ones
// equal to it, at least k together, into keys[0, n). Returns n (more than kPlaces: too many, the keys are void). All
// threads, behind a barrier; ends with one.
template <typename T, int THREADS, int U>
__device__ __noinline__ int collect_from_bound(const RowSpan<T> span, uint32_t least, int groups, int per_group, int k,
                                               TopBuffer<THREADS>& t) {
    constexpr int E = Vec<T>::kElems, kPlaces = TopBuffer<THREADS>::kPlaces, kStep = 4;
    static_assert(kMaxTop + kStep * THREADS <= kPlaces, "fewer than k keys and all of a step fit");
    const int tid = threadIdx.x;
    auto offer = [&](float x, int offset) {
        const int at = atomicAdd(&t.count, 1);
        if (at < kPlaces) t.keys[at] = element_key(x, span.start + offset);
    };
    if (tid == 0) t.count = t.notes = 0;
    __syncthreads();
    if (tid < span.edges) {
        const int offset = span.edge_offset(tid);
        const float x = Vec<T>::load(span.first + offset);
        if (ordered_image(x) > least) offer(x, offset);
    }
    for (int g = 0; g < groups; ++g)
        if (ordered_image(t.group[g][tid]) > least) {
            const int at = atomicAdd(&t.notes, 1);
            if (at < kPlaces) t.noted[at] = g * THREADS + tid;
        }
    __syncthreads();
    const int notes = t.notes, vectors = U * per_group;
    if (notes > kPlaces) return notes;   // an element each at least
    for (int i = tid; i < notes * vectors; i += THREADS) {
        const int note = t.noted[i / vectors];
        const int v = ((note / THREADS * per_group) * U + i % vectors) * THREADS + note % THREADS;
        if (v >= span.nvec) continue;
        float x[E];
        Vec<T>::unpack(span.vectors()[v], x);
#pragma unroll
        for (int j = 0; j < E; ++j)
            if (ordered_image(x[j]) > least) offer(x[j], span.head + v * E + j);
    }
    __syncthreads();
    int n = t.count;
    __syncthreads();
    for (int base = 0; base < span.local && n < k; base += kStep * THREADS) {
#pragma unroll
        for (int j = 0; j < kStep; ++j) {
            const int i = base + j * THREADS + tid;
            const float x = i < span.local ? Vec<T>::load(span.first + i) : -CUDART_INF_F;
            if (ordered_image(x) == least) offer(x, i);
        }
        __syncthreads();
        n = t.count;
        __syncthreads();
    }
    return n;
}

// One CTA's groups while its slice streams by, in chunks of U vectors a thread.
template <typename T, int THREADS, int U>
struct TopCollector {
    static constexpr int E = Vec<T>::kElems, kWarps = THREADS / 32, kPlaces = TopBuffer<THREADS>::kPlaces;
    TopBuffer<THREADS>& t;
    const int k;
    int chunks, per_group;
    float running;

    __device__ __forceinline__ TopCollector(TopBuffer<THREADS>& t_, int k_, int chunks_)
        : t(t_), k(k_), chunks(chunks_), per_group((chunks_ + kTopGroups - 1) / kTopGroups), running(-INFINITY) {}

    // The thread's maximum of chunk `it`.
    __device__ __forceinline__ void add(float top, int it) {
        running = max_nan(running, top);
        const int g = per_group == 1 ? it : it / per_group;
        if (per_group == 1 || it + 1 == (g + 1) * per_group || it + 1 == chunks) {
            t.group[g][threadIdx.x] = running;
            running = -CUDART_INF_F;
        }
    }

    __device__ __forceinline__ void offer(float x, int column) {
        const int at = atomicAdd(&t.count, 1);
        if (at < kPlaces) t.keys[at] = element_key(x, column);
    }

    // An element outside the vectors competes in any case.
    __device__ __forceinline__ void add_edge(float x, int column) {
        if (x != -CUDART_INF_F) offer(x, column);
    }

    // The k largest of the slice in keys[0, fill), sorted, behind a barrier. `thread_max`: over all of the
    // thread's elements, edges included.
    __device__ __forceinline__ void finish(const RowSpan<T>& span, float thread_max) {
        const int tid = threadIdx.x, lane = tid & 31;
        const uint32_t mine = ordered_image(thread_max);
        uint32_t m = 0;
        bool taken = false;
#pragma unroll 1
        for (int i = 0; i < (k + kWarps - 1) / kWarps; ++i) {
            m = __reduce_max_sync(0xffffffffu, taken ? 0u : mine);
            taken |= lane == __ffs(__ballot_sync(0xffffffffu, !taken && mine == m)) - 1;
        }
        if (lane == 0) t.floor[tid >> 5] = m;
        __syncthreads();
        const uint32_t least = max(__reduce_min_sync(0xffffffffu, t.floor[lane & (kWarps - 1)]),
                                   static_cast<uint32_t>(kLowestKey >> 32));
        const float floor = image_value(least);   // NaN: only NaN reaches it
        const bool nan = floor != floor;
        const int groups = (chunks + per_group - 1) / max(per_group, 1);
        uint32_t reach = 0;   // groups, a bit each
#pragma unroll
        for (int g = 0; g < kTopGroups; ++g) {
            const float x = g < groups ? t.group[g][tid] : -CUDART_INF_F;
            if (nan ? x != x : !(x < floor)) reach |= 1u << g;
        }
        if (reach != 0) {
            int at = atomicAdd(&t.notes, __popc(reach));
            for (; reach != 0; reach &= reach - 1, ++at)
                if (at < kPlaces) t.noted[at] = (__ffs(reach) - 1) * THREADS + tid;
        }
        __syncthreads();
        const int notes = t.notes, vectors = U * per_group;
        bool overflow = notes > kPlaces;
        if (!overflow) {
#pragma unroll 1
            for (int i = tid; i < notes * vectors; i += THREADS) {
                const int which = per_group == 1 ? i / U : i / vectors, place = i - which * vectors, note = t.noted[which];
                const int v = ((note / THREADS * per_group) * U + place) * THREADS + note % THREADS;
                if (v >= span.nvec) continue;
                float x[E];
                Vec<T>::unpack(span.vectors()[v], x);
                uint32_t hits = 0;
#pragma unroll
                for (int j = 0; j < E; ++j)
                    if (nan ? x[j] != x[j] : !(x[j] < floor)) hits |= 1u << j;
                if (hits == 0) continue;
                int at = atomicAdd(&t.count, __popc(hits));
                const int column = span.vector_column(v);
#pragma unroll
                for (int j = 0; j < E; ++j)
                    if (hits >> j & 1u) {
                        if (at < kPlaces) t.keys[at] = element_key(x[j], column + j);
                        ++at;
                    }
            }
        }
        __syncthreads();
        int n = t.count;
        if (overflow || n > kPlaces) {
            __syncthreads();
            n = collect_from_bound<T, THREADS, U>(span, least, groups, per_group, k, t);
            if (n > kPlaces) {
                __syncthreads();
                select_from_slice(span.first, span.start, span.local, k, t);
                n = t.fill;
                __syncthreads();
            }
        }
        rank_largest(t, n, k);
    }
};

// Smallest 64-bit key over a warp.
__device__ __forceinline__ uint64_t warp_min_key(uint64_t key) {
    const uint32_t hi = static_cast<uint32_t>(key >> 32), lo = static_cast<uint32_t>(key);
    const uint32_t m = __reduce_min_sync(0xffffffffu, hi);
    const uint32_t l = __reduce_min_sync(0xffffffffu, hi == m ? lo : 0xffffffffu);
    return (static_cast<uint64_t>(m) << 32) | l;
}

// Rank 0: the k largest of `lists` sorted lists of k keys (zeros at their ends) into t.keys[0, fill), sorted. Of
// every list the first ceil(k / lists) entries are k together, so nothing below the smallest of those can
// be among the k largest. All threads, behind a barrier.
template <int THREADS>
__device__ __forceinline__ void merge_lists(TopBuffer<THREADS>& t, const unsigned long long* gathered, int lists, int k) {
    static_assert(TopBuffer<THREADS>::kPlaces >= kMaxClusterSize * kMaxTop, "every gathered key may be a candidate");
    const int share = (k + lists - 1) / lists - 1;
    const int lane = threadIdx.x & 31;
    const uint64_t floor = warp_min_key(lane < lists ? gathered[lane * k + share] : ~0ull);
    if (threadIdx.x == 0) t.count = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < lists * k; i += THREADS) {
        const uint64_t key = gathered[i];
        if (key != 0 && key >= floor) t.keys[atomicAdd(&t.count, 1)] = key;   // at most 16 * 128 of them
    }
    __syncthreads();
    const int n = t.count;
    rank_largest(t, n, k);
}

}  // namespace credit
