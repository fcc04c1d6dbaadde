// What the kernels of a paged key-value cache share: the arguments, where a token's rows lie,
// which keys a token sees, and the attention of one row by one warp.
//
// The cache is two pools [pages][kv_heads][page_size][dim] of fp32, fp16 or bf16 numbers: a page
// of a kv head is one run of memory.  Token j of a sequence lies in page tables[slot][j /
// page_size], at row j % page_size.
#pragma once

#include <cuda_bf16.h>

#include "b200w4_internal.cuh"

namespace paged {

struct Args {
    void *k, *v;
    const int32_t *tables, *lengths, *slots_of, *starts;
    int pages, kv_heads, page_size;
    int slots, table_len, sequences, rows, max_length;
    int* status;
    int first_item, items;  // paged::item: of a launch
    // x / page_size for 0 <= x < 2^31 (Granlund and Montgomery, Division by invariant integers
    // using multiplication, 1994): t = x multiplier >> 32, (t + (x - t >> shift1)) >> shift2
    uint32_t multiplier;
    int shift1, shift2;
};
inline void set_division(Args& a) {
    int l = 0;
    while (l < 31 && (1u << l) < (uint32_t)a.page_size)
        ++l;
    a.multiplier = (uint32_t)((((uint64_t)1 << 32) * (((uint64_t)1 << l) - a.page_size)) /
                                  a.page_size +
                              1);
    a.shift1 = l < 1 ? l : 1;
    a.shift2 = l < 1 ? 0 : l - 1;
}
inline __host__ __device__ int page_of(const Args& a, int x) {
    const uint32_t t = (uint32_t)(((uint64_t)a.multiplier * (uint32_t)x) >> 32);
    return (int)((t + (((uint32_t)x - t) >> a.shift1)) >> a.shift2);
}

// A sequence of the batch: its table, its tokens, its first row of the call and how many.
struct Sequence {
    const int32_t* table;
    int length, first, count;
};

inline __host__ __device__ int at_most(int a, int b) { return a < b ? a : b; }

// Everything that the device arrays say is bounded here, so that no call reads or writes out of
// its tables, rows or pools; *bad: a slot or a row count that the call does not have.
inline __host__ __device__ Sequence sequence(const Args& a, int i, bool* bad) {
    Sequence s;
    int slot = a.slots_of ? a.slots_of[i] : i;
    if (slot < 0 || slot >= a.slots) {
        *bad |= slot != -1;  // that names no slot
        slot = 0;
        s.length = 0;
    } else {
        s.length = a.lengths[slot];
    }
    // table_len * page_size may pass 32 bits
    const long long room = (long long)a.table_len * a.page_size;
    int most = a.max_length;
    if (room < most)
        most = (int)room;
    if (s.length < 0 || s.length > most) {
        *bad = true;
        s.length = s.length < 0 ? 0 : most;
    }
    s.table = a.tables + (size_t)slot * a.table_len;
    s.first = a.starts ? a.starts[i] : i;
    s.count = a.starts ? a.starts[i + 1] - s.first : 1;
    if (s.first < 0 || s.count < 0 || s.first > a.rows || s.count > a.rows - s.first) {
        *bad = true;
        s.first = s.count = 0;
    }
    return s;
}

// As the kernels take it: a sequence whose length is not one that the call can have has no token in
// it.  (With its length only bounded, a new key would be written over a good one further ahead.)
inline __host__ __device__ Sequence taken(const Args& a, int i, bool* bad) {
    bool wrong = false;
    Sequence s = sequence(a, i, &wrong);
    if (wrong)
        s.length = 0;
    *bad |= wrong;
    return s;
}

// The sequence that row `row` of the call belongs to: the last one that begins at or before it;
// -1 where the row lies before the first sequence or behind the last.
inline __host__ __device__ int sequence_of(const Args& a, int row) {
    if (!a.starts)
        return row < a.sequences ? row : -1;
    if (row < a.starts[0] || row >= a.starts[a.sequences])
        return -1;
    int lo = 0, hi = a.sequences;  // starts[lo] <= row < starts[hi]
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a.starts[mid] <= row)
            lo = mid;
        else
            hi = mid;
    }
    return lo;
}

// What is attended one token at a time: the sequences, with their last token, or with BY_ROW the
// rows of all, each as a sequence that ends with its token (length 0: it has none; count 0: there
// is no such row).  i: counted from the launch's first.
template <bool BY_ROW>
inline __host__ __device__ Sequence item(const Args& a, int i, bool* bad) {
    i += a.first_item;
    if (!BY_ROW)
        return taken(a, i, bad);
    const int n = sequence_of(a, i);
    if (n < 0)
        return {a.tables, 0, 0, 0};
    Sequence s = taken(a, n, bad);
    const int in = i - s.first;
    if (in >= s.count)
        return {a.tables, 0, 0, 0};
    const int length = s.length - s.count + in + 1;
    return {s.table, length < 0 ? 0 : length, i, 1};
}

// Row of the pools (of dim numbers) where token j of a sequence lies, kv head h; -1: its page is
// not one of the pool's.  A device holds fewer than 2^31 rows of 64 numbers or more.
inline __host__ __device__ int cache_row(const Args& a, const int32_t* table, int j, int h) {
    const int n = page_of(a, j);
    const int page = table[n];
    if ((unsigned)page >= (unsigned)a.pages)
        return -1;
    return (page * a.kv_heads + h) * a.page_size + (j - n * a.page_size);
}

// The keys that a token at position p sees: [0, sinks) and [from, p].
struct Window {
    int size, sinks;
    inline __host__ __device__ int from(int p) const {
        return size > 0 && p >= size ? p - size + 1 : 0;
    }
    inline __host__ __device__ bool sees(int p, int j) const {
        return j <= p && (j >= from(p) || j < sinks);
    }
};

#ifdef __CUDACC__
template <typename T>
__device__ __forceinline__ float number(T x) {
    if constexpr (sizeof(T) == 4)
        return x;
    else if constexpr (std::is_same_v<T, __half>)
        return __half2float(x);
    else
        return __bfloat162float(x);
}
// rounded to the cache's type, to nearest even
template <typename T>
__device__ __forceinline__ T stored(float x) {
    if constexpr (sizeof(T) == 4)
        return x;
    else if constexpr (std::is_same_v<T, __half>)
        return __float2half_rn(x);
    else
        return __float2bfloat16_rn(x);
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int off = 16; off > 0; off >>= 1)
        v = __fadd_rn(v, __shfl_xor_sync(0xffffffffu, v, off));
    return v;
}

// Attention of one query row (a token's head) at position p by one warp, key by key with a
// running softmax in 32 bits: the form for any input.  A key whose probability is zero
// contributes nothing, whatever its value row holds; one whose page is not the pool's is left
// out (and reported).  q, out: DIM numbers; p < 0: zeros.
template <typename T, int DIM>
__device__ void attend_row(const Args& a, const Sequence& s, const float* __restrict__ q, int p,
                           int h, float scale, const Window& w, float* __restrict__ out) {
    constexpr int kOwn = DIM / 32;
    const int lane = threadIdx.x & 31;
    float x[kOwn], o[kOwn], m = -INFINITY, l = 0.f;
#pragma unroll
    for (int i = 0; i < kOwn; ++i) {
        x[i] = q[lane + 32 * i];
        o[i] = 0.f;
    }
    const T* k = static_cast<const T*>(a.k);
    const T* v = static_cast<const T*>(a.v);
    const int from = w.from(p);
    bool any = false;
    for (int j = from > 0 && w.sinks <= 0 ? from : 0; j <= p; ++j) {
        if (j < from && j >= w.sinks)
            j = from;
        const int row = cache_row(a, s.table, j, h);
        if (row < 0) {
            b2w4_report(a.status, B2W4_E_INVALID);
            continue;
        }
        any = true;
        float dot = 0.f;
#pragma unroll
        for (int i = 0; i < kOwn; ++i)
            dot = __fmaf_rn(x[i], number(k[(size_t)row * DIM + lane + 32 * i]), dot);
        const float score = __fmul_rn(warp_sum(dot), scale);
        const float top = fmaxf(m, score), base = top == -INFINITY ? 0.f : top;
        const float alpha = expf(__fsub_rn(m, base)), e = expf(__fsub_rn(score, base));
        m = top;
        l = __fmaf_rn(l, alpha, e);
#pragma unroll
        for (int i = 0; i < kOwn; ++i)
            o[i] = __fmul_rn(o[i], alpha);
        if (e != 0.f) {
#pragma unroll
            for (int i = 0; i < kOwn; ++i)
                o[i] = __fmaf_rn(e, number(v[(size_t)row * DIM + lane + 32 * i]), o[i]);
        }
    }
#pragma unroll
    for (int i = 0; i < kOwn; ++i)
        out[lane + 32 * i] = any ? __fdiv_rn(o[i], l) : 0.f;
}
#endif

}  // namespace paged
