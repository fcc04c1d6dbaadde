// Log probabilities of given tokens, the entropy of their distributions, and the most likely
// tokens: one pass over the logits.
//
// With M the row's maximum, S = sum exp(x - M) and T = sum exp(x - M) (x - M):
//   log p(t) = x_t - M - log S,   entropy = log S - T / S   (a sum of two terms >= 0).
// Every thread keeps a running maximum m and sums relative to it, in 32 bits; two such triples
// join as M = max, S = S1 e^(m1 - M) + S2 e^(m2 - M), T likewise of T_i + (m_i - M) S_i.
//
// The k largest: a number below which the k-th largest cannot lie comes from the first tile (the
// k-th largest of the maxima of 128 groups of its numbers, all different), and what is not below
// it goes to a list in shared memory, about a hundred numbers of a chunk of 19,000.  The list's
// first k are found by counting, for each, how many are before it.
#include "b200w4_internal.cuh"

#include <climits>

#include <cooperative_groups.h>

namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kVecs = 4;                    // of four numbers, a thread's share of a tile
constexpr int kTile = kThreads * kVecs * 4;
constexpr int kMostTop = 32;
constexpr int kGroups = kThreads / 2;       // two threads each
constexpr int kTrim = 256;                  // a longer list is cut back to the k largest
constexpr int kList = kTrim + kTile;
constexpr int kMostCluster = 8;

struct Args {
    const float* x;
    const int32_t* target;
    float *logprob, *entropy, *values;
    int32_t* indices;
    int ld, rows, vocab, top;
    int* status;
};

// Larger word: larger number, among equals the lower index; NaN below everything, then -inf.
__device__ __forceinline__ unsigned long long word(float v, int i) {
    unsigned bits = __float_as_uint(v);
    if (bits == 0x80000000u)
        bits = 0u;  // -0 equals 0
    const unsigned key = v != v ? 0u : (bits & 0x80000000u) ? ~bits : bits | 0x80000000u;
    return ((unsigned long long)key << 32) | (0xffffffffu - (unsigned)i);
}
__device__ __forceinline__ int index_of(unsigned long long w) {
    return (int)(0xffffffffu - (unsigned)w);
}
// The smallest number that may have this word's key: what is below it need not be looked at.
__device__ __forceinline__ float floor_of(unsigned long long w) {
    const unsigned key = (unsigned)(w >> 32);
    if (key < 0x00800000u)  // NaN, or no number at all
        return -INFINITY;
    return __uint_as_float((key & 0x80000000u) ? key ^ 0x80000000u : ~key);
}

struct Sums {
    float m, s, t;
};
__device__ __forceinline__ Sums join(const Sums& a, const Sums& b) {
    const float m = fmaxf(a.m, b.m), base = m == -INFINITY ? 0.f : m;
    const float da = fmaxf(__fsub_rn(a.m, base), -1e30f), db = fmaxf(__fsub_rn(b.m, base), -1e30f);
    const float ea = expf(da), eb = expf(db);
    Sums r;
    r.m = m;
    r.s = __fmaf_rn(a.s, ea, __fmul_rn(b.s, eb));
    // a side without numbers, or without any that count, has s = 0 and t = 0
    const float ta = ea == 0.f ? __fmul_rn(a.s, 0.f) : __fmul_rn(__fmaf_rn(a.s, da, a.t), ea);
    const float tb = eb == 0.f ? __fmul_rn(b.s, 0.f) : __fmul_rn(__fmaf_rn(b.s, db, b.t), eb);
    r.t = __fadd_rn(ta, tb);
    return r;
}

struct Shared {
    unsigned long long list[kList];
    unsigned long long group[kGroups];
    unsigned long long first[kMostTop];
    unsigned long long best[kMostCluster][kMostTop];  // of the cluster's blocks, in block 0
    Sums part[kMostCluster];                          // likewise
    Sums warp[kWarps];
    unsigned long long kth;
    int count;
};

// Cuts the list to its `top` largest, in order (or to all that there are); whole block.
__device__ void trim(Shared& s, int top) {
    __syncthreads();
    const int n = s.count;
    for (int i = threadIdx.x; i < n; i += kThreads) {
        const unsigned long long w = s.list[i];
        int before = 0;
        for (int j = 0; j < n && before < top; ++j)
            before += s.list[j] > w;
        if (before < top)
            s.first[before] = w;
    }
    __syncthreads();
    if ((int)threadIdx.x < min(n, top))
        s.list[threadIdx.x] = s.first[threadIdx.x];
    if (threadIdx.x == 0) {
        s.count = min(n, top);
        s.kth = n >= top ? s.first[top - 1] : 0ull;
    }
    __syncthreads();
}

// A cluster per row, a chunk of the row per block.
__global__ void __launch_bounds__(kThreads)
logprobs_kernel(const Args a, bool aligned) {
    namespace cg = cooperative_groups;
    b2w4_pdl_chain_entry();
    __shared__ Shared s;
    cg::cluster_group cluster = cg::this_cluster();
    const int blocks = (int)cluster.num_blocks(), block = (int)cluster.block_rank();
    const int row = blockIdx.x / blocks;
    const float* x = a.x + (size_t)row * a.ld;
    const int chunk = ((a.vocab + blocks - 1) / blocks + 3) & ~3;
    const int lo = min(a.vocab, block * chunk), hi = min(a.vocab, lo + chunk);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 0) {
        s.count = 0;
        s.kth = 0ull;
    }
    // number e of the thread's vector u of the tile at `base`
    auto place = [&](int base, int u) { return base + (tid + u * kThreads) * 4; };
    auto load = [&](int base, float4 (&v)[kVecs]) {
#pragma unroll
        for (int u = 0; u < kVecs; ++u) {
            const int i = place(base, u);
            if (aligned && i + 4 <= hi) {
                v[u] = __ldcs(reinterpret_cast<const float4*>(x + i));
            } else {
                v[u].x = i < hi ? __ldcs(x + i) : -INFINITY;
                v[u].y = i + 1 < hi ? __ldcs(x + i + 1) : -INFINITY;
                v[u].z = i + 2 < hi ? __ldcs(x + i + 2) : -INFINITY;
                v[u].w = i + 3 < hi ? __ldcs(x + i + 3) : -INFINITY;
            }
        }
    };
    float m = -INFINITY, sum = 0.f, t = 0.f;
    unsigned long long kth = 0ull;
    float limit = -INFINITY;
    float4 next[kVecs];
    load(lo, next);
    for (int base = lo; base < hi; base += kTile) {
        float v[kVecs * 4];
#pragma unroll
        for (int u = 0; u < kVecs; ++u) {
            v[4 * u] = next[u].x;
            v[4 * u + 1] = next[u].y;
            v[4 * u + 2] = next[u].z;
            v[4 * u + 3] = next[u].w;
        }
        load(base + kTile, next);
        float top = m;
#pragma unroll
        for (int i = 0; i < kVecs * 4; ++i)
            top = fmaxf(top, v[i]);
        if (top > m) {
            if (m > -INFINITY) {
                const float d = __fsub_rn(m, top), e = expf(d);
                // (below, d may be -inf where top is)
                t = e == 0.f ? 0.f : __fmul_rn(__fmaf_rn(sum, d, t), e);
                sum = __fmul_rn(sum, e);
            }
            m = top;
        }
        const float from = m == -INFINITY ? 0.f : m;
#pragma unroll
        for (int i = 0; i < kVecs * 4; ++i) {
            const float d = __fsub_rn(v[i], from);
            float e;
            asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(__fmul_rn(d, 1.4426950408889634f)));
            sum = __fadd_rn(sum, e);
            t = __fmaf_rn(e, fmaxf(d, -200.f), t);  // e = 0 where d = -inf
        }
        if (a.top > 0) {
            if (base == lo) {
                unsigned long long w = 0ull;
#pragma unroll
                for (int i = 0; i < kVecs * 4; ++i) {
                    const int at = place(base, i / 4) + i % 4;
                    if (at < hi)
                        w = max(w, word(v[i], at));
                }
                w = max(w, __shfl_xor_sync(0xffffffffu, w, 1));
                if (!(tid & 1))
                    s.group[tid >> 1] = w;
                __syncthreads();
                if (tid < kGroups) {
                    w = s.group[tid];
                    int before = 0;
                    for (int j = 0; j < kGroups; ++j)
                        before += s.group[j] > w;
                    if (before == a.top - 1 && w)
                        s.kth = w;
                }
                __syncthreads();
                kth = s.kth;
                limit = floor_of(kth);
            }
            bool some = false;
#pragma unroll
            for (int i = 0; i < kVecs * 4; ++i)
                some |= !(v[i] < limit);
            bool over = false;
            if (some) {
#pragma unroll
                for (int i = 0; i < kVecs * 4; ++i) {
                    const int at = place(base, i / 4) + i % 4;
                    if (!(v[i] < limit) && at < hi) {
                        const unsigned long long w = word(v[i], at);
                        if (w >= kth) {
                            const int n = atomicAdd(&s.count, 1);
                            s.list[n] = w;
                            over |= n >= kTrim;
                        }
                    }
                }
            }
            if (__syncthreads_or(over)) {
                trim(s, a.top);
                kth = s.kth;
                limit = floor_of(kth);
            }
        }
    }
    // the block's sums, in a fixed order
    Sums mine = {m, sum, t};
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
        Sums o;
        o.m = __shfl_xor_sync(0xffffffffu, mine.m, off);
        o.s = __shfl_xor_sync(0xffffffffu, mine.s, off);
        o.t = __shfl_xor_sync(0xffffffffu, mine.t, off);
        mine = lane & off ? join(o, mine) : join(mine, o);
    }
    if (lane == 0)
        s.warp[warp] = mine;
    trim(s, max(a.top, 1));
    Shared* out = cluster.map_shared_rank(&s, 0);
    if (tid == 0) {
        Sums all = s.warp[0];
        for (int w = 1; w < kWarps; ++w)
            all = join(all, s.warp[w]);
        out->part[block] = all;
    }
    if (tid < a.top)
        out->best[block][tid] = tid < s.count ? s.list[tid] : 0ull;
    cluster.sync();
    if (block != 0)
        return;
    Sums all = s.part[0];
    for (int b = 1; b < blocks; ++b)
        all = join(all, s.part[b]);
    const float log_s = logf(all.s);
    auto answer = [&](float v) { return __fsub_rn(__fsub_rn(v, all.m), log_s); };
    if (tid == 0) {
        if (a.logprob) {
            const int token = a.target[row];
            float v = 0.f;  // no token
            if (token >= a.vocab) {
                b2w4_report(a.status, B2W4_E_INVALID);
                v = __int_as_float(0x7fc00000);
            } else if (token >= 0) {
                v = answer(x[token]);
            }
            a.logprob[row] = v;
        }
        if (a.entropy)
            a.entropy[row] = __fsub_rn(log_s, __fdiv_rn(all.t, all.s));
    }
    for (int i = tid; i < blocks * a.top; i += kThreads) {
        const unsigned long long w = s.best[i / a.top][i % a.top];
        if (!w)
            continue;
        int before = 0;
        for (int b = 0; b < blocks; ++b)
            for (int j = 0; j < a.top; ++j)
                before += s.best[b][j] > w;
        if (before < a.top) {
            const size_t at = (size_t)row * a.top + before;
            if (a.indices)
                a.indices[at] = index_of(w);
            if (a.values)
                a.values[at] = answer(x[index_of(w)]);
        }
    }
}

// Blocks that share a row.
int cluster_for(int vocab) {
    int blocks = kMostCluster;
    while (blocks > 1 && vocab < blocks * 2 * kTile)
        blocks /= 2;
    return blocks;
}

}  // namespace

extern "C" int b2w4_logprobs(b2w4_ctx* ctx, const float* logits_dev, int ld, int rows, int vocab,
                             const int32_t* targets_dev, float* logprob_dev, float* entropy_dev,
                             int top, float* top_values_dev, int32_t* top_indices_dev) {
    if (!ctx)
        return B2W4_E_INVALID;
    if (!logits_dev || rows <= 0 || vocab <= 0 || ld < vocab || rows > INT_MAX / kMostCluster ||
        vocab > INT_MAX - 2 * kTile || (reinterpret_cast<uintptr_t>(logits_dev) & 3))
        return b2w4_fail(ctx, B2W4_E_INVALID, "logprobs: bad logits (rows %d, vocab %d, ld %d)",
                         rows, vocab, ld);
    if ((logprob_dev != nullptr) != (targets_dev != nullptr))
        return b2w4_fail(ctx, B2W4_E_INVALID, "logprobs: targets and logprob go together");
    if (top < 0 || top > kMostTop || top > vocab || (top == 0 && (top_values_dev || top_indices_dev)) ||
        (top > 0 && !top_values_dev && !top_indices_dev))
        return b2w4_fail(ctx, B2W4_E_INVALID,
                         "logprobs: top must be 0 to %d tokens of the vocabulary, with outputs "
                         "(got %d)", kMostTop, top);
    if (!logprob_dev && !entropy_dev && !top)
        return b2w4_fail(ctx, B2W4_E_INVALID, "logprobs: nothing is asked for");
    const b2w4_device_guard device(ctx);
    const Args a = {logits_dev,     targets_dev,     logprob_dev, entropy_dev,
                    top_values_dev, top_indices_dev, ld,          rows,
                    vocab,          top,             ctx->status_dev};
    const bool aligned = !((reinterpret_cast<uintptr_t>(logits_dev) & 15) || (ld & 3));
    const int blocks = cluster_for(vocab);
    B2W4_CUDA(ctx, b2w4_launch_chained_cluster(ctx->pdl, logprobs_kernel,
                                               dim3((unsigned)rows * blocks), dim3(kThreads),
                                               blocks, 0, ctx->stream, a, aligned));
    ctx->launches++;
    return B2W4_OK;
}
