// Log probabilities of given tokens, the entropy of their distributions, and the most likely
// tokens: one pass over the logits.
//
// With M the row's maximum, S = sum exp(x - M) and T = sum exp(x - M) (x - M):
//   log p(t) = x_t - M - log S,   entropy = log S - T / S   (a sum of two terms >= 0).
// Every warp keeps a running maximum m, every thread sums relative to its warp's, in 32 bits; two such
// triples join as M = max, S = S1 e^(m1 - M) + S2 e^(m2 - M), T likewise of T_i + (m_i - M) S_i.  The
// largest number's own term is 1 without a rounding, no term of T is above zero, so that S >= 1, T <= 0,
// no log probability is above zero and no entropy below, and a likely token's log probability, which
// is -log S, is as good as the sum of the others' terms.  (A maximum per thread would change in nearly
// every tile for some thread of a warp; a warp's changes about ln(tiles) times.)
//
// The k largest: a number below which the k-th largest cannot lie comes from the block's first tile
// (the k-th largest of the maxima of 64 groups of its numbers), and what is not below it goes to a
// list of its warp in shared memory.  After two tiles, four, eight, .. of a long chunk the lists are
// cut back to the k largest so far, by counting for each entry how many are before it, and the k-th
// is the new limit: about k numbers come between one time and the next.
//
// What bounds it: issue slots (64 % busy), about nine instructions for a number that takes four bytes
// of the card's bandwidth; sums take two numbers an instruction, and a warp looks for numbers above
// the limit only where a thread's largest of 16 is.  600 rows of 151,936 with the 20 largest: 87 us,
// 4.2 TB/s; 160 with 100 tokens left by a mask, 410 of equal numbers (first tiles without a useful
// limit).  One row of as many: 9.6 us, a first tile, its limit and the joins one after the other.
#include "b200w4_internal.cuh"

#include <math.h>

#include <climits>
#include <utility>

#include <cooperative_groups.h>

namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kVecs = 4;                    // of four numbers, a thread's share of a tile
constexpr int kTile = kThreads * kVecs * 4;
constexpr int kMostTop = 32;
constexpr int kGroups = 64;                 // of four threads each
constexpr int kTrim = 64;                   // a longer list is cut back to the k largest
constexpr int kList = kTrim + 32 * kVecs * 4;
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
// The smallest number above this word's: of the tiles behind it what is below that has no place ahead
// of the word, equal numbers included, whose indices are higher.  (With equal ones let through, every
// number of a row of equal logits, or of -inf where a mask leaves few tokens, went to the lists.)
__device__ __forceinline__ float above(unsigned long long w) {
    const unsigned key = (unsigned)(w >> 32);
    if (key == 0u)  // NaN, or no number at all
        return -INFINITY;
    if (key >= 0xff800000u)  // inf
        return INFINITY;
    return __uint_as_float((key + 1u & 0x80000000u) ? key + 1u ^ 0x80000000u : ~(key + 1u));
}

struct Sums {
    float m, s, t;
};
struct alignas(16) Shared {
    unsigned long long flat[kWarps * kTrim + kMostTop + 8];
    unsigned long long kept[kMostTop];  // the largest so far, in order; 0: there are not so many
    unsigned long long list[kWarps][kList];
    unsigned long long first[kWarps][kMostTop];
    unsigned long long best[kMostCluster][kMostTop];  // of the cluster's blocks, in block 0
    Sums part[kMostCluster];                          // likewise
    Sums warp[kWarps];
    float group[kGroups];
    float limit;
    int count[kWarps];
};

// Cuts the warp's list to its `top` largest, in order (or to all that there are); whole warp.
// Returns the least word that may still be wanted.
__device__ unsigned long long trim(Shared& s, int warp, int& n, int top) {
    const int lane = threadIdx.x & 31;
    unsigned long long *list = s.list[warp], *first = s.first[warp];
    __syncwarp();
    for (int i = lane; i < n; i += 32) {
        const unsigned long long w = list[i];
        int before = 0;
        for (int j = 0; j < n && before < top; ++j)
            before += list[j] > w;
        if (before < top)
            first[before] = w;
    }
    __syncwarp();
    const int left = min(n, top);
    if (lane < left)
        list[lane] = first[lane];
    const unsigned long long least = n >= top ? first[top - 1] : 0ull;
    n = left;
    __syncwarp();
    return least;
}

// The lists and what was kept before, cut to the `top` largest in s.kept; the lists are empty then.
// Whole block.
__device__ void settle(Shared& s, int warp, int& n, int top) {
    const int tid = threadIdx.x, lane = tid & 31;
    if (lane == 0)
        s.count[warp] = n;
    __syncthreads();
    int all = 0, mine = 0;
#pragma unroll
    for (int k = 0; k < kWarps; ++k) {
        mine += k < warp ? s.count[k] : 0;
        all += s.count[k];
    }
    for (int i = lane; i < n; i += 32)
        s.flat[mine + i] = s.list[warp][i];
    if (tid < top)
        s.flat[all + tid] = s.kept[tid];
    all += top;
    if (tid < 8)
        s.flat[all + tid] = 0ull;
    __syncthreads();
    if (tid < top)
        s.kept[tid] = 0ull;
    if (lane == 0)
        s.count[warp] = 0;
    n = 0;
    __syncthreads();
    for (int i = tid; i < all; i += kThreads) {
        const unsigned long long w = s.flat[i];
        int before = 0;
        for (int j = 0; j < all; j += 8)
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
                const ulonglong2 o = *reinterpret_cast<const ulonglong2*>(s.flat + j + e);
                before += (o.x > w) + (o.y > w);
            }
        if (before < top && w)
            s.kept[before] = w;
    }
    __syncthreads();
}

// The lanes' sums as one, in all lanes: n lanes, a power of two, next to each other.
__device__ __forceinline__ Sums join_lanes(Sums v, int n) {
    float m = v.m;
    for (int off = n / 2; off > 0; off >>= 1)
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
    const float base = m == -INFINITY ? 0.f : m;
    const float d = fmaxf(__fsub_rn(v.m, base), -1e30f), e = expf(d);
    // a side without numbers, or without any that count, has s = 0 and t = 0
    float t = e == 0.f ? __fmul_rn(v.s, 0.f) : __fmul_rn(__fmaf_rn(v.s, d, v.t), e);
    float sum = __fmul_rn(v.s, e);
    for (int off = n / 2; off > 0; off >>= 1) {
        sum = __fadd_rn(sum, __shfl_xor_sync(0xffffffffu, sum, off));
        t = __fadd_rn(t, __shfl_xor_sync(0xffffffffu, t, off));
    }
    return {m, sum, t};
}

// A cluster per row, a chunk of the row per block.
__global__ void __launch_bounds__(kThreads, 4)
logprobs_kernel(const Args a, bool aligned) {
    namespace cg = cooperative_groups;
    b2w4_pdl_chain_entry();
    extern __shared__ __align__(16) uint8_t s_dyn[];
    Shared& s = *reinterpret_cast<Shared*>(s_dyn);
    cg::cluster_group cluster = cg::this_cluster();
    const int blocks = (int)cluster.num_blocks(), block = (int)cluster.block_rank();
    // that every block of the cluster has begun is asked for before one writes to another
    auto begun = cluster.barrier_arrive();
    const int row = blockIdx.x / blocks;
    const float* x = a.x + (size_t)row * a.ld;
    const int chunk = ((a.vocab + blocks - 1) / blocks + 3) & ~3;
    const int lo = min(a.vocab, block * chunk), hi = min(a.vocab, lo + chunk);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    // number e of the thread's vector u of the tile at `base`
    auto place = [&](int base, int u) { return base + (tid + u * kThreads) * 4; };
    auto load = [&](int base, float4 (&v)[kVecs]) {
        if (aligned && base + kTile <= hi) {
#pragma unroll
            for (int u = 0; u < kVecs; ++u)
                v[u] = __ldg(reinterpret_cast<const float4*>(x + place(base, u)));
            return;
        }
#pragma unroll
        for (int u = 0; u < kVecs; ++u) {
            const int i = place(base, u);
            if (aligned && i + 4 <= hi) {
                v[u] = __ldg(reinterpret_cast<const float4*>(x + i));
            } else {
                v[u].x = i < hi ? __ldg(x + i) : -INFINITY;
                v[u].y = i + 1 < hi ? __ldg(x + i + 1) : -INFINITY;
                v[u].z = i + 2 < hi ? __ldg(x + i + 2) : -INFINITY;
                v[u].w = i + 3 < hi ? __ldg(x + i + 3) : -INFINITY;
            }
        }
    };
    if (tid < kWarps)
        s.count[tid] = 0;
    if (tid < kMostTop)
        s.kept[tid] = 0ull;
    __syncthreads();
    float m = -INFINITY;
    uint64_t sum2 = 0ull, t2 = 0ull;  // two sums each
    float limit = -INFINITY;  // what is below it is not among the largest
    int n = 0;  // of the warp's list; the same in all lanes
    float4 next[kVecs];
    load(lo, next);
    int tile = 0;
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
        float top = v[0];
#pragma unroll
        for (int i = 1; i < kVecs * 4; ++i)
            top = fmaxf(top, v[i]);
        if (__any_sync(0xffffffffu, top > m)) {
            float up = fmaxf(m, top);
#pragma unroll
            for (int off = 16; off > 0; off >>= 1)
                up = fmaxf(up, __shfl_xor_sync(0xffffffffu, up, off));
            if (m > -INFINITY) {
                const float d = __fsub_rn(m, up), e = expf(d);
                float s0, s1, t0, t1;
                b2w4_unpack2(sum2, s0, s1);
                b2w4_unpack2(t2, t0, t1);
                // (d may be -inf where up is inf)
                t2 = e == 0.f ? 0ull : b2w4_pack2(__fmul_rn(__fmaf_rn(s0, d, t0), e),
                                                  __fmul_rn(__fmaf_rn(s1, d, t1), e));
                sum2 = b2w4_pack2(__fmul_rn(s0, e), __fmul_rn(s1, e));
            }
            m = up;
        }
        const float from = m == -INFINITY ? 0.f : m;
        const uint64_t from2 = b2w4_pack2(from, from);
        const uint64_t log2e = b2w4_pack2(1.4426950408889634f, 1.4426950408889634f);
#pragma unroll
        for (int i = 0; i < kVecs * 4; i += 2) {
            const uint64_t d = b2w4_sub2(b2w4_pack2(v[i], v[i + 1]), from2);
            float d0, d1, z0, z1, e0, e1;
            b2w4_unpack2(d, d0, d1);
            b2w4_unpack2(b2w4_mul2(d, log2e), z0, z1);
            asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e0) : "f"(z0));
            asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e1) : "f"(z1));
            const uint64_t e = b2w4_pack2(e0, e1);
            asm("add.rn.f32x2 %0, %0, %1;" : "+l"(sum2) : "l"(e));
            // e = 0 where d = -inf
            t2 = b2w4_fma2(e, b2w4_pack2(fmaxf(d0, -200.f), fmaxf(d1, -200.f)), t2);
        }
        if (a.top > 0) {
            if (base == lo) {  // the whole block, if any of it is here
                float g = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                g = fmaxf(g, __shfl_xor_sync(0xffffffffu, g, 2));
                if (!(tid & 3))
                    s.group[tid >> 2] = g;
                if (tid == 0)
                    s.limit = -INFINITY;
                __syncthreads();
                if (tid < kGroups) {
                    const float mine = s.group[tid];
                    int above = 0, level = 0;
#pragma unroll 8
                    for (int j = 0; j < kGroups; ++j) {
                        above += s.group[j] > mine;
                        level += s.group[j] >= mine;
                    }
                    if (above < a.top && a.top <= level)
                        s.limit = mine;  // the same number from every thread that writes
                }
                __syncthreads();
                limit = s.limit;
            }
            auto cut = [&]() {
                __syncwarp();
                n = s.count[warp];
                __syncwarp();
                if (n > kTrim) {
                    limit = fmaxf(limit, above(trim(s, warp, n, a.top)));
                    if (lane == 0)
                        s.count[warp] = n;
                    __syncwarp();
                }
            };
            if (limit == -INFINITY) {
                // No limit yet (the whole warp): everything comes in, NaN too, which nothing else
                // wants.  A quarter at a time: a trim takes the square of what it finds (600 rows with
                // 100 tokens left 480 us with the tile's 512 at once).
#pragma unroll 1
                for (int u = 0; u < kVecs; ++u) {
#pragma unroll 1
                    for (int at = place(base, u), to = min(hi, at + 4); at < to; ++at) {
                        const float number = __ldg(x + at);
                        if (!(number < limit))
                            s.list[warp][atomicAdd(&s.count[warp], 1)] = word(number, at);
                    }
                    cut();
                }
            } else if (top >= limit) {
                unsigned mine = 0;
#pragma unroll
                for (int i = 0; i < kVecs * 4; ++i)
                    mine |= (unsigned)!(v[i] < limit) << i;
                // the number from memory again: one or two, where the registers would want a look
                // at each of the 16
                for (; mine; mine &= mine - 1) {
                    const int i = __ffs(mine) - 1;
                    const int at = place(base, i >> 2) + (i & 3);
                    if (at < hi)
                        s.list[warp][atomicAdd(&s.count[warp], 1)] = word(__ldg(x + at), at);
                }
            }
            cut();
            ++tile;
            // (worth its barriers where as much again and more is to come)
            if (tile > 1 && !(tile & (tile - 1)) && hi - base > 2 * tile * kTile) {
                settle(s, warp, n, a.top);
                limit = fmaxf(limit, above(s.kept[a.top - 1]));
            }
        }
    }
    float sum, t, sum_odd, t_odd;
    b2w4_unpack2(sum2, sum, sum_odd);
    b2w4_unpack2(t2, t, t_odd);
    sum = __fadd_rn(sum, sum_odd);
    t = __fadd_rn(t, t_odd);
    // the block's sums, in a fixed order
    const Sums mine = join_lanes({m, sum, t}, 32);
    if (lane == 0)
        s.warp[warp] = mine;
    if (a.top > 0)
        settle(s, warp, n, a.top);
    else
        __syncthreads();
    cluster.barrier_wait(std::move(begun));
    Shared* out = cluster.map_shared_rank(&s, 0);
    if (warp == 0) {
        const Sums all = join_lanes(s.warp[lane % kWarps], kWarps);
        if (lane == 0)
            out->part[block] = all;
    }
    if (tid < a.top)
        out->best[block][tid] = s.kept[tid];
    cluster.sync();
    if (block != 0)
        return;
    const Sums all = join_lanes(s.part[lane % blocks], blocks);
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

// Blocks that share a row.  A block's work is its numbers and a share of its own, about that of
// kFixed numbers (a limit, lists, the join); a multiprocessor's blocks are done side by side as fast
// as one up to kBeside of them, from where on they share it.
constexpr int kFixed = 8000;
constexpr double kBeside = 3.5;
int cluster_for(int rows, int vocab, int sm_count) {
    int best = 1;
    double least = 0;
    for (int blocks = 1; blocks <= kMostCluster; blocks *= 2) {
        if (blocks > 1 && vocab < blocks * kTile)
            break;
        const double each = ceil((double)rows * blocks / sm_count) / kBeside;
        const double time = (each > 1 ? each : 1) * (vocab / blocks + kFixed);
        if (blocks == 1 || time < least) {
            best = blocks;
            least = time;
        }
    }
    return best;
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
    static b2w4_smem_optin cfg;
    B2W4_CUDA(ctx, b2w4_opt_in_smem(ctx, logprobs_kernel, sizeof(Shared), cfg));
    const int blocks = cluster_for(rows, vocab, ctx->sm_count);
    B2W4_CUDA(ctx, b2w4_launch_chained_cluster(ctx->pdl, logprobs_kernel,
                                               dim3((unsigned)rows * blocks), dim3(kThreads),
                                               blocks, sizeof(Shared), ctx->stream, a, aligned));
    ctx->launches++;
    return B2W4_OK;
}
