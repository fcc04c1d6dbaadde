// The pages of a paged key-value cache: handing them out, sharing them between sequences, giving
// them back, moving them together, and copying them.
//
// A pool's state is on the device: how many tables hold a page (refs, 0: free), the sequences'
// tables and their lengths.  There is no list of free pages to keep in step with it: the free
// pages are those with refs 0, and they are handed out lowest first, so that what a call does
// follows from the state alone.  Nothing here needs the host, so a captured decode step takes its
// next page by itself.
//
// What bounds it: the bytes that move, each read and written once.  Compaction of a pool of 2048
// pages in 16 planes, 64 KB a page of a plane, 491 of which move: 184 us, 5.6 TB/s both ways.  Eight
// children of a sequence of 1001 tokens, their last pages copied in 72 planes, and given back: 19 to
// 22 us, the plan's and the commit's chains of lookups rather than the 38 MB.  A step's extend takes 4.9
// us where no sequence needs a page; where one does, one block looks through the counts from page 0: 11
// to 37 us in pools of 65,536 pages, 0.3 ms behind 900,000 pages in use.
//
// Only full pages are ever shared: a fork copies a last page that is not full.  So the page that
// a sequence's next token goes to is its own.
#include "b200w4_internal.cuh"

#include <climits>

namespace {

constexpr int kMostItems = 1024;  // sequences of a call
constexpr int kPlanes = 256;      // planes of a launch

struct Pool {
    int32_t *refs, *tables, *lengths;
    int pages, page_size, slots, table_len;
    int* status;
};

struct Planes {
    uint4* at[kPlanes];
    int count, pages;
    size_t vectors;  // of 16 bytes, in a page of a plane
};

__device__ __forceinline__ void bad(const Pool& p) { b2w4_report(p.status, B2W4_E_INVALID); }

__device__ __forceinline__ int pages_of(const Pool& p, int tokens) {
    return tokens / p.page_size + (tokens % p.page_size != 0);
}
// Tokens that slot's table can hold at most; table_len * page_size may pass 32 bits.
__device__ __forceinline__ int room(const Pool& p) {
    const long long r = (long long)p.table_len * p.page_size;
    return r < INT_MAX ? (int)r : INT_MAX;
}

// Sum of the threads' values before this one's; total: of all.  s_part: a word per warp.
template <int THREADS, typename N>
__device__ N scan(N v, N* s_part, N* total) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    N x = v;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
        const N y = __shfl_up_sync(0xffffffffu, x, off);
        if (lane >= off)
            x += y;
    }
    __syncthreads();  // s_part may still be read
    if (lane == 31)
        s_part[warp] = x;
    __syncthreads();
    N before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 32; ++w) {
        before += w < warp ? s_part[w] : 0;
        all += s_part[w];
    }
    *total = all;
    return before + x - v;
}

// Calls take(rank, page) for the first `want` free pages, lowest first, from the threads of the
// block; returns how many there are (the whole block has the same answer).
template <int THREADS, typename F>
__device__ int free_pages(const Pool& p, int want, int* s_part, F take) {
    constexpr int kEach = 16;
    int found = 0;
    for (int base = 0; base < p.pages && found < want; base += THREADS * kEach) {
        const int at = base + threadIdx.x * kEach;
        unsigned mask = 0;
#pragma unroll
        for (int i = 0; i < kEach; ++i)
            mask |= (unsigned)(at + i < p.pages && p.refs[at + i] == 0) << i;
        int total;
        int rank = found + scan<THREADS>(__popc(mask), s_part, &total);
        for (; mask && rank < want; mask &= mask - 1, ++rank)
            take(rank, at + __ffs(mask) - 1);
        found += total;
    }
    __syncthreads();
    return min(found, want);
}

// ---- extend ----------------------------------------------------------------------------

// lengths[slot] += count, with the pages that takes.  One block: thread i has item i; pages go
// out in the order of the list, to a sequence all that it needs or none.
__global__ void __launch_bounds__(kMostItems)
pages_extend_kernel(const Pool p, const int32_t* __restrict__ slots,
                    const int32_t* __restrict__ counts, int n, int32_t* __restrict__ granted) {
    b2w4_pdl_chain_entry();
    __shared__ int s_part[32], s_slot[kMostItems], s_first[kMostItems];
    // (what the sequences ask for may pass 32 bits)
    __shared__ long long s_sum[32], s_off[kMostItems + 1];
    const int i = threadIdx.x;
    const int slot = i < n ? (slots ? slots[i] : i) : -1;
    const int count = i < n ? (counts ? counts[i] : 1) : 0;
    s_slot[i] = slot;
    __syncthreads();
    bool good = i < n && slot >= 0 && slot < p.slots && count >= 0;
    if (slots && good)
        for (int j = 0; j < i; ++j)
            good &= s_slot[j] != slot;
    int length = 0, need = 0;
    if (good) {
        length = p.lengths[slot];
        good = length >= 0 && length <= room(p) && count <= room(p) - length;
        if (good)
            need = pages_of(p, length + count) - pages_of(p, length);
    }
    if (i < n && !good && slot != -1)
        bad(p);
    long long total;
    const long long off = scan<kMostItems>((long long)need, s_sum, &total);
    s_off[i] = off;
    s_first[i] = good ? pages_of(p, length) : 0;
    if (i == 0)
        s_off[kMostItems] = total;
    __syncthreads();
    int have = 0;
    const int want = (int)min(total, (long long)p.pages);
    if (want > 0)
        have = free_pages<kMostItems>(p, want, s_part, [&](int rank, int page) {
            int lo = 0, hi = kMostItems;  // the last item that begins at or before the rank
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (s_off[mid] <= rank)
                    lo = mid;
                else
                    hi = mid;
            }
            p.tables[(size_t)s_slot[lo] * p.table_len + s_first[lo] + rank - (int)s_off[lo]] =
                page;
            p.refs[page] = 1;
        });
    const bool fits = good && (need == 0 || off + need <= have);
    if (granted && i < n)
        granted[i] = fits ? slot : -1;
    if (!good)
        return;
    if (!fits) {  // back with what it got
        const int32_t* row = p.tables + (size_t)slot * p.table_len + s_first[i];
        for (long long r = off; r < have; ++r)
            p.refs[row[r - off]] = 0;
        b2w4_report(p.status, B2W4_E_NOMEM);
        return;
    }
    p.lengths[slot] = length + count;
}

// ---- copying ---------------------------------------------------------------------------

constexpr int kCopyThreads = 256, kCopyEach = 8;
constexpr size_t kPiece = kCopyThreads * kCopyEach;  // vectors that a block moves at a time

__device__ __forceinline__ void copy_piece(uint4* __restrict__ dst, const uint4* __restrict__ src,
                                           size_t from, size_t vectors) {
    uint4 v[kCopyEach];
    if (from + kPiece <= vectors) {
#pragma unroll
        for (int i = 0; i < kCopyEach; ++i)
            v[i] = src[from + threadIdx.x + i * kCopyThreads];
#pragma unroll
        for (int i = 0; i < kCopyEach; ++i)
            dst[from + threadIdx.x + i * kCopyThreads] = v[i];
    } else {
        for (size_t i = from + threadIdx.x; i < vectors; i += kCopyThreads)
            dst[i] = src[i];
    }
}

// Pages src(i) -> dst(i), i < n, of every plane; the blocks share the pieces.
template <typename F>
__device__ __forceinline__ void copy_pages(const Planes& planes, int n, F pair) {
    const size_t pieces = (planes.vectors + kPiece - 1) / kPiece;
    const size_t all = (size_t)n * planes.count * pieces;
    for (size_t w = blockIdx.x; w < all; w += gridDim.x) {
        const size_t page = w / pieces;
        const int plane = (int)(page % planes.count), i = (int)(page / planes.count);
        int src, dst;
        if (!pair(i, &src, &dst))
            continue;
        uint4* base = planes.at[plane];
        copy_piece(base + dst * planes.vectors, base + src * planes.vectors,
                   (w - page * pieces) * kPiece, planes.vectors);
    }
}

__global__ void __launch_bounds__(kCopyThreads)
pages_copy_kernel(const __grid_constant__ Planes planes, const int32_t* __restrict__ src,
                  const int32_t* __restrict__ dst, int n, int* status) {
    b2w4_pdl_chain_entry();
    copy_pages(planes, n, [&](int i, int* s, int* d) {
        *s = src[i];
        *d = dst[i];
        const bool good = (unsigned)*s < (unsigned)planes.pages &&
                          (unsigned)*d < (unsigned)planes.pages;
        if (!good)
            b2w4_report(status, B2W4_E_INVALID);
        return good && *s != *d;
    });
}

// ---- fork ------------------------------------------------------------------------------

// What a fork does, worked out from the pool's state by every block that needs it: parents are
// read as they were before the call, and what the copying kernel changes (the children's tables,
// counts of pages in use) is nothing that this reads.
template <int THREADS>
struct ForkPlan {
    static constexpr int kEach = kMostItems / THREADS;
    int part[32];
    int parent[kMostItems], child[kMostItems];  // child -1: the item does nothing
    int length[kMostItems];
    int page[kMostItems];  // the copy of the parent's last page; -1: that is full
    int free[kMostItems];

    __device__ void make(const Pool& p, const int32_t* parents, const int32_t* children, int n,
                         bool report) {
        const int first = threadIdx.x * kEach;  // the thread's items
        for (int i = threadIdx.x; i < n; i += THREADS) {
            parent[i] = parents[i];
            child[i] = children[i];
        }
        __syncthreads();
        unsigned wrong = 0, quiet = 0, need = 0;  // a bit per item
#pragma unroll
        for (int e = 0; e < kEach; ++e) {
            const int i = first + e;
            if (i >= n)
                break;
            bool good = (unsigned)parent[i] < (unsigned)p.slots &&
                        (unsigned)child[i] < (unsigned)p.slots;
            for (int j = 0; j < i && good; ++j)
                good = child[j] != child[i];
            int len = 0;
            if (good) {
                len = p.lengths[parent[i]];
                good = p.lengths[child[i]] == 0 && len >= 0 && len <= room(p);
            }
            length[i] = good ? len : 0;
            wrong |= (unsigned)!good << e;
            quiet |= (unsigned)(parent[i] == -1 || child[i] == -1) << e;
            need |= (unsigned)(good && len % p.page_size != 0) << e;
        }
        int total;  // the barriers of the sum: every thread has compared the children
        int rank = scan<THREADS>(__popc(need), part, &total);
        const int have = total ? free_pages<THREADS>(p, total, part,
                                                     [&](int r, int f) { free[r] = f; })
                               : 0;
#pragma unroll
        for (int e = 0; e < kEach; ++e) {
            const int i = first + e;
            if (i >= n)
                break;
            const bool wants = need >> e & 1, gets = wants && rank < have;
            page[i] = gets ? free[rank] : -1;
            rank += wants;
            if ((wrong >> e & 1) || (wants && !gets)) {
                child[i] = -1;
                if (report && !(quiet >> e & 1))
                    b2w4_report(p.status, wants ? B2W4_E_NOMEM : B2W4_E_INVALID);
            }
        }
        __syncthreads();
    }
};

// The copies of last pages; with `tables`, the children's rows and the counts of shared pages.
__global__ void __launch_bounds__(kCopyThreads)
pages_fork_kernel(const Pool p, const __grid_constant__ Planes planes,
                  const int32_t* __restrict__ parents, const int32_t* __restrict__ children, int n,
                  bool tables) {
    b2w4_pdl_chain_entry();
    __shared__ ForkPlan<kCopyThreads> plan;
    plan.make(p, parents, children, n, false);
    if (tables)
        for (int i = blockIdx.x; i < n; i += gridDim.x) {
            if (plan.child[i] < 0)
                continue;
            const int full = plan.length[i] / p.page_size;
            const int32_t* from = p.tables + (size_t)plan.parent[i] * p.table_len;
            int32_t* to = p.tables + (size_t)plan.child[i] * p.table_len;
            for (int j = threadIdx.x; j < full; j += kCopyThreads) {
                const int page = from[j];
                to[j] = page;
                if ((unsigned)page < (unsigned)p.pages)
                    atomicAdd(p.refs + page, 1);
                else
                    bad(p);
            }
            if (threadIdx.x == 0 && plan.page[i] >= 0)
                to[full] = plan.page[i];
        }
    copy_pages(planes, n, [&](int i, int* s, int* d) {
        if (plan.child[i] < 0 || plan.page[i] < 0)
            return false;
        *s = p.tables[(size_t)plan.parent[i] * p.table_len + plan.length[i] / p.page_size];
        *d = plan.page[i];
        if ((unsigned)*s < (unsigned)p.pages)
            return true;
        bad(p);
        return false;
    });
}

// Behind it: the children's lengths, and their own pages in use.
__global__ void __launch_bounds__(kMostItems)
pages_fork_commit_kernel(const Pool p, const int32_t* __restrict__ parents,
                         const int32_t* __restrict__ children, int n) {
    b2w4_pdl_chain_entry();
    __shared__ ForkPlan<kMostItems> plan;
    plan.make(p, parents, children, n, true);
    const int i = threadIdx.x;
    if (i < n && plan.child[i] >= 0) {
        p.lengths[plan.child[i]] = plan.length[i];
        if (plan.page[i] >= 0)
            p.refs[plan.page[i]] = 1;
    }
}

// ---- free ------------------------------------------------------------------------------

// A block per item.  A slot that is named twice is free when the second comes.
__global__ void __launch_bounds__(256)
pages_free_kernel(const Pool p, const int32_t* __restrict__ slots) {
    b2w4_pdl_chain_entry();
    __shared__ int s_length;
    const int slot = slots ? slots[blockIdx.x] : (int)blockIdx.x;
    if ((unsigned)slot >= (unsigned)p.slots) {
        if (threadIdx.x == 0 && slot != -1)
            bad(p);
        return;
    }
    if (threadIdx.x == 0) {
        int length = atomicExch(p.lengths + slot, 0);
        if (length < 0 || length > room(p)) {
            bad(p);
            length = length < 0 ? 0 : room(p);
        }
        s_length = length;
    }
    __syncthreads();
    const int held = pages_of(p, s_length);
    for (int j = threadIdx.x; j < held; j += blockDim.x) {
        const int page = p.tables[(size_t)slot * p.table_len + j];
        if ((unsigned)page >= (unsigned)p.pages) {
            bad(p);
        } else if (atomicSub(p.refs + page, 1) <= 0) {  // nobody held it
            atomicAdd(p.refs + page, 1);
            bad(p);
        }
    }
}

// ---- compact ---------------------------------------------------------------------------

// Which pages move: work [pages / 2] | [pages / 2], the pages in use at or beyond the count of
// pages in use, ascending, and the free ones below it that they go to; -1 behind the last.  There
// are as many of one as of the other, and never more than half of the pool.
__global__ void __launch_bounds__(1024)
pages_compact_plan_kernel(const Pool p, int32_t* __restrict__ work, int32_t* __restrict__ used) {
    b2w4_pdl_chain_entry();
    constexpr int kEach = 16, kStep = 1024 * kEach;
    __shared__ int s_part[32];
    const int half = p.pages / 2;
    auto in_use = [&](int base) {
        const int at = base + threadIdx.x * kEach;
        unsigned mask = 0;
#pragma unroll
        for (int i = 0; i < kEach; ++i)
            mask |= (unsigned)(at + i < p.pages && p.refs[at + i] != 0) << i;
        return mask;
    };
    int mine = 0, count;
    for (int base = 0; base < p.pages; base += kStep)
        mine += __popc(in_use(base));
    scan<1024>(mine, s_part, &count);
    int holes = 0, movers = 0;
    for (int base = 0; base < p.pages; base += kStep) {
        const int at = base + threadIdx.x * kEach;
        const unsigned use = in_use(base);
        // pages below the count, of the thread's
        const int below = max(0, min(kEach, count - at));
        const unsigned low = (1u << below) - 1u;
        const unsigned exist = (1u << max(0, min(kEach, p.pages - at))) - 1u;
        unsigned hole = ~use & low & exist, mover = use & ~low;
        int all;
        int h = holes + scan<1024>(__popc(hole), s_part, &all);
        holes += all;
        int m = movers + scan<1024>(__popc(mover), s_part, &all);
        movers += all;
        for (; hole; hole &= hole - 1)
            work[half + h++] = at + __ffs(hole) - 1;
        for (; mover; mover &= mover - 1)
            work[m++] = at + __ffs(mover) - 1;
    }
    for (int i = movers + threadIdx.x; i < half; i += 1024)
        work[i] = -1;
    if (used && threadIdx.x == 0)
        *used = count;
}

// The moves; with `tables`, the tables' entries and the counts too.
__global__ void __launch_bounds__(kCopyThreads)
pages_compact_move_kernel(const Pool p, const __grid_constant__ Planes planes,
                          const int32_t* __restrict__ work, bool tables) {
    b2w4_pdl_chain_entry();
    const int half = p.pages / 2;
    int n = 0;  // how many move: the first -1
    for (int lo = 0, hi = half; lo < hi; n = lo) {
        const int mid = (lo + hi) >> 1;
        if (work[mid] >= 0)
            lo = mid + 1;
        else
            hi = mid;
    }
    if (n == 0)
        return;
    if (tables) {
        const size_t threads = (size_t)gridDim.x * kCopyThreads;
        const size_t first = (size_t)blockIdx.x * kCopyThreads + threadIdx.x;
        for (size_t i = first; i < (size_t)n; i += threads) {
            p.refs[work[half + i]] = p.refs[work[i]];
            p.refs[work[i]] = 0;
        }
        for (size_t i = first; i < (size_t)p.slots * p.table_len; i += threads) {
            const int slot = (int)(i / p.table_len), j = (int)(i - (size_t)slot * p.table_len);
            const int length = min(max(p.lengths[slot], 0), room(p));
            if (j >= pages_of(p, length))
                continue;
            const int page = p.tables[i];
            int lo = 0, hi = n;
            while (lo < hi) {
                const int mid = (lo + hi) >> 1;
                if (work[mid] < page)
                    lo = mid + 1;
                else
                    hi = mid;
            }
            if (lo < n && work[lo] == page)
                p.tables[i] = work[half + lo];
        }
    }
    copy_pages(planes, n, [&](int i, int* s, int* d) {
        *s = work[i];
        *d = work[half + i];
        return true;
    });
}

Pool pool_of(b2w4_ctx* ctx, const b2w4_page_pool& p) {
    return {p.refs_dev, p.tables_dev, p.lengths_dev, p.pages,
            p.page_size, p.slots, p.table_len, ctx->status_dev};
}

// The planes in groups that a launch takes: f(group, whether it is the first).
template <typename F>
int by_group(const b2w4_page_planes& pl, F f) {
    for (int first = 0; first < pl.count; first += kPlanes) {
        Planes g = {};
        g.count = pl.count - first < kPlanes ? pl.count - first : kPlanes;
        g.pages = pl.pages;
        g.vectors = pl.page_bytes / 16;
        for (int i = 0; i < g.count; ++i)
            g.at[i] = static_cast<uint4*>(pl.planes[first + i]);
        const int rc = f(g, first == 0);
        if (rc != B2W4_OK)
            return rc;
    }
    return B2W4_OK;
}

// Blocks for n pages of a group's planes: every piece one, up to what is resident at once.
unsigned copy_blocks(const b2w4_ctx* ctx, const Planes& g, size_t n) {
    const size_t pieces = n * g.count * ((g.vectors + kPiece - 1) / kPiece);
    const size_t most = (size_t)ctx->sm_count * 8;
    return (unsigned)(pieces < 1 ? 1 : pieces < most ? pieces : most);
}

}  // namespace

// What a pool and its planes must be; the text of what is wrong, or NULL.  Host only.
extern "C" const char* b2w4_pages_refusal(const b2w4_page_pool* p, const b2w4_page_planes* pl,
                                          int wants_pool, int wants_planes) {
    if (wants_pool) {
        if (!p || !p->refs_dev || !p->tables_dev || !p->lengths_dev)
            return "no pool";
        if (p->pages <= 0 || p->page_size <= 0 || p->slots <= 0 || p->table_len <= 0)
            return "pages, page_size, slots and table_len must be positive";
        if (p->pages > INT_MAX / 2)
            return "fewer than 2^30 pages";
    }
    if (wants_planes) {
        if (!pl || !pl->planes || pl->count <= 0 || pl->pages <= 0)
            return "no planes";
        if (!pl->page_bytes || pl->page_bytes % 16)
            return "a page of a plane is a positive multiple of 16 bytes";
        if (wants_pool && pl->pages != p->pages)
            return "the planes have another number of pages than the pool";
        for (int i = 0; i < pl->count; ++i)
            if (!pl->planes[i] || (reinterpret_cast<uintptr_t>(pl->planes[i]) & 15))
                return "planes must be 16-byte aligned device memory";
    }
    return nullptr;
}

extern "C" {

int b2w4_pages_extend(b2w4_ctx* ctx, const b2w4_page_pool* pool, const int32_t* slots_dev,
                      const int32_t* counts_dev, int n, int32_t* granted_dev) {
    if (!ctx)
        return B2W4_E_INVALID;
    if (const char* why = b2w4_pages_refusal(pool, nullptr, 1, 0))
        return b2w4_fail(ctx, B2W4_E_INVALID, "pages_extend: %s", why);
    if (n <= 0 || n > kMostItems || (!slots_dev && n > pool->slots))
        return b2w4_fail(ctx, B2W4_E_INVALID, "pages_extend: 1 to %d sequences (got %d)",
                         kMostItems, n);
    const b2w4_device_guard device(ctx);
    B2W4_CUDA(ctx, b2w4_launch_chained(ctx->pdl, pages_extend_kernel, dim3(1), dim3(kMostItems), 0,
                                       ctx->stream, pool_of(ctx, *pool), slots_dev, counts_dev,
                                       n, granted_dev));
    ctx->launches++;
    return B2W4_OK;
}

int b2w4_pages_fork(b2w4_ctx* ctx, const b2w4_page_pool* pool, const b2w4_page_planes* planes,
                    const int32_t* parents_dev, const int32_t* children_dev, int n) {
    if (!ctx)
        return B2W4_E_INVALID;
    if (const char* why = b2w4_pages_refusal(pool, planes, 1, 1))
        return b2w4_fail(ctx, B2W4_E_INVALID, "pages_fork: %s", why);
    if (!parents_dev || !children_dev || n <= 0 || n > kMostItems)
        return b2w4_fail(ctx, B2W4_E_INVALID, "pages_fork: 1 to %d parents and children (got %d)",
                         kMostItems, n);
    const b2w4_device_guard device(ctx);
    const Pool p = pool_of(ctx, *pool);
    const int rc = by_group(*planes, [&](const Planes& g, bool first) {
        B2W4_CUDA(ctx, b2w4_launch_chained(ctx->pdl, pages_fork_kernel,
                                           dim3(copy_blocks(ctx, g, n)), dim3(kCopyThreads), 0,
                                           ctx->stream, p, g, parents_dev, children_dev, n, first));
        ctx->launches++;
        return (int)B2W4_OK;
    });
    if (rc != B2W4_OK)
        return rc;
    B2W4_CUDA(ctx, b2w4_launch_chained(ctx->pdl, pages_fork_commit_kernel, dim3(1),
                                       dim3(kMostItems), 0, ctx->stream, p, parents_dev,
                                       children_dev, n));
    ctx->launches++;
    return B2W4_OK;
}

int b2w4_pages_free(b2w4_ctx* ctx, const b2w4_page_pool* pool, const int32_t* slots_dev, int n) {
    if (!ctx)
        return B2W4_E_INVALID;
    if (const char* why = b2w4_pages_refusal(pool, nullptr, 1, 0))
        return b2w4_fail(ctx, B2W4_E_INVALID, "pages_free: %s", why);
    if (n <= 0 || (!slots_dev && n > pool->slots))
        return b2w4_fail(ctx, B2W4_E_INVALID, "pages_free: no slots (got %d)", n);
    const b2w4_device_guard device(ctx);
    B2W4_CUDA(ctx, b2w4_launch_chained(ctx->pdl, pages_free_kernel, dim3(n), dim3(256), 0,
                                       ctx->stream, pool_of(ctx, *pool), slots_dev));
    ctx->launches++;
    return B2W4_OK;
}

int b2w4_pages_compact(b2w4_ctx* ctx, const b2w4_page_pool* pool, const b2w4_page_planes* planes,
                       int32_t* work_dev, int32_t* used_dev) {
    if (!ctx)
        return B2W4_E_INVALID;
    if (const char* why = b2w4_pages_refusal(pool, planes, 1, 1))
        return b2w4_fail(ctx, B2W4_E_INVALID, "pages_compact: %s", why);
    if (!work_dev)
        return b2w4_fail(ctx, B2W4_E_INVALID, "pages_compact: no work area");
    const b2w4_device_guard device(ctx);
    const Pool p = pool_of(ctx, *pool);
    B2W4_CUDA(ctx, b2w4_launch_chained(ctx->pdl, pages_compact_plan_kernel, dim3(1), dim3(1024), 0,
                                       ctx->stream, p, work_dev, used_dev));
    ctx->launches++;
    return by_group(*planes, [&](const Planes& g, bool first) {
        B2W4_CUDA(ctx, b2w4_launch_chained(ctx->pdl, pages_compact_move_kernel,
                                           dim3(copy_blocks(ctx, g, pool->pages / 2 + 1)),
                                           dim3(kCopyThreads), 0, ctx->stream, p, g, work_dev,
                                           first));
        ctx->launches++;
        return (int)B2W4_OK;
    });
}

int b2w4_pages_copy(b2w4_ctx* ctx, const b2w4_page_planes* planes, const int32_t* src_dev,
                    const int32_t* dst_dev, int n) {
    if (!ctx)
        return B2W4_E_INVALID;
    if (const char* why = b2w4_pages_refusal(nullptr, planes, 0, 1))
        return b2w4_fail(ctx, B2W4_E_INVALID, "pages_copy: %s", why);
    if (!src_dev || !dst_dev || n <= 0)
        return b2w4_fail(ctx, B2W4_E_INVALID, "pages_copy: no pages (got %d)", n);
    const b2w4_device_guard device(ctx);
    return by_group(*planes, [&](const Planes& g, bool) {
        B2W4_CUDA(ctx, b2w4_launch_chained(ctx->pdl, pages_copy_kernel,
                                           dim3(copy_blocks(ctx, g, n)), dim3(kCopyThreads), 0,
                                           ctx->stream, g, src_dev, dst_dev, n, ctx->status_dev));
        ctx->launches++;
        return (int)B2W4_OK;
    });
}

}  // extern "C"
