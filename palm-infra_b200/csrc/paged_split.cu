// Attention of one new token per sequence over a paged cache, or of a run's tokens one by one, split
// over the cache's length and joined.
//
// For the heads of a kv head, with the keys of a part of the cache: m = max s_j, l = sum
// exp(s_j - m), o = sum exp(s_j - m) v_j; parts join by scaling with exp(m_part - m).
//
// What bounds it: the bytes of the cache.  So the keys that the batch sees, in blocks of 16, lie
// in one line over sequences, kv heads and sets of 8 or 16 heads, of which every warp of the chip
// takes an equal share, whatever the lengths: one long sequence fills the chip as well as many
// short ones.  A warp streams its blocks through a cp.async ring of its own, across the ends of
// sequences, and meets no other warp.  A part of the cache that began or ended inside another
// warp's share goes to the work area; a second launch joins those.  (Joined by each thread block
// first, what its warps have of a tile costs more than it saves: 64 sequences of 1028 keys 36 -> 37
// us, two of 120,001 and 58,650 85 -> 93.)
// 120,001 and 58,650 keys of 64 heads over 4 of 128, bf16: 83 us (4.4 TB/s; 255 registers leave two
// warps a scheduler, whose latencies show); 64 sequences under a window of 1024, 64 heads over 8 of 64,
// fp16: 32 us; one of 300 tokens: 11 us, 7 of them lookups and first loads, 3 the join.
//
// Products are mma.sync m16n8k16, the heads as the rows: with 16 heads a key costs 8192
// multiply-adds, more than the fp32 pipe has in the time that the key's bytes take.  Every operand
// of 32 bits is a sum of pieces of the cache's 16-bit type, products small ones first, sums in 32
// bits: three bf16 pieces (24 bits) beside a bf16 cache; two fp16 pieces (22 bits) of the row's
// query or probabilities times a power of two beside an fp16 cache, the second one of what is left
// times 2^12 (paged_kernels.cuh); three pieces of both sides beside an fp32 cache, six products of the
// nine.  A sum in the tensor core truncates, so an output's sum over a block of keys starts from zero
// and is added to the running one with one rounding.
//
// What pieces cannot hold -- infinities, NaN, results that are not finite -- is done key by key in
// 32 bits (paged::attend_row), which has the rule for values of probability zero.
#include "paged_kernels.cuh"

#include <math.h>

#include <climits>

namespace {

using paged::add2;
using paged::Args;
using paged::Attend;
using paged::cp16;
using paged::exp2_neg;
using paged::kDown;
using paged::kHalf;
using paged::kLift;
using paged::kTop;
using paged::Sequence;

constexpr int kKeys = 16;  // of a block

template <typename T>
struct Pieces {  // of a query or probability, and of a key or value
    static constexpr int kQ = 3, kK = 1;
};
template <>
struct Pieces<__half> {
    static constexpr int kQ = 2, kK = 1;
};
template <>
struct Pieces<float> {
    static constexpr int kQ = 3, kK = 3;
};

// Operands of a product's rows.  SET 16: a row for each of 16 heads, an operand for each piece.  SET
// 8: eight heads, their first pieces in rows 0 to 7 and their second ones in rows 8 to 15 of one
// operand, their third ones, if any, in a second: two thirds or half of the products, and of the
// registers, for groups of up to eight heads; a score is the sum of two rows.
template <typename T, int SET>
constexpr int kOperands = SET == 16 ? Pieces<T>::kQ : Pieces<T>::kQ - 1;

constexpr int kMostWarps = 16;
template <typename T, int DIM, int SET>
struct Ring {
    static constexpr int kRow = DIM * sizeof(T);       // bytes
    static constexpr int kHalf = kKeys * kRow;          // keys; the values behind them
    static constexpr int kSlot = 2 * kHalf;
    static constexpr int kWarps = kSlot > 24576   ? 3
                                  : kSlot > 16384 ? 4
                                  : DIM > 128     ? 7
                                  : kSlot > 8192  ? 7
                                  : SET == 16     ? 8
                                  : kSlot > 4096  ? 12
                                                  : 16;
    static constexpr int kSlots = 208 * 1024 / (kWarps * kSlot) < 2
                                      ? 2
                                      : 208 * 1024 / (kWarps * kSlot) > 5
                                            ? 5
                                            : 208 * 1024 / (kWarps * kSlot);
    static constexpr int kBytes = kWarps * kSlots * kSlot;
    static_assert(kWarps <= kMostWarps, "the work area");
};

// Keys that the one token of a sequence sees: [0, low) and [from, length).
struct Seen {
    int low, from, count;
};
__device__ __forceinline__ Seen seen_by(const Sequence& s, const paged::Window& w) {
    Seen v = {0, 0, 0};
    if (s.count != 1 || s.length <= 0)
        return v;
    v.from = w.from(s.length - 1);
    v.low = min(w.sinks, v.from);
    v.count = v.low + s.length - v.from;
    return v;
}
template <bool BY_ROW>
__device__ __forceinline__ int blocks_of(const Args& a, const paged::Window& w, int i, bool report) {
    bool bad = false;
    const Sequence s = paged::item<BY_ROW>(a, i, &bad);
    if (report && (bad || s.count > 1))
        b2w4_report(a.status, B2W4_E_INVALID);
    return (seen_by(s, w).count + kKeys - 1) / kKeys;
}

// Whole warp.  Blocks of all sequences; every tile (kv head and set of heads) of a sequence has as
// many.  mine: those of sequence `lane`.
template <bool BY_ROW>
__device__ int line_of(const Args& a, const paged::Window& w, int tiles, bool report, int* mine) {
    const int lane = threadIdx.x & 31;
    *mine = lane < a.items ? blocks_of<BY_ROW>(a, w, lane, report) : 0;
    int sum = *mine;
#pragma unroll 4
    for (int i = lane + 32; i < a.items; i += 32)
        sum += blocks_of<BY_ROW>(a, w, i, report);
    return __reduce_add_sync(0xffffffffu, sum) * tiles;
}

// Whole warp.  The sequence whose blocks hold block `at` of the line, and where they begin.
template <bool BY_ROW>
__device__ int find(const Args& a, const paged::Window& w, int tiles, int at, int mine, int* begin) {
    const int lane = threadIdx.x & 31;
    int before = 0;
    for (int base = 0; base < a.items; base += 32) {
        int n = mine * tiles;
        if (base > 0)
            n = base + lane < a.items ? blocks_of<BY_ROW>(a, w, base + lane, false) * tiles : 0;
        int x = n;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, x, off);
            if (lane >= off)
                x += y;
        }
        const unsigned past = __ballot_sync(0xffffffffu, before + x > at);
        if (past) {
            const int l = __ffs(past) - 1;
            *begin = before + __shfl_sync(0xffffffffu, x - n, l);
            return base + l;
        }
        before += __shfl_sync(0xffffffffu, x, 31);
    }
    *begin = before;
    return a.items;
}

// A part: m and l of its SET rows, then their outputs.
template <int DIM, int SET>
struct Part {
    static constexpr int kFloats = 2 * SET + SET * DIM;
};
// Whose part it is: the tile's heads, in the rows of q and out of its sequence, and the warps that
// have parts of it, the first's in its second place if `second`.  heads 0: no part.
struct Owner {
    int seq, head0, heads, row;
    int first, last, second, pad;
};
// The work area: two parts of every warp, and their owners.
template <int DIM, int SET>
__host__ __device__ constexpr size_t owners_at(int blocks) {
    return sizeof(float) * 2 * Part<DIM, SET>::kFloats * (size_t)kMostWarps * blocks;
}
// Where a warp's stream of blocks is: what its next blocks' tile needs.
struct Stream {
    const int32_t* table;
    int low, from, count, blocks, seq;
    int tile, kv_row;  // kv_row: of the tile's kv head, in a page
};

template <int N>
__device__ __forceinline__ void cp_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldmatrix(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(at));
}
__device__ __forceinline__ void ldmatrix_trans(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(at));
}
__device__ __forceinline__ float4 lds128(uint32_t at) {
    float4 v;
    asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                 : "r"(at));
    return v;
}
// bf16 products except beside an fp16 cache
template <typename T>
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                    uint32_t b1) {
    if constexpr (std::is_same_v<T, __half>)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, "
            "%7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, "
            "%7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// The next piece of two numbers; they keep what is left, times kUp beside an fp16 cache.
template <typename T>
__device__ __forceinline__ uint32_t take_piece(float& lo, float& hi) {
    uint64_t v = b2w4_pack2(lo, hi);
    const uint32_t p = paged::take_piece<T>(v, kHalf<T> ? paged::kUp : 1.f);
    b2w4_unpack2(v, lo, hi);
    return p;
}
// Sums of products of first pieces, and of second ones, as one.
template <typename T>
__device__ __forceinline__ float joined(float second, float first) {
    return kHalf<T> ? __fmaf_rn(second, kDown, first) : __fadd_rn(second, first);
}
template <typename T>
__device__ __forceinline__ uint64_t joined2(uint64_t second, uint64_t first) {
    return kHalf<T> ? b2w4_fma2(second, b2w4_pack2(kDown, kDown), first) : add2(second, first);
}

// Pieces of a row's column pairs (2t and 2t + 8, of rows r and r + 8) as operands: at(i, e) is
// register e of operand i.
template <int Q, int N, typename At>
__device__ __forceinline__ void operands(const uint32_t (&piece)[Q][N], At at) {
    if constexpr (N == 4) {
#pragma unroll
        for (int i = 0; i < Q; ++i) {
            at(i, 0) = piece[i][0];
            at(i, 1) = piece[i][2];
            at(i, 2) = piece[i][1];
            at(i, 3) = piece[i][3];
        }
    } else {
        at(0, 0) = piece[0][0];
        at(0, 1) = piece[1][0];
        at(0, 2) = piece[0][1];
        at(0, 3) = piece[1][1];
        if constexpr (Q == 3) {
            at(1, 0) = piece[2][0];
            at(1, 1) = 0u;
            at(1, 2) = piece[2][1];
            at(1, 3) = 0u;
        }
    }
}
// A row's sums over parts, by one warp: lane + 32 i are its features.
template <int DIM, int SET>
struct Joined {
    static constexpr int kOwn = DIM / 32;
    float m = -INFINITY, l = 0.f, o[kOwn] = {};
    // parts w, w + step, .. up to `last`, kBatch of them on their way together
    template <typename PartOf>
    __device__ __forceinline__ void add(PartOf part_of, int w, int last, int step, int row) {
        constexpr int kBatch = 10;
        const int lane = threadIdx.x & 31;
        for (; w <= last; w += kBatch * step) {
            float pm[kBatch], pl[kBatch], x[kBatch][kOwn];
#pragma unroll
            for (int b = 0; b < kBatch; ++b) {
                const bool in = w + b * step <= last;
                const float* part = part_of(in ? w + b * step : w);
                pm[b] = in ? part[row] : -INFINITY;
                pl[b] = in ? part[SET + row] : 0.f;
#pragma unroll
                for (int i = 0; i < kOwn; ++i)
                    x[b][i] = in ? part[2 * SET + row * DIM + lane + 32 * i] : 0.f;
            }
            float top = m;
#pragma unroll
            for (int b = 0; b < kBatch; ++b)
                top = fmaxf(top, pm[b]);
            const float base = top == -INFINITY ? 0.f : top;
            const float before = exp2_neg(__fsub_rn(m, base));
            m = top;
            l = __fmul_rn(l, before);
#pragma unroll
            for (int i = 0; i < kOwn; ++i)
                o[i] = __fmul_rn(o[i], before);
#pragma unroll
            for (int b = 0; b < kBatch; ++b) {
                const float e = exp2_neg(__fsub_rn(pm[b], base));
                l = __fmaf_rn(pl[b], e, l);
#pragma unroll
                for (int i = 0; i < kOwn; ++i)
                    o[i] = __fmaf_rn(x[b][i], e, o[i]);
            }
        }
    }
    __device__ __forceinline__ void store(float* part, int row) const {
        const int lane = threadIdx.x & 31;
        if (lane == 0) {
            part[row] = m;
            part[SET + row] = l;
        }
#pragma unroll
        for (int i = 0; i < kOwn; ++i)
            part[2 * SET + row * DIM + lane + 32 * i] = o[i];
    }
    // the result of one of the owner's heads
    template <typename T, bool BY_ROW>
    __device__ __forceinline__ void finish(const Args& a, const Attend& p, const Owner& t, int head) {
        const int lane = threadIdx.x & 31;
        float* out = p.out + (size_t)t.row * p.ldo + (size_t)head * DIM;
        const float over = __fdiv_rn(1.f, l);
        bool odd = false;
#pragma unroll
        for (int i = 0; i < kOwn; ++i) {
            const float x = __fmul_rn(o[i], over);
            odd |= paged::odd_result<T>(x);
            out[lane + 32 * i] = x;
        }
        __syncwarp();
        if (__any_sync(0xffffffffu, odd)) {
            bool bad = false;
            const Sequence s = paged::item<BY_ROW>(a, t.seq, &bad);
            paged::attend_row<T, DIM>(a, s, p.q + (size_t)t.row * p.ldq + (size_t)head * DIM,
                                      s.length - 1, head / (p.heads / a.kv_heads), p.scale,
                                      p.window, out);
        }
    }
};

template <typename T, int DIM, int SET, bool BY_ROW>
__global__ void __launch_bounds__(Ring<T, DIM, SET>::kWarps * 32, 1)
paged_split_kernel(const Args a, const Attend p, float* __restrict__ parts,
                   Owner* __restrict__ owners) {
    using R = Ring<T, DIM, SET>;
    constexpr int kQ = Pieces<T>::kQ, kK = Pieces<T>::kK, kSteps = DIM / 16, kTiles = DIM / 8;
    constexpr int kHalves = SET / 8;  // of a product's rows, heads
    constexpr int kA = kOperands<T, SET>;
    constexpr bool kWide = sizeof(T) == 4;  // an fp32 cache
    extern __shared__ __align__(1024) uint8_t smem[];
    b2w4_pdl_chain_entry();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int r = lane >> 2, t = lane & 3;  // row of the products' operands, column pair
    const int group = p.heads / a.kv_heads, sets = (group + SET - 1) / SET;
    const int tiles = a.kv_heads * sets;
    Stream& stream = reinterpret_cast<Stream*>(smem + R::kBytes)[warp];
    int mine;
    const int total = line_of<BY_ROW>(a, p.window, tiles, blockIdx.x + warp == 0, &mine);
    // a share for every warp, or, where there are fewer blocks, for some warps of every thread block
    const int active = min(R::kWarps, max(1, (total + (int)gridDim.x - 1) / (int)gridDim.x));
    const int warps = gridDim.x * active, share = max(1, (total + warps - 1) / warps);
    const int me = warp * gridDim.x + blockIdx.x;
    int at = warp < active ? min(total, me * share) : total;
    const int end = min(total, at + share);
    // sequences that see no key
    for (int i = warp * gridDim.x + blockIdx.x; i < a.items; i += gridDim.x * R::kWarps) {
        bool bad = false;
        const Sequence s = paged::item<BY_ROW>(a, i, &bad);
        if (s.count == 1 && seen_by(s, p.window).count == 0)
            for (int d = lane; d < p.heads * DIM; d += 32)
                p.out[(size_t)s.first * p.ldo + d] = 0.f;
    }
    // (of the warps behind those at work too)
    if (lane < 2)
        owners[2 * me + lane].heads = 0;
    if (at >= end)
        return;
    const uint32_t ring = (uint32_t)__cvta_generic_to_shared(smem) + warp * R::kSlots * R::kSlot;
    const int first = at;
    int begin;
    int seq = find<BY_ROW>(a, p.window, tiles, at, mine, &begin);
    auto prefetch_queries = [&](int row, int kvh, int head0) {
        const float* q = p.q + (size_t)row * p.ldq + (size_t)head0 * DIM;
        for (int d = lane * 32; d < min(SET, (kvh + 1) * group - head0) * DIM; d += 1024)
            asm volatile("prefetch.global.L1 [%0];" ::"l"(q + d));
    };

    // ---- the stream of blocks --------------------------------------------------------
    // It is ahead of the blocks that are worked on, in the next tile or sequence too.
    int f_at = at, f_b = 0;  // the next block, in the line and in its tile
    const int page_stride = a.kv_heads * a.page_size;
    auto to_tile = [&](int tile) {  // of the stream's sequence
        __syncwarp();
        const int kvh = tile / sets;
        if (lane == 0) {
            stream.tile = tile;
            stream.kv_row = kvh * a.page_size;
        }
        bool bad = false;
        prefetch_queries(paged::item<BY_ROW>(a, stream.seq, &bad).first, kvh,
                         kvh * group + (tile - kvh * sets) * SET);
        __syncwarp();
    };
    auto to_sequence = [&](int i) {  // the first from sequence i on that sees a key
        bool bad = false;
        Sequence s = paged::item<BY_ROW>(a, i, &bad);
        Seen seen = seen_by(s, p.window);
        while (seen.count == 0 && i + 1 < a.items) {
            s = paged::item<BY_ROW>(a, ++i, &bad);
            seen = seen_by(s, p.window);
        }
        __syncwarp();
        if (lane == 0)
            stream = {s.table, seen.low, seen.from, seen.count,
                      (seen.count + kKeys - 1) / kKeys, i, 0, 0};
        __syncwarp();
    };
    // Lane j < 16 learns where key j of the next block lies; -1: there is no such key.
    auto next_row_of = [&]() {
        if (f_at >= end)
            return -1;
        if (f_b == stream.blocks) {
            f_b = 0;
            int tile = stream.tile + 1;
            if (tile == tiles) {
                to_sequence(stream.seq + 1);
                tile = 0;
            }
            to_tile(tile);
        }
        const int i = f_b * kKeys + (lane & 15);
        ++f_b;
        ++f_at;
        if (i >= stream.count)
            return -1;
        const int low = stream.low, j = i < low ? i : i - low + stream.from;
        const int n = paged::page_of(a, j), page = stream.table[n];
        if ((unsigned)page >= (unsigned)a.pages) {
            b2w4_report(a.status, B2W4_E_INVALID);
            return -1;
        }
        return page * page_stride + stream.kv_row + j - n * a.page_size;
    };
    constexpr int kChunks = R::kRow / 16, kRows = kChunks >= 32 ? 1 : 32 / kChunks;
    auto swizzled = [&](int key, int chunk, bool values) {
        const int x = kWide ? (values ? key & 6 : (key & 1) << 2) : key & 7;
        return (uint32_t)(key * R::kRow + ((chunk ^ x) << 4));
    };
    auto fetch = [&](int slot, int row) {
        const uint32_t dst = ring + slot * R::kSlot;
#pragma unroll
        for (int i = 0; i < kKeys / kRows; ++i) {
            const int key = i * kRows + (kRows > 1 ? lane / kChunks : 0);
            const int from = __shfl_sync(0xffffffffu, row, key);
            const size_t off = (size_t)max(from, 0) * R::kRow;
#pragma unroll
            for (int c = lane % kChunks; c < kChunks; c += 32) {
                cp16(dst + swizzled(key, c, false), static_cast<const uint8_t*>(a.k) + off + c * 16,
                     from >= 0);
                cp16(dst + R::kHalf + swizzled(key, c, true),
                     static_cast<const uint8_t*>(a.v) + off + c * 16, from >= 0);
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        return __ballot_sync(0xffffffffu, row >= 0) & 0xffffu;
    };
    // of the keys of the blocks on their way, those that exist: the next block's first
    unsigned there[R::kSlots - 1];
    int slot = 0, into = R::kSlots - 1;
    to_sequence(seq);
    f_b = (at - begin) % stream.blocks;
    to_tile((at - begin) / stream.blocks);
    int rows[R::kSlots];
#pragma unroll
    for (int i = 0; i < R::kSlots; ++i)
        rows[i] = next_row_of();
#pragma unroll
    for (int i = 0; i < R::kSlots - 1; ++i)
        there[i] = fetch(i, rows[i]);
    int next_row = rows[R::kSlots - 1];

    while (at < end) {
        bool bad = false;
        const Sequence s = paged::item<BY_ROW>(a, seq, &bad);
        const Seen seen = seen_by(s, p.window);
        const int blocks = (seen.count + kKeys - 1) / kKeys;
        if (blocks == 0) {
            ++seq;
            continue;
        }
        // the tile, and the share's blocks of it
        const int tile = (at - begin) / blocks;
        const int b0 = at - begin - tile * blocks, b1 = min(blocks, b0 + end - at);
        const int kvh = tile / sets, head0 = kvh * group + (tile - kvh * sets) * SET;
        const int heads = min(SET, (kvh + 1) * group - head0);

        // ---- the heads' queries as operands ------------------------------------------
        uint32_t q[kA][kSteps][4];
        float unscale[kHalves];
        {
            const float* row = p.q + (size_t)s.first * p.ldq + (size_t)head0 * DIM;
            float x[kSteps][4 * kHalves];
#pragma unroll
            for (int k = 0; k < kSteps; ++k)
#pragma unroll
                for (int h = 0; h < kHalves; ++h) {
                    const bool in = r + 8 * h < heads;
                    const float* src = row + (r + 8 * h) * DIM + 16 * k;
                    if (kWide) {  // column pairs 2t and 2t + 8 hold features 4t .. 4t + 3
                        const float4 v = in ? *reinterpret_cast<const float4*>(src + 4 * t)
                                            : make_float4(0.f, 0.f, 0.f, 0.f);
                        x[k][4 * h] = v.x;
                        x[k][4 * h + 1] = v.y;
                        x[k][4 * h + 2] = v.z;
                        x[k][4 * h + 3] = v.w;
                    } else {
                        const float2 z = make_float2(0.f, 0.f);
                        const float2 v = in ? *reinterpret_cast<const float2*>(src + 2 * t) : z;
                        const float2 w = in ? *reinterpret_cast<const float2*>(src + 2 * t + 8) : z;
                        x[k][4 * h] = v.x;
                        x[k][4 * h + 1] = v.y;
                        x[k][4 * h + 2] = w.x;
                        x[k][4 * h + 3] = w.y;
                    }
                }
#pragma unroll
            for (int h = 0; h < kHalves; ++h) {
                unscale[h] = 1.f;
                if constexpr (kHalf<T>) {
                    float top = 0.f;
#pragma unroll
                    for (int k = 0; k < kSteps; ++k)
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            top = fmaxf(top, fabsf(x[k][4 * h + e]));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                    int e = (int)(__float_as_uint(top) >> 23) - 127;
                    e = top == 0.f ? kTop : min(max(e, -100), 120);
                    const float up = __uint_as_float((unsigned)(127 + kTop - e) << 23);
                    unscale[h] = __uint_as_float((unsigned)(127 - kTop + e) << 23);
#pragma unroll
                    for (int k = 0; k < kSteps; ++k)
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            x[k][4 * h + i] = __fmul_rn(x[k][4 * h + i], up);
                }
            }
#pragma unroll
            for (int k = 0; k < kSteps; ++k) {
                uint32_t piece[kQ][2 * kHalves];
#pragma unroll
                for (int i = 0; i < kQ; ++i)
#pragma unroll
                    for (int e = 0; e < 2 * kHalves; ++e)
                        piece[i][e] = take_piece<T>(x[k][2 * e], x[k][2 * e + 1]);
                operands(piece, [&](int i, int e) -> uint32_t& { return q[i][k][e]; });
            }
        }

        float m[kHalves], l[kHalves], factor[kHalves];
#pragma unroll
        for (int h = 0; h < kHalves; ++h) {
            m[h] = -INFINITY;
            l[h] = 0.f;
            factor[h] = __fmul_rn(__fmul_rn(p.scale, 1.4426950408889634f), unscale[h]);
        }
        uint64_t o[kTiles][kHalves];  // two columns each
#pragma unroll
        for (int i = 0; i < kTiles; ++i)
#pragma unroll
            for (int h = 0; h < kHalves; ++h)
                o[i][h] = 0ull;

        auto block = [&](int slot, unsigned keys) {
            const uint32_t ks = ring + slot * R::kSlot, vs = ks + R::kHalf;
            // sums of their own for products of different sizes: more chains side by side
            float by[kA][2][4] = {};
#pragma unroll
            for (int k = 0; k < kSteps; ++k) {
                if constexpr (kWide) {
#pragma unroll
                    for (int n = 0; n < 2; ++n) {
                        const float4 f = lds128(ks + swizzled(n * 8 + r, 4 * k + t, false));
                        float v[4] = {f.x, f.y, f.z, f.w};
                        uint32_t b[kK][2];
#pragma unroll
                        for (int i = 0; i < kK; ++i) {
                            b[i][0] = take_piece<T>(v[0], v[1]);
                            b[i][1] = take_piece<T>(v[2], v[3]);
                        }
                        if constexpr (SET == 16) {
                            mma<T>(by[2][n], q[2][k], b[0][0], b[0][1]);
                            mma<T>(by[1][n], q[1][k], b[0][0], b[0][1]);
                            mma<T>(by[0][n], q[0][k], b[0][0], b[0][1]);
                            mma<T>(by[2][n], q[1][k], b[1][0], b[1][1]);
                            mma<T>(by[1][n], q[0][k], b[1][0], b[1][1]);
                            mma<T>(by[2][n], q[0][k], b[2][0], b[2][1]);
                        } else {
                            mma<T>(by[1][n], q[1][k], b[0][0], b[0][1]);
                            mma<T>(by[0][n], q[0][k], b[2][0], b[2][1]);
                            mma<T>(by[0][n], q[0][k], b[1][0], b[1][1]);
                            mma<T>(by[0][n], q[0][k], b[0][0], b[0][1]);
                        }
                    }
                } else {
                    // matrices: keys 0-7 and 8-15, features 0-7 and 8-15 of the step
                    uint32_t b[4];
                    ldmatrix(b, ks + swizzled((lane & 7) + (lane >> 4) * 8,
                                              2 * k + ((lane >> 3) & 1), false));
#pragma unroll
                    for (int i = kA - 1; i >= 0; --i) {
                        mma<T>(by[i][0], q[i][k], b[0], b[1]);
                        mma<T>(by[i][1], q[i][k], b[2], b[3]);
                    }
                }
            }
            float alpha[kHalves], pr[kHalves][4];  // of keys 2t, 2t + 1 and those behind 8
#pragma unroll
            for (int h = 0; h < kHalves; ++h) {
                float sc[4], top = m[h];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int n = e >> 1, c = e & 1;
                    if constexpr (SET == 16) {
                        sc[e] = by[kA - 1][n][2 * h + c];
#pragma unroll
                        for (int i = kA - 2; i >= 0; --i)
                            sc[e] = joined<T>(sc[e], by[i][n][2 * h + c]);
                    } else {
                        sc[e] = by[0][n][2 + c];
                        if (kA > 1)
                            sc[e] = __fadd_rn(by[kA - 1][n][c], sc[e]);
                        sc[e] = joined<T>(sc[e], by[0][n][c]);
                    }
                    sc[e] = __fmul_rn(sc[e], factor[h]);
                    if (!(keys >> (8 * n + 2 * t + c) & 1))
                        sc[e] = -INFINITY;
                    top = fmaxf(top, sc[e]);
                }
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                const float base = top == -INFINITY ? 0.f : top;
                alpha[h] = exp2_neg(__fsub_rn(m[h], base));
                m[h] = top;
                const float shift = __fsub_rn(kLift<T>, base);
                float sum = 0.f;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    pr[h][e] = exp2_neg(__fadd_rn(sc[e], shift));
                    sum = __fadd_rn(sum, pr[h][e]);
                }
                l[h] = __fmaf_rn(l[h], alpha[h], sum);
            }
            uint32_t pp[kA][4];
            {
                uint32_t piece[kQ][2 * kHalves];
#pragma unroll
                for (int i = 0; i < kQ; ++i)
#pragma unroll
                    for (int e = 0; e < 2 * kHalves; ++e)
                        piece[i][e] = take_piece<T>(pr[e >> 1][2 * (e & 1)],
                                                    pr[e >> 1][2 * (e & 1) + 1]);
                operands(piece, [&](int i, int e) -> uint32_t& { return pp[i][e]; });
            }
            uint64_t alpha2[kHalves];
#pragma unroll
            for (int h = 0; h < kHalves; ++h)
                alpha2[h] = b2w4_pack2(alpha[h], alpha[h]);
            auto add = [&](int n, const float (&x)[4]) {
                const uint64_t x0 = b2w4_pack2(x[0], x[1]), x1 = b2w4_pack2(x[2], x[3]);
                if constexpr (SET == 16) {
                    o[n][0] = b2w4_fma2(o[n][0], alpha2[0], x0);
                    o[n][1] = b2w4_fma2(o[n][1], alpha2[1], x1);
                } else {
                    o[n][0] = b2w4_fma2(o[n][0], alpha2[0], joined2<T>(x1, x0));
                }
            };
            // sums of two fp16 pieces that are apart, rows of first ones in x, of second ones in y
            auto join_rows = [&](float (&x)[4], const float (&y)[4]) {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    x[e] = joined<T>(y[e], x[e]);
            };
            if constexpr (kWide) {
                // a group of 32 features: lane's four of each of its keys, one per tile
#pragma unroll
                for (int j = 0; j < DIM / 32; ++j) {
                    float v[4][4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float4 f =
                            lds128(vs + swizzled(2 * t + (e & 1) + (e >> 1) * 8, 8 * j + r, true));
                        v[e][0] = f.x;
                        v[e][1] = f.y;
                        v[e][2] = f.z;
                        v[e][3] = f.w;
                    }
                    float x[4][4] = {};
                    uint32_t b[4][kK][2];
#pragma unroll
                    for (int n = 0; n < 4; ++n)
#pragma unroll
                        for (int i = 0; i < kK; ++i) {
                            b[n][i][0] = take_piece<T>(v[0][n], v[1][n]);
                            b[n][i][1] = take_piece<T>(v[2][n], v[3][n]);
                        }
                    constexpr int kPairs = SET == 16 ? 6 : 4;
                    constexpr int kPa[2][6] = {{2, 0, 1, 1, 0, 0}, {1, 0, 0, 0}};
                    constexpr int kPb[2][6] = {{0, 2, 1, 0, 1, 0}, {0, 2, 1, 0}};
#pragma unroll
                    for (int i = 0; i < kPairs; ++i)
#pragma unroll
                        for (int n = 0; n < 4; ++n)
                            mma<T>(x[n], pp[kPa[SET == 8][i]], b[n][kPb[SET == 8][i]][0],
                                   b[n][kPb[SET == 8][i]][1]);
#pragma unroll
                    for (int n = 0; n < 4; ++n)
                        add(4 * j + n, x[n]);
                }
            } else {
#pragma unroll
                for (int n = 0; n < kTiles; n += 4) {
                    // keys 0-7 and 8-15, features 8n .. 8n + 7 and the next eight
                    uint32_t b[2][4];
#pragma unroll
                    for (int j = 0; j < 2; ++j)
                        ldmatrix_trans(b[j], vs + swizzled((lane & 7) + ((lane >> 3) & 1) * 8,
                                                           n + 2 * j + (lane >> 4), true));
                    float x[4][4] = {};
                    if constexpr (kHalf<T> && SET == 16) {
                        float y[4][4] = {};
#pragma unroll
                        for (int i = kA - 1; i >= 0; --i)
#pragma unroll
                            for (int j = 0; j < 4; ++j)
                                mma<T>(i ? y[j] : x[j], pp[i], b[j >> 1][(j & 1) * 2],
                                       b[j >> 1][(j & 1) * 2 + 1]);
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            join_rows(x[j], y[j]);
                    } else {
#pragma unroll
                        for (int i = kA - 1; i >= 0; --i)
#pragma unroll
                            for (int j = 0; j < 4; ++j)
                                mma<T>(x[j], pp[i], b[j >> 1][(j & 1) * 2],
                                       b[j >> 1][(j & 1) * 2 + 1]);
                    }
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        add(n + j, x[j]);
                }
            }
        };

        // One copy of the body: unrolled over the slots, its code came from beyond the
        // instruction cache.
#pragma unroll 1
        for (int b = b0; b < b1; ++b) {
            cp_wait<R::kSlots - 2>();
            __syncwarp();
            const unsigned keys = there[0];
#pragma unroll
            for (int i = 0; i + 1 < R::kSlots - 1; ++i)
                there[i] = there[i + 1];
            there[R::kSlots - 2] = fetch(into, next_row);  // the slot that the block before left
            next_row = next_row_of();
            block(slot, keys);
            __syncwarp();
            into = slot;
            slot = slot + 1 == R::kSlots ? 0 : slot + 1;
        }

        // ---- the part, or the result -------------------------------------------------
#pragma unroll
        for (int h = 0; h < kHalves; ++h) {
            l[h] = __fadd_rn(l[h], __shfl_xor_sync(0xffffffffu, l[h], 1));
            l[h] = __fadd_rn(l[h], __shfl_xor_sync(0xffffffffu, l[h], 2));
        }
        const bool whole = b0 == 0 && b1 == blocks;
        float* part = parts + ((size_t)2 * me + (at != first)) * Part<DIM, SET>::kFloats;
        if (!whole && lane == 0) {
            const int from = begin + tile * blocks, w0 = from / share;
            owners[2 * me + (at != first)] = {seq, head0, heads, s.first, w0,
                                              (from + blocks - 1) / share, from != w0 * share, 0};
        }
        bool odd = false;
#pragma unroll
        for (int h = 0; h < kHalves; ++h) {
            const int row = r + 8 * h;
            if (row >= heads)
                continue;
            float* dst = whole ? p.out + (size_t)s.first * p.ldo + (size_t)(head0 + row) * DIM
                               : part + 2 * SET + row * DIM;
            if (!whole && t == 0) {
                part[row] = m[h];
                part[SET + row] = l[h];
            }
            auto final = [&](float x) {
                if (!whole)
                    return x;
                x = __fdiv_rn(x, l[h]);
                odd |= paged::odd_result<T>(x);
                return x;
            };
            if constexpr (kWide) {
#pragma unroll
                for (int j = 0; j < DIM / 32; ++j) {
                    float x[4][2];
#pragma unroll
                    for (int n = 0; n < 4; ++n)
                        b2w4_unpack2(o[4 * j + n][h], x[n][0], x[n][1]);
#pragma unroll
                    for (int e = 0; e < 2; ++e)
                        *reinterpret_cast<float4*>(dst + 32 * j + 8 * t + 4 * e) = make_float4(
                            final(x[0][e]), final(x[1][e]), final(x[2][e]), final(x[3][e]));
                }
            } else {
#pragma unroll
                for (int n = 0; n < kTiles; ++n) {
                    float x, y;
                    b2w4_unpack2(o[n][h], x, y);
                    *reinterpret_cast<float2*>(dst + 8 * n + 2 * t) = make_float2(final(x), final(y));
                }
            }
        }
        __syncwarp();
        if (__any_sync(0xffffffffu, odd)) {
            for (int h = 0; h < heads; ++h)
                paged::attend_row<T, DIM>(a, s, p.q + (size_t)s.first * p.ldq +
                                                    (size_t)(head0 + h) * DIM,
                                          s.length - 1, kvh, p.scale, p.window,
                                          p.out + (size_t)s.first * p.ldo +
                                              (size_t)(head0 + h) * DIM);
        }
        at += b1 - b0;
        if (at - begin == blocks * tiles) {
            begin = at;
            ++seq;
        }
    }
    cp_wait<0>();
}

// Joins what several warps' shares hold of a tile.  A warp has an owner's place in the work area:
// with the other owners of the same tile it shares out the tile's heads.  Where a tile has more than
// kFew parts its heads are shared out to the blocks that have a place of it, and a block's warps take
// the parts in turn.
constexpr int kJoinWarps = 16, kFew = 20;
template <typename T, int DIM, int SET, bool BY_ROW>
__global__ void __launch_bounds__(kJoinWarps * 32)
paged_join_kernel(const Args a, const Attend p, const float* __restrict__ parts,
                  const Owner* __restrict__ owners, int places) {
    b2w4_pdl_chain_entry();
    __shared__ float s_part[kJoinWarps][Part<DIM, 1>::kFloats];
    __shared__ Owner s_own[kJoinWarps];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int place = blockIdx.x * kJoinWarps + warp;
    Owner mine = {};
    if (place < places)
        mine = owners[place];
    if (lane == 0)
        s_own[warp] = mine;
    auto part = [&](const Owner& t, int w) {
        return parts + (size_t)(2 * w + (w == t.first && t.second)) * Part<DIM, SET>::kFloats;
    };
    if (mine.heads && mine.last - mine.first < kFew) {
        for (int row = place / 2 - mine.first; row < mine.heads; row += mine.last - mine.first + 1) {
            Joined<DIM, SET> sum;
            sum.add([&](int w) { return part(mine, w); }, mine.first, mine.last, 1, row);
            sum.template finish<T, BY_ROW>(a, p, mine, mine.head0 + row);
        }
    }
    __syncthreads();
    // the first place in this block of every tile with many parts; a tile's places are neighbours
    // or have one without a part between them
    bool leads = false;
    if (lane < kJoinWarps) {
        const Owner& t = s_own[lane];
        leads = t.heads && t.last - t.first >= kFew;
        for (int back = 1; back <= 2 && back <= lane && leads; ++back) {
            const Owner& o = s_own[lane - back];
            leads = !(o.heads && o.seq == t.seq && o.head0 == t.head0);
        }
    }
    for (unsigned m = __ballot_sync(0xffffffffu, leads); m; m &= m - 1) {
        const Owner t = s_own[__ffs(m) - 1];
        const int b0 = (2 * t.first + t.second) / kJoinWarps, b1 = 2 * t.last / kJoinWarps;
        for (int row = blockIdx.x - b0; row < t.heads; row += b1 - b0 + 1) {
            Joined<DIM, SET> sum;
            sum.add([&](int w) { return part(t, w); }, t.first + warp, t.last, kJoinWarps, row);
            Joined<DIM, 1> all, one;
            one.m = sum.m;
            one.l = sum.l;
#pragma unroll
            for (int d = 0; d < DIM / 32; ++d)
                one.o[d] = sum.o[d];
            __syncthreads();  // of the row before
            one.store(s_part[warp], 0);
            __syncthreads();
            if (warp != 0)
                continue;
            all.add([&](int w) { return s_part[w]; }, 0, kJoinWarps - 1, 1, 0);
            all.template finish<T, BY_ROW>(a, p, t, t.head0 + row);
        }
    }
}

template <typename T, int DIM, int SET, bool BY_ROW>
int launch_set(b2w4_ctx* ctx, const Args& a, const Attend& p, void* work) {
    using R = Ring<T, DIM, SET>;
    static b2w4_smem_optin cfg;
    auto kern = paged_split_kernel<T, DIM, SET, BY_ROW>;
    constexpr size_t smem = R::kBytes + R::kWarps * sizeof(Stream);
    static_assert(smem <= 227 * 1024, "shared memory");
    B2W4_CUDA(ctx, b2w4_opt_in_smem(ctx, kern, smem, cfg));
    const int blocks = ctx->sm_count;
    float* parts = static_cast<float*>(work);
    Owner* owners =
        reinterpret_cast<Owner*>(static_cast<uint8_t*>(work) + owners_at<DIM, SET>(blocks));
    B2W4_CUDA(ctx, b2w4_launch_chained(ctx->pdl, kern, dim3(blocks), dim3(R::kWarps * 32), smem,
                                       ctx->stream, a, p, parts, owners));
    ctx->launches++;
    B2W4_CUDA(ctx, b2w4_launch_chained(ctx->pdl, paged_join_kernel<T, DIM, SET, BY_ROW>,
                                       dim3((2 * blocks * R::kWarps + kJoinWarps - 1) / kJoinWarps),
                                       dim3(kJoinWarps * 32), 0,
                                       ctx->stream, a, p, static_cast<const float*>(parts),
                                       static_cast<const Owner*>(owners),
                                       2 * blocks * R::kWarps));
    ctx->launches++;
    return B2W4_OK;
}
// Heads of a set: the registers of wide heads have no room for sixteen.
int set_of(int dim, int group) { return dim <= 128 && group > 8 ? 16 : 8; }
template <typename T, int DIM, bool BY_ROW>
int launch(b2w4_ctx* ctx, const Args& a, const Attend& p, void* work) {
    if constexpr (DIM <= 128)
        if (set_of(DIM, p.heads / a.kv_heads) == 16)
            return launch_set<T, DIM, 16, BY_ROW>(ctx, a, p, work);
    return launch_set<T, DIM, 8, BY_ROW>(ctx, a, p, work);
}
template <typename T, bool BY_ROW>
int launch_dim(b2w4_ctx* ctx, int dim, const Args& a, const Attend& p, void* work) {
    switch (dim) {
    case 64: return launch<T, 64, BY_ROW>(ctx, a, p, work);
    case 128: return launch<T, 128, BY_ROW>(ctx, a, p, work);
    case 192: return launch<T, 192, BY_ROW>(ctx, a, p, work);
    default: return launch<T, 256, BY_ROW>(ctx, a, p, work);
    }
}
template <bool BY_ROW>
int launch_type(b2w4_ctx* ctx, int type, int dim, const Args& a, const Attend& p, void* work) {
    return type == B2W4_F16    ? launch_dim<__half, BY_ROW>(ctx, dim, a, p, work)
           : type == B2W4_BF16 ? launch_dim<__nv_bfloat16, BY_ROW>(ctx, dim, a, p, work)
                               : launch_dim<float, BY_ROW>(ctx, dim, a, p, work);
}

}  // namespace

// The most that a set of eight heads or of sixteen takes.
size_t b2w4_paged_split_work(int sm_count, int dim) {
    const size_t parts = dim <= 64    ? owners_at<64, 16>(sm_count)
                         : dim <= 128 ? owners_at<128, 16>(sm_count)
                                      : owners_at<256, 8>(sm_count);
    return parts + 2 * sizeof(Owner) * (size_t)kMostWarps * sm_count;
}

// A launch counts its blocks of keys in 32 bits: the items (paged::item) that it may have, each of
// `keys` keys at most; 0: not even one.
extern "C" int b2w4_paged_split_items(int items, double keys, int dim, int heads, int kv_heads) {
    const int set = set_of(dim, heads / kv_heads);
    const double tiles = (double)kv_heads * ((heads / kv_heads + set - 1) / set);
    const double most = floor(0x40000000 / (ceil(keys / kKeys) * tiles));
    return most < items ? (int)most : items;
}

int b2w4_launch_paged_split(b2w4_ctx* ctx, int type, int dim, Args a, const Attend& p,
                            bool by_row, void* work) {
    const int items = by_row ? a.rows : a.sequences;
    double keys = a.max_length < (double)a.table_len * a.page_size
                      ? a.max_length
                      : (double)a.table_len * a.page_size;
    if (p.window.size > 0 && (double)p.window.size + p.window.sinks < keys)
        keys = (double)p.window.size + p.window.sinks;
    const int most = b2w4_paged_split_items(items, keys, dim, p.heads, a.kv_heads);
    if (most == 0)
        return b2w4_fail(ctx, B2W4_E_INVALID, "paged_attention: max_length is too large (%d)",
                         a.max_length);
    for (int first = 0; first < items; first += a.items) {
        a.first_item = first;
        a.items = most < items - first ? most : items - first;
        const int rc = by_row ? launch_type<true>(ctx, type, dim, a, p, work)
                              : launch_type<false>(ctx, type, dim, a, p, work);
        if (rc != B2W4_OK)
            return rc;
    }
    return B2W4_OK;
}
