// Attention of runs of new tokens (prompts, chunks of prompts, several sequences at once) over a
// paged cache, on tcgen05.mma kind::f16.
//
// A block takes 128 rows -- the heads of one kv head for consecutive tokens of a sequence --
// against blocks of kKeys keys with a running softmax in 32 bits (base 2): m the running maximum,
// p = 2^(s - m), o = o 2^(m_old - m) + p V.  The keys that any of its rows sees, the first ones
// that stay visible and those from the first row's window on, are taken as one list; what a row
// does not see of them is masked.
//
// Operands of 32 bits are sums of pieces of the cache's 16-bit type, as in paged_split.cu: three
// bf16 pieces of queries and probabilities beside a bf16 cache, two fp16 pieces of a row's queries
// times a power of two and of its probabilities beside an fp16 cache, the second one of what is left
// times 2^12 (paged_kernels.cuh); three pieces of both sides, six products, beside an fp32 cache; small
// products first.  The first product behind those of the second fp16 pieces takes their sum times
// 2^-12 (an MMA's scale of its input).  Sums in tensor memory truncate, so those of an output are of
// one block of keys, and the running output is in registers, one rounding per block.
//
// What bounds it: a step's rows, then the MMAs, which the pieces multiply.  128 rows x 128 keys x 128
// features in three pieces are 48 MMAs of about 58 cycles, 2800 cycles; the rows' part of a step --
// scores out of tensor memory, 2^x, the sum, three pieces, the running output -- is about 3500
// beside them, and a step about 4000 (clock readings; the tensor pipe is 64 % busy).  6000 tokens of
// 32 heads over 8 of 128, bf16, a window of 2048: 408 to 473 us from one GPU to another, 0.4 PFLOP/s
// of the formula's products and 1.2 with the pieces'.  A tile's start and end take about 17,000
// cycles: queries in 3600 and into pieces 1500, the first scores 2500, the last P V 2250, results out
// 5500.  They tell where rows see few keys: 333 tokens behind 900, fp32, 64 us; six chunks of 50 to
// 700, fp16, 64 / 8 heads of 64 under a window of 512, 82.
//
// Blocks stay and take one tile after the other, so that a tile's first keys and values are on their
// way while the one before is finished (6000 tokens as above with a block per tile: 455 to 498 us).
//
// Roles: warps of rows, two or four threads to a row; a warp that issues the MMAs, the scores' up to
// two blocks ahead; one that looks the tiles up, two ahead; the rest bring keys and values.  Both lie
// in shared memory as they lie in the cache, a key's features in 128-byte rows: the keys are the
// scores' B operand with features running fastest, the values P V's with them running slowest, so
// neither is transposed.  Rows come one by one with their pages' addresses, so a page may end
// anywhere.
//
// A row whose result is not finite is done again key by key (paged::attend_row): a key that it does
// not see, or that has no probability, may hold anything.  That takes as long as the cache is (a warp
// does a row, 0.6 us a key), so it waits until the block's other warps are done: every wait is bounded
// (2 s), and within the tiles none is for more than a tile's steps.
#include "paged_kernels.cuh"
#include "tcgen05_ops.cuh"

namespace {

using paged::add2;
using paged::Args;
using paged::Attend;
using paged::cp16;
using paged::exp2_neg;
using paged::kHalf;
using paged::kLift;
using paged::kTop;
using paged::Sequence;
using paged::take_piece;

constexpr int kRows = 128;

template <typename T, int DIM>
struct Cfg {
    static constexpr bool kWide = sizeof(T) == 4;
    // heads of 64 in 16 bits: two smaller blocks to a multiprocessor, one's softmax, start and end
    // beside the other's products
    static constexpr bool kTwo = !kWide && DIM == 64;
    static constexpr int kKeys = kWide || kTwo ? 64 : 128;
    static constexpr int kK = kWide ? 3 : 1;                             // pieces of a key
    static constexpr int kQ = kHalf<T> ? 2 : 3;                          // of a query
    // of them in tensor memory, as many as it holds beside the rest (an MMA with both operands in
    // shared memory takes as long, but the pieces' place there is wanted too)
    static constexpr int kQTmem = kWide ? 2 : kQ == 3 ? 1 : kQ;
    // what of a query or probability its first piece leaves is taken times 2^kUpBits
    static constexpr int kUpBits = kHalf<T> ? paged::kUpBits : 0;
    static constexpr float kUp = kUpBits ? paged::kUp : 1.f;
    static constexpr int kParts = kWide || kTwo ? 2 : 4;  // threads to a row
    static constexpr int kRowWarps = 4 * kParts, kMmaWarp = kRowWarps;
    // for the keys, and as many for the values
    static constexpr int kLoadWarp0 = kRowWarps + 1, kLoadWarps = kWide ? 9 : 1;
    static constexpr int kTileWarp = kLoadWarp0 + 2 * kLoadWarps, kThreads = (kTileWarp + 1) * 32;
    static_assert(kThreads % 128 == 0, "warpgroups");
    static constexpr int kBlocks = kTwo ? 2 : 1;  // of a multiprocessor
    static constexpr int kRegsStart = kWide ? 72 : kTwo ? 80 : 96;
    static constexpr int kRegsRows = kWide ? 128 : kTwo ? 96 : 104;
    static constexpr int kRegsOther = kWide ? 48 : kTwo ? 48 : 64;
    static_assert(kParts * kRegsRows + (kThreads / 128 - kParts) * kRegsOther <=
                      kThreads / 128 * kRegsStart,
                  "registers of the block");
    // A piece of a block of keys or values: 64 features' rows of 128 bytes, then the next 64's.
    static constexpr int kPart = kKeys * 128, kPiece = kPart * (DIM / 64);
    static constexpr int kBuf = kK * kPiece;
    static constexpr int kQPart = kRows * 128, kQPiece = kQPart * (DIM / 64);
    static constexpr int kKs = 0, kVs = 2 * kBuf, kQs = 4 * kBuf;
    // The rows' queries and results in 32 bits pass through the place of the queries' pieces, beside
    // an fp32 cache through the values'.
    static constexpr int kStageBytes = kRows * DIM * 4, kQBytes = (kQ - kQTmem) * kQPiece;
    static constexpr bool kStageInValues = kWide;
    static constexpr int kStage = kStageInValues ? kVs : kQs;
    static_assert(!kStageInValues || kStageBytes <= 2 * kBuf);
    static constexpr int kMax = kQs + (kStageInValues || kQBytes > kStageBytes ? kQBytes : kStageBytes);
    static constexpr int kBar = kMax + 2 * kParts * kRows * 4;  // kMax: float [2][kParts][kRows]
    static constexpr int kTotal = kBar + 512;
    static_assert(kTotal <= (228 / kBlocks - 1) * 1024, "shared memory");
    // tensor memory, columns
    static constexpr int kTq = 0, kTs = kTq + kQTmem * DIM / 2, kTp = kTs + kKeys;
    static constexpr int kTo = kTp + kQ * kKeys / 2;
    static constexpr int kColumns = 512 / kBlocks;
    static_assert(kTo + DIM <= kColumns, "tensor memory");
};

// fp32 accumulate, M = 128, N = n; type 0: fp16, 1: bf16; b_slow: B's columns run fastest
__host__ __device__ constexpr uint32_t idesc(int type, int n, bool b_slow) {
    return (1u << 4) | ((uint32_t)type << 7) | ((uint32_t)type << 10) | ((uint32_t)b_slow << 16) |
           ((uint32_t)(n >> 3) << 17) | ((uint32_t)(kRows >> 4) << 24);
}
// B with its columns (features) fastest, 128-byte swizzle: 64 columns of eight k rows are an atom
// of 1024 bytes; `next` bytes to the next 64 columns, 1024 to the next eight rows
__device__ __forceinline__ uint64_t desc_slow(uint32_t at, uint32_t next) {
    return (uint64_t)((at & 0x3FFFF) >> 4) | (uint64_t)(next >> 4) << 16 |
           (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
// DOWN > 0: what is there already counts 2^-DOWN
template <int DOWN = 0>
__device__ __forceinline__ void umma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t id,
                                        uint32_t accumulate) {
    if constexpr (DOWN > 0)
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p, %5;\n\t}"
            ::"r"(d), "r"(a), "l"(b), "r"(id), "r"(accumulate), "n"(DOWN)
            : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
            ::"r"(d), "r"(a), "l"(b), "r"(id), "r"(accumulate)
            : "memory");
}
__device__ __forceinline__ void umma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t id,
                                        uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(d), "l"(a), "l"(b), "r"(id), "r"(accumulate)
        : "memory");
}
#define B2W4_W8(r, o) "=r"(r[o]), "=r"(r[o + 1]), "=r"(r[o + 2]), "=r"(r[o + 3]),            \
                      "=r"(r[o + 4]), "=r"(r[o + 5]), "=r"(r[o + 6]), "=r"(r[o + 7])
#define B2W4_RW8(r, o) "+r"(r[o]), "+r"(r[o + 1]), "+r"(r[o + 2]), "+r"(r[o + 3]),           \
                       "+r"(r[o + 4]), "+r"(r[o + 5]), "+r"(r[o + 6]), "+r"(r[o + 7])
#define B2W4_R8(r, o) "r"(r[o]), "r"(r[o + 1]), "r"(r[o + 2]), "r"(r[o + 3]), "r"(r[o + 4]), \
                      "r"(r[o + 5]), "r"(r[o + 6]), "r"(r[o + 7])
__device__ __forceinline__ void tmem_ld16(uint32_t at, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, "
        "%11, %12, %13, %14, %15}, [%16];"
        : B2W4_W8(r, 0), B2W4_W8(r, 8)
        : "r"(at)
        : "memory");
}
// the wait that makes columns readable, and waits for none that is used later
__device__ __forceinline__ void tmem_ld_wait(uint32_t (&a)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;" : B2W4_RW8(a, 0), B2W4_RW8(a, 8) : : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t at, const uint32_t (&r)[8]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x8.b32 [%8], {%0, %1, %2, %3, %4, %5, %6, %7};" ::B2W4_R8(
            r, 0),
        "r"(at)
        : "memory");
}
__device__ __forceinline__ void tmem_st_wait() {
    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}
// row, chunk of 16 bytes -> bytes in 128-byte rows: 8-row atoms, chunks swizzled with the row
__device__ __forceinline__ uint32_t place(int row, int chunk) {
    return (uint32_t)((row >> 3) * 1024 + (row & 7) * 128 + ((chunk ^ (row & 7)) << 4));
}

// Whole warp.  Tile `at` of the call's, counted from the last sequence's last tile; false: there is
// none.  t0: its first token of the sequence's rows.
__device__ bool find_tile(const Args& a, int tq, int at, int* seq, int* t0) {
    const int lane = threadIdx.x & 31;
    for (int base = a.sequences; base > 0; base -= 32) {
        const int i = base - 1 - lane;
        int n = 0;
        if (i >= 0) {
            bool bad = false;
            n = (paged::taken(a, i, &bad).count + tq - 1) / tq;
            if (bad)
                b2w4_report(a.status, B2W4_E_INVALID);
        }
        int x = n;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, x, off);
            if (lane >= off)
                x += y;
        }
        const unsigned past = __ballot_sync(0xffffffffu, x > at);
        if (past) {
            const int l = __ffs(past) - 1;
            *seq = base - 1 - l;
            *t0 = (__shfl_sync(0xffffffffu, x, l) - 1 - at) * tq;
            return true;
        }
        at -= __shfl_sync(0xffffffffu, x, 31);
    }
    return false;
}

// A tile: its sequence and kv head, its first token of the sequence's rows, and the keys that its
// rows see, [0, low) and [from, ..), as one list.
struct Tile {
    const int32_t* table;
    int seq, first, count, length, kvh, t0;
    int low, from, keys, pad;
    __device__ __forceinline__ int p0() const { return length - count + t0; }  // its position
};

// Rows of a tile to be done again: bit r of `rows` is row r of the quarter.  In the work area a list
// for every quarter of every block's rows, an entry a tile.
struct alignas(16) Again {
    int seq, t0, kvh;
    unsigned rows;
};
// The most tiles of a call: a sequence's last one may be short, one more for each.
long tiles_of(int rows, int sequences, int heads, int kv_heads) {
    return ((long)rows / (kRows / (heads / kv_heads)) + sequences) * kv_heads;
}
constexpr int kMostBlocks = 2;  // of a multiprocessor

template <typename T, int DIM>
__global__ void __launch_bounds__(Cfg<T, DIM>::kThreads, Cfg<T, DIM>::kBlocks)
paged_runs_kernel(const Args a, const Attend p, int tq, Again* __restrict__ lists,
                  int most_tiles) {
    using C = Cfg<T, DIM>;
    constexpr int kKeys = C::kKeys, kParts = C::kParts, kRowWarps = C::kRowWarps;
    constexpr int kMmaWarp = C::kMmaWarp, kLoadWarp0 = C::kLoadWarp0;
    constexpr int kType = std::is_same_v<T, __half> ? 0 : 1;
    extern __shared__ __align__(1024) uint8_t smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::kBar);
    uint64_t* q_full = bars;        // the queries' pieces
    uint64_t* s_full = bars + 1;    // scores of a block complete
    uint64_t* s_free = bars + 2;    // ... and in registers
    uint64_t* p_full = bars + 3;    // probabilities' pieces in tensor memory, the last P V out of it
    uint64_t* o_full = bars + 4;    // P V of a block complete (and P read)
    uint64_t* drained = bars + 6;   // every MMA retired
    uint64_t* k_full = bars + 8;    // [2]
    uint64_t* k_free = bars + 10;   // [2]
    uint64_t* v_full = bars + 12;   // [2]
    uint64_t* v_free = bars + 14;   // [2]
    uint64_t* tile_full = bars + 16;  // [2] what the tile is
    uint64_t* tile_free = bars + 18;  // [2]
    Tile* s_tile = reinterpret_cast<Tile*>(bars + 20);  // [2]
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(s_tile + 2);
    volatile int* s_abort = reinterpret_cast<volatile int*>(tmem_slot + 1);
    uint32_t* s_bad = tmem_slot + 2;  // [2] a page that is not the pool's
    uint32_t* s_odd = tmem_slot + 4;  // [4] rows to be done again
    int* s_listed = reinterpret_cast<int*>(tmem_slot + 8);  // [4] tiles with such rows
    static_assert(20 * 8 + 2 * sizeof(Tile) + 12 * 4 <= 512);
    float* s_max = reinterpret_cast<float*>(smem + C::kMax);

    if (threadIdx.x == 0) {
        mbar_init(q_full, kRowWarps);
        mbar_init(s_full, 1);
        mbar_init(s_free, kRowWarps);
        mbar_init(p_full, kRowWarps);
        mbar_init(o_full, 1);
        mbar_init(drained, 1);
        for (int b = 0; b < 2; ++b) {
            // (a lane's copies arrive by themselves)
            mbar_init(&k_full[b], C::kWide ? C::kLoadWarps : 32);
            mbar_init(&k_free[b], 1);
            mbar_init(&v_full[b], C::kWide ? C::kLoadWarps : 32);
            mbar_init(&v_free[b], 1);
            mbar_init(&tile_full[b], 1);
            mbar_init(&tile_free[b], kRowWarps + 1 + 2 * C::kLoadWarps);
            s_bad[b] = 0;
        }
        *s_abort = 0;
        for (int i = 0; i < 4; ++i)
            s_odd[i] = s_listed[i] = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    b2w4_pdl_wait();
    if (warp == kMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                     ::"r"(smem_u32(tmem_slot)), "r"(C::kColumns)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = *tmem_slot;
    // Not before tensor memory is this block's: a block of the next kernel beside it, which may
    // take tensor memory ahead of its wait for this kernel, would wait for the one that waits.
    b2w4_pdl_launch_dependents();
    auto fail = [&]() {
        *s_abort = 1;
        b2w4_report_timeout(a.status);
    };
    auto wait = [&](uint64_t* bar, uint32_t parity) {
        return mbar_try_wait(bar, parity) || (!*s_abort && mbar_wait(bar, parity));
    };
    auto warp_wait = [&](uint64_t* bar, uint32_t parity) {
        return __all_sync(0xffffffffu, wait(bar, parity)) != 0;
    };
    auto warp_arrive = [&](uint64_t* bar) {
        __syncwarp();
        if (lane == 0)
            mbar_arrive(bar);
    };

    const int rep = p.heads / a.kv_heads;
    // r / rep for r < 128: a division for every row of the tile was 5000 cycles of it
    const int inverse = (65536 + rep - 1) / rep;
    auto token_of = [&](int r) { return (r * inverse) >> 16; };
    // The block's n-th tile; false: there is none, or a wait ran out.
    auto next_tile = [&](int n) {
        if (!warp_wait(&tile_full[n & 1], (n >> 1) & 1)) {
            fail();
            return false;
        }
        return s_tile[n & 1].seq >= 0;
    };

    if (warp < kRowWarps) {
        // ================================== rows =====================================
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::kRegsRows));
        // a quarter of the tensor memory's lanes; a part of the keys and of the features
        const int quarter = warp & 3, part = warp >> 2;
        const int row = quarter * 32 + lane;
        const uint32_t lane_addr = tmem + ((uint32_t)(quarter * 32) << 16);
        auto row_sync = [&]() {  // the threads of a quarter's rows have come here
            asm volatile("bar.sync %0, %1;" ::"r"(3 + quarter), "n"(32 * kParts) : "memory");
        };
        auto all_rows_any = [&](bool v) {  // all row warps have come here
            int r;
            asm volatile(
                "{\n\t.reg .pred p, q;\n\t"
                "setp.ne.s32 p, %1, 0;\n\t"
                "barrier.cta.red.or.pred q, 2, %2, p;\n\t"
                "selp.s32 %0, 1, 0, q;\n\t}"
                : "=r"(r)
                : "r"((int)v), "n"(kRowWarps * 32)
                : "memory");
            return r != 0;
        };
        // the threads' values of the row, through words that alternate
        int turn = 0;
        auto share = [&](float v, auto join) {
            float* mx = s_max + (turn++ & 1) * kParts * kRows + row;
            mx[part * kRows] = v;
            row_sync();
            float r = mx[0];
#pragma unroll
            for (int i = 1; i < kParts; ++i)
                r = join(r, mx[i * kRows]);
            return r;
        };
        auto larger = [](float x, float y) { return fmaxf(x, y); };
        constexpr int kOwn = DIM / kParts, kMine = kKeys / kParts;  // features, keys
        // a tile of fp32 rows in shared memory: a warp moves some of its quarter's rows whole, where
        // a thread's own accesses would be a line each (5000 cycles of the load path)
        constexpr int kRowChunks = DIM / 4, kRowsAtOnce = 32 / kRowChunks;
        constexpr int kMoves = 32 / kParts / kRowsAtOnce;
        uint8_t* const stage = smem + C::kStage;
        auto staged = [](int r, int chunk) { return (r * kRowChunks + (chunk ^ (r & 7))) * 16; };
        const int stage_chunk = lane % kRowChunks;
        auto stage_row = [&](int i) {
            return quarter * 32 + (part * kMoves + i) * kRowsAtOnce + lane / kRowChunks;
        };
        bool live = true;  // no way out of a tile: the threads of a row meet once a step
        auto await = [&](uint64_t* bar, uint32_t parity) {
            if (live && !warp_wait(bar, parity)) {
                live = false;
                fail();
            }
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        };
        int g = 0;  // steps of the tiles before
        auto list_of = [&]() { return lists + (size_t)(blockIdx.x * 4 + quarter) * most_tiles; };
        for (int n = 0;; ++n) {
            const bool more = next_tile(n);
            // one answer for all rows
            if (all_rows_any(!more || !live || *s_abort))
                break;
            const Tile& t = s_tile[n & 1];  // read where it is wanted, it costs no registers
            const int steps = (t.keys + kKeys - 1) / kKeys;
            auto row_offset = [&](int r, int ld) {
                const int k = token_of(r);
                return (size_t)(t.first + t.t0 + k) * ld + (size_t)(t.kvh * rep + r - k * rep) * DIM;
            };
            auto row_exists = [&](int r) { return r < tq * rep && t.t0 + token_of(r) < t.count; };
            const bool exists = row_exists(row);
            const int pos = exists ? t.p0() + token_of(row) : -1;
            // The factor of the scores, in base 2.  It is positive: the queries take a negative
            // sign, and zero is as small a number as can be, so that a masked score stays below all
            // others.
            const float scale = __fmul_rn(p.scale, 1.4426950408889634f);
            float factor = fmaxf(fabsf(scale), 0x1p-100f);
            if (steps > 0) {
                // all loads ahead of the first store, which might be to where a load is from for
                // all that the compiler knows
                float4 v[kMoves];
#pragma unroll
                for (int i = 0; i < kMoves; ++i) {
                    const int r = stage_row(i);
                    v[i] = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (row_exists(r))
                        v[i] = *reinterpret_cast<const float4*>(p.q + row_offset(r, p.ldq) +
                                                                stage_chunk * 4);
                }
#pragma unroll
                for (int i = 0; i < kMoves; ++i)
                    *reinterpret_cast<float4*>(stage + staged(stage_row(i), stage_chunk)) = v[i];
                row_sync();
                float4 f[kOwn / 4];
#pragma unroll
                for (int i = 0; i < kOwn / 4; ++i)
                    f[i] =
                        *reinterpret_cast<const float4*>(stage + staged(row, part * (kOwn / 4) + i));
                if (!C::kStageInValues)
                    all_rows_any(false);  // the pieces go where the rows were
                float up = scale < 0.f ? -1.f : 1.f;
                if constexpr (kHalf<T>) {
                    float top = 0.f;
#pragma unroll
                    for (int i = 0; i < kOwn / 4; ++i)
                        top = fmaxf(
                            fmaxf(fmaxf(top, fabsf(f[i].x)), fmaxf(fabsf(f[i].y), fabsf(f[i].z))),
                            fabsf(f[i].w));
                    top = share(top, larger);
                    int e = (int)(__float_as_uint(top) >> 23) - 127;
                    e = top == 0.f ? kTop : min(max(e, -100), 120);
                    up = __fmul_rn(up, __uint_as_float((unsigned)(127 + kTop - e) << 23));
                    factor = __fmul_rn(factor, __uint_as_float((unsigned)(127 - kTop + e) << 23));
                    factor = fmaxf(factor, 0x1p-100f);
                }
                const uint64_t up2 = b2w4_pack2(up, up);
#pragma unroll
                for (int c = 0; c < kOwn; c += 16) {
                    uint64_t v[8];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        v[2 * i] = b2w4_mul2(b2w4_pack2(f[c / 4 + i].x, f[c / 4 + i].y), up2);
                        v[2 * i + 1] = b2w4_mul2(b2w4_pack2(f[c / 4 + i].z, f[c / 4 + i].w), up2);
                    }
                    const int at = part * kOwn + c;  // first feature
#pragma unroll
                    for (int i = 0; i < C::kQ; ++i) {
                        uint32_t r[8];
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            r[e] = take_piece<T>(v[e], C::kUp, i == C::kQ - 1);
                        if (i < C::kQTmem) {
                            tmem_st8(lane_addr + C::kTq + i * (DIM / 2) + at / 2, r);
                        } else {
                            uint8_t* to = smem + C::kQs + (i - C::kQTmem) * C::kQPiece +
                                          at / 64 * C::kQPart;
#pragma unroll
                            for (int e = 0; e < 2; ++e)
                                *reinterpret_cast<uint4*>(to + place(row, at % 64 / 8 + e)) =
                                    make_uint4(r[4 * e], r[4 * e + 1], r[4 * e + 2], r[4 * e + 3]);
                        }
                    }
                }
                tmem_st_wait();
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                warp_arrive(q_full);
            }
            // m: the row's largest score, mf: times the factor, as it is taken from the exponents
            float m = -INFINITY, mf = -INFINITY, l = 0.f, alpha = 1.f;
            uint64_t acc[kOwn / 2];
#pragma unroll
            for (int i = 0; i < kOwn / 2; ++i)
                acc[i] = 0ull;
            // 16 of the thread's features of P V, on their way; and into the running output
            auto output_ld = [&](int c, uint32_t (&r)[16]) {
                tmem_ld16(lane_addr + C::kTo + part * kOwn + 16 * c, r);
            };
            auto output_add = [&](int c, uint32_t (&r)[16]) {
                const uint64_t al = b2w4_pack2(alpha, alpha);
                tmem_ld_wait(r);
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    acc[8 * c + i] = b2w4_fma2(acc[8 * c + i], al,
                                               b2w4_pack2(__uint_as_float(r[2 * i]),
                                                          __uint_as_float(r[2 * i + 1])));
            };
            // of the list, the row sees [0, sinks) and [lo, hi)
            const int hi = pos < 0 ? 0 : pos - t.from + t.low + 1;
            const int lo = p.window.from(max(pos, 0)) - t.from + t.low;
            for (int j = 0; j < steps; ++j) {
                await(s_full, (g + j) & 1);
                uint32_t sr[kMine / 16][16];
#pragma unroll
                for (int h = 0; h < kMine / 16; ++h)
                    tmem_ld16(lane_addr + C::kTs + part * kMine + 16 * h, sr[h]);
#pragma unroll
                for (int h = 0; h < kMine / 16; ++h)
                    tmem_ld_wait(sr[h]);
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                warp_arrive(s_free);
                float sc[kMine];
#pragma unroll
                for (int i = 0; i < kMine; ++i)
                    sc[i] = __uint_as_float(sr[i / 16][i % 16]);
                const int first = j * kKeys + part * kMine;  // the thread's first key of the list
                if (first + kMine > hi || (first < lo && first + kMine > p.window.sinks)) {
                    static_assert(kMine <= 32);
                    auto below = [](int k) { return k <= 0 ? 0u : k >= 32 ? ~0u : (1u << k) - 1u; };
                    const unsigned seen = below(hi - first) &
                                          (~below(lo - first) | below(p.window.sinks - first));
#pragma unroll
                    for (int i = 0; i < kMine; ++i)
                        if (!(seen >> i & 1))
                            sc[i] = -INFINITY;
                }
                float top = m;
#pragma unroll
                for (int i = 0; i < kMine; i += 2)
                    top = fmaxf(fmaxf(top, sc[i]), sc[i + 1]);
                m = share(top, larger);
                const float next_mf = m == -INFINITY ? 0.f : __fmul_rn(m, factor);
                const float shift = __fsub_rn(kLift<T>, next_mf);
                const uint64_t factor2 = b2w4_pack2(factor, factor);
                const uint64_t shift2 = b2w4_pack2(shift, shift);
                uint64_t pr[kMine / 2];
#pragma unroll
                for (int i = 0; i < kMine / 2; ++i) {
                    float x, y;
                    b2w4_unpack2(b2w4_fma2(b2w4_pack2(sc[2 * i], sc[2 * i + 1]), factor2, shift2), x,
                                 y);
                    pr[i] = b2w4_pack2(exp2_neg(x), exp2_neg(y));
                }
                uint64_t sum[4] = {pr[0], pr[1], pr[2], pr[3]};
#pragma unroll
                for (int i = 4; i < kMine / 2; ++i)
                    sum[i & 3] = add2(sum[i & 3], pr[i]);
                sum[0] = add2(add2(sum[0], sum[1]), add2(sum[2], sum[3]));
                float sum0, sum1;
                b2w4_unpack2(sum[0], sum0, sum1);
                const float next_alpha = exp2_neg(__fsub_rn(mf, next_mf));
                mf = m == -INFINITY ? -INFINITY : next_mf;
                l = __fmaf_rn(l, next_alpha, __fadd_rn(sum0, sum1));
                // The pieces that fit the registers are taken ahead of the wait for the product
                // before, which reads the probabilities: the MMAs of the next one wait for what is
                // behind it.
                constexpr int kPs = kMine / 16, kOs = kOwn / 16, kTurns = kPs > kOs ? kPs : kOs;
                uint32_t pieces[C::kQ][8];
                auto take = [&](int u) {
#pragma unroll
                    for (int i = 0; i < C::kQ; ++i)
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            pieces[i][e] = take_piece<T>(pr[8 * u + e], C::kUp, i == C::kQ - 1);
                };
                take(0);
                if (j)
                    await(o_full, (g + j - 1) & 1);
#pragma unroll
                for (int u = 0; u < kTurns; ++u) {
                    uint32_t ro[16];
                    if (j && u < kOs)
                        output_ld(u, ro);
                    if (u < kPs) {
                        if (u)
                            take(u);
#pragma unroll
                        for (int i = 0; i < C::kQ; ++i)
                            tmem_st8(lane_addr + C::kTp + i * (kKeys / 2) + part * (kMine / 2) +
                                         8 * u,
                                     pieces[i]);
                    }
                    if (j && u < kOs)
                        output_add(u, ro);
                }
                alpha = next_alpha;
                tmem_st_wait();
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                warp_arrive(p_full);
            }
            if (steps > 0) {
                await(o_full, (g + steps - 1) & 1);
#pragma unroll
                for (int u = 0; u < kOwn / 16; ++u) {
                    uint32_t ro[16];
                    output_ld(u, ro);
                    output_add(u, ro);
                }
            }
            g += steps;
            const float total = share(l, [](float x, float y) { return __fadd_rn(x, y); });
            bool odd = false;
            const float over = pos < 0 ? 0.f : __fdiv_rn(1.f, total);
#pragma unroll
            for (int i = 0; i < kOwn / 2; ++i) {
                float x, y;
                b2w4_unpack2(acc[i], x, y);
                x = pos < 0 ? 0.f : __fmul_rn(x, over);
                y = pos < 0 ? 0.f : __fmul_rn(y, over);
                odd |= paged::odd_result<T>(x) || paged::odd_result<T>(y);
                acc[i] = b2w4_pack2(x, y);
            }
            // out through shared memory too: every product that read it has retired
#pragma unroll
            for (int i = 0; i < kOwn / 4; ++i)
                *reinterpret_cast<ulonglong2*>(stage + staged(row, part * (kOwn / 4) + i)) =
                    make_ulonglong2(acc[2 * i], acc[2 * i + 1]);
            const unsigned again =
                __ballot_sync(0xffffffffu, exists && (odd || s_bad[n & 1]));
            if (lane == 0 && again)
                atomicOr(&s_odd[quarter], again);
            row_sync();
            {
                float4 v[kMoves];
#pragma unroll
                for (int i = 0; i < kMoves; ++i)
                    v[i] = *reinterpret_cast<const float4*>(stage +
                                                            staged(stage_row(i), stage_chunk));
                const bool good = live && !*s_abort;
#pragma unroll
                for (int i = 0; i < kMoves; ++i) {
                    const int r = stage_row(i);
                    if (good && row_exists(r))
                        *reinterpret_cast<float4*>(p.out + row_offset(r, p.ldo) + stage_chunk * 4) =
                            v[i];
                }
            }
            row_sync();
            if (const unsigned mine = s_odd[quarter]) {
                row_sync();  // all have looked
                if (part == 0 && lane == 0) {
                    // (more tiles than the call's rows make: starts that are wrong)
                    const int at = s_listed[quarter];
                    if (at < most_tiles) {
                        list_of()[at] = {t.seq, t.t0, t.kvh, mine};
                        s_listed[quarter] = at + 1;
                    } else {
                        b2w4_report(a.status, B2W4_E_INVALID);
                    }
                    s_odd[quarter] = 0;
                }
                row_sync();
            }
            // every row has looked at the word
            if (all_rows_any(false), threadIdx.x == 0)
                s_bad[n & 1] = 0;
            warp_arrive(&tile_free[n & 1]);
        }
        // No warp waits for this with a limit: the others stand at the block's last barrier.
#pragma unroll 1
        for (int i = 0; i < s_listed[quarter] && live && !*s_abort; ++i) {
            const Again t = list_of()[i];
            bool bad = false;
            const Sequence s = paged::taken(a, t.seq, &bad);
#pragma unroll 1
            for (int r = part; r < 32; r += kParts) {
                if (!(t.rows >> r & 1))
                    continue;
                const int token = t.t0 + token_of(quarter * 32 + r);
                const int head = t.kvh * rep + quarter * 32 + r - (token - t.t0) * rep;
                const size_t row = s.first + token;
                paged::attend_row<T, DIM>(a, s, p.q + row * p.ldq + (size_t)head * DIM,
                                          s.length - s.count + token, t.kvh, p.scale, p.window,
                                          p.out + row * p.ldo + (size_t)head * DIM);
            }
        }
    } else {
      asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::kRegsOther));
      if (warp == kMmaWarp) {
        // ================================= MMA issue =================================
        // One warp, so that P V of a block goes ahead of the scores of the next but one, which
        // become possible at the same time: the rows wait for the former.  The warp stays together
        // and one lane issues: what the MMAs are given is then the same for all lanes and is
        // worked out once a warp.
        {
            const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
            const uint64_t k_desc0 = umma_desc_k_sw128(smem_u32(smem + C::kKs));
            const uint64_t q_desc = umma_desc_k_sw128(smem_u32(smem + C::kQs));
            const uint64_t v_desc0 = desc_slow(smem_u32(smem + C::kVs), C::kPart);
            constexpr uint32_t score_id = idesc(kType, kKeys, false);
            constexpr uint32_t out_id = idesc(kType, DIM, true);
            // sizes of products, the smallest first: pieces i of Q and size - i of K
            auto scores = [&](int j) {
                const uint64_t d = k_desc0 + (uint64_t)((j & 1) * (C::kBuf >> 4));
                bool more = false;
#pragma unroll
                for (int size = C::kQ - 1; size >= 0; --size)
#pragma unroll
                    for (int i = size; i >= 0; --i) {
                        if (size - i >= C::kK)
                            continue;
#pragma unroll
                        for (int k = 0; k < DIM / 16; ++k) {
                            const uint64_t kd =
                                d + (uint64_t)(((size - i) * C::kPiece + k / 4 * C::kPart +
                                                k % 4 * 32) >> 4);
                            if (C::kUpBits && size == 0 && k == 0)
                                umma_ts<C::kUpBits>(tm + C::kTs, tm + C::kTq, kd, score_id, 1);
                            else if (i < C::kQTmem)
                                umma_ts(tm + C::kTs, tm + C::kTq + i * (DIM / 2) + k * 8, kd,
                                        score_id, more);
                            else
                                umma_ss(tm + C::kTs,
                                        q_desc + (uint64_t)(((i - C::kQTmem) * C::kQPiece +
                                                             k / 4 * C::kQPart + k % 4 * 32) >> 4),
                                        kd, score_id, more);
                            more = true;
                        }
                    }
                umma_commit(s_full);
                umma_commit(&k_free[j & 1]);
            };
            // products of one size
            auto output = [&](int j, int size) {
                const uint64_t d = v_desc0 + (uint64_t)((j & 1) * (C::kBuf >> 4));
#pragma unroll
                for (int i = size; i >= 0; --i) {
                    if (size - i >= C::kK)
                        continue;
#pragma unroll
                    for (int k = 0; k < kKeys / 16; ++k)
                        if (C::kUpBits && size == 0 && k == 0)
                            umma_ts<C::kUpBits>(tm + C::kTo, tm + C::kTp, d, out_id, 1);
                        else
                            umma_ts(tm + C::kTo, tm + C::kTp + i * (kKeys / 2) + k * 8,
                                    d + (uint64_t)(((size - i) * C::kPiece + k * 2048) >> 4), out_id,
                                    size < C::kQ - 1 || i < size || k > 0);
                }
            };
            // what the loaders' asynchronous copies wrote is for the tensor core to read; where they
            // write it themselves they say so
            auto copied = [&]() {
                if (!C::kWide)
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            };
            auto scores_wait = [&](int j) {
                const bool ok = __all_sync(0xffffffffu, wait(&k_full[j & 1], (j >> 1) & 1) &&
                                                            (j == 0 || wait(s_free, (j - 1) & 1)));
                copied();
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                return ok;
            };
            // P V of block j, then the scores of block `next`, unless that is -1.  What the scores
            // wait for comes a little after the probabilities: the warp asks for it with a part of
            // P V on its way, so that no gap is left between the products.
            auto step = [&](int j, int next) {
                if (!__all_sync(0xffffffffu,
                                wait(&v_full[j & 1], (j >> 1) & 1) && wait(p_full, j & 1)))
                    return false;
                copied();
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                if (elect_one())
                    output(j, C::kQ - 1);
                __syncwarp();
                const bool ok = next < 0 || scores_wait(next);
                if (elect_one()) {
#pragma unroll
                    for (int size = C::kQ - 2; size >= 0; --size)
                        output(j, size);
                    umma_commit(o_full);
                    umma_commit(&v_free[j & 1]);
                    if (next >= 0 && ok)
                        scores(next);
                }
                __syncwarp();
                return ok;
            };
            auto first_scores = [&](int j) {
                const bool ok = scores_wait(j);
                if (ok && elect_one())
                    scores(j);
                __syncwarp();
                return ok;
            };
            int g = 0, queries = 0;
            for (int n = 0;; ++n) {
                if (!next_tile(n))
                    break;
                const int steps = (s_tile[n & 1].keys + kKeys - 1) / kKeys;
                warp_arrive(&tile_free[n & 1]);
                if (steps == 0)
                    continue;
                bool ok = warp_wait(q_full, queries++ & 1) && first_scores(g) &&
                          (steps == 1 || first_scores(g + 1));
#pragma unroll 1
                for (int j = 0; j < steps && ok; ++j)
                    ok = step(g + j, j + 2 < steps ? g + j + 2 : -1);
                g += steps;
                if (!ok) {
                    fail();
                    break;
                }
            }
            if (elect_one())
                umma_commit(drained);
            __syncwarp();
            if (!mbar_wait(drained, 0))
                fail();
        }
      } else if (warp == C::kTileWarp) {
        // ================================ tiles =====================================
        for (int n = 0;; ++n) {
            if (n >= 2 && !warp_wait(&tile_free[n & 1], ((n >> 1) - 1) & 1)) {
                fail();
                break;
            }
            const int at = blockIdx.x + n * gridDim.x;
            Tile t = {};
            t.kvh = at % a.kv_heads;
            if (find_tile(a, tq, at / a.kv_heads, &t.seq, &t.t0)) {
                bool bad = false;
                const Sequence s = paged::taken(a, t.seq, &bad);
                t.table = s.table;
                t.first = s.first;
                t.count = s.count;
                t.length = s.length;
                const int p1 = s.length - s.count + min(t.t0 + tq, s.count) - 1;  // its last token
                t.from = p.window.from(max(t.p0(), 0));
                t.low = min(p.window.sinks, t.from);
                t.keys = p1 < 0 ? 0 : t.low + p1 + 1 - t.from;
            } else {
                t.seq = -1;
            }
            if (lane == 0)
                s_tile[n & 1] = t;
            warp_arrive(&tile_full[n & 1]);
            if (t.seq < 0)
                break;
        }
      } else {
        // ============================== keys and values ==============================
        auto full = [&](uint64_t* bar) {  // make it visible to the tensor core
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            warp_arrive(bar);
        };
        // Half of the warps have the keys, the others the values.
        const bool values = warp >= kLoadWarp0 + C::kLoadWarps;
        const int w0 = (warp - kLoadWarp0) % C::kLoadWarps;
        uint64_t *filled = values ? v_full : k_full, *freed = values ? v_free : k_free;
        const T* pool = static_cast<const T*>(values ? a.v : a.k);
        uint8_t* ring = smem + (values ? C::kVs : C::kKs);
        constexpr int kChunks = DIM / 8, kPer = 32 / kChunks;  // of eight features; rows at a time
        const int c = lane % kChunks, sub = lane / kChunks;
        uint8_t* const mine = ring + (c >> 3) * C::kPart;
        int g = 0, queries = 0;
        bool ok = true;
        for (int n = 0; ok; ++n) {
            if (!next_tile(n))
                break;
            const Tile& t = s_tile[n & 1];
            const int steps = (t.keys + kKeys - 1) / kKeys;
            // Where key i of the list lies; -1: it does not exist.  One whose page is not the
            // pool's is left out, which a masked row cannot be: the tile's rows are done again.
            auto row_of = [&](int i) {
                if (i >= t.keys)
                    return -1;
                const int row =
                    paged::cache_row(a, t.table, i < t.low ? i : i - t.low + t.from, t.kvh);
                if (row < 0) {
                    b2w4_report(a.status, B2W4_E_INVALID);
                    atomicOr(&s_bad[n & 1], 1u);
                }
                return row;
            };
            auto free = [&](int i) {
                ok = i < 2 || warp_wait(&freed[i & 1], ((i >> 1) - 1) & 1);
                if (!ok)
                    fail();
                return ok;
            };
            // (the values' place holds the queries at first)
            if (C::kStageInValues && values && steps > 0 && !warp_wait(q_full, queries++ & 1)) {
                fail();
                break;
            }
            if constexpr (C::kWide) {
                // A warp has every kLoadWarps-th set of kPer rows of a block.  Its lanes know where a
                // block's rows lie, a block ahead, and the numbers of the next kDepth sets are on
                // their way: as many as 48 registers hold (all five sets of seven warps in 56, some
                // in local memory: 333 tokens behind 900 70 us, so 63).
                constexpr int kSets = kKeys / kPer;
                constexpr int kMine = (kSets + C::kLoadWarps - 1) / C::kLoadWarps, kDepth = 2;
                static_assert(kMine * kPer <= 32 && kMine % kDepth == 0);
                ulonglong2 next[kDepth][2];
                auto look = [&](int j) {
                    const int set = w0 + lane / kPer * C::kLoadWarps;
                    return set < kSets ? row_of(j * kKeys + set * kPer + lane % kPer) : -1;
                };
                auto load = [&](int rows, int u) {
                    const int row = __shfl_sync(0xffffffffu, rows, u * kPer + sub);
#pragma unroll
                    for (int h = 0; h < 2; ++h)
                        next[u % kDepth][h] = row >= 0 ? reinterpret_cast<const ulonglong2*>(
                                                             pool + (size_t)row * DIM + c * 8)[h]
                                                       : make_ulonglong2(0ull, 0ull);
                };
                int rows = look(0), ahead = look(1);
#pragma unroll
                for (int u = 0; u < kDepth; ++u)
                    load(rows, u);
                for (int j = 0; j < steps && free(g + j); ++j) {
#pragma unroll
                    for (int u = 0; u < kMine; ++u) {
                        const int set = w0 + u * C::kLoadWarps;
                        const ulonglong2 (&n)[2] = next[u % kDepth];
                        uint64_t x[4] = {n[0].x, n[0].y, n[1].x, n[1].y};
                        uint8_t* dst =
                            mine + ((g + j) & 1) * C::kBuf + place(set * kPer + sub, c & 7);
                        if (u + kDepth < kMine)
                            load(rows, u + kDepth);
                        else
                            load(ahead, u + kDepth - kMine);
                        if (set >= kSets)
                            continue;
#pragma unroll
                        for (int i = 0; i < C::kK; ++i) {
                            uint4 o;
                            o.x = take_piece<T>(x[0], 1.f, i == C::kK - 1);
                            o.y = take_piece<T>(x[1], 1.f, i == C::kK - 1);
                            o.z = take_piece<T>(x[2], 1.f, i == C::kK - 1);
                            o.w = take_piece<T>(x[3], 1.f, i == C::kK - 1);
                            *reinterpret_cast<uint4*>(dst + i * C::kPiece) = o;
                        }
                    }
                    full(&filled[(g + j) & 1]);
                    rows = ahead;
                    ahead = look(j + 2);
                }
            } else {
                // The warp's lanes know where some of a block's keys lie each, a block ahead.  A copy
                // is a shuffle, an address and the copy: what of its place depends on the lane is
                // the same for every eighth row, and whether a row exists is asked once for a block.
                static_assert(C::kWide || C::kLoadWarps == 1);
                constexpr int kEach = kKeys / 32, kPeriod = 8 / kPer;
                uint32_t place_of[kPeriod];
#pragma unroll
                for (int e = 0; e < kPeriod; ++e)
                    place_of[e] = smem_u32(mine) + place(e * kPer + sub, c & 7);
                const T* const source = pool + c * 8;
                int next[kEach], rows[kEach];
                auto look = [&](int j) {
#pragma unroll
                    for (int u = 0; u < kEach; ++u)
                        next[u] = row_of(j * kKeys + u * 32 + lane);
                };
                look(0);
                for (int j = 0; j < steps && free(g + j); ++j) {
                    bool whole = true;
#pragma unroll
                    for (int u = 0; u < kEach; ++u) {
                        rows[u] = next[u];
                        whole &= rows[u] >= 0;
                    }
                    whole = __all_sync(0xffffffffu, whole);
                    look(j + 1);
                    const uint32_t to = ((g + j) & 1) * C::kBuf;
                    // the rows of eight copies are fetched ahead of them: one by one, every copy
                    // waited for its shuffle (80 cycles each)
                    auto copy = [&](int rows, int i0, int first, bool whole) {
                        int r[8];
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            r[e] = __shfl_sync(0xffffffffu, rows, (i0 + e) * kPer + sub);
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            const int at = first + (i0 + e) * kPer;
                            const bool there = whole || r[e] >= 0;
                            cp16(place_of[e % kPeriod] + to + at / 8 * 1024,
                                 source + (size_t)(there ? (unsigned)r[e] : 0u) * DIM, there);
                        }
                    };
                    if (whole) {
#pragma unroll
                        for (int u = 0; u < kEach; ++u)
#pragma unroll
                            for (int i = 0; i < 32 / kPer; i += 8)
                                copy(rows[u], i, u * 32, true);
                    } else {
#pragma unroll
                        for (int u = 0; u < kEach; ++u)
#pragma unroll 1
                            for (int i = 0; i < 32 / kPer; i += 8)
                                copy(rows[u], i, u * 32, false);
                    }
                    // when they have all come; the warp goes on with the next block
                    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];"
                                 ::"r"(smem_u32(&filled[(g + j) & 1]))
                                 : "memory");
                }
            }
            g += steps;
            warp_arrive(&tile_free[n & 1]);
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
      }
    }

    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (warp == kMmaWarp) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;"
                     ::"r"(tmem), "r"(C::kColumns)
                     : "memory");
    }
}

template <typename T, int DIM>
int launch(b2w4_ctx* ctx, const Args& a, const Attend& p, void* work) {
    using C = Cfg<T, DIM>;
    static_assert(C::kBlocks <= kMostBlocks);
    static b2w4_smem_optin cfg;
    auto kern = paged_runs_kernel<T, DIM>;
    const int tq = kRows / (p.heads / a.kv_heads);
    const long tiles = tiles_of(a.rows, a.sequences, p.heads, a.kv_heads);
    const long resident = (long)ctx->sm_count * C::kBlocks;
    const unsigned blocks = (unsigned)(tiles < resident ? tiles : resident);
    const int most_tiles = (int)((tiles + blocks - 1) / blocks);
    B2W4_CUDA(ctx, b2w4_opt_in_smem(ctx, kern, C::kTotal, cfg));
    B2W4_CUDA(ctx, b2w4_launch_chained(ctx->pdl, kern, dim3(blocks), dim3(C::kThreads),
                                       C::kTotal, ctx->stream, a, p, tq, static_cast<Again*>(work),
                                       most_tiles));
    ctx->launches++;
    return B2W4_OK;
}

}  // namespace

// keys: the most that a tile sees.  Tiles are counted in 32 bits; the work area holds an entry of every block's lists for each, and a
// tile of 2^24 keys takes 0.7 s of a wait's 2.
bool b2w4_paged_runs_takes(int sm_count, int dim, int heads, int kv_heads, int rows, int sequences,
                           double keys) {
    if (dim > 128 || heads / kv_heads > kRows || keys > 1 << 24)
        return false;
    const long tiles = tiles_of(rows, sequences, heads, kv_heads);
    return tiles < 0x3fffffff && 4 * sizeof(Again) * (tiles + (long)sm_count * kMostBlocks) <=
                                     b2w4_paged_split_work(sm_count, dim);
}

int b2w4_launch_paged_runs(b2w4_ctx* ctx, int type, int dim, const Args& a, const Attend& p,
                           void* work) {
    if (dim == 64)
        return type == B2W4_F16    ? launch<__half, 64>(ctx, a, p, work)
               : type == B2W4_BF16 ? launch<__nv_bfloat16, 64>(ctx, a, p, work)
                                   : launch<float, 64>(ctx, a, p, work);
    return type == B2W4_F16    ? launch<__half, 128>(ctx, a, p, work)
           : type == B2W4_BF16 ? launch<__nv_bfloat16, 128>(ctx, a, p, work)
                               : launch<float, 128>(ctx, a, p, work);
}
