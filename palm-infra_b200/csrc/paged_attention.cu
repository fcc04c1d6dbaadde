// Paged key-value cache: the step between the qkv matmul and attention (Q/K norm, rotary
// embedding, append to the pages), and attention over the pages.
#include "paged_kernels.cuh"

#include <math.h>

#include <climits>

namespace {

using paged::Args;
using paged::Attend;
using paged::Sequence;
using paged::Window;

constexpr int kWarps = 8;

// Whether sequence i's slot is that of an earlier sequence too (whole warp).
__device__ __forceinline__ bool slot_again(const Args& a, int i) {
    if (!a.slots_of)
        return false;
    const int mine = a.slots_of[i];
    bool again = false;
    for (int j = threadIdx.x & 31; j < i; j += 32)
        again |= a.slots_of[j] == mine;
    return __any_sync(0xffffffffu, again);
}

struct Prepare {
    const float *qkv, *q_weight, *k_weight, *cosv, *sinv;
    float* q_out;
    float eps;
    int ld, ldq, heads;
};

// A block has a row and a warp EACH heads of it at a time, all their loads on the way together;
// what the row needs -- its sequence, position, cosines and sines -- is looked up once.  The
// arithmetic is that of b2w4_qkv_prepare, operation for operation; keys and values are rounded to
// the cache's type as they are stored.
// What bounds it: memory traffic, for a few rows the chain of lookups.  3208 rows of 32 / 8 heads of
// 128 into an fp32 cache take 35 us (4.5 TB/s), 48 with a warp for every head and a lookup in each;
// 64 rows 3 us with a warp for every head.
template <typename T, int DIM, int EACH>
__global__ void __launch_bounds__(32 * kWarps)
paged_prepare_kernel(const Args a, const Prepare p) {
    b2w4_pdl_chain_entry();
    constexpr int kPer = DIM / 32, kHi = kPer / 2;  // v[i] pairs with v[i + kHi]
    const int slots = p.heads + 2 * a.kv_heads;
    const int row = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int first = (blockIdx.y * kWarps + warp) * EACH;
    if (first >= slots)
        return;
    float v[EACH][kPer];
    const float* x = p.qkv + (size_t)row * p.ld + (size_t)first * DIM;
#pragma unroll
    for (int e = 0; e < EACH; ++e)
#pragma unroll
        for (int d = 0; d < kPer; ++d)
            v[e][d] = first + e < slots ? x[e * DIM + lane + 32 * d] : 0.f;
    const int i = paged::sequence_of(a, row);
    if (i < 0)
        return;
    bool bad = false;
    const Sequence s = paged::taken(a, i, &bad);
    if (bad)
        b2w4_report(a.status, B2W4_E_INVALID);
    const int in = row - s.first;
    const int pos = s.length - s.count + in;
    const bool token = in < s.count && pos >= 0;
    float c[kHi], sn[kHi];
    int page_row = -1;  // of kv head 0
    if (token) {
#pragma unroll
        for (int d = 0; d < kHi; ++d) {
            c[d] = p.cosv[(size_t)pos * (DIM / 2) + lane + 32 * d];
            sn[d] = p.sinv[(size_t)pos * (DIM / 2) + lane + 32 * d];
        }
        if (first + EACH > p.heads) {  // keys or values among the warp's
            page_row = slot_again(a, i) ? -1 : paged::cache_row(a, s.table, pos, 0);
            if (page_row < 0)
                b2w4_report(a.status, B2W4_E_INVALID);
        }
    }
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
        const int slot = first + e;
        if (slot >= slots)
            break;
        const bool query = slot < p.heads, key = !query && slot < p.heads + a.kv_heads;
        float* q = p.q_out + (size_t)row * p.ldq + (size_t)slot * DIM;
        if (!token) {
            if (query)
#pragma unroll
                for (int d = 0; d < DIM; d += 32)
                    q[lane + d] = 0.f;
            continue;
        }
        T* dst = nullptr;
        if (!query) {
            if (page_row < 0)
                continue;
            const int h = slot - p.heads - (key ? 0 : a.kv_heads);
            dst = static_cast<T*>(key ? a.k : a.v) +
                  ((size_t)page_row + (size_t)h * a.page_size) * DIM;
            if (!key) {
#pragma unroll
                for (int d = 0; d < kPer; ++d)
                    dst[lane + 32 * d] = paged::stored<T>(v[e][d]);
                continue;
            }
        }
        const float* w = query ? p.q_weight : p.k_weight;
        if (w) {
            float ss = 0.f;
#pragma unroll
            for (int d = 0; d < kPer; ++d)
                ss = __fadd_rn(ss, __fmul_rn(v[e][d], v[e][d]));
            ss = paged::warp_sum(ss);
            const float r = __fdiv_rn(1.f, sqrtf(__fadd_rn(__fdiv_rn(ss, (float)DIM), p.eps)));
#pragma unroll
            for (int d = 0; d < kPer; ++d)
                v[e][d] = __fmul_rn(__fmul_rn(v[e][d], r), w[lane + 32 * d]);
        }
#pragma unroll
        for (int d = 0; d < kHi; ++d) {
            const int j = lane + 32 * d;
            const float x0 = v[e][d], x1 = v[e][d + kHi];
            const float lo = __fsub_rn(__fmul_rn(x0, c[d]), __fmul_rn(x1, sn[d]));
            const float hi = __fadd_rn(__fmul_rn(x0, sn[d]), __fmul_rn(x1, c[d]));
            if (query) {
                q[j] = lo;
                q[j + DIM / 2] = hi;
            } else {
                dst[j] = paged::stored<T>(lo);
                dst[j + DIM / 2] = paged::stored<T>(hi);
            }
        }
    }
}

bool misaligned(const void* p, int ld = 0) {
    return (reinterpret_cast<uintptr_t>(p) & 15) || (ld & 3);
}

// Calls f with a null pointer of the cache's type and its head size.
template <typename F>
int by_type(int type, int dim, F f) {
    auto by_dim = [&](auto* t) {
        switch (dim) {
        case 64: return f(t, std::integral_constant<int, 64>());
        case 128: return f(t, std::integral_constant<int, 128>());
        case 192: return f(t, std::integral_constant<int, 192>());
        default: return f(t, std::integral_constant<int, 256>());
        }
    };
    switch (type) {
    case B2W4_F16: return by_dim(static_cast<__half*>(nullptr));
    case B2W4_BF16: return by_dim(static_cast<__nv_bfloat16*>(nullptr));
    default: return by_dim(static_cast<float*>(nullptr));
    }
}

Args args_of(b2w4_ctx* ctx, const b2w4_paged_cache& c, const b2w4_paged_batch& b) {
    Args a = {c.k_dev,   c.v_dev,  b.tables_dev, b.lengths_dev, b.slots_dev,
              b.starts_dev, c.pages, c.kv_heads,   c.page_size,   b.slots,
              b.table_len, b.sequences, b.rows,    b.max_length,
              ctx ? ctx->status_dev : nullptr, 0, 0, 0, 0, 0};
    paged::set_division(a);
    return a;
}

}  // namespace

// Runs of rows go to the kernel that takes 128 (row, head) pairs together, or row by row to the one
// that shares the cache's bytes out over the chip: long runs and many sequences to the former, a few
// rows behind a long cache to the latter, by their times in us.  A tile's steps are those of
// paged_runs.cu; row by row every token has its keys read again, from the second level cache for the
// most part.  Heads of 192 and 256 numbers, groups of more than 128, and what
// b2w4_paged_runs_takes has no room or time for, go row by row whatever that costs (a prompt of 2000 of
// 16 / 4 heads of 256: 7.1 ms in fp32, 2.5 in bf16, 1.8 in fp16; of 128, together, 0.14, 0.07, 0.06).
// Measured, us together / row by row, 32 heads over 8 of 128 in bf16: 2 rows behind 30,000 keys 506 /
// 52; 16 behind 2000 44 / 33; 32 behind 4000 75 / 81; 64 behind 8000 138 / 278; 128 behind 4000 75 /
// 278; under a window of 512 16 rows 21.5 / 18, 64 rows 22.5 / 33.  In fp32: 16 behind 2000 92 / 55; 32
// behind 4000 172 / 180; 128 behind 4000 184 / 669.  Of 174 shapes (three types, four head layouts,
// 54 of them under windows of 512 and 2048) three take the one that is slower by more than 5 %: 64 rows
// of 64 / 4 heads of 128 in fp16 behind 8000 keys (166, together 122), 64 of 64 / 8 of 64 in fp16 under
// a window of 512 (20.5, 18.0), 32 of 32 / 8 of 128 in bf16 behind 4000 (81, 75).
extern "C" int b2w4_paged_runs_wanted_by(int sm_count, int type, int dim, int heads, int kv_heads,
                                         int rows, int sequences, int max_length, int window,
                                         int sinks) {
    const int rep = heads / kv_heads;
    if (rep > 128)
        return 0;
    const bool wide = type == B2W4_F32, two = !wide && dim == 64;
    const int tq = 128 / rep, per = wide || two ? 64 : 128;
    double keys = max_length;
    if (window > 0 && (double)window + sinks + tq < keys)
        keys = (double)window + sinks + tq;
    if (!b2w4_paged_runs_takes(sm_count, dim, heads, kv_heads, rows, sequences, keys))
        return 0;
    const double tiles = ((double)rows / tq + 0.5 * sequences) * kv_heads;
    const double waves = ceil(tiles / (sm_count * (two ? 2 : 1)));
    // (two blocks beside each other share the products' rate)
    const double step = wide ? (dim == 64 ? 1.6 : 2.8)
                        : two ? (tiles <= sm_count ? 1.25 : 1.9) : 2.2;
    const double together = 6. + waves * (4. + keys / per * step);
    // row by row: bytes a microsecond, by what their products cost
    const double sets = rep <= 8 ? 1 : (rep + 15) / 16;
    const double bytes = (double)rows * kv_heads * sets * keys * 2 * dim * (wide ? 4 : 2);
    const double rate = (wide ? 6.8e6 : type == B2W4_F16 ? 12e6 : 8e6) * (rep <= 8 ? 1 : 0.66);
    return together <= 12. + bytes / rate;
}

bool b2w4_paged_runs_wanted(int sm_count, const b2w4_paged_cache& c, const b2w4_paged_batch& b,
                            int heads, int window, int sinks) {
    const double room = (double)b.table_len * c.page_size;  // a table's tokens
    return b2w4_paged_runs_wanted_by(sm_count, c.type, c.dim, heads, c.kv_heads, b.rows, b.sequences,
                                     room < b.max_length ? (int)room : b.max_length, window,
                                     sinks) != 0;
}

// What a cache and a batch must be, whatever is done with them; the text of what is wrong, or
// NULL.  Host only, for the entry points and for checks without a device.
extern "C" const char* b2w4_paged_refusal(const b2w4_paged_cache* c, const b2w4_paged_batch* b,
                                          int heads) {
    if (!c || !b)
        return "no cache or no batch";
    if (!c->k_dev || !c->v_dev || misaligned(c->k_dev) || misaligned(c->v_dev))
        return "the pools must be 16-byte aligned device memory";
    if (c->type != B2W4_F32 && c->type != B2W4_F16 && c->type != B2W4_BF16)
        return "the cache's type is fp32, fp16 or bf16";
    if (c->dim <= 0 || c->dim > 256 || c->dim % 64)
        return "heads of 64, 128, 192 or 256 numbers";
    if (c->pages <= 0 || c->kv_heads <= 0 || c->page_size <= 0 ||
        (double)c->pages * c->kv_heads * c->page_size > INT_MAX)
        return "pages, kv_heads and page_size must be positive, with fewer than 2^31 rows";
    if (heads <= 0 || heads % c->kv_heads || (double)heads * c->dim > INT_MAX / 4)
        return "heads must be a multiple of kv_heads";
    if (!b->tables_dev || !b->lengths_dev || b->slots <= 0 || b->table_len <= 0 ||
        b->sequences <= 0 || b->max_length <= 0 || b->max_new <= 0)
        return "tables, lengths, slots, table_len, sequences, max_new and max_length are wanted";
    if (!b->slots_dev && b->sequences > b->slots)
        return "more sequences than slots";
    if (b->rows <= 0 || (!b->starts_dev && b->rows != b->sequences))
        return "without starts every sequence has one row";
    if ((double)b->rows * heads > INT_MAX / 64)
        return "too many rows";
    return nullptr;
}

// Where token j of a sequence lies, by the kernels' own arithmetic: for checks without a device
// (every pointer of the batch is host memory).  The row of the pools, -1 for a page that is not
// theirs, -2 where the sequence is not one of the batch's or has no such token; length, first
// and count as they are bounded (what is out of bounds has no token: paged::taken).
extern "C" int b2w4_paged_row(const b2w4_paged_cache* c, const b2w4_paged_batch* b, int i, int j,
                              int h, int* length, int* first, int* count) {
    const Args a = args_of(nullptr, *c, *b);
    bool bad = false;
    const Sequence s = paged::sequence(a, i, &bad);
    *length = s.length;
    *first = s.first;
    *count = s.count;
    if (bad || j < 0 || j >= s.length)
        return -2;
    return paged::cache_row(a, s.table, j, h);
}

extern "C" {

int b2w4_paged_prepare(b2w4_ctx* ctx, const b2w4_paged_cache* cache,
                       const b2w4_paged_batch* batch, const float* qkv_dev, int ld, int heads,
                       const float* q_weight_dev, const float* k_weight_dev, float eps,
                       const float* cos_dev, const float* sin_dev, float* q_out_dev, int ldq) {
    if (!ctx)
        return B2W4_E_INVALID;
    if (const char* why = b2w4_paged_refusal(cache, batch, heads))
        return b2w4_fail(ctx, B2W4_E_INVALID, "paged_prepare: %s", why);
    const int slots = heads + 2 * cache->kv_heads;
    if (!qkv_dev || !cos_dev || !sin_dev || !q_out_dev || ld < slots * cache->dim ||
        ldq < heads * cache->dim || slots > 65535)
        return b2w4_fail(ctx, B2W4_E_INVALID, "paged_prepare: bad rows (ld %d, ldq %d)", ld, ldq);
    if (b2w4_overlap(q_out_dev, sizeof(float) * ((size_t)(batch->rows - 1) * ldq +
                                                 heads * cache->dim),
                     qkv_dev, sizeof(float) * ((size_t)(batch->rows - 1) * ld +
                                               slots * cache->dim)))
        return b2w4_fail(ctx, B2W4_E_INVALID, "paged_prepare: q_out lies over qkv");
    const b2w4_device_guard device(ctx);
    const Args a = args_of(ctx, *cache, *batch);
    const Prepare p = {qkv_dev, q_weight_dev, k_weight_dev, cos_dev, sin_dev,
                       q_out_dev, eps, ld, ldq, heads};
    // few rows: a head per warp, so that more of the chip works on them
    const bool few = (long)batch->rows * slots <= 64l * ctx->sm_count;
    return by_type(cache->type, cache->dim, [&](auto* t, auto dim) {
        using T = std::remove_pointer_t<decltype(t)>;
        auto launch = [&](auto kern, int each) {
            const dim3 grid(batch->rows, (slots + kWarps * each - 1) / (kWarps * each));
            B2W4_CUDA(ctx, b2w4_launch_chained(ctx->pdl, kern, grid, dim3(32 * kWarps), 0,
                                               ctx->stream, a, p));
            ctx->launches++;
            return (int)B2W4_OK;
        };
        return few ? launch(paged_prepare_kernel<T, dim(), 1>, 1)
                   : launch(paged_prepare_kernel<T, dim(), 4>, 4);
    });
}

size_t b2w4_paged_attention_work(const b2w4_ctx* ctx, int heads, int dim) {
    return ctx && heads > 0 && dim > 0 ? b2w4_paged_split_work(ctx->sm_count, dim) : 0;
}

int b2w4_paged_attention(b2w4_ctx* ctx, const b2w4_paged_cache* cache,
                         const b2w4_paged_batch* batch, const float* q_dev, int ldq, int heads,
                         float scale, int window, int sinks, float* out_dev, int ldo,
                         void* work_dev, size_t work_bytes) {
    if (!ctx)
        return B2W4_E_INVALID;
    if (const char* why = b2w4_paged_refusal(cache, batch, heads))
        return b2w4_fail(ctx, B2W4_E_INVALID, "paged_attention: %s", why);
    const int width = heads * cache->dim;
    if (!q_dev || !out_dev || ldq < width || ldo < width || misaligned(q_dev, ldq) ||
        misaligned(out_dev, ldo))
        return b2w4_fail(ctx, B2W4_E_INVALID,
                         "paged_attention: q and out are 16-byte aligned rows of %d numbers",
                         width);
    if (window < 0 || sinks < 0)
        return b2w4_fail(ctx, B2W4_E_INVALID, "paged_attention: a negative window or sinks");
    const size_t span = sizeof(float) * (size_t)(batch->rows - 1);
    if (b2w4_overlap(q_dev, span * ldq + sizeof(float) * width, out_dev,
                     span * ldo + sizeof(float) * width))
        return b2w4_fail(ctx, B2W4_E_INVALID, "paged_attention: out lies over q");
    if (!work_dev || misaligned(work_dev) ||
        work_bytes < b2w4_paged_attention_work(ctx, heads, cache->dim))
        return b2w4_fail(ctx, B2W4_E_INVALID, "paged_attention: the work area is too small");
    const b2w4_device_guard device(ctx);
    const Args a = args_of(ctx, *cache, *batch);
    const Attend p = {q_dev, out_dev, scale, {window, sinks}, ldq, ldo, heads};
    const bool runs = batch->max_new > 1;
    if (runs && b2w4_paged_runs_wanted(ctx->sm_count, *cache, *batch, heads, window, sinks))
        return b2w4_launch_paged_runs(ctx, cache->type, cache->dim, a, p, work_dev);
    return b2w4_launch_paged_split(ctx, cache->type, cache->dim, a, p, runs, work_dev);
}

}  // extern "C"
