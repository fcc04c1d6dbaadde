// The kernels of attention over a paged cache, as the entry point calls them.
#pragma once

#include "paged.cuh"

namespace paged {

// q and out: rows of ldq and ldo numbers, heads * dim of them used.
struct Attend {
    const float* q;
    float* out;
    float scale;
    Window window;
    int ldq, ldo, heads;
};

#ifdef __CUDACC__
// A result that the pieces of its operands may have lost: done again key by key.  Pieces of 32-bit
// numbers below 2^-133 are no bf16 numbers any more.
template <typename T>
__device__ __forceinline__ bool odd_result(float x) {
    return !(fabsf(x) < INFINITY) || (sizeof(T) == 4 && x != 0.f && fabsf(x) < 0x1p-100f);
}

// Operands of 32 bits as sums of pieces of the cache's 16-bit type (bf16 beside an fp32 cache).
// bf16 has fp32's exponents: three pieces are all 24 bits, whatever the number's size.  fp16 has
// not: a second piece that is what the first one left falls among the numbers below 2^-14, whose
// step does not shrink with them, from 2^-3 of the largest on.  So what is left is taken times kUp,
// about as large again as the first piece, and the sum of its products times kDown.  Two pieces are then 22 bits (off by 2^-23 of the number) down to 2^-14, and below that a
// multiple of 2^-36.  Largest numbers lie just below 2^15: what is left of them is below 2^3.
template <typename T>
constexpr bool kHalf = std::is_same_v<T, __half>;
constexpr int kUpBits = 12;
constexpr float kUp = 0x1p12f, kDown = 0x1p-12f;
// 2^kLift times a row's probabilities are what is taken apart and summed: a multiple of 2^-51 of the
// row's largest.
template <typename T>
constexpr float kLift = kHalf<T> ? 15.f : 0.f;
// The exponents of a row's largest query, taken to [2^kTop, 2^(kTop + 1)).
constexpr int kTop = 14;

// The next piece of two numbers, low half = lo; they keep what is left (exact), times `up` if that
// is not 1, but not behind the last piece.
template <typename T>
__device__ __forceinline__ uint32_t take_piece(uint64_t& v, float up = 1.f, bool last = false) {
    float lo, hi;
    b2w4_unpack2(v, lo, hi);
    uint32_t p;
    if constexpr (kHalf<T>) {
        asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(p) : "f"(hi), "f"(lo));
        if (last)
            return p;
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&p));
        v = b2w4_sub2(v, b2w4_pack2(f.x, f.y));
    } else {
        asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(p) : "f"(hi), "f"(lo));
        if (last)
            return p;
        v = b2w4_sub2(v, b2w4_pack2(__uint_as_float(p << 16), __uint_as_float(p & 0xffff0000u)));
    }
    if (up != 1.f)
        v = b2w4_mul2(v, b2w4_pack2(up, up));
    return p;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ float exp2_neg(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool there) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src),
                 "r"(there ? 16 : 0)
                 : "memory");
}
#endif

}  // namespace paged

// Runs of rows (paged_runs.cu): heads of 64 or 128 numbers.  work: as the split kernel's.
bool b2w4_paged_runs_takes(int sm_count, int dim, int heads, int kv_heads, int rows, int sequences,
                           double keys);
int b2w4_launch_paged_runs(b2w4_ctx* ctx, int type, int dim, const paged::Args& a,
                           const paged::Attend& p, void* work);

bool b2w4_paged_runs_wanted(int sm_count, const b2w4_paged_cache& c, const b2w4_paged_batch& b,
                            int heads, int window, int sinks);

// One row per sequence, or row by row (paged_split.cu).
size_t b2w4_paged_split_work(int sm_count, int dim);
int b2w4_launch_paged_split(b2w4_ctx* ctx, int type, int dim, paged::Args a,
                            const paged::Attend& p, bool by_row, void* work);
