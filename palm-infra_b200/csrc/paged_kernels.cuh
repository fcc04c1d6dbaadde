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
#endif

}  // namespace paged

// Runs of rows (paged_runs.cu): heads of 64 or 128 numbers.
bool b2w4_paged_runs_takes(int dim, int heads, int kv_heads, int rows, int sequences);
int b2w4_launch_paged_runs(b2w4_ctx* ctx, int type, int dim, const paged::Args& a,
                           const paged::Attend& p);

bool b2w4_paged_runs_wanted(int sm_count, const b2w4_paged_cache& c, const b2w4_paged_batch& b,
                            int heads, int window, int sinks);

// One row per sequence, or row by row (paged_split.cu).
size_t b2w4_paged_split_work(int sm_count, int dim);
int b2w4_launch_paged_split(b2w4_ctx* ctx, int type, int dim, paged::Args a,
                            const paged::Attend& p, bool by_row, void* work);
