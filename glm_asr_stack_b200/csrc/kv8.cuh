// The 8-bit paged KV cache: what its kernels share.
//
//   codes   e4m3 [num_blocks][kv_heads][block_size][128], K and V each
//   scales  fp32 [num_blocks][kv_heads][block_size / 16], K and V each: one power of two per 16 tokens of a head
//   value   code * scale
//
// The tokens of a page lie together per head (the bf16 pool interleaves the heads), so that 16 tokens of one head, the unit every
// kernel here works in, are 2 KB in one piece.  A scale is the smallest 2^e, e >= -126, with amax <= 448 * 2^e.  Powers of two make
// what follows exact: a block whose scale grows is rescaled without a second rounding (but where a code leaves e4m3's normal
// range), and code * scale is a bf16 number.  A block that got a value that is not finite, or one beyond 448 * 2^60, has the scale
// NaN and zero codes until its first token is written again, and every query that sees a token of it gets NaN.
//
// A batch: sequence s has the packed rows [cu_new[s], cu_new[s + 1]) as its new tokens and seq_lens[s] tokens with them, so row i
// of it is at position seq_lens[s] - n_s + i.  Rows outside [0, total_new), positions below zero or behind the block table, and
// pages outside [0, num_blocks) are skipped.
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace glmasr {

static constexpr int kKv8Group = 16;               // tokens under one scale
static constexpr int kKv8Dim = 128;                // head_dim
static constexpr int kKv8MaxExp = 60;              // largest exponent of a scale

// Division by a number that the host knows, for dividends below 2^31: a 32 x 32 bit product and a shift.  With s the smallest power of two
// not below d, m = ceil(2^(31 + log2 s) / d) exceeds the true factor by less than 2^-31 of it, too little to reach the next integer.
struct FastDiv {
    uint32_t d, mul, shift;
    FastDiv() = default;
    explicit FastDiv(int by) {
        d = (uint32_t)by;
        uint32_t log2 = 0;
        while ((1ull << log2) < d) ++log2;
        mul = (uint32_t)(((1ull << (31 + log2)) + d - 1) / d);
        shift = log2 + 31;
    }
#ifdef __CUDACC__
    __device__ __forceinline__ int div(int x) const { return (int)(((unsigned long long)(uint32_t)x * mul) >> shift); }
#endif
};

struct Kv8Batch {
    FastDiv by_kv_heads, by_page;     // by_page: groups of a page
    const int *block_tables;      // [num_seqs, max_blocks]
    const int *seq_lens;          // [num_seqs]
    const int *cu_new;            // [num_seqs + 1]
    int num_seqs, max_blocks, num_blocks, block_size, kv_heads, q_heads, total_new;
    int max_tokens;               // that a row of the table has pages for
};

#ifdef __CUDACC__
// First token of a group in rows of 128 codes; -1 where there is no page for it.
__device__ __forceinline__ long long kv8_group_row(const Kv8Batch &b, int seq, int head, int group) {
    if (group < 0) return -1;
    const int page = b.by_page.div(group);
    if (page >= b.max_blocks) return -1;
    const int blk = b.block_tables[(size_t)seq * b.max_blocks + page];
    if (blk < 0 || blk >= b.num_blocks) return -1;
    return ((long long)blk * b.kv_heads + head) * b.block_size + (long long)(group - page * (int)b.by_page.d) * kKv8Group;
}

// The last s in [0, n) with key(s) <= x for a non-decreasing key, or -1: a whole warp looks 32 places up per round.
template <typename Key>
__device__ __forceinline__ int warp_last_not_above(int n, long long x, Key key) {
    const int lane = threadIdx.x & 31;
    int lo = -1, hi = n;                           // key(lo) <= x < key(hi)
    while (hi - lo > 1) {
        const int step = (hi - lo - 1 + 31) / 32;
        const int s = lo + 1 + lane * step;
        const bool le = s < hi && key(s) <= x;
        const unsigned m = __ballot_sync(0xFFFFFFFFu, le);
        if (m == 0u) return lo;
        const int top = lo + 1 + (31 - __clz((int)m)) * step;
        hi = min(hi, top + step);
        lo = top;
    }
    return lo;
}
#endif

int kv8_take_status();             // first status code of these kernels on the current device, cleared; 0 if none
int kv8_status();                  // the same, without asking a device that none of them was launched on

bool kv8_append_launch(uint8_t *k_cache, uint8_t *v_cache, float *k_scale, float *v_scale, const __nv_bfloat16 *key, long long ldk,
                       const __nv_bfloat16 *value, long long ldv, const __nv_bfloat16 *query, long long ldq, __nv_bfloat16 *query_out,
                       long long ldqo, const Kv8Batch &b, double theta, cudaStream_t st);

}  // namespace glmasr
