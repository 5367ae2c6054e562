// Attention over the 8-bit paged cache (kv8.cuh): what its kernels share.
//   o_i = sum_j softmax_j(scale q_i . k_j) v_j  over the positions j <= p_i with  window == 0 or p_i - j < window or j < sinks;
//   zeros where no position is left.
#pragma once
#include "kv8.cuh"

namespace glmasr {

struct Kv8Attend {
    const uint8_t *k_cache, *v_cache;
    const float *k_scale, *v_scale;
    const __nv_bfloat16 *query;
    __nv_bfloat16 *out;
    long long ldq, ldo;
    Kv8Batch b;
    int group;                    // query heads per kv head
    FastDiv by_group, by_q_heads;
    int window, sinks;            // window 0: no limit
    float scale_log2;             // softmax scale * log2(e)
};

#ifdef __CUDACC__
// What the queries at positions [p0, p1] of a sequence with `len` tokens see, in groups of 16 tokens: groups [0, sink) and
// [from, to).  count = all of them.
struct Kv8Span {
    int sink, from, count;
    __device__ __forceinline__ int group_of(int i) const { return i < sink ? i : from + (i - sink); }
};
__device__ __forceinline__ Kv8Span kv8_span(const Kv8Attend &a, int len, int p0, int p1) {
    const int end = min(min(len, p1 + 1), a.b.max_tokens);               // tokens [0, end) exist for them
    Kv8Span s = {0, 0, 0};
    if (end <= 0) return s;
    const int to = (end + kKv8Group - 1) / kKv8Group;
    if (a.window > 0) {
        s.sink = (min(a.sinks, end) + kKv8Group - 1) / kKv8Group;
        s.from = max(max(0, p0 - a.window + 1) / kKv8Group, s.sink);
    }
    s.count = s.sink + max(0, to - s.from);
    return s;
}
__device__ __forceinline__ bool kv8_sees(const Kv8Attend &a, int pos, int tok) {
    return tok <= pos && (a.window == 0 || pos - tok < a.window || tok < a.sinks);
}
#endif

// Bytes of workspace the launch may use (partial results of contexts that several warps share), on the current device.
size_t kv8_attention_workspace_bytes();
bool kv8_attention_launch(const Kv8Attend &a, int max_new, int max_len, void *workspace, cudaStream_t st, int &launches);

}  // namespace glmasr
