// Attention over the 8-bit paged cache (kv8.cuh): what its kernels share.
//   o_i = sum_j softmax_j(scale q_i . k_j) v_j  over the positions j <= p_i with  window == 0 or p_i - j < window or j < sinks;
//   zeros where no position is left.
#pragma once
#include <cuda_fp16.h>

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
    FastDiv by_group;
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

constexpr float kNothing = -3.4028234664e38f;     // a running maximum before the first term: every term is above it, and 2^(it - m) is 0

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float lg2(float x) {
    float y;
    asm("lg2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float pow2(int e) { return __int_as_float((e + 127) << 23); }      // e in [-126, 127]
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    const __nv_bfloat162 b = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&b);
}
// two values -> two e4m3 codes, nearest (the first in the low byte), and what is left of each
__device__ __forceinline__ uint32_t e4m3_split(float &a, float &b) {
    uint16_t c;
    uint32_t h;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(c) : "f"(b), "f"(a));
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(c));
    const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&h));
    a -= f.x, b -= f.y;
    return c;
}
__device__ __forceinline__ uint32_t e4m3x2(float a, float b) {
    uint16_t c;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(c) : "f"(b), "f"(a));
    return c;
}
// byte b (0..127) of row r of an operand with 128-byte rows under the 128-byte swizzle
__device__ __forceinline__ uint32_t swizzled(int r, int b) { return (uint32_t)(r * 128 + ((((b >> 4) ^ (r & 7)) << 4) | (b & 15))); }
#endif

// Bytes of workspace the launch may use (partial results of contexts that several warps share), on the current device.
size_t kv8_attention_workspace_bytes();
bool kv8_attention_launch(const Kv8Attend &a, int max_new, int max_len, void *workspace, cudaStream_t st, int &launches);
// Many queries per sequence (kv8_prefill.cu): a tile of 128 (query, head of the group) rows per CTA.
bool kv8_prefill_launch(const Kv8Attend &a, cudaStream_t st);
int kv8_prefill_take_status();     // as kv8_take_status(), for kv8_prefill.cu alone

}  // namespace glmasr
