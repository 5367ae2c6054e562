// New tokens into the 8-bit paged cache: queries and keys rotated to their positions, keys and values quantised.
//
//   x'[d]      = x[d] cos a - x[d + 64] sin a,  x'[d + 64] = x[d] sin a + x[d + 64] cos a,   a = p * theta^(-d / 64)
//   e(block)   = max over the block's tokens of the exponent above; a block whose earlier tokens came with a smaller scale has
//                their codes rescaled: code' = rn(code * old / new)
//   code       = rn(x' / 2^e)
//
// A block of 16 tokens is read and written by one CTA, so that its scale needs no atomics and no second pass.  All heads of a block
// use the same 16 x 64 angles: they are evaluated once per CTA into shared memory.
//
// Angles and keys are computed in 64 bits.  A key decides by comparison which code, and which scale, it gets; in 32 bits about one
// value in a million falls on the wrong side of a border, and a position of 100000 has lost 7 bits of its angle before the
// cosine.  The 64-bit value is cut to 32 bits with the last bit set if anything was cut off, which keeps every later comparison
// and rounding to 4 bits exact.
#include <math.h>

#include "kv8.cuh"
#include "runtime.cuh"

namespace glmasr {

namespace {

constexpr int THREADS = 256;
constexpr int HALF = kKv8Dim / 2;

struct AppendParams {
    uint8_t *cache[2];            // K, V
    float *scale[2];
    const __nv_bfloat16 *in[2];
    long long ld[2];
    const __nv_bfloat16 *query;   // NULL: none
    __nv_bfloat16 *query_out;
    long long ldq, ldqo;
    Kv8Batch b;
    double turns[HALF];           // theta^(-d / 64) / (2 pi)
};

// 64 bits -> 32 bits, cut towards zero, the last bit set if anything was cut ("round to odd").
__device__ __forceinline__ float cut_odd(double x) {
    const uint32_t hi = (uint32_t)__double2hiint(x), lo = (uint32_t)__double2loint(x);
    const uint32_t mag = hi & 0x7FFFFFFFu;
    if (mag < 0x38100000u || mag >= 0x47F00000u) return (float)x;        // below 2^-126 (nothing there is near a border), or not finite
    const uint32_t r = __funnelshift_l(lo, hi, 3) - (384u << 23);        // nine exponent bits and 23 of the mantissa, exponent re-biased
    return __uint_as_float((hi & 0x80000000u) | (r & 0x7FFFFFFFu) | ((lo & 0x1FFFFFFFu) != 0u ? 1u : 0u));
}

__device__ __forceinline__ float bf16_lo(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t w) { return __uint_as_float(w & 0xFFFF0000u); }

// two values -> two e4m3 codes, nearest, ties to even, saturating (the first in the low byte)
__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) { return e4m3x2(a, b) | (e4m3x2(c, d) << 16); }
// an e4m3 code's value times 2^-120: its bits are those of a bf16 number with another exponent bias
__device__ __forceinline__ float e4m3_value(uint32_t c) { return __uint_as_float(((c & 0x7Fu) << 20) | ((c & 0x80u) << 24)) * 0x1p120f; }

// Exponent of the scale for a block whose largest absolute value has the given bits (finite, at most 448 * 2^60): 448 = 1.75 * 2^8.
__device__ __forceinline__ int scale_exponent(uint32_t amax) {
    const int e = (int)(amax >> 23) - 127 - 8 + ((amax & 0x7FFFFFu) > 0x600000u ? 1 : 0);
    return max(e, -126);
}
__device__ __forceinline__ float pow2f(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }     // e in [-126, 127]

// Angle tables: entry [token][j][i] is dim pair 8 i + j, so that the eight lanes that share a row read side by side.
__device__ __forceinline__ int angle_at(int token, int d) { return token * HALF + (d & 7) * 8 + (d >> 3); }

// One head of one block, K (rotated) or V, by a warp.  Half a warp per token: lane c (0..15) of it has dims 8c .. 8c + 7, two tokens
// per step.
template <bool KEY>
__device__ __forceinline__ void quantise_head(const AppendParams &p, int head, int first_row, int first, int n, int kept, long long row,
                                              const double2 *angles) {
    constexpr int which = KEY ? 0 : 1;
    const int lane = threadIdx.x & 31, c = lane & 15, sub = lane >> 4;
    const __nv_bfloat16 *src = p.in[which] + (size_t)head * kKv8Dim + c * 8;
    float x[8][8];
    uint32_t amax = 0u;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int t = 2 * i + sub;                               // token, from the first new one of the block
        uint4 w = make_uint4(0u, 0u, 0u, 0u);
        const int r = first_row + t;
        if (t < n && r >= 0 && r < p.b.total_new) w = *reinterpret_cast<const uint4 *>(src + (long long)r * p.ld[which]);
        const uint32_t own[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            x[i][2 * j] = bf16_lo(own[j]);
            x[i][2 * j + 1] = bf16_hi(own[j]);
        }
        if (KEY && 2 * i < n) {
            // the other half of the dims is eight lanes away; y = own * cos -+ other * sin
            const double sign = c < 8 ? -1.0 : 1.0;
            const double2 *a = angles + min(t, n - 1) * HALF + (c & 7);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t other = __shfl_xor_sync(0xFFFFFFFFu, own[j], 8);
                const double2 a0 = a[16 * j], a1 = a[16 * j + 8];
                x[i][2 * j] = cut_odd(fma((double)x[i][2 * j], a0.x, sign * a0.y * (double)bf16_lo(other)));
                x[i][2 * j + 1] = cut_odd(fma((double)x[i][2 * j + 1], a1.x, sign * a1.y * (double)bf16_hi(other)));
            }
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) amax = max(amax, __float_as_uint(x[i][j]) & 0x7FFFFFFFu);
    }
    amax = __reduce_max_sync(0xFFFFFFFFu, amax);
    if (row < 0) return;                                         // no page: nowhere to write
    uint8_t *dst = p.cache[which] + row * kKv8Dim;
    float *scale = p.scale[which] + row / kKv8Group;
    const float old = kept > 0 ? *scale : 0.0f;
    const bool poisoned = amax > __float_as_uint(448.0f * 0x1p60f) || (kept > 0 && !(old >= 0.0f && old <= pow2f(kKv8MaxExp)));
    float now = 0.0f, inv = 0.0f;
    if (!poisoned) {
        now = pow2f(scale_exponent(amax));
        if (old > now) now = old;
        inv = 1.0f / now;                                        // exact: a power of two, at most 2^126
    }
    __syncwarp();                                                // every lane has the old scale
    if (lane == 0) *scale = poisoned ? __uint_as_float(0x7FFFFFFFu) : now;
    if (kept > 0 && (poisoned || now != old)) {                  // the earlier tokens of the block, under the new scale
        const float ratio = poisoned ? 0.0f : old * inv;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int t = 2 * i + sub;
            if (t >= kept) continue;
            uint2 *at = reinterpret_cast<uint2 *>(dst + t * kKv8Dim + c * 8);
            uint2 w = *at;
            uint32_t v[2] = {w.x, w.y};
#pragma unroll
            for (int j = 0; j < 2; ++j)
                v[j] = poisoned ? 0u
                                : e4m3x4(e4m3_value(v[j] & 0xFFu) * ratio, e4m3_value((v[j] >> 8) & 0xFFu) * ratio,
                                         e4m3_value((v[j] >> 16) & 0xFFu) * ratio, e4m3_value(v[j] >> 24) * ratio);
            *at = make_uint2(v[0], v[1]);
        }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int t = 2 * i + sub;
        const int r = first_row + t;
        if (t >= n || r < 0 || r >= p.b.total_new) continue;
        uint2 w = make_uint2(0u, 0u);
        if (!poisoned)
            w = make_uint2(e4m3x4(x[i][0] * inv, x[i][1] * inv, x[i][2] * inv, x[i][3] * inv),
                           e4m3x4(x[i][4] * inv, x[i][5] * inv, x[i][6] * inv, x[i][7] * inv));
        *reinterpret_cast<uint2 *>(dst + (first + t) * kKv8Dim + c * 8) = w;
    }
}

__global__ void __launch_bounds__(THREADS, 2) kv8_append_kernel(const __grid_constant__ AppendParams p) {
    __shared__ double2 angles[kKv8Group * HALF];                 // cos, sin
    __shared__ float2 angles_q[kKv8Group * HALF];                // the same, rounded
    pdl_launch_dependents();
    pdl_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    // CTA i takes block i of the batch, where sequence s has its blocks from cu_new[s] / 16 + 2 s on: n tokens touch at most
    // n / 16 + 2 blocks, so this bound needs no pass over the lengths.
    const int *cu = p.b.cu_new;
    const int seq = warp_last_not_above(p.b.num_seqs, (long long)blockIdx.x, [&](int s) { return (long long)(cu[s] >> 4) + 2LL * s; });
    if (seq < 0) return;
    const int row0 = cu[seq], n_new = cu[seq + 1] - row0;
    const int start = p.b.seq_lens[seq] - n_new;                 // position of the sequence's first new token
    const int group = (start >> 4) + ((int)blockIdx.x - (row0 >> 4) - 2 * seq);
    if (n_new <= 0 || group < 0) return;
    const int pos = max(start, group * kKv8Group);               // first new token in this block
    const int n = min(start + n_new, (group + 1) * kKv8Group) - pos;
    if (n <= 0) return;
    const int first = pos & (kKv8Group - 1);                     // its row in the block
    const int first_row = row0 + (pos - start);

    for (int i = threadIdx.x; i < n * HALF; i += THREADS) {
        const double turn = (double)(pos + i / HALF) * p.turns[i % HALF];
        double s, c;
        sincospi(2.0 * (turn - rint(turn)), &s, &c);
        const int at = angle_at(i / HALF, i % HALF);
        angles[at] = make_double2(c, s);
        angles_q[at] = make_float2((float)c, (float)s);
    }
    __syncthreads();

    const int heads = p.b.kv_heads;
    for (int task = warp; task < 2 * heads; task += THREADS / 32) {
        const int head = task >> 1;
        // tokens that were in the block before; with a start inside the block they are the rows below `first`
        const long long row = kv8_group_row(p.b, seq, head, group);
        if (task & 1) quantise_head<false>(p, head, first_row, first, n, first, row, angles);
        else quantise_head<true>(p, head, first_row, first, n, first, row, angles);
    }
    if (p.query == nullptr) return;
    // Queries: half a warp per token with its angles in registers, several tokens' share of the heads each where the block has few
    // tokens.  Nothing is decided by comparison here: 32-bit arithmetic on rounded angles.
    const int c = lane & 15, half_warp = warp * 2 + (lane >> 4);
    const int t = half_warp % n, at = first_row + t;
    const int shares = THREADS / 16 / n, share = half_warp / n;
    const bool there = share < shares && at >= 0 && at < p.b.total_new;
    float2 cs[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) cs[j] = angles_q[t * HALF + j * 8 + (c & 7)];
    if (c < 8)
#pragma unroll
        for (int j = 0; j < 8; ++j) cs[j].y = -cs[j].y;
    const int step = max(1, shares);
    for (int head0 = 0; head0 < p.b.q_heads; head0 += 4 * step) {
        uint4 w[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int head = head0 + u * step + share;
            w[u] = make_uint4(0u, 0u, 0u, 0u);
            if (there && head < p.b.q_heads) w[u] = *reinterpret_cast<const uint4 *>(p.query + (long long)at * p.ldq + (size_t)head * kKv8Dim + c * 8);
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int head = head0 + u * step + share;
            uint32_t own[4] = {w[u].x, w[u].y, w[u].z, w[u].w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t other = __shfl_xor_sync(0xFFFFFFFFu, own[j], 8);
                const float y0 = fmaf(bf16_lo(own[j]), cs[2 * j].x, cs[2 * j].y * bf16_lo(other));
                const float y1 = fmaf(bf16_hi(own[j]), cs[2 * j + 1].x, cs[2 * j + 1].y * bf16_hi(other));
                const __nv_bfloat162 y = __floats2bfloat162_rn(y0, y1);
                own[j] = *reinterpret_cast<const uint32_t *>(&y);
            }
            if (there && head < p.b.q_heads)
                *reinterpret_cast<uint4 *>(p.query_out + (long long)at * p.ldqo + (size_t)head * kKv8Dim + c * 8) = make_uint4(own[0], own[1], own[2], own[3]);
        }
    }
}

}  // namespace

bool kv8_append_launch(uint8_t *k_cache, uint8_t *v_cache, float *k_scale, float *v_scale, const __nv_bfloat16 *key, long long ldk,
                       const __nv_bfloat16 *value, long long ldv, const __nv_bfloat16 *query, long long ldq, __nv_bfloat16 *query_out,
                       long long ldqo, const Kv8Batch &b, double theta, cudaStream_t st) {
    AppendParams p;
    memset(&p, 0, sizeof(p));
    p.cache[0] = k_cache, p.cache[1] = v_cache;
    p.scale[0] = k_scale, p.scale[1] = v_scale;
    p.in[0] = key, p.in[1] = value;
    p.ld[0] = ldk, p.ld[1] = ldv;
    p.query = query, p.query_out = query_out;
    p.ldq = ldq, p.ldqo = ldqo;
    p.b = b;
    // a function of theta alone, kept for the next layer's call
    static double known = -1.0, turns[HALF];
    if (theta != known) {
        for (int d = 0; d < HALF; ++d) turns[d] = theta > 0.0 ? pow(theta, -(double)d / HALF) / 6.283185307179586476925 : 0.0;
        known = theta;
    }
    memcpy(p.turns, turns, sizeof(turns));
    const long long blocks = (long long)b.total_new / 16 + 2LL * b.num_seqs;
    return launch_chained(kv8_append_kernel, dim3((unsigned)blocks), dim3(THREADS), 0, st, p) == cudaSuccess;
}

}  // namespace glmasr
