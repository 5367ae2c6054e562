// New tokens into the 8-bit paged cache: queries and keys rotated to their positions, keys and values quantised.
//
//   x'[d]      = x[d] cos a - x[d + 64] sin a,  x'[d + 64] = x[d] sin a + x[d + 64] cos a,   a = p * theta^(-d / 64)
//   e(block)   = max over the block's tokens of the exponent above; a block whose earlier tokens came with a smaller scale has
//                their codes rescaled: code' = rn(code * old / new)
//   code       = rn(x' / 2^e)
//
// A block of 16 tokens of K and V is read and written by one CTA, so that its scale needs no atomics and no second pass; others (grid.y)
// rotate the queries of the block, 16 heads each.  All heads of a block use the same 16 x 64 angles: a CTA evaluates them once, into
// shared memory, while its first rows are on their way.
//
// Bound: the rows' bytes for many tokens, but every CTA is a chain (its sequence, lengths, rows, angles, scale, stores), so there are
// three CTAs per SM (80 registers, eight tokens of a head per warp): 10000 tokens of 25 prompts take 27.8 us (62% of the copy
// bandwidth); 46 us with two CTAs of 128 registers whose warps had sixteen tokens, and the queries as well.  256 sequences
// with a token each take 6.6 us (7.3), one token 3.4 us (4.9).
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

constexpr int THREADS = 256, CTAS = 3;     // per SM
constexpr int QUERY_HEADS = 16;            // of a CTA that has queries
constexpr size_t SPREAD = 64 * 1024;       // of shared memory: with it two CTAs fit an SM, not three
constexpr int HALF = kKv8Dim / 2;
// Keys are computed times 2^40, which their angles bring along: numbers below 2^-126, where 32 bits have fewer digits, are then below
// 2^-166, and the smallest one with a code other than 0 is 2^-136.  At the other end 448 * 2^60 still has 2^19 above it.
constexpr int KEY_EXP = 40;
constexpr double KEY_UNIT = (double)(1ull << KEY_EXP);

struct AppendParams {
    uint8_t *cache[2];            // K, V
    float *scale[2];
    const __nv_bfloat16 *in[2];
    long long ld[2];
    const __nv_bfloat16 *query;   // NULL: none
    __nv_bfloat16 *query_out;
    long long ldq, ldqo;
    Kv8Batch b;
    double turns[HALF];           // theta^(-d / 64) / (2 pi); zeros: no rotation
};

// 64 bits -> 32 bits, cut towards zero, the last bit set if anything was cut ("round to odd").
__device__ __forceinline__ float cut_odd(double x) {
    const uint32_t hi = (uint32_t)__double2hiint(x), lo = (uint32_t)__double2loint(x);
    const uint32_t mag = hi & 0x7FFFFFFFu;
    if (mag < 0x38100000u || mag >= 0x47F00000u) return (float)x;        // below 2^-126 (there is no border there: see KEY_UNIT), or not finite
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

// Exponent of the scale for a block whose largest absolute value, times 2^unit, has the given bits (finite, at most 448 * 2^60 without the
// unit): 448 = 1.75 * 2^8.
__device__ __forceinline__ int scale_exponent(uint32_t amax, int unit) {
    const int e = (int)(amax >> 23) - 127 - 8 - unit + ((amax & 0x7FFFFFu) > 0x600000u ? 1 : 0);
    return max(e, -126);
}
__device__ __forceinline__ float pow2f(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }     // e in [-126, 127]

// Angle tables: entry [token][j][i] is dim pair 8 i + j, so that the eight lanes that share a row read side by side.
__device__ __forceinline__ int angle_at(int token, int d) { return token * HALF + (d & 7) * 8 + (d >> 3); }

// What a warp does of a block: half a warp per token, lane c (0..15) of it has dims 8c .. 8c + 7, two tokens per step and eight in all.
// A head of a block with more new tokens takes two warps.
constexpr int STEPS = 4;
struct Part {
    int first_row, n;             // row of the block's first new token in the batch, new tokens of the block
    int first;                    // the first one's place in the block; places before it have earlier tokens
    int from;                     // of the new tokens, this warp's first
};

__device__ __forceinline__ void load_rows(const AppendParams &p, const Part &b, int which, int head, uint4 (&w)[STEPS]) {
    const int lane = threadIdx.x & 31;
    const __nv_bfloat16 *src = p.in[which] + (size_t)head * kKv8Dim + (lane & 15) * 8;
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
        const int t = b.from + 2 * i + (lane >> 4), r = b.first_row + t;
        w[i] = make_uint4(0u, 0u, 0u, 0u);
        if (t < b.n && r >= 0 && r < p.b.total_new) w[i] = *reinterpret_cast<const uint4 *>(src + (long long)r * p.ld[which]);
    }
}

// The two warps of a head meet.
__device__ __forceinline__ void meet(int pair) { asm volatile("barrier.cta.sync %0, 64;" ::"r"(1 + pair) : "memory"); }

// One head of one block, K (rotated) or V.  shared_max: where the two warps of a head find each other's largest value (NULL: one warp)
template <bool KEY>
__device__ __forceinline__ void quantise_head(const AppendParams &p, const Part &b, long long row, const uint4 (&w)[STEPS], const double2 *angles, volatile uint32_t *shared_max) {
    constexpr int which = KEY ? 0 : 1;
    constexpr float unit = KEY ? (float)KEY_UNIT : 1.0f;         // that x is taken times
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, c = lane & 15, sub = lane >> 4;
    float *scale = p.scale[which] + row / kKv8Group;
    const float old = b.first > 0 && row >= 0 ? *scale : 0.0f;
    float x[STEPS][8];
    uint32_t amax = 0u;
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
        const uint32_t own[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            x[i][2 * j] = bf16_lo(own[j]);
            x[i][2 * j + 1] = bf16_hi(own[j]);
        }
        if (KEY && b.from + 2 * i < b.n) {
            // the other half of the dims is eight lanes away; y = own * cos -+ other * sin
            const double sign = c < 8 ? -1.0 : 1.0;
            const double2 *a = angles + min(b.from + 2 * i + sub, b.n - 1) * HALF + (c & 7);
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
    if (shared_max != nullptr) {
        if (lane == 0) shared_max[warp] = amax;
        meet(warp >> 1);
        amax = max(amax, shared_max[warp ^ 1]);
    } else {
        __syncwarp();
    }
    // every lane has the old scale
    if (row < 0) return;                                         // no page: nowhere to write
    uint8_t *dst = p.cache[which] + row * kKv8Dim;
    const bool poisoned = amax > __float_as_uint(448.0f * 0x1p60f * unit) || (b.first > 0 && !(old >= 0.0f && old <= pow2f(kKv8MaxExp)));
    float now = 0.0f, inv = 0.0f;
    if (!poisoned) {
        now = pow2f(scale_exponent(amax, KEY ? KEY_EXP : 0));
        if (old > now) now = old;
        inv = 1.0f / now;                                        // exact: a power of two, at most 2^126
    }
    const float quantum = inv / unit;
    if (b.from == 0) {
        if (lane == 0) *scale = poisoned ? __uint_as_float(0x7FFFFFFFu) : now;
        if (b.first > 0 && (poisoned || now != old)) {           // the earlier tokens of the block, under the new scale
            const float ratio = poisoned ? 0.0f : old * inv;
#pragma unroll 1
            for (int t = sub; t < b.first; t += 2) {
                uint2 *at = reinterpret_cast<uint2 *>(dst + t * kKv8Dim + c * 8);
                const uint2 codes = *at;
                uint32_t v[2] = {codes.x, codes.y};
#pragma unroll
                for (int j = 0; j < 2; ++j)
                    v[j] = poisoned ? 0u
                                    : e4m3x4(e4m3_value(v[j] & 0xFFu) * ratio, e4m3_value((v[j] >> 8) & 0xFFu) * ratio,
                                             e4m3_value((v[j] >> 16) & 0xFFu) * ratio, e4m3_value(v[j] >> 24) * ratio);
                *at = make_uint2(v[0], v[1]);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
        const int t = b.from + 2 * i + sub, r = b.first_row + t;
        if (t >= b.n || r < 0 || r >= p.b.total_new) continue;
        uint2 codes = make_uint2(0u, 0u);
        if (!poisoned)
            codes = make_uint2(e4m3x4(x[i][0] * quantum, x[i][1] * quantum, x[i][2] * quantum, x[i][3] * quantum),
                               e4m3x4(x[i][4] * quantum, x[i][5] * quantum, x[i][6] * quantum, x[i][7] * quantum));
        *reinterpret_cast<uint2 *>(dst + (b.first + t) * kKv8Dim + c * 8) = codes;
    }
}

__global__ void __launch_bounds__(THREADS, CTAS) kv8_append_kernel(const __grid_constant__ AppendParams p) {
    __shared__ double2 angles[kKv8Group * HALF];                 // cos, sin
    __shared__ uint32_t shared_max[2][THREADS / 32];
    pdl_launch_dependents();
    pdl_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    // CTA i takes block i of the batch, where sequence s has its blocks from cu_new[s] / 16 + 2 s on: n tokens touch at most
    // n / 16 + 2 blocks, so this bound needs no pass over the lengths.
    const int *cu = p.b.cu_new;
    const int seq = warp_last_not_above(p.b.num_seqs, (long long)blockIdx.x, [&](int s) { return (long long)(cu[s] >> 4) + 2LL * s; });
    if (seq < 0) return;
    const int row0 = cu[seq], n_new = cu[seq + 1] - row0;
    const int len = p.b.seq_lens[seq];
    const int start = len - n_new;                               // position of the sequence's first new token
    const int group = (start >> 4) + ((int)blockIdx.x - (row0 >> 4) - 2 * seq);
    if (n_new <= 0 || len <= 0 || (uint32_t)group >= 1u << 27) return;           // before the first position, or behind the last there is
    const int pos = max(start, group * kKv8Group);               // first new token in this block
    const int n = min(len - group * kKv8Group, kKv8Group) - (pos - group * kKv8Group);
    if (n <= 0) return;
    // tokens that were in the block before: with a start inside the block they are the places below `first`
    Part part = {row0 + (pos - start), n, pos & (kKv8Group - 1), 0};

    auto find_angles = [&](double unit) {
#pragma unroll 1                     // two at once take registers from the rest: 28.4 us instead of 27.9
        for (int i = threadIdx.x; i < n * HALF; i += THREADS) {
            const double turn = (double)(pos + i / HALF) * p.turns[i % HALF];
            double s, c;
            sincospi(2.0 * (turn - rint(turn)), &s, &c);
            angles[angle_at(i / HALF, i % HALF)] = make_double2(c * unit, s * unit);
        }
        __syncthreads();
    };
    uint4 w[STEPS];
    if (blockIdx.y == 0) {
        // Tasks: head, K or V; K has all the arithmetic, so they are dealt out in turn.
        const bool shared = n > 2 * STEPS;
        const int units = shared ? THREADS / 64 : THREADS / 32, heads = p.b.kv_heads;
        int task = shared ? warp >> 1 : warp;
        if (shared) part.from = (warp & 1) * 2 * STEPS;
        auto is_value = [&](int i) { return (i ^ (i / units)) & 1; };
        if (task < 2 * heads) load_rows(p, part, is_value(task), task >> 1, w);  // on their way under the angles
        find_angles(KEY_UNIT);
        for (int round = 0; task < 2 * heads; task += units, ++round) {
            const long long row = kv8_group_row(p.b, seq, task >> 1, group);
            volatile uint32_t *max_here = shared ? shared_max[round & 1] : nullptr;
            if (is_value(task)) quantise_head<false>(p, part, row, w, angles, max_here);
            else quantise_head<true>(p, part, row, w, angles, max_here);
            if (task + units < 2 * heads) load_rows(p, part, is_value(task + units), (task + units) >> 1, w);
        }
        return;
    }
    // Queries: half a warp per token with its angles in registers, several tokens' share of the heads each where the block has few
    // tokens.  Nothing is decided by comparison here: 32-bit arithmetic on rounded angles.
    const int c = lane & 15, half_warp = warp * 2 + (lane >> 4);
    const int t = half_warp % n, at = part.first_row + t, shares = THREADS / 16 / n, share = half_warp / n;
    const bool there = share < shares && at >= 0 && at < p.b.total_new;
    const int end = min(p.b.q_heads, (int)blockIdx.y * QUERY_HEADS);
    int head = ((int)blockIdx.y - 1) * QUERY_HEADS + share;
    const __nv_bfloat16 *from = p.query + (long long)at * p.ldq + c * 8;
    __nv_bfloat16 *to = p.query_out + (long long)at * p.ldqo + c * 8;
    auto load_heads = [&](int first) {
#pragma unroll
        for (int u = 0; u < STEPS; ++u) {
            const int h = first + u * shares;
            w[u] = make_uint4(0u, 0u, 0u, 0u);
            if (there && h < end) w[u] = *reinterpret_cast<const uint4 *>(from + (size_t)h * kKv8Dim);
        }
    };
    load_heads(head);
    find_angles(1.0);
    const bool rotated = p.turns[0] != 0.0;                      // else as they are: 0 * inf is not 0, and -0 + 0 not -0
    float2 cs[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const double2 a = angles[t * HALF + j * 8 + (c & 7)];
        cs[j] = make_float2((float)a.x, c < 8 ? -(float)a.y : (float)a.y);
    }
    for (int first = head - share; first < end; first += STEPS * shares, head += STEPS * shares) {          // the same for a whole warp
        uint4 y[STEPS];
#pragma unroll
        for (int u = 0; u < STEPS; ++u) {
            uint32_t own[4] = {w[u].x, w[u].y, w[u].z, w[u].w};
            if (rotated) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t other = __shfl_xor_sync(0xFFFFFFFFu, own[j], 8);
                    const float y0 = fmaf(bf16_lo(own[j]), cs[2 * j].x, cs[2 * j].y * bf16_lo(other));
                    const float y1 = fmaf(bf16_hi(own[j]), cs[2 * j + 1].x, cs[2 * j + 1].y * bf16_hi(other));
                    const __nv_bfloat162 b = __floats2bfloat162_rn(y0, y1);
                    own[j] = *reinterpret_cast<const uint32_t *>(&b);
                }
            }
            y[u] = make_uint4(own[0], own[1], own[2], own[3]);
        }
        load_heads(head + STEPS * shares);
#pragma unroll
        for (int u = 0; u < STEPS; ++u) {
            const int h = head + u * shares;
            if (there && h < end) *reinterpret_cast<uint4 *>(to + (size_t)h * kKv8Dim) = y[u];
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
    thread_local double known = -1.0, turns[HALF];
    if (theta != known) {
        for (int d = 0; d < HALF; ++d) turns[d] = theta > 0.0 ? pow(theta, -(double)d / HALF) / 6.283185307179586476925 : 0.0;
        known = theta;
    }
    memcpy(p.turns, turns, sizeof(turns));
    static PerDevice<bool> configured;
    const cudaError_t ready = once_per_device(configured, [] { return cudaFuncSetAttribute(kv8_append_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)SPREAD); });
    if (ready != cudaSuccess) return false;
    const long long blocks = (long long)b.total_new / 16 + 2LL * b.num_seqs;
    const int parts = query != nullptr ? 1 + (b.q_heads + QUERY_HEADS - 1) / QUERY_HEADS : 1;
    // Where three would go to an SM while another has one, the slowest SM counts: two at most, if about that many have work
    // (7 sequences of 33 to 601 tokens: 8.8 us instead of 11.0; forced on 10000 tokens it costs 34.8 us instead of 27.9).
    const bool few = ((long long)b.total_new / 16 + b.num_seqs) * parts <= 2LL * num_sms();
    return launch_chained(kv8_append_kernel, dim3((unsigned)blocks, (unsigned)parts), dim3(THREADS), few ? SPREAD : 0, st, p) == cudaSuccess;
}

}  // namespace glmasr
