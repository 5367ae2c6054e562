// Attention of a few queries per sequence over the 8-bit paged cache: decode steps and drafted tokens.
//
// Such a call reads every visible byte of the cache once and has 4 * rows multiply-adds for it, so the bound is HBM; what has to be
// kept off its way is the work per byte.  The cache goes to the tensor cores as it lies in memory, as the 128-row operand, and the
// queries are the narrow one:
//   S^T [128 tokens, rows] = K Q^T,    O^T [128 dims, rows] += V^T P^T      (tcgen05, e4m3 x e4m3, sums in fp32)
// so no code is ever converted and no thread touches a key or a value.  (Warp-level products of the same formulas on converted
// codes took 450 instructions per 32 tokens and warp, and 29 us where this kernel takes TIME_256 us for 256 sequences of 200 to 450 tokens.)
//   queries  A row is taken times a power of two that brings its largest element to 2^7 and split into two e4m3 numbers,
//            q = hi + 2^-5 lo, side by side as columns: a bf16 number has 8 bits, each of them carries 4, so the split is exact for
//            elements down to 2^-14 of the largest, and off by 2^-22 of the largest below.
//   weights  2^(x_j - m) v_scale_j, x_j the score in log2, spans more than 8 bits have, so the accumulator has a reference of its own
//            beside the running maximum m of the softmax: W, the running maximum of x_j + log2 v_scale_j.  The weight
//            2^(x_j + log2 v_scale_j - W + 6), at most 2^8, is split as p = hi + 2^-4 lo: off by 6.6e-4 of its size (rms; bf16: 1.6e-3) or 2^-20
//            of the largest, whichever is more.
//   lazily   m and W are touched when a term has grown past 2^8 m or 2^2 W: an ordinary tile needs one vote of its four warps.
//   split    All visible groups of 16 tokens of all (sequence, kv head) pairs form one line, cut into equal pieces, one per CTA:
//            uneven lengths cost nothing.  A piece that ends inside a context leaves m, W, the sum and the accumulator in the
//            workspace, and a second launch joins those.
// A CTA walks its piece context by context in tiles of up to eight groups: warp 4 copies (a TMA box of 2 KB per group, K or V; the
// groups of a tile may lie anywhere), warp 5 issues the products, warp 6 prepares the queries of the next context, warps 0-3 are the
// softmax, one thread per token, and write the results.
#include <cuda_fp16.h>
#include <math.h>

#include "kv8_attention.cuh"
#include "ptx.cuh"
#include "runtime.cuh"

namespace glmasr {

__device__ int g_kv8_status[4];

namespace {

constexpr int SOFTMAX = 128;                                  // threads; also tokens of a tile and lanes of tensor memory
constexpr int THREADS = SOFTMAX + 96;
constexpr int TILE_GROUPS = SOFTMAX / kKv8Group;
constexpr int GROUP_BYTES = kKv8Group * kKv8Dim;
constexpr int TILE_BYTES = TILE_GROUPS * GROUP_BYTES;         // 16 KB of K, or V
constexpr int MAX_SEQS = 4096;                                // the line's table lies in shared memory
constexpr float kNothing = -3.4028234664e38f;                 // m and W before the first term: every term is above it, and 2^(it - m) is 0
constexpr float kTop = 8.0f, kWeightTop = 2.0f, kWeightBase = 6.0f;
constexpr float kQLo = 1.0f / 32.0f, kPLo = 1.0f / 16.0f;

enum : int { B_KFULL = 0, B_KEMPTY = 2, B_VFULL = 4, B_SFULL = 6, B_PFULL = 8, B_PVDONE = 10, B_QFULL = 12, B_QEMPTY = 14, B_OFREE = 16, B_COUNT = 17 };

// Shared memory; R = query rows of a context.
template <int R>
struct Smem {
    uint8_t k[2][TILE_BYTES], v[2][TILE_BYTES];
    uint8_t q[2][2 * R * kKv8Dim];        // B operand of S^T: rows hi, then lo
    uint8_t p[2][2 * R * SOFTMAX];        // B operand of O^T: rows hi, then lo
    float qscale[2][R];                   // softmax scale * log2(e) / the power of two in the row's queries
    float top[R], wtop[R];
    float red[4][R][2], factor[R][2];
    float2 scales[2][TILE_GROUPS];        // K, V
    int tokens[2][TILE_GROUPS];           // of each group that exist
    unsigned long long bars[B_COUNT];
    uint32_t tmem;
    int abort, warp_sum[8];
    int prefix[1];                        // num_seqs entries: units before each sequence
};

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
// Whether any of the softmax threads says so (and a barrier among them).
__device__ __forceinline__ bool any_of_softmax(bool x) {
    uint32_t r;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.u32 p, %1, 0;\n\t"
        "barrier.cta.red.or.pred q, 1, 128, p;\n\t"
        "selp.u32 %0, 1, 0, q;\n\t}"
        : "=r"(r) : "r"(x ? 1u : 0u) : "memory");
    return r != 0;
}
// byte b (0..127) of row r of an operand with 128-byte rows under the 128-byte swizzle
__device__ __forceinline__ uint32_t swizzled(int r, int b) { return (uint32_t)(r * 128 + ((((b >> 4) ^ (r & 7)) << 4) | (b & 15))); }

// The line of work.  rows = query rows (new token, head of the group) a context has at most; a sequence with more of them has
// several row tiles.  Unit = one visible group of 16 tokens (or the one empty unit of a context in which nothing is visible) of
// (sequence, row tile, kv head), in that order.
struct SeqWork {
    int row0, n, len, start, tiles;   // first packed row, new tokens, tokens in all, position of the first new one, row tiles
    Kv8Span span;                     // what any of its queries sees
    int units;                        // per (row tile, kv head)
};
__device__ __forceinline__ SeqWork seq_work(const Kv8Attend &a, int s, int rows) {
    SeqWork w;
    w.row0 = a.b.cu_new[s];
    const int end = a.b.cu_new[s + 1];
    w.len = a.b.seq_lens[s];
    w.n = w.row0 < 0 ? 0 : max(0, min(end, a.b.total_new) - w.row0);
    w.start = w.len - (end - w.row0);
    w.tiles = (w.n * a.group + rows - 1) / rows;
    w.span = kv8_span(a, w.len, w.start, w.len - 1);
    w.units = max(1, w.span.count);
    return w;
}
// A context of a piece: the row tile and kv head that unit `at` belongs to, and its groups [from, to) in the piece.
struct Context {
    SeqWork w;
    int seq, head, row_tile;
    int unit0, unit1;                 // its units on the line
    int from, to;                     // its groups in this piece, of w.span.count
    __device__ __forceinline__ int tiles() const { return (to - from + TILE_GROUPS - 1) / TILE_GROUPS; }
};
__device__ __forceinline__ Context context_at(const Kv8Attend &a, const int *prefix, int rows, int seq, int at, int end) {
    Context c;
    while (seq + 1 < a.b.num_seqs && prefix[seq + 1] <= at) ++seq;
    c.seq = seq;
    c.w = seq_work(a, seq, rows);
    const int x = (at - prefix[seq]) / c.w.units;
    c.unit0 = prefix[seq] + x * c.w.units;
    c.unit1 = c.unit0 + c.w.units;
    c.row_tile = a.b.by_kv_heads.div(x);
    c.head = x - c.row_tile * a.b.kv_heads;
    c.from = min(at - c.unit0, c.w.span.count);
    c.to = min(min(end, c.unit1) - c.unit0, c.w.span.count);
    return c;
}

struct Partial {                  // workspace layout
    float4 *stats;                // [2 * CTAs][rows]: m, sum, W, -
    float *acc;                   // [2 * CTAs][rows][128]
    int *prefix;                  // [num_seqs + 2]: units before each sequence, units in all, units per CTA
};
inline size_t partial_bytes(int ctas, int rows, int num_seqs, void *base, Partial *out) {
    size_t off = 0;
    auto take = [&](size_t bytes) {
        const size_t at = off;
        off = (off + bytes + 255) & ~(size_t)255;
        return (char *)base + at;
    };
    char *stats = take((size_t)2 * ctas * rows * sizeof(float4));
    char *acc = take((size_t)2 * ctas * rows * kKv8Dim * sizeof(float));
    char *prefix = take((size_t)(num_seqs + 2) * sizeof(int));
    if (out != nullptr) out->stats = (float4 *)stats, out->acc = (float *)acc, out->prefix = (int *)prefix;
    return off;
}

struct Params {
    CUtensorMap tm_k, tm_v;       // [groups * 16 rows][128 bytes], boxes of 16 rows
    Kv8Attend a;
    Partial part;
    int min_units;
};

template <int R>
__global__ void __launch_bounds__(THREADS, R == 8 ? 3 : 2) kv8_attend_kernel(const __grid_constant__ Params p) {
    constexpr int N = 2 * R;                                  // columns of both products
    constexpr int TMEM_COLS = 3 * N <= 64 ? 64 : 3 * N <= 128 ? 128 : 256;     // two score buffers, the accumulator
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    Smem<R> &sm = *reinterpret_cast<Smem<R> *>(smem_raw);
    const Kv8Attend &a = p.a;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t sbase = smem_u32(smem_raw);
    auto bar = [&](int i) { return smem_u32(&sm.bars[i]); };
    if ((sbase & 1023u) != 0) {                               // the swizzled tiles need a 1024-byte aligned base
        if (threadIdx.x == 0) atomicCAS(&g_kv8_status[0], 0, ST_BAD_LAYOUT);
        return;
    }
    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(bar(B_KFULL + i), 1);
            mbar_init(bar(B_KEMPTY + i), 1);
            mbar_init(bar(B_VFULL + i), 1);
            mbar_init(bar(B_SFULL + i), 1);
            mbar_init(bar(B_PFULL + i), SOFTMAX);
            mbar_init(bar(B_PVDONE + i), 1);
            mbar_init(bar(B_QFULL + i), 1);
            mbar_init(bar(B_QEMPTY + i), 1 + SOFTMAX);        // the last product and the last look at the scales
        }
        mbar_init(bar(B_OFREE), SOFTMAX);
        sm.abort = 0;
        fence_mbar_init();
        tma_prefetch_desc(&p.tm_k);
        tma_prefetch_desc(&p.tm_v);
    }
    if (warp == 5) {
        tmem_alloc(smem_u32(&sm.tmem), TMEM_COLS);
        tmem_relinquish();
    }
    pdl_wait();
    pdl_launch_dependents();          // after the wait: the join may look at the batch before its own

    // ---- units before each sequence: two sequences of a thread at a time, their loads together ----
    constexpr int EACH = 2;
    int carry = 0;
    for (int s0 = 0; s0 < a.b.num_seqs; s0 += THREADS * EACH) {
        const int s = s0 + (int)threadIdx.x * EACH;
        int mine[EACH], sum = 0;
#pragma unroll
        for (int e = 0; e < EACH; ++e) {
            mine[e] = 0;
            if (s + e < a.b.num_seqs) {
                const SeqWork w = seq_work(a, s + e, R);
                mine[e] = w.units * w.tiles * a.b.kv_heads;
            }
            sum += mine[e];
        }
        const int own_sum = sum;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int up = __shfl_up_sync(0xFFFFFFFFu, sum, d);
            if (lane >= d) sum += up;
        }
        if (lane == 31) sm.warp_sum[warp] = sum;
        __syncthreads();
        int before = carry + sum - own_sum;
#pragma unroll
        for (int w = 0; w < THREADS / 32; ++w) {
            if (w < warp) before += sm.warp_sum[w];
            carry += sm.warp_sum[w];
        }
#pragma unroll
        for (int e = 0; e < EACH; ++e)
            if (s + e < a.b.num_seqs) {
                sm.prefix[s + e] = before;
                before += mine[e];
            }
        __syncthreads();
    }
    const int total = carry;
    const int quota = max(p.min_units, (total + (int)gridDim.x - 1) / (int)gridDim.x);
    if (blockIdx.x == 0) {
        for (int s = threadIdx.x; s < a.b.num_seqs; s += THREADS) p.part.prefix[s] = sm.prefix[s];
        if (threadIdx.x == 0) p.part.prefix[a.b.num_seqs] = total, p.part.prefix[a.b.num_seqs + 1] = quota;
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t *>(&sm.tmem);
    const long long begin_l = (long long)blockIdx.x * quota;
    const int begin = (int)min(begin_l, (long long)total), end = (int)min((long long)total, begin_l + quota);
    volatile int *abort_word = &sm.abort;
    int seq0 = 0;                     // the sequence of the first unit
    {
        int hi = a.b.num_seqs;
        while (hi - seq0 > 1) {
            const int mid = (seq0 + hi) >> 1;
            if (sm.prefix[mid] <= begin) seq0 = mid;
            else hi = mid;
        }
    }

    if (warp == 4) {
        // ================================ copies ================================
        const bool leader = elect_one();
        uint32_t t = 0;               // tiles started
        bool ok = true;
        int seq = seq0;
        for (int at = begin; ok && at < end;) {
            const Context c = context_at(a, sm.prefix, R, seq, at, end);
            seq = c.seq;
            at = min(end, c.unit1);
            // groups of a tile by lane; those of the next tile are looked up while this one's copies run
            auto look_up = [&](int g, int &place, int &tokens, float2 &scale) {
                place = -1, tokens = 0;
                scale = make_float2(0.0f, 0.0f);
                if (lane < TILE_GROUPS && g + lane < c.to) {
                    const int group = c.w.span.group_of(g + lane);
                    const long long row = kv8_group_row(a.b, c.seq, c.head, group);
                    if (row >= 0) {
                        place = (int)(row / kKv8Group);
                        tokens = min(kKv8Group, c.w.len - group * kKv8Group);
                        scale = make_float2(a.k_scale[place], a.v_scale[place]);
                    }
                }
            };
            int place, tokens;
            float2 scale;
            look_up(c.from, place, tokens, scale);
            for (int g = c.from; g < c.to; g += TILE_GROUPS, ++t) {
                const int s = (int)(t & 1u);
                const uint32_t free_phase = ((t >> 1) & 1u) ^ 1u;
                const uint32_t there = __ballot_sync(0xFFFFFFFFu, place >= 0);
                const uint32_t bytes = (uint32_t)__popc(there) * GROUP_BYTES;
                if (!mbar_wait_warp(bar(B_KEMPTY + s), free_phase, abort_word, ST_TIMEOUT_ATTENTION)) { ok = false; break; }
                if (leader) mbar_expect_tx(bar(B_KFULL + s), bytes);
                __syncwarp();
                if (place >= 0) tma_load_2d(smem_u32(sm.k[s]) + lane * GROUP_BYTES, &p.tm_k, bar(B_KFULL + s), 0, place * kKv8Group);
                if (!mbar_wait_warp(bar(B_PVDONE + s), free_phase, abort_word, ST_TIMEOUT_ATTENTION)) { ok = false; break; }
                if (lane < TILE_GROUPS) {
                    sm.scales[s][lane] = scale;
                    sm.tokens[s][lane] = tokens;
                }
                __syncwarp();
                if (leader) mbar_expect_tx(bar(B_VFULL + s), bytes);
                __syncwarp();
                if (place >= 0) tma_load_2d(smem_u32(sm.v[s]) + lane * GROUP_BYTES, &p.tm_v, bar(B_VFULL + s), 0, place * kKv8Group);
                look_up(g + TILE_GROUPS, place, tokens, scale);
            }
        }
    } else if (warp == 5) {
        // ================================ products ==============================
        const bool leader = elect_one();
        constexpr uint32_t idesc_s = idesc_e4m3(128, N);
        constexpr uint32_t idesc_o = idesc_e4m3(128, N) | kIdescAMnMajor;
        const uint32_t t_o = tmem + 2 * N;
        uint32_t t = 0, contexts = 0;
        bool ok = true;
        int seq = seq0;
        // O^T of tile u: `steps` of 32 tokens; the first tile of a context overwrites the accumulator once the last result has been read
        auto weigh = [&](uint32_t u, int steps, bool first) {
            const int s = (int)(u & 1u);
            const uint32_t ph = (u >> 1) & 1u;
            if (!mbar_wait_warp(bar(B_VFULL + s), ph, abort_word, ST_TIMEOUT_ATTENTION)) return false;
            if (!mbar_wait_warp(bar(B_PFULL + s), ph, abort_word, ST_TIMEOUT_ATTENTION)) return false;
            if (first && !mbar_wait_warp(bar(B_OFREE), ((contexts - 1) & 1u) ^ 1u, abort_word, ST_TIMEOUT_ATTENTION)) return false;
            tc_fence_after();
            if (leader) {
                const uint64_t ad = smem_desc_sw128_mn(smem_u32(sm.v[s]), TILE_BYTES), bd = smem_desc_sw128(smem_u32(sm.p[s]));
                for (int k = 0; k < steps; ++k)
                    umma_f8(t_o, ad + (uint64_t)((k * 4096) >> 4), bd + (uint64_t)((k * 32) >> 4), idesc_o, !first || k > 0 ? 1u : 0u);
                umma_commit(bar(B_PVDONE + s));
            }
            __syncwarp();
            return true;
        };
        for (int at = begin; ok && at < end;) {
            const Context c = context_at(a, sm.prefix, R, seq, at, end);
            seq = c.seq;
            at = min(end, c.unit1);
            const int n = c.tiles();
            if (n == 0) continue;
            const int qs = (int)(contexts & 1u);
            if (!mbar_wait_warp(bar(B_QFULL + qs), (contexts >> 1) & 1u, abort_word, ST_TIMEOUT_ATTENTION)) break;
            ++contexts;
            for (int j = 0; j <= n; ++j) {
                if (j < n) {
                    const int s = (int)(t & 1u);
                    // the score buffer is free: the weights of two tiles ago came after its last read, and their product was issued
                    if (!mbar_wait_warp(bar(B_KFULL + s), (t >> 1) & 1u, abort_word, ST_TIMEOUT_ATTENTION)) { ok = false; break; }
                    tc_fence_after();
                    if (leader) {
                        const uint64_t ad = smem_desc_sw128(smem_u32(sm.k[s])), bd = smem_desc_sw128(smem_u32(sm.q[qs]));
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            umma_f8(tmem + (uint32_t)s * N, ad + (uint64_t)((k * 32) >> 4), bd + (uint64_t)((k * 32) >> 4), idesc_s, k > 0 ? 1u : 0u);
                        umma_commit(bar(B_KEMPTY + s));
                        umma_commit(bar(B_SFULL + s));
                        if (j == n - 1) umma_commit(bar(B_QEMPTY + qs));
                    }
                    __syncwarp();
                    ++t;
                }
                if (j >= 1) {
                    const int groups = min(TILE_GROUPS, c.to - c.from - (j - 1) * TILE_GROUPS);
                    const uint32_t u = j < n ? t - 2 : t - 1;
                    if (!weigh(u, (groups + 1) / 2, j == 1)) { ok = false; break; }
                }
            }
        }
    } else if (warp == 6) {
        // ================================ queries ===============================
        uint32_t contexts = 0;
        int seq = seq0;
        for (int at = begin; at < end;) {
            const Context c = context_at(a, sm.prefix, R, seq, at, end);
            seq = c.seq;
            at = min(end, c.unit1);
            if (c.tiles() == 0) continue;
            const int qs = (int)(contexts & 1u);
            if (!mbar_wait_warp(bar(B_QEMPTY + qs), ((contexts >> 1) & 1u) ^ 1u, abort_word, ST_TIMEOUT_ATTENTION)) break;
            ++contexts;
#pragma unroll 4
            for (int r = 0; r < R; ++r) {
                const int row = c.row_tile * R + r, tok = a.by_group.div(row);
                uint2 v = make_uint2(0u, 0u);                 // lane: dims 4 lane .. 4 lane + 3
                if (tok < c.w.n)
                    v = *reinterpret_cast<const uint2 *>(a.query + (long long)(c.w.row0 + tok) * a.ldq + (size_t)(c.head * a.group + row - tok * a.group) * kKv8Dim + lane * 4);
                uint32_t most = max(max(v.x & 0x7FFF0000u, (v.x << 16) & 0x7FFF0000u), max(v.y & 0x7FFF0000u, (v.y << 16) & 0x7FFF0000u));
                most = __reduce_max_sync(0xFFFFFFFFu, most);
                // 2^shift brings the largest element to [2^7, 2^8); a row that is not finite gets NaN scores by its scale
                const int expo = max(1, (int)(most >> 23));
                const int shift = expo == 255 ? 0 : 7 + 127 - expo;
                const float up0 = pow2(shift / 2), up1 = pow2(shift - shift / 2);
                float x0 = __uint_as_float(v.x << 16) * up0 * up1, x1 = __uint_as_float(v.x & 0xFFFF0000u) * up0 * up1;
                float x2 = __uint_as_float(v.y << 16) * up0 * up1, x3 = __uint_as_float(v.y & 0xFFFF0000u) * up0 * up1;
                const uint32_t hi0 = e4m3_split(x0, x1), hi1 = e4m3_split(x2, x3);
                *reinterpret_cast<uint32_t *>(sm.q[qs] + swizzled(r, lane * 4)) = hi0 | (hi1 << 16);
                *reinterpret_cast<uint32_t *>(sm.q[qs] + swizzled(R + r, lane * 4)) =
                    e4m3x2(x0 / kQLo, x1 / kQLo) | (e4m3x2(x2 / kQLo, x3 / kQLo) << 16);
                if (lane == 0)
                    sm.qscale[qs][r] = expo == 255 ? __int_as_float(0x7FFFFFFF) : a.scale_log2 * pow2(-(shift / 2)) * pow2(shift / 2 - shift);
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(B_QFULL + qs));
        }
    } else {
        // ================================ softmax ===============================
        const int me = (int)threadIdx.x;                      // token of the tile, lane of tensor memory, dim of the result
        const uint32_t t_lane = tmem + ((uint32_t)(warp * 32) << 16);
        const uint32_t t_o = t_lane + 2 * N;
        uint32_t t = 0, contexts = 0;
        bool ok = true;
        int seq = seq0;
        for (int at = begin; at < end;) {
            const Context c = context_at(a, sm.prefix, R, seq, at, end);
            seq = c.seq;
            const int first_unit = at;
            at = min(end, c.unit1);
            const int n = c.tiles(), qs = (int)(contexts & 1u);
            const int pos_lo = c.w.start + a.by_group.div(c.row_tile * R);
            const int pos_hi = c.w.start + min(c.w.n - 1, a.by_group.div(c.row_tile * R + R - 1));
            float sum[R];
#pragma unroll
            for (int r = 0; r < R; ++r) sum[r] = 0.0f;
            if (me < R) sm.top[me] = sm.wtop[me] = kNothing;
            if (n > 0) {
                ok = mbar_wait_warp(bar(B_QFULL + qs), (contexts >> 1) & 1u, abort_word, ST_TIMEOUT_ATTENTION);
                ++contexts;
            }
            if (any_of_softmax(!ok)) { ok = false; break; }
            for (int j = 0; j < n; ++j, ++t) {
                const int s = (int)(t & 1u);
                const uint32_t ph = (t >> 1) & 1u;
                ok = mbar_wait_warp(bar(B_VFULL + s), ph, abort_word, ST_TIMEOUT_ATTENTION);
                ok = ok && mbar_wait_warp(bar(B_SFULL + s), ph, abort_word, ST_TIMEOUT_ATTENTION);
                // the weights of two tiles ago have been read
                ok = ok && mbar_wait_warp(bar(B_PVDONE + s), ph ^ 1u, abort_word, ST_TIMEOUT_ATTENTION);
                tc_fence_after();
                const int g = c.from + j * TILE_GROUPS + me / kKv8Group;
                const bool there = me % kKv8Group < sm.tokens[s][me / kKv8Group];
                const int tok = c.w.span.group_of(g) * kKv8Group + me % kKv8Group;
                const float2 sc = sm.scales[s][me / kKv8Group];
                const float vs = lg2(sc.y);
                const bool all = there && tok <= pos_lo && (a.window == 0 || pos_hi - tok < a.window || tok < a.sinks);
                float x[R];
#pragma unroll
                for (int r0 = 0; r0 < R; r0 += 8) {
                    uint32_t hi[8], lo[8];
                    tmem_ld_x8(t_lane + (uint32_t)(s * N + r0), hi);
                    tmem_ld_x8(t_lane + (uint32_t)(s * N + R + r0), lo);
                    tmem_ld_wait();
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        x[r0 + e] = fmaf(__uint_as_float(lo[e]), kQLo, __uint_as_float(hi[e])) * (sm.qscale[qs][r0 + e] * sc.x);
                }
                if (!all) {
#pragma unroll
                    for (int r = 0; r < R; ++r)
                        if (!there || !kv8_sees(a, c.w.start + a.by_group.div(c.row_tile * R + r), tok)) x[r] = -INFINITY;
                }
                bool grown = !ok;
#pragma unroll
                for (int r = 0; r < R; ++r) grown = grown || x[r] > fminf(sm.top[r] + kTop, sm.wtop[r] + kWeightTop - vs);
                if (any_of_softmax(grown)) {
                    // the maxima over the tile's tokens: order-preserving integers within a warp, shared memory between the warps
#pragma unroll
                    for (int r = 0; r < R; ++r) {
                        const int m = __float_as_int(fmaxf(x[r], kNothing)), w = __float_as_int(fmaxf(x[r] + vs, kNothing));
                        const int mm = __reduce_max_sync(0xFFFFFFFFu, m ^ ((m >> 31) & 0x7FFFFFFF)), ww = __reduce_max_sync(0xFFFFFFFFu, w ^ ((w >> 31) & 0x7FFFFFFF));
                        if (lane == 0) {
                            sm.red[warp][r][0] = __int_as_float(mm ^ ((mm >> 31) & 0x7FFFFFFF));
                            sm.red[warp][r][1] = __int_as_float(ww ^ ((ww >> 31) & 0x7FFFFFFF));
                        }
                    }
                    // the accumulator is expressed against the new W: the product before has to be complete
                    if (j > 0) ok = ok && mbar_wait_warp(bar(B_PVDONE + (s ^ 1)), ((t - 1) >> 1) & 1u, abort_word, ST_TIMEOUT_ATTENTION);
                    if (any_of_softmax(!ok)) { ok = false; break; }
                    if (me < R) {
                        const float m = fmaxf(fmaxf(fmaxf(sm.red[0][me][0], sm.red[1][me][0]), fmaxf(sm.red[2][me][0], sm.red[3][me][0])), sm.top[me]);
                        const float w = fmaxf(fmaxf(fmaxf(sm.red[0][me][1], sm.red[1][me][1]), fmaxf(sm.red[2][me][1], sm.red[3][me][1])), sm.wtop[me]);
                        sm.factor[me][0] = ex2(sm.top[me] - m);
                        sm.factor[me][1] = ex2(sm.wtop[me] - w);
                        sm.top[me] = m;
                        sm.wtop[me] = w;
                    }
                    if (any_of_softmax(false)) {}
#pragma unroll
                    for (int r = 0; r < R; ++r) sum[r] *= sm.factor[r][0];
                    if (j > 0) {
                        tc_fence_after();
#pragma unroll
                        for (int r0 = 0; r0 < N; r0 += 8) {
                            uint32_t o[8];
                            tmem_ld_x8(t_o + (uint32_t)r0, o);
                            tmem_ld_wait();
#pragma unroll
                            for (int e = 0; e < 8; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * sm.factor[(r0 + e) % R][1]);
                            tmem_st_x8(t_o + (uint32_t)r0, o);
                        }
                        tmem_st_wait();
                    }
                }
                const uint32_t pb = smem_u32(sm.p[s]);
#pragma unroll
                for (int r = 0; r < R; r += 2) {
                    float w[2];
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        sum[r + e] += ex2(x[r + e] - sm.top[r + e]);
                        // a token that is not seen weighs 0 whatever its block's scale is
                        w[e] = !all && x[r + e] == -INFINITY ? 0.0f : ex2(x[r + e] + (vs + kWeightBase - sm.wtop[r + e]));
                    }
                    const uint32_t hi = e4m3_split(w[0], w[1]);
                    const uint32_t lo = e4m3x2(w[0] / kPLo, w[1] / kPLo);
                    asm volatile("st.shared.u8 [%0], %1;" ::"r"(pb + swizzled(r, me)), "r"(hi & 0xFFu) : "memory");
                    asm volatile("st.shared.u8 [%0], %1;" ::"r"(pb + swizzled(r + 1, me)), "r"(hi >> 8) : "memory");
                    asm volatile("st.shared.u8 [%0], %1;" ::"r"(pb + swizzled(R + r, me)), "r"(lo & 0xFFu) : "memory");
                    asm volatile("st.shared.u8 [%0], %1;" ::"r"(pb + swizzled(R + r + 1, me)), "r"(lo >> 8) : "memory");
                }
                // a token that does not exist weighs 0, but what lies in its place may be anything, and 0 * NaN is not 0
                if (!there) {
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(smem_u32(sm.v[s]) + me * kKv8Dim + i * 16), "r"(0) : "memory");
                }
                fence_proxy_async_smem();
                tc_fence_before();
                mbar_arrive(bar(B_PFULL + s));
            }
            if (!ok) break;
            if (n > 0) mbar_arrive(bar(B_QEMPTY + qs));

            // ---- the result of these groups ----
            if (n > 0) ok = mbar_wait_warp(bar(B_PVDONE + (int)((t - 1) & 1u)), ((t - 1) >> 1) & 1u, abort_word, ST_TIMEOUT_ATTENTION);
#pragma unroll
            for (int r = 0; r < R; ++r) {
                float v = sum[r];
#pragma unroll
                for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, d);
                if (lane == 0) sm.red[warp][r][0] = v;
            }
            if (any_of_softmax(!ok)) { ok = false; break; }
            tc_fence_after();
            const bool whole = first_unit == c.unit0 && at == c.unit1;
            const int slot = 2 * (int)blockIdx.x + (c.unit0 > begin ? 1 : 0);
            const int rows = min(R, c.w.n * a.group - c.row_tile * R);
#pragma unroll
            for (int r0 = 0; r0 < R; r0 += 8) {
                uint32_t hi[8], lo[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) hi[e] = lo[e] = 0u;
                if (n > 0) {
                    tmem_ld_x8(t_o + (uint32_t)r0, hi);
                    tmem_ld_x8(t_o + (uint32_t)(R + r0), lo);
                    tmem_ld_wait();
                }
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int r = r0 + e;
                    if (r >= rows) break;
                    const float o = fmaf(__uint_as_float(lo[e]), kPLo, __uint_as_float(hi[e]));
                    const float l = (sm.red[0][r][0] + sm.red[1][r][0]) + (sm.red[2][r][0] + sm.red[3][r][0]);
                    if (whole) {
                        // a row that sees nothing has the sum 0 and the result 0; a NaN sum stays one
                        const float inv = l == 0.0f ? 0.0f : ex2(sm.wtop[r] - kWeightBase - sm.top[r]) / l;
                        const int row = c.row_tile * R + r, tk = a.by_group.div(row);
                        a.out[(long long)(c.w.row0 + tk) * a.ldo + (size_t)(c.head * a.group + row - tk * a.group) * kKv8Dim + me] = __float2bfloat16(o * inv);
                    } else {
                        const size_t to = (size_t)slot * R + r;
                        p.part.acc[to * kKv8Dim + me] = o;
                        if (me == 0) p.part.stats[to] = make_float4(sm.top[r], l, sm.wtop[r] - kWeightBase, 0.0f);
                    }
                }
            }
            tc_fence_before();
            if (n > 0) mbar_arrive(bar(B_OFREE));
            if (any_of_softmax(false)) {}                     // the state in shared memory is free for the next context
        }
    }

    // ================================ teardown ==========================================
    tc_fence_before();
    __syncthreads();
    if (*abort_word != 0) {
        for (int i = 0; i < 64; ++i) __nanosleep(1000);      // let copies in flight land
        if (threadIdx.x == 0) atomicCAS(&g_kv8_status[0], 0, *abort_word);
    }
    if (warp == 5) {
        __syncwarp();
        tmem_dealloc(tmem, TMEM_COLS);
    }
}

// The terms of one row joined: each part's sum and accumulator under the larger of the two references.
struct Joined {
    float m = kNothing, l = 0.0f, w = kNothing;
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    __device__ __forceinline__ void add(const float4 &st, const float4 &x) {
        const float mn = fmaxf(m, st.x), wn = fmaxf(w, st.z);
        const float f = ex2(m == mn ? 0.0f : m - mn), fx = ex2(st.x == mn ? 0.0f : st.x - mn);
        const float h = ex2(w == wn ? 0.0f : w - wn), hx = ex2(st.z == wn ? 0.0f : st.z - wn);
        l = l * f + st.y * fx;
        o.x = o.x * h + x.x * hx, o.y = o.y * h + x.y * hx, o.z = o.z * h + x.z * hx, o.w = o.w * h + x.w * hx;
        m = mn, w = wn;
    }
};

// Contexts that several pieces share.  A CTA of eight warps takes 8 / per rows, `per` warps each: the row's parts are dealt out to
// them, every one joins its own, and the first joins those.
__global__ void __launch_bounds__(256) kv8_join_kernel(const __grid_constant__ Kv8Attend a, const Partial part, int rows, int per) {
    __shared__ float4 stats[8], acc[8][kKv8Dim / 4];
    pdl_launch_dependents();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int mine = warp % per;
    const int item = (int)blockIdx.x * (8 / per) + warp / per;
    const int token = a.by_q_heads.div(item), q_head = item - token * a.b.q_heads;
    Joined j;
    bool shared_row = token < a.b.total_new;
    int seq = -1, head = 0, r = 0;
    SeqWork w;
    if (shared_row) {
        const int *cu = a.b.cu_new;
        seq = warp_last_not_above(a.b.num_seqs + 1, (long long)token, [&](int s) { return (long long)cu[s]; });
        shared_row = seq >= 0 && seq < a.b.num_seqs;
    }
    if (shared_row) {
        w = seq_work(a, seq, rows);
        head = a.by_group.div(q_head);
        r = (token - w.row0) * a.group + q_head - head * a.group;
        shared_row = token - w.row0 < w.n;
    }
    pdl_wait();                       // the parts are there
    if (shared_row) {
        const int quota = part.prefix[a.b.num_seqs + 1];
        const int first = part.prefix[seq] + (r / rows * a.b.kv_heads + head) * w.units;
        const int w0 = first / quota, w1 = (first + w.units - 1) / quota;
        shared_row = w0 != w1;
        if (shared_row) {
#pragma unroll 4
            for (int p = w0 + mine; p <= w1; p += per) {
                const size_t at = (size_t)(2 * p + (first > p * quota ? 1 : 0)) * rows + r % rows;
                j.add(part.stats[at], *reinterpret_cast<const float4 *>(part.acc + at * kKv8Dim + lane * 4));
            }
        }
    }
    if (per > 1) {
        if (mine != 0) {
            if (lane == 0) stats[warp] = make_float4(j.m, j.l, j.w, 0.0f);
            acc[warp][lane] = j.o;
        }
        __syncthreads();
        if (mine != 0 || !shared_row) return;
        for (int p = 1; p < per; ++p) j.add(stats[warp + p], acc[warp + p][lane]);
    }
    if (!shared_row) return;
    const float inv = j.l == 0.0f ? 0.0f : ex2(j.w - j.m) / j.l;
    *reinterpret_cast<uint2 *>(a.out + (long long)token * a.ldo + (size_t)q_head * kKv8Dim + lane * 4) =
        make_uint2(pack2(j.o.x * inv, j.o.y * inv), pack2(j.o.z * inv, j.o.w * inv));
}

constexpr int kSmemPerSm = 228 * 1024, kSmemReserved = 1024;       // of an SM; taken by the system from each CTA

template <int R>
size_t smem_bytes(int num_seqs) { return sizeof(Smem<R>) + (size_t)num_seqs * sizeof(int); }
// CTAs per SM that the launch bounds and the shared memory allow
template <int R>
int ctas_per_sm(int num_seqs) {
    const int fit = (int)(kSmemPerSm / (smem_bytes<R>(num_seqs) + kSmemReserved));
    return fit < 1 ? 1 : fit > (R == 8 ? 3 : 2) ? (R == 8 ? 3 : 2) : fit;
}

template <int R>
bool launch_rows(Params &p, void *workspace, int num_seqs, cudaStream_t st, int &grid) {
    static PerDevice<bool> configured;
    const cudaError_t ready = once_per_device(configured, [] {
        const cudaError_t e = cudaFuncSetAttribute(kv8_attend_kernel<R>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem_bytes<R>(MAX_SEQS));
        if (e != cudaSuccess) return e;
        return cudaFuncSetAttribute(kv8_attend_kernel<R>, cudaFuncAttributePreferredSharedMemoryCarveout, (int)cudaSharedmemCarveoutMaxShared);
    });
    if (ready != cudaSuccess) return false;
    grid = num_sms() * ctas_per_sm<R>(num_seqs);
    partial_bytes(grid, R, num_seqs, workspace, &p.part);
    return launch_chained(kv8_attend_kernel<R>, dim3(grid), dim3(THREADS), smem_bytes<R>(num_seqs), st, p) == cudaSuccess;
}

}  // namespace

size_t kv8_attention_workspace_bytes(int num_seqs) {
    const size_t one = partial_bytes(num_sms() * 3, 8, num_seqs, nullptr, nullptr);
    const size_t more = partial_bytes(num_sms() * 2, 32, num_seqs, nullptr, nullptr);
    return one > more ? one : more;
}

bool kv8_attention_launch(const Kv8Attend &a, int max_new, int max_len, void *workspace, cudaStream_t st, int &launches) {
    if (a.b.num_seqs > MAX_SEQS) return false;
    const long long want = (long long)max_new * a.group;
    const int rows = want <= 8 ? 8 : want <= 16 ? 16 : 32;
    // units are counted in 32 bits
    const long long groups = (long long)a.b.max_blocks * a.b.block_size / kKv8Group + 1;
    const long long most = ((long long)a.b.total_new * a.group / rows + a.b.num_seqs) * a.b.kv_heads;
    if (most > 0x7FFFFFFFLL / groups) return false;
    Params p;
    memset(&p, 0, sizeof(p));
    const uint64_t pool_rows = (uint64_t)a.b.num_blocks * a.b.kv_heads * a.b.block_size;
    if (!make_u8_tmap_sw128(&p.tm_k, a.k_cache, kKv8Dim, pool_rows, kKv8Dim, kKv8Dim, kKv8Group)) return false;
    if (!make_u8_tmap_sw128(&p.tm_v, a.v_cache, kKv8Dim, pool_rows, kKv8Dim, kKv8Dim, kKv8Group)) return false;
    p.a = a;
    p.min_units = 4;
    int grid = 0;
    bool ok = false;
    switch (rows) {
        case 8: ok = launch_rows<8>(p, workspace, a.b.num_seqs, st, grid); break;
        case 16: ok = launch_rows<16>(p, workspace, a.b.num_seqs, st, grid); break;
        default: ok = launch_rows<32>(p, workspace, a.b.num_seqs, st, grid); break;
    }
    if (!ok) return false;
    // warps per row of the join: about four parts for each, as many parts as there are CTAs for a context
    const long long parts = (long long)grid / ((long long)a.b.num_seqs * a.b.kv_heads);
    const int per = parts <= 4 ? 1 : parts <= 8 ? 2 : parts <= 16 ? 4 : 8;
    const long long items = (long long)a.b.total_new * a.b.q_heads;
    const long long ctas = (items + 8 / per - 1) / (8 / per);
    if (launch_chained(kv8_join_kernel, dim3((unsigned)ctas), dim3(256), 0, st, a, p.part, rows, per) != cudaSuccess) return false;
    launches = 2;
    return true;
}

int kv8_take_status() {
    int code[4] = {0, 0, 0, 0};
    if (cudaMemcpyFromSymbol(code, g_kv8_status, sizeof(code)) != cudaSuccess) return -1;
    if (code[0] != 0) {
        const int zero[4] = {0, 0, 0, 0};
        (void)cudaMemcpyToSymbol(g_kv8_status, zero, sizeof(zero));
    }
    return code[0];
}

}  // namespace glmasr
