// Attention of a few queries per sequence over the 8-bit paged cache: decode steps and drafted tokens.
//
// One decode step reads every cached byte once and does 4 * group multiply-adds with it, so the bound is HBM.  What has to be kept
// off its way is the work per byte: the codes become bf16 by moving bits, and the tensor cores get the CACHE as their 16-row operand and the
// queries as the 8-column one (S^T = K Q^T, O^T = V^T P^T): a group of 4 or 8 query heads fills the tile, where queries
// as rows would leave half of it or more empty.
//
//   bits     An e4m3 code's seven low bits are the top of a bf16 number's exponent and mantissa, 2^120 too small.  The queries are taken times
//            2^64 and so are the weights of V, and 2^56 is left for the scores' factor and the end: no code is ever multiplied.
//   K        ldmatrix gives a lane four consecutive codes of a token; their even and odd ones are the two halves of an A operand whose
//            k index runs over the dims in another order, and the queries are laid out in that order.
//   V        ldmatrix.trans gives a lane two dims of two tokens; even and odd codes are rows g and g + 8 of V^T.
//   scores   the running maximum is only touched when a score has grown past 2^8 times the value the weights are expressed
//            against, so that an ordinary step needs one vote and no shuffle.
//   split    All visible groups of 16 tokens of all (sequence, head) pairs form one line, cut into equal pieces, one per warp:
//            uneven lengths cost nothing.  A piece that ends inside a context leaves its maximum, sum and accumulator in the
//            workspace, and a second launch joins those.  A warp stages its groups through its own ring of cp.async copies (4 KB each) and
//            never waits for another warp.
#include <math.h>

#include "kv8_attention.cuh"
#include "ptx.cuh"
#include "runtime.cuh"

namespace glmasr {

namespace {

constexpr int WARPS = 4;
constexpr int STAGES = 4;
constexpr int TILE_BYTES = kKv8Group * kKv8Dim;               // 2 KB: 16 tokens of one head, K or V
constexpr int WARP_SMEM = STAGES * 2 * TILE_BYTES;
constexpr int MAX_SEQS = 4096;                                // the line's table lies in shared memory
constexpr float kLazy = 8.0f;                                 // log2

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    const __nv_bfloat162 b = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&b);
}
// codes 0 and 2 / 1 and 3 of a word as bf16 pairs, times 2^-120
__device__ __forceinline__ uint32_t even_codes(uint32_t w) { return ((w & 0x007F007Fu) << 4) | ((w & 0x00800080u) << 8); }
__device__ __forceinline__ uint32_t odd_codes(uint32_t w) { return ((w >> 4) & 0x07F007F0u) | (w & 0x80008000u); }

__device__ __forceinline__ void ldsm_x4(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ void ldsm_x4_trans(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ void mma_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// 16-byte chunk c (0..7) of token r of a tile; the chunks of a row are permuted so that ldmatrix meets every bank once
__device__ __forceinline__ uint32_t tile_at(int r, int c) { return (uint32_t)(r * kKv8Dim + ((c ^ (r & 7)) << 4)); }

// The line of work.  rows = query rows (new token, head of the group) a warp takes at once; a sequence with more of them has
// several row tiles.  Unit = one visible group of 16 tokens (or the one empty unit of a context in which nothing is visible) of
// (sequence, row tile, kv head), in that order.
struct SeqWork {
    int row0, n, start, tiles;    // first packed row, new tokens, position of the first, row tiles
    Kv8Span span;                 // what any of its queries sees
    int units;                    // per (row tile, kv head)
};
__device__ __forceinline__ SeqWork seq_work(const Kv8Attend &a, int s, int rows) {
    SeqWork w;
    w.row0 = a.b.cu_new[s];
    w.n = max(0, min(a.b.cu_new[s + 1], a.b.total_new) - max(0, w.row0));
    if (w.row0 < 0) w.n = 0;
    const int len = a.b.seq_lens[s];
    w.start = len - (a.b.cu_new[s + 1] - w.row0);
    w.tiles = (int)(((long long)w.n * a.group + rows - 1) / rows);
    w.span = kv8_span(a, len, w.start, len - 1);
    w.units = max(1, w.span.count);
    return w;
}

struct Partial {                  // workspace layout
    float *stats;                 // [2 * warps][rows][2]: maximum (log2 domain), sum
    float *acc;                   // [2 * warps][rows][128], 2^-56 of the accumulator
    int *prefix;                  // [num_seqs + 2]: units before each sequence, units in all, units per warp
};
__host__ __device__ inline size_t partial_bytes(int warps, int rows, int num_seqs, void *base, Partial *out) {
    size_t off = 0;
    auto take = [&](size_t bytes) {
        const size_t at = off;
        off = (off + bytes + 255) & ~(size_t)255;
        return (char *)base + at;
    };
    char *stats = take((size_t)2 * warps * rows * 2 * sizeof(float));
    char *acc = take((size_t)2 * warps * rows * kKv8Dim * sizeof(float));
    char *prefix = take((size_t)(num_seqs + 2) * sizeof(int));
    if (out != nullptr) out->stats = (float *)stats, out->acc = (float *)acc, out->prefix = (int *)prefix;
    return off;
}

// NT = row tiles of eight query rows
template <int NT>
__global__ void __launch_bounds__(WARPS * 32, NT == 1 ? 3 : 2) kv8_attend_kernel(const __grid_constant__ Kv8Attend a, const Partial part, int min_units) {
    constexpr int ROWS = NT * 8;
    extern __shared__ __align__(1024) uint8_t smem[];
    __shared__ int warp_sum[WARPS];
    int *prefix = reinterpret_cast<int *>(smem + WARPS * WARP_SMEM);
    pdl_launch_dependents();
    pdl_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = lane >> 2, tq = lane & 3;

    // ---- units before each sequence ----
    int carry = 0;
    for (int s0 = 0; s0 < a.b.num_seqs; s0 += WARPS * 32) {
        const int s = s0 + threadIdx.x;
        int mine = 0;
        if (s < a.b.num_seqs) {
            const SeqWork w = seq_work(a, s, ROWS);
            mine = w.units * w.tiles * a.b.kv_heads;
        }
        int sum = mine;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int up = __shfl_up_sync(0xFFFFFFFFu, sum, d);
            if (lane >= d) sum += up;
        }
        if (lane == 31) warp_sum[warp] = sum;
        __syncthreads();
        int before = carry, all = 0;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
            if (w < warp) before += warp_sum[w];
            all += warp_sum[w];
        }
        if (s < a.b.num_seqs) prefix[s] = before + sum - mine;
        carry += all;
        __syncthreads();
    }
    const int total = carry;
    const int workers = (int)gridDim.x * WARPS;
    const int quota = max(min_units, (total + workers - 1) / workers);
    if (blockIdx.x == 0) {
        for (int s = threadIdx.x; s < a.b.num_seqs; s += WARPS * 32) part.prefix[s] = prefix[s];
        if (threadIdx.x == 0) part.prefix[a.b.num_seqs] = total, part.prefix[a.b.num_seqs + 1] = quota;
    }
    __syncthreads();

    const int worker = warp * (int)gridDim.x + (int)blockIdx.x;      // the first pieces go to different SMs
    const long long begin_l = (long long)worker * quota;
    if (begin_l >= total) return;
    const int begin = (int)begin_l, end = min(total, begin + quota);
    const uint32_t ring = smem_u32(smem) + (uint32_t)warp * WARP_SMEM;

    // ---- units of this piece, 32 at a time, one per lane: where its codes are, and its scales ----
    long long l_row = -1;             // first row of codes (128 bytes each), -1: nothing to see
    float l_ks = 0.0f, l_vs = 0.0f;
    long long n_row = -1;
    float n_ks = 0.0f, n_vs = 0.0f;
    auto resolve = [&](int unit, long long &row, float &ks, float &vs) {
        row = -1;
        ks = vs = 0.0f;
        if (unit >= end) return;
        int lo = 0, hi = a.b.num_seqs;                                // prefix[lo] <= unit < prefix[hi]
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (prefix[mid] <= unit) lo = mid;
            else hi = mid;
        }
        const SeqWork w = seq_work(a, lo, ROWS);
        if (w.span.count == 0) return;
        const int x = unit - prefix[lo];
        const int head = (x / w.units) % a.b.kv_heads;
        row = kv8_group_row(a.b, lo, head, w.span.group_of(x % w.units));
        if (row >= 0) {
            ks = a.k_scale[row / kKv8Group];
            vs = a.v_scale[row / kKv8Group];
        }
    };
    resolve(begin + lane, l_row, l_ks, l_vs);
    if (begin + 32 < end) resolve(begin + 32 + lane, n_row, n_ks, n_vs);

    auto load = [&](int i) {          // unit begin + i of this piece into its slot
        const long long row = __shfl_sync(0xFFFFFFFFu, ((i >> 5) & 1) ? n_row : l_row, i & 31);
        if (row < 0) return;
        const uint32_t dst = ring + (uint32_t)(i % STAGES) * (2 * TILE_BYTES);
        const size_t off = (size_t)row * kKv8Dim + (size_t)(lane >> 3) * kKv8Dim + (size_t)(lane & 7) * 16;
#pragma unroll
        for (int j = 0; j < 4; ++j) {                                 // four tokens per step, eight lanes each
            const uint32_t at = tile_at(j * 4 + (lane >> 3), lane & 7);
            cp_async16_zfill(dst + at, a.k_cache + off + j * 4 * kKv8Dim, true);
            cp_async16_zfill(dst + TILE_BYTES + at, a.v_cache + off + j * 4 * kKv8Dim, true);
        }
    };
    const int count = end - begin;
#pragma unroll
    for (int i = 0; i < STAGES - 1; ++i) {
        if (i < count) load(i);
        cp_async_commit();
    }

    // ---- the context this piece is in ----
    int seq = 0, unit0 = 0;           // its sequence; first unit of the (row tile, kv head)
    SeqWork w;
    int head = 0, row_tile = 0;
    int pos[NT][2];                   // positions of this lane's query rows 8 nt + 2 tq and + 1; -1: no such row
    int pos_lo = 0, pos_hi = 0;       // over all rows of the tile
    uint32_t qb[NT][8][2];
    float acc[NT][8][4], base[NT][2], top[NT][2], sum[NT][2];
    auto enter = [&](int unit) {
        while (seq + 1 < a.b.num_seqs && prefix[seq + 1] <= unit) ++seq;
        w = seq_work(a, seq, ROWS);
        const int x = (unit - prefix[seq]) / w.units;
        unit0 = prefix[seq] + x * w.units;
        head = x % a.b.kv_heads;
        row_tile = x / a.b.kv_heads;
        pos_lo = 0x7FFFFFFF, pos_hi = -1;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int t = (row_tile * ROWS + nt * 8 + tq * 2 + e) / a.group;
                pos[nt][e] = t < w.n ? w.start + t : -1;
                base[nt][e] = 0.0f;
                top[nt][e] = -INFINITY;
                sum[nt][e] = 0.0f;
            }
            // the B operand's column is row 8 nt + g
            const int r = row_tile * ROWS + nt * 8 + g;
            const int t = r / a.group;
            const bool there = t < w.n;
            const __nv_bfloat16 *q = a.query + (long long)(w.row0 + (there ? t : 0)) * a.ldq + (size_t)(head * a.group + r - t * a.group) * kKv8Dim + tq * 4;
#pragma unroll
            for (int c = 0; c < 8; ++c) {
                uint2 v = make_uint2(0u, 0u);
                if (there) v = *reinterpret_cast<const uint2 *>(q + c * 16);
                const float x0 = __uint_as_float(v.x << 16) * 0x1p64f, x1 = __uint_as_float(v.x & 0xFFFF0000u) * 0x1p64f;
                const float x2 = __uint_as_float(v.y << 16) * 0x1p64f, x3 = __uint_as_float(v.y & 0xFFFF0000u) * 0x1p64f;
                qb[nt][c][0] = pack2(x0, x2);
                qb[nt][c][1] = pack2(x1, x3);
            }
#pragma unroll
            for (int c = 0; c < 8; ++c) acc[nt][c][0] = acc[nt][c][1] = acc[nt][c][2] = acc[nt][c][3] = 0.0f;
        }
        const int t0 = row_tile * ROWS / a.group, t1 = min(w.n - 1, (row_tile * ROWS + ROWS - 1) / a.group);
        pos_lo = w.start + t0, pos_hi = w.start + t1;
    };
    // the result of units [from, to) of the present context
    auto leave = [&](int from, int to) {
        const bool whole = from == unit0 && to == unit0 + w.units;
        const int slot = 2 * worker + (unit0 > begin ? 1 : 0);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float s = sum[nt][e];
                s += __shfl_xor_sync(0xFFFFFFFFu, s, 4);
                s += __shfl_xor_sync(0xFFFFFFFFu, s, 8);
                s += __shfl_xor_sync(0xFFFFFFFFu, s, 16);
                const int r_in = nt * 8 + tq * 2 + e;
                const int r = row_tile * ROWS + r_in;
                const int t = r / a.group;
                if (t >= w.n) continue;
                if (whole) {
                    // a row that sees nothing has the sum 0 and the result 0; a NaN sum stays one
                    const float inv = s == 0.0f ? 0.0f : 0x1p56f / s;
                    __nv_bfloat16 *o = a.out + (long long)(w.row0 + t) * a.ldo + (size_t)(head * a.group + r - t * a.group) * kKv8Dim + g * 2;
#pragma unroll
                    for (int c = 0; c < 8; ++c)
                        *reinterpret_cast<uint32_t *>(o + c * 16) = pack2(acc[nt][c][e] * inv, acc[nt][c][2 + e] * inv);
                } else {
                    const size_t at = (size_t)slot * ROWS + r_in;
                    if (g == 0) *reinterpret_cast<float2 *>(part.stats + at * 2) = make_float2(top[nt][e], s);
                    float *o = part.acc + at * kKv8Dim + g * 2;
#pragma unroll
                    for (int c = 0; c < 8; ++c) *reinterpret_cast<float2 *>(o + c * 16) = make_float2(acc[nt][c][e], acc[nt][c][2 + e]);
                }
            }
        }
    };
    enter(begin);
    int from = begin;

    const float f0 = a.scale_log2 * 0x1p56f;
    for (int i = 0; i < count; ++i) {
        const int unit = begin + i;
        if (i + STAGES - 1 < count) load(i + STAGES - 1);
        cp_async_commit();
        if (unit >= unit0 + w.units) {
            leave(from, unit);
            enter(unit);
            from = unit;
        }
        const bool second = ((i >> 5) & 1) != 0;
        const long long row = __shfl_sync(0xFFFFFFFFu, second ? n_row : l_row, i & 31);
        const float ks = __shfl_sync(0xFFFFFFFFu, second ? n_ks : l_ks, i & 31) * f0;
        const float vs = __shfl_sync(0xFFFFFFFFu, second ? n_vs : l_vs, i & 31) * 0x1p64f;
        // the 32 units just finished make room for those after the next 32 (load() looks STAGES - 1 units ahead, into the others)
        if ((i & 31) == 31) {
            if (second) resolve(begin + i + 33 + lane, n_row, n_ks, n_vs);
            else resolve(begin + i + 33 + lane, l_row, l_ks, l_vs);
        }
        cp_async_wait<STAGES - 1>();
        __syncwarp();
        if (row >= 0) {
            const uint32_t kt = ring + (uint32_t)(i % STAGES) * (2 * TILE_BYTES), vt = kt + TILE_BYTES;
            float s[NT][4];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.0f;
#pragma unroll
            for (int c = 0; c < 8; c += 2) {
                uint32_t k[4];       // tokens 0-7 and 8-15 of chunk c, then of chunk c + 1
                ldsm_x4(kt + tile_at(lane & 15, c + (lane >> 4)), k);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint32_t a0 = even_codes(k[2 * h]), a1 = even_codes(k[2 * h + 1]), a2 = odd_codes(k[2 * h]), a3 = odd_codes(k[2 * h + 1]);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) mma_16816(s[nt], a0, a1, a2, a3, qb[nt][c + h][0], qb[nt][c + h][1]);
                }
            }
            // lane: tokens g and g + 8 (s[.][0..1] and s[.][2..3]) of rows 2 tq and 2 tq + 1
            const int tok0 = w.span.group_of(unit - unit0) * kKv8Group;
            const bool all = tok0 + kKv8Group - 1 <= pos_lo && (a.window == 0 || pos_hi - tok0 < a.window || tok0 + kKv8Group <= a.sinks);
            bool grown = false;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float x = s[nt][e] * ks;
                    if (!all && !kv8_sees(a, pos[nt][e & 1], tok0 + g + (e >> 1) * 8)) x = -INFINITY;
                    s[nt][e] = x;
                    grown = grown || x > top[nt][e & 1] + kLazy;
                }
            if (__any_sync(0xFFFFFFFFu, grown)) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float m = fmaxf(top[nt][e], fmaxf(s[nt][e], s[nt][2 + e]));
                        m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, 4));
                        m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, 8));
                        m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, 16));
                        const float alpha = top[nt][e] == -INFINITY ? 0.0f : ex2(top[nt][e] - m);
                        top[nt][e] = m;
                        base[nt][e] = m == -INFINITY ? 0.0f : m;
                        if (sum[nt][e] != 0.0f) sum[nt][e] *= alpha;
#pragma unroll
                        for (int c = 0; c < 8; ++c) {
                            acc[nt][c][e] *= alpha;
                            acc[nt][c][2 + e] *= alpha;
                        }
                    }
            }
            uint32_t pb[NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                float p[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    p[e] = ex2(s[nt][e] - base[nt][e & 1]);
                    sum[nt][e & 1] += p[e];
                    // a token that is not seen weighs 0 whatever its block's scale is
                    p[e] = !all && s[nt][e] == -INFINITY ? 0.0f : p[e] * vs;
                }
                pb[nt][0] = transpose_8x8(pack2(p[0], p[1]));
                pb[nt][1] = transpose_8x8(pack2(p[2], p[3]));
            }
#pragma unroll
            for (int c = 0; c < 8; c += 2) {
                uint32_t v[4];       // tokens 0-7 and 8-15 of chunk c, then of chunk c + 1
                ldsm_x4_trans(vt + tile_at(lane & 15, c + (lane >> 4)), v);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint32_t a0 = even_codes(v[2 * h]), a1 = odd_codes(v[2 * h]), a2 = even_codes(v[2 * h + 1]), a3 = odd_codes(v[2 * h + 1]);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) mma_16816(acc[nt][c + h], a0, a1, a2, a3, pb[nt][0], pb[nt][1]);
                }
            }
        }
        __syncwarp();                 // every lane is done with the slot before it is filled again
    }
    leave(from, end);
    cp_async_wait<0>();
}

// Contexts that several pieces share.  A CTA of eight warps takes 8 / per rows, `per` warps each: the row's parts are dealt out to
// them, every one joins its own, and the first joins those.
__global__ void __launch_bounds__(256) kv8_join_kernel(const __grid_constant__ Kv8Attend a, const Partial part, int rows, int per) {
    __shared__ float joined[8][2 + kKv8Dim];
    pdl_launch_dependents();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int mine = warp % per;
    const long long item = (long long)blockIdx.x * (8 / per) + warp / per;
    pdl_wait();
    const int token = (int)(item / a.b.q_heads), q_head = (int)(item % a.b.q_heads);
    bool shared_row = item < (long long)a.b.total_new * a.b.q_heads;
    float m = -INFINITY, l = 0.0f;
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (shared_row) {
        const int *cu = a.b.cu_new;
        const int seq = warp_last_not_above(a.b.num_seqs + 1, (long long)token, [&](int s) { return (long long)cu[s]; });
        shared_row = seq >= 0 && seq < a.b.num_seqs;
        if (shared_row) {
            const SeqWork w = seq_work(a, seq, rows);
            const int head = q_head / a.group;
            const int r = (token - w.row0) * a.group + q_head % a.group;
            const int quota = part.prefix[a.b.num_seqs + 1];
            const int first = part.prefix[seq] + ((r / rows) * a.b.kv_heads + head) * w.units;
            const int w0 = first / quota, w1 = (first + w.units - 1) / quota;
            shared_row = w0 != w1 && token - w.row0 < w.n;
            if (shared_row) {
                for (int p = w0 + mine; p <= w1; p += per) {
                    const size_t at = (size_t)(2 * p + (first > p * quota ? 1 : 0)) * rows + r % rows;
                    const float2 st = *reinterpret_cast<const float2 *>(part.stats + at * 2);
                    const float4 x = *reinterpret_cast<const float4 *>(part.acc + at * kKv8Dim + lane * 4);
                    const float mn = fmaxf(m, st.x);
                    const float f = m == -INFINITY ? 0.0f : ex2(m - mn), fx = st.x == -INFINITY ? (st.y == 0.0f ? 0.0f : 1.0f) : ex2(st.x - mn);
                    m = mn;
                    l = (l == 0.0f ? 0.0f : l * f) + st.y * fx;
                    o.x = o.x * f + x.x * fx, o.y = o.y * f + x.y * fx, o.z = o.z * f + x.z * fx, o.w = o.w * f + x.w * fx;
                }
            }
        }
    }
    if (per > 1) {
        if (mine != 0) {
            if (lane == 0) joined[warp][0] = m, joined[warp][1] = l;
            joined[warp][2 + lane * 4] = o.x, joined[warp][3 + lane * 4] = o.y, joined[warp][4 + lane * 4] = o.z, joined[warp][5 + lane * 4] = o.w;
        }
        __syncthreads();
        if (mine != 0 || !shared_row) return;
        for (int p = 1; p < per; ++p) {
            const float *x = joined[warp + p];
            const float mn = fmaxf(m, x[0]);
            const float f = m == -INFINITY ? 0.0f : ex2(m - mn), fx = x[0] == -INFINITY ? (x[1] == 0.0f ? 0.0f : 1.0f) : ex2(x[0] - mn);
            m = mn;
            l = (l == 0.0f ? 0.0f : l * f) + x[1] * fx;
            o.x = o.x * f + x[2 + lane * 4] * fx, o.y = o.y * f + x[3 + lane * 4] * fx;
            o.z = o.z * f + x[4 + lane * 4] * fx, o.w = o.w * f + x[5 + lane * 4] * fx;
        }
    }
    if (!shared_row) return;
    const float inv = l == 0.0f ? 0.0f : 0x1p56f / l;
    *reinterpret_cast<uint2 *>(a.out + (long long)token * a.ldo + (size_t)q_head * kKv8Dim + lane * 4) =
        make_uint2(pack2(o.x * inv, o.y * inv), pack2(o.z * inv, o.w * inv));
}

template <int NT>
bool launch_rows(const Kv8Attend &a, const Partial &part, int grid, size_t smem, int min_units, cudaStream_t st) {
    static PerDevice<bool> configured;
    const cudaError_t ready = once_per_device(configured, [] {
        const cudaError_t e = cudaFuncSetAttribute(kv8_attend_kernel<NT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                   WARPS * WARP_SMEM + MAX_SEQS * (int)sizeof(int));
        if (e != cudaSuccess) return e;
        return cudaFuncSetAttribute(kv8_attend_kernel<NT>, cudaFuncAttributePreferredSharedMemoryCarveout, (int)cudaSharedmemCarveoutMaxShared);
    });
    if (ready != cudaSuccess) return false;
    return launch_chained(kv8_attend_kernel<NT>, dim3(grid), dim3(WARPS * 32), smem, st, a, part, min_units) == cudaSuccess;
}

constexpr int CTAS_PER_SM = 3;

}  // namespace

size_t kv8_attention_workspace_bytes(int num_seqs) {
    const size_t one = partial_bytes(num_sms() * CTAS_PER_SM * WARPS, 8, num_seqs, nullptr, nullptr);
    const size_t more = partial_bytes(num_sms() * 2 * WARPS, 32, num_seqs, nullptr, nullptr);
    return one > more ? one : more;
}

bool kv8_attention_launch(const Kv8Attend &a, int max_new, int max_len, void *workspace, cudaStream_t st, int &launches) {
    if (a.b.num_seqs > MAX_SEQS) return false;
    const long long want = (long long)max_new * a.group;
    const int nt = want <= 8 ? 1 : want <= 16 ? 2 : want <= 24 ? 3 : 4;
    const int rows = nt * 8;
    // units are counted in 32 bits
    const long long tiles = (long long)a.b.max_blocks * a.b.block_size / kKv8Group + 1;
    const long long most = ((long long)a.b.total_new * a.group / rows + a.b.num_seqs) * a.b.kv_heads;
    if (most > 0x7FFFFFFFLL / tiles) return false;
    const int grid = num_sms() * (nt == 1 ? CTAS_PER_SM : 2);
    Partial part;
    partial_bytes(grid * WARPS, rows, a.b.num_seqs, workspace, &part);
    const size_t smem = (size_t)WARPS * WARP_SMEM + (size_t)a.b.num_seqs * sizeof(int);
    const int min_units = 2;
    bool ok = false;
    switch (nt) {
        case 1: ok = launch_rows<1>(a, part, grid, smem, min_units, st); break;
        case 2: ok = launch_rows<2>(a, part, grid, smem, min_units, st); break;
        case 3: ok = launch_rows<3>(a, part, grid, smem, min_units, st); break;
        default: ok = launch_rows<4>(a, part, grid, smem, min_units, st); break;
    }
    if (!ok) return false;
    const int per = 8;
    const long long items = (long long)a.b.total_new * a.b.q_heads;
    const long long ctas = (items + 8 / per - 1) / (8 / per);
    if (launch_chained(kv8_join_kernel, dim3((unsigned)ctas), dim3(256), 0, st, a, part, rows, per) != cudaSuccess) return false;
    launches = 2;
    return true;
}

}  // namespace glmasr
