// Attention of a few queries per sequence over the 8-bit paged cache: decode steps and drafted tokens.
//
// Such a call reads every visible byte of the cache once and has 4 * rows multiply-adds for it, so the bound is HBM; what has to be
// kept off its way is the work per byte.  The cache goes to the tensor cores as it lies in memory, as the 128-row operand, and the
// queries are the narrow one:
//   S^T [128 tokens, rows] = K Q^T,    O^T [128 dims, rows] += V^T P^T      (tcgen05, e4m3 x e4m3, sums in fp32)
// so no code is ever converted and no thread touches a key or a value.  (Warp-level products of the same formulas on converted
// codes took 450 instructions per 32 tokens and warp, and 29 us where this kernel takes 24.7 us for 256 sequences of 200 to 450 tokens.)
//   queries  A row is taken times a power of two that brings its largest element to 2^7 and split into two e4m3 numbers,
//            q = hi + 2^-5 lo, side by side as columns: a bf16 number has 8 bits, each of them carries 4, so the split is exact for
//            elements down to 2^-14 of the largest, and off by 2^-22 of the largest below.
//   weights  2^(x_j - m) v_scale_j, x_j the score in log2, spans more than 8 bits have, so the accumulator has a reference of its own
//            beside the running maximum m of the softmax: W, the running maximum of x_j + log2 v_scale_j.  The weight
//            2^(x_j + log2 v_scale_j - W + 12), at most 2^14, is rounded to f16, whose upper byte is an e5m2 number: that byte, the upper byte of
//            8 times what it leaves, and of 8 times what is left then, side by side as columns: p = hi + 2^-3 mid + 2^-6 lo.  That is off by 2^-9
//            of the weight, or 2^-35 of the largest, whichever is more: a long tail of small weights beside one token that has
//            nearly all of it, with little V, is what counts then.  (Two e4m3 numbers per weight end at 2^-20 of the largest: 5000
//            weights of 2^-20.6 beside one came out 26% short.)
//   lazily   m and W are touched when a term has grown past 2^8 m or 2^2 W: an ordinary tile needs one vote of the softmax's warps.
//   split    Two ways to deal out the work, chosen on the host (see deal_whole()).  Whole: one CTA of the grid for each (sequence, kv
//            head); those that run take over the work of those that have not started, and there is nothing to join.  Pieces: all
//            visible groups of 16 tokens of all (sequence, kv head) pairs form one line, cut into equal pieces, one per CTA, so that
//            uneven lengths cost little; a piece that ends inside a context leaves m, W, the sum and the accumulator in the
//            workspace, and a second launch joins those.
// A CTA walks its piece context by context in tiles of up to eight groups: one warp copies (a TMA box of 2 KB per group, K or V; the
// groups of a tile may lie anywhere), prepares the queries of the next context and says where its results go, one issues the
// products, and the others are the softmax and write the results: a thread per token, or two where there are more than 8 rows, each
// with half of them (64 sequences of 200 to 2000 tokens with 8 new ones, 32 rows: 50 us instead of 54).
// K and V have two buffers each.  A tile's chain of waits, products and softmax is about 2000 cycles, and a copy takes as long: three
// CTAs with 64 KB of tiles each keep HBM busy.  (Four with one buffer of each: every copy waits for a product, 4000 cycles a tile.)
#include <math.h>

#include "kv8_attention.cuh"
#include "ptx.cuh"
#include "runtime.cuh"

namespace glmasr {

static __device__ int g_kv8_status[4];

namespace {

constexpr int SOFTMAX = 128;                                  // tokens of a tile, lanes of tensor memory
// Softmax threads of a token, each of which has as many of the rows; then two more warps.
constexpr int split(int rows) { return rows <= 8 ? 1 : 2; }
constexpr int threads(int rows) { return split(rows) * SOFTMAX + 64; }
constexpr int TILE_GROUPS = SOFTMAX / kKv8Group;
constexpr int GROUP_BYTES = kKv8Group * kKv8Dim;
constexpr int TILE_BYTES = TILE_GROUPS * GROUP_BYTES;         // 16 KB of K, or V
constexpr int MAX_SEQS = 4096;                                // the line's table lies in shared memory
constexpr float kTop = 8.0f, kWeightTop = 2.0f, kWeightBase = 12.0f;
constexpr float kQLo = 1.0f / 32.0f, kPMid = 1.0f / 8.0f, kPLo = 1.0f / 64.0f;
constexpr int PARTS = 3;                                      // numbers per weight
constexpr int weight_columns(int used) { return (PARTS * used + 15) / 16 * 16; }

enum : int { B_KFULL = 0, B_KEMPTY = 2, B_VFULL = 4, B_PVDONE = 6, B_SFULL = 8, B_SCALES = 10, B_CFULL = 12, B_CEMPTY = 14, B_PFULL = 16, B_OFREE = 17, B_NEXT = 18, B_FIRST = 19, B_COUNT = 20 };

// What the products and the softmax have to know of a context.
template <int R>
struct ContextInfo {
    int groups;                           // in this piece; 0: the piece is done
    int rows;                             // query rows that exist
    int first, sink, from;                // group i of the piece is group first + i of the context; Kv8Span
    int pos_lo, pos_hi;                   // positions of its queries
    int slot;                             // of its parts in the workspace; -1: it is whole
    float qscale[R];                      // softmax scale * log2(e) / the power of two in the row's queries
    int pos[R];
    __nv_bfloat16 *out[R];
};
// Shared memory; R = query rows of a context as the scores have them, U those that the weights have.
template <int R, int U>
struct Smem {
    uint8_t k[2][TILE_BYTES], v[2][TILE_BYTES];
    uint8_t q[2][2 * R * kKv8Dim];        // B operand of S^T: rows hi, then lo
    uint8_t p[weight_columns(U) * SOFTMAX];   // B operand of O^T: per 16 columns (rows hi, then mid, then lo) 16 bytes of each token
    ContextInfo<R> ctx[2];
    float4 row[R];                        // m + kTop, W + kWeightTop, -m, kWeightBase - W
    float red[4][R][2], factor[R][2];
    float2 scales[2][TILE_GROUPS];        // K, V
    int tokens[2][TILE_GROUPS];           // of each group that exist
    uint4 next;                           // answer to the question for more work
    struct { int row0, head, first_token, start; } begin;      // whose queries the CTA's first context has: see split_row
    unsigned long long bars[B_COUNT];
    uint32_t tmem;
    int abort, warp_sum[threads(R) / 32];
    int prefix[1];                        // num_seqs entries: units before each sequence
};

// Whether any of the softmax threads says so (and a barrier among them).
template <int COUNT>
__device__ __forceinline__ bool any_of_softmax(bool x) {
    uint32_t r;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.u32 p, %1, 0;\n\t"
        "barrier.cta.red.or.pred q, 1, %2, p;\n\t"
        "selp.u32 %0, 1, 0, q;\n\t}"
        : "=r"(r) : "r"(x ? 1u : 0u), "n"(COUNT) : "memory");
    return r != 0;
}
// Two weights (at least 0) as f16, in the upper byte of each half: an e5m2 number, the one of 8 times the rest, and the rounded one of 8 times
// what is left of that.  All steps but the first and the last are exact.
__device__ __forceinline__ void split_weights(float a, float b, uint32_t &hi, uint32_t &mid, uint32_t &lo) {
    auto bits = [](__half2 h) { return *reinterpret_cast<const uint32_t *>(&h); };
    auto upper = [&](uint32_t w) {
        const uint32_t u = w & 0xFF00FF00u;
        return *reinterpret_cast<const __half2 *>(&u);
    };
    const __half2 eight = __float2half2_rn(8.0f), w = __floats2half2_rn(a, b);
    hi = bits(w);
    const __half2 m = __hmul2(__hsub2(w, upper(hi)), eight);
    mid = bits(m);
    lo = bits(__hmul2(__hsub2(m, upper(mid)), eight)) + 0x00800080u;
}
// Query rows are split by QL lanes each (all rows of a small tile at a time, or eight): a lane has dims 8 QL i + 8 (lane % QL) .. + 7.
constexpr int query_lanes(int rows) { return rows <= 4 ? 8 : 4; }
// Row r of context cs, which is row `row` of its sequence.
template <int QL, int R, int U>
__device__ __forceinline__ void split_row(const Kv8Attend &a, Smem<R, U> &sm, int cs, int r, bool exists, const uint4 (&q)[16 / QL], int row, int head, int first_token, int start) {
    const int part = (int)threadIdx.x % QL;
    uint32_t most = 0u;
#pragma unroll
    for (int i = 0; i < 16 / QL; ++i)
        most = __vmaxu2(most, __vmaxu2(__vmaxu2(q[i].x & 0x7FFF7FFFu, q[i].y & 0x7FFF7FFFu), __vmaxu2(q[i].z & 0x7FFF7FFFu, q[i].w & 0x7FFF7FFFu)));
#pragma unroll
    for (int d = 1; d < QL; d <<= 1) most = __vmaxu2(most, __shfl_xor_sync(0xFFFFFFFFu, most, d));
    most = max(most >> 16, most & 0xFFFFu);
    // 2^shift brings the largest element to [2^7, 2^8) (one below 2^-119 less far); a row that is not finite gets NaN scores by its scale
    const int expo = (int)(most >> 7), shift = expo == 255 ? 0 : min(7 + 127 - expo, 126);
    const float up = pow2(shift);
#pragma unroll
    for (int i = 0; i < 16 / QL; ++i) {
        const uint32_t w[4] = {q[i].x, q[i].y, q[i].z, q[i].w};
        uint32_t hi[2] = {0u, 0u}, lo[2] = {0u, 0u};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            float x0 = __uint_as_float(w[e] << 16) * up, x1 = __uint_as_float(w[e] & 0xFFFF0000u) * up;
            hi[e >> 1] |= e4m3_split(x0, x1) << (16 * (e & 1));
            lo[e >> 1] |= e4m3x2(x0 / kQLo, x1 / kQLo) << (16 * (e & 1));
        }
        const int b = i * 8 * QL + part * 8;
        *reinterpret_cast<uint2 *>(sm.q[cs] + swizzled(r, b)) = make_uint2(hi[0], hi[1]);
        *reinterpret_cast<uint2 *>(sm.q[cs] + swizzled(R + r, b)) = make_uint2(lo[0], lo[1]);
    }
    if (part == 0) {
        const int tok = a.by_group.div(row);
        ContextInfo<R> &info = sm.ctx[cs];
        info.qscale[r] = expo == 255 ? __int_as_float(0x7FFFFFFF) : a.scale_log2 * pow2(-shift);
        info.pos[r] = exists ? start + tok : -1;
        info.out[r] = a.out + (long long)(first_token + tok) * a.ldo + (size_t)(head * a.group + row - tok * a.group) * kKv8Dim;
    }
}
template <int QL>
__device__ __forceinline__ void load_row(const Kv8Attend &a, bool exists, uint4 (&q)[16 / QL], int row, int head, int first_token) {
    const int tok = a.by_group.div(row);
    const __nv_bfloat16 *src = a.query + (long long)(first_token + tok) * a.ldq + (size_t)(head * a.group + row - tok * a.group) * kKv8Dim + threadIdx.x % QL * 8;
#pragma unroll
    for (int i = 0; i < 16 / QL; ++i) q[i] = exists ? *reinterpret_cast<const uint4 *>(src + i * 8 * QL) : make_uint4(0u, 0u, 0u, 0u);
}
// V columns of tensor memory, 32 bits of this lane each
template <int V>
__device__ __forceinline__ void load_columns(uint32_t t, uint32_t (&r)[V]) {
    static_assert(V == 4 || V == 8 || V == 12 || V == 16, "columns");
    if constexpr (V >= 8) {
        if constexpr (V == 16) tmem_ld_x16(t, r);
        else tmem_ld_x8(t, *reinterpret_cast<uint32_t(*)[8]>(&r[0]));
    }
    if constexpr (V % 8 == 4) tmem_ld_x4(t + V / 8 * 8, *reinterpret_cast<uint32_t(*)[4]>(&r[V / 8 * 8]));
}
template <int V>
__device__ __forceinline__ void store_columns(uint32_t t, const uint32_t (&r)[V]) {
    if constexpr (V >= 8) {
        if constexpr (V == 16) tmem_st_x16(t, r);
        else tmem_st_x8(t, *reinterpret_cast<const uint32_t(*)[8]>(&r[0]));
    }
    if constexpr (V % 8 == 4) tmem_st_x4(t + V / 8 * 8, *reinterpret_cast<const uint32_t(*)[4]>(&r[V / 8 * 8]));
}
// The line of work.  rows = query rows (new token, head of the group) a context has at most; a sequence with more of them has
// several row tiles.  Units of (sequence, row tile, kv head), in that order: its visible groups of 16 tokens, and behind them as many
// empty ones as its last tile lacks and one more tile has, for what a context costs by itself.  (Without those a piece of
// short contexts takes twice as long as the others: 47 us instead of 29 for 19 sequences of 40 to 4450 tokens, 5 new.)
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
    w.units = (w.span.count + 2 * TILE_GROUPS - 1) / TILE_GROUPS * TILE_GROUPS;
    return w;
}
// A context of a piece: the row tile and kv head that unit `at` belongs to, and its groups [from, to) in the piece.
struct Context {
    SeqWork w;
    int seq, head, row_tile;
    int unit0, unit1, real1;          // its units on the line; those with groups (one if it has none) end at real1
    int from, to;                     // its groups in this piece, of w.span.count
};
// x / d for x >= 0, d > 0: the fp32 quotient of rounded numbers is off by 2^-22 of itself, so its floor by one below 2^22; beyond, exactly.
__device__ __forceinline__ int quotient(int x, int d) {
    if (x >= (1 << 22)) return x / d;
    int q = (int)__fdividef((float)x, (float)d);
    const int r = x - q * d;
    if (r < 0) --q;
    if (r >= d) ++q;
    return q;
}
__device__ __forceinline__ Context context_at(const Kv8Attend &a, const int *prefix, int rows, int seq, int at, int end) {
    Context c;
    while (seq + 1 < a.b.num_seqs && prefix[seq + 1] <= at) ++seq;
    c.seq = seq;
    c.w = seq_work(a, seq, rows);
    const int x = quotient(at - prefix[seq], c.w.units);
    c.unit0 = prefix[seq] + x * c.w.units;
    c.unit1 = c.unit0 + c.w.units;
    c.real1 = c.unit0 + max(1, c.w.span.count);
    c.row_tile = a.b.by_kv_heads.div(x);
    c.head = x - c.row_tile * a.b.kv_heads;
    c.from = min(at - c.unit0, c.w.span.count);
    c.to = min(min(end, c.unit1) - c.unit0, c.w.span.count);
    return c;
}

// A context that begins in a piece and ends in a later one.
struct JoinInfo {
    int last;                     // the piece it ends in; -1: there is none
    int slot;                     // of its first part; those of the others are 2 * piece
    int rows, row0, head;         // its query rows: row0 + r counts (new token, head of the group) of the sequence
    int first_token;              // packed row of the sequence's first new token
};
struct Partial {                  // workspace layout
    float4 *stats;                // [2 * CTAs][rows]: m, sum, W, -
    float *acc;                   // [2 * CTAs][rows][128]
    JoinInfo *join;               // [CTAs]: the context that begins in the CTA's piece and ends in another
};
inline size_t partial_bytes(int ctas, int rows, void *base, Partial *out) {
    size_t off = 0;
    auto take = [&](size_t bytes) {
        const size_t at = off;
        off = (off + bytes + 255) & ~(size_t)255;
        return (char *)base + at;
    };
    char *stats = take((size_t)2 * ctas * rows * sizeof(float4));
    char *acc = take((size_t)2 * ctas * rows * kKv8Dim * sizeof(float));
    char *join = take((size_t)ctas * sizeof(JoinInfo));
    if (out != nullptr) out->stats = (float4 *)stats, out->acc = (float *)acc, out->join = (JoinInfo *)join;
    return off;
}

struct Params {
    CUtensorMap tm_k, tm_v;       // [groups * 16 rows][128 bytes], boxes of 16 rows
    Kv8Attend a;
    Partial part;
    int whole;                    // how the work is dealt out
    int min_units;                // of a piece
};

// CTAs on an SM: what registers, tensor memory and the tiles allow
constexpr int max_ctas(int rows) { return rows <= 8 ? 3 : 2; }

// R = query rows of a context as the products have them, U <= R how many the softmax works on (a group of four heads fills half
// of the narrowest product).
template <int R, int U>
__global__ void __launch_bounds__(threads(R), max_ctas(R)) kv8_attend_kernel(const __grid_constant__ Params p) {
    constexpr int N = 2 * R, NP = weight_columns(U);          // columns of the two products
    constexpr int SPLIT = split(R), THREADS = threads(R), WORKERS = SPLIT * SOFTMAX, COPIES = WORKERS / 32, PRODUCTS = COPIES + 1;       // the last two: warps
    // The softmax's warps split the queries of the first context, all rows at once (19 sequences with 4 new tokens behind 300, 16 rows:
    // 12.1 -> 11.4 us).  Up to 8 rows the copying warp is as quick, and nobody has to be told (6.3 us, 6.6 for one of 60 tokens).
    constexpr bool SHARED_FIRST = U > 8;
    constexpr int TMEM_COLS = 2 * N + NP <= 64 ? 64 : 2 * N + NP <= 128 ? 128 : 256;     // two score buffers, the accumulator
    static_assert(2 * N + NP <= 256, "tensor memory of a CTA");
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    Smem<R, U> &sm = *reinterpret_cast<Smem<R, U> *>(smem_raw);
    const Kv8Attend &a = p.a;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t sbase = smem_u32(smem_raw);
    auto bar = [&](int i) { return smem_u32(&sm.bars[i]); };
    if ((sbase & 1023u) != 0) {                               // the swizzled tiles need a 1024-byte aligned base
        pdl_wait();
        if (threadIdx.x == 0) {
            atomicCAS(&g_kv8_status[0], 0, ST_BAD_LAYOUT);
            if (!p.whole) p.part.join[blockIdx.x].last = -1;      // else the join would take what lies there for work
        }
        return;
    }
    if (threadIdx.x == 0) {
        mbar_init(bar(B_PFULL), WORKERS / 32);
        mbar_init(bar(B_OFREE), WORKERS / 32);
        mbar_init(bar(B_NEXT), 1);
        mbar_init(bar(B_FIRST), 1);
        for (int i = 0; i < 2; ++i) {
            mbar_init(bar(B_KFULL + i), 1);
            mbar_init(bar(B_KEMPTY + i), 1);
            mbar_init(bar(B_VFULL + i), 1);
            mbar_init(bar(B_PVDONE + i), 1);
            mbar_init(bar(B_SFULL + i), 1);
            mbar_init(bar(B_SCALES + i), 1);
            mbar_init(bar(B_CFULL + i), 1);
            mbar_init(bar(B_CEMPTY + i), 1 + WORKERS / 32);        // the last product of scores and the results
        }
        sm.abort = 0;
        fence_mbar_init();
        tma_prefetch_desc(&p.tm_k);
        tma_prefetch_desc(&p.tm_v);
    }
    // Tensor memory is asked for, without a limit to the wait, when no earlier kernel can be about to, and later ones start when this one
    // has it: two kernels that each have a part and wait for the other cannot come about.
    pdl_wait();
    if (warp == PRODUCTS) {
        tmem_alloc(smem_u32(&sm.tmem), TMEM_COLS);
        tmem_relinquish();
    }

    // rows of the queries' operand that no row of a context fills stay zero
    if constexpr (U < R) {
        constexpr int SPARE = R - U;
        const int i = (int)threadIdx.x / 8, row = i % SPARE + U + (i / SPARE & 1 ? R : 0);
        if (i < 4 * SPARE) *reinterpret_cast<uint4 *>(sm.q[i / SPARE / 2] + row * kKv8Dim + threadIdx.x % 8 * 16) = make_uint4(0u, 0u, 0u, 0u);
        fence_proxy_async_smem();
    }
    int begin = 0, end = 0, quota = 1, seq0 = 0;          // the piece, and the sequence of its first unit
    if (!p.whole) {
        // units before each sequence: two sequences of a thread at a time, their loads together
        constexpr int EACH = 2;
        int carry = 0;
        for (int s0 = 0; s0 < a.b.num_seqs; s0 += THREADS * EACH) {
            const int s = s0 + (int)threadIdx.x * EACH;
            int mine[EACH], sum = 0;
#pragma unroll
            for (int e = 0; e < EACH; ++e) {
                mine[e] = 0;
                if (s + e < a.b.num_seqs) {
                    const SeqWork w = seq_work(a, s + e, U);
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
        quota = max(p.min_units, (carry + (int)gridDim.x - 1) / (int)gridDim.x);
        const long long at = (long long)blockIdx.x * quota;
        begin = (int)min(at, (long long)carry), end = (int)min((long long)carry, at + quota);
        int hi = a.b.num_seqs;
        while (hi - seq0 > 1) {
            const int mid = (seq0 + hi) >> 1;
            if (sm.prefix[mid] <= begin) seq0 = mid;
            else hi = mid;
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    pdl_launch_dependents();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t *>(&sm.tmem);
    volatile int *abort_word = &sm.abort;

    if (warp == COPIES) {
        // ================================ copies, queries =======================
        const bool leader = elect_one();
        uint32_t t = 0, contexts = 0; // tiles and contexts started
        bool ok = true, have = false, first = false, more = true;
        int at = begin, first_unit = begin, g = 0, rows = 0, item = -1;
        uint32_t asked = 0;           // for more work
        JoinInfo join = {-1, 0, 0, 0, 0, 0};
        Context c;
        c.seq = seq0, c.to = 0, c.row_tile = 0, c.w.tiles = 0;
        // the next context of the piece, or the next row tile of a whole (sequence, kv head), or the next one that has any
        auto next_context = [&]() {
            if (!p.whole) {
                if (at >= end) return false;
                c = context_at(a, sm.prefix, U, c.seq, at, end);
                first_unit = at;
                at = min(end, c.unit1);
                if (first_unit == c.unit0 && at < c.real1)
                    join = {(c.real1 - 1) / quota, 2 * (int)blockIdx.x + (c.unit0 > begin ? 1 : 0), 0, c.row_tile * U, c.head, c.w.row0};
            } else if (++c.row_tile >= c.w.tiles) {
                do {
                    if (item < 0) {
                        item = (int)blockIdx.x;
                    } else {
                        ok = mbar_wait_short(bar(B_NEXT), (asked - 1) & 1u, abort_word, ST_TIMEOUT_ATTENTION);
                        if (!ok) return false;
                        item = cancelled_cta(smem_u32(&sm.next));
                        if (item < 0) return false;
                        fence_proxy_async_smem();             // the answer has been read before the next one is written
                        __syncwarp();
                    }
                    if (leader) {
                        mbar_expect_tx(bar(B_NEXT), 16);
                        ask_cancelled_cta(smem_u32(&sm.next), bar(B_NEXT));
                    }
                    __syncwarp();
                    ++asked;
                    c.seq = a.b.by_kv_heads.div(item);
                    c.head = item - c.seq * a.b.kv_heads;
                    c.w = seq_work(a, c.seq, U);
                } while (c.w.tiles == 0);
                c.row_tile = c.from = 0;
                c.to = c.w.span.count;
            }
            return true;
        };
        // of the coming tile, by lane: place in the pool in groups (-1: none) and existing tokens of a group, its scales
        int place = -1, tokens = 0;
        float2 scale = make_float2(0.0f, 0.0f);
        // Queries of a context, under the tiles of the one before; the first rows are asked for when it is entered.
        constexpr int QL = query_lanes(U), QROWS = 32 / QL, QI = 16 / QL;
        uint4 q[QI];
        auto place_of = [&](int r, int &tok) {                // first element of the row's head in a packed row, and the row
            const int row = c.row_tile * U + r;
            tok = a.by_group.div(row);
            return (size_t)(c.head * a.group + row - tok * a.group) * kKv8Dim;
        };
        for (;;) {
            have = false;
            while (!have && more) {
                first = g >= c.to;
                if (first) {
                    more = next_context();
                    if (!more) break;
                    rows = min(U, c.w.n * a.group - c.row_tile * U);
                    join.rows = rows;
                    g = c.from;
                    if (!SHARED_FIRST || contexts > 0) load_row<QL>(a, lane / QL < rows, q, c.row_tile * U + lane / QL, c.head, c.w.row0);
                }
                if (g == c.to) {                              // empty units, or a context in which nothing is visible
                    if (c.w.span.count > 0 || (!p.whole && first_unit != c.unit0)) continue;
                    for (int r = 0; r < rows; ++r) {
                        int tok;
                        const size_t col = place_of(r, tok);
                        *reinterpret_cast<uint2 *>(a.out + (long long)(c.w.row0 + tok) * a.ldo + col + lane * 4) = make_uint2(0u, 0u);
                    }
                    continue;
                }
                have = true;
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
                g += TILE_GROUPS;
            }
            if (!have) break;
            const int s = (int)(t & 1u);
            const uint32_t free_phase = ((t >> 1) & 1u) ^ 1u, bytes = (uint32_t)__popc(__ballot_sync(0xFFFFFFFFu, place >= 0)) * GROUP_BYTES;
            ++t;
            ok = mbar_wait_short(bar(B_KEMPTY + s), free_phase, abort_word, ST_TIMEOUT_ATTENTION);
            if (!ok) break;
            if (leader) mbar_expect_tx(bar(B_KFULL + s), bytes);
            __syncwarp();
            if (place >= 0) tma_load_2d(smem_u32(sm.k[s]) + lane * GROUP_BYTES, &p.tm_k, bar(B_KFULL + s), 0, place * kKv8Group);
            // V, and the scales: the tile of two before, whose places they take, has to be summed
            auto put_v = [&]() {
                ok = mbar_wait_short(bar(B_PVDONE + s), free_phase, abort_word, ST_TIMEOUT_ATTENTION);
                if (!ok) return false;
                if (leader) mbar_expect_tx(bar(B_VFULL + s), bytes);
                __syncwarp();
                if (place >= 0) tma_load_2d(smem_u32(sm.v[s]) + lane * GROUP_BYTES, &p.tm_v, bar(B_VFULL + s), 0, place * kKv8Group);
                if (lane < TILE_GROUPS) {
                    sm.scales[s][lane] = scale;
                    sm.tokens[s][lane] = tokens;
                }
                __syncwarp();
                if (leader) mbar_arrive(bar(B_SCALES + s));
                __syncwarp();
                return true;
            };
            if (!first) {
                if (!put_v()) break;
                continue;
            }
            const int cs = (int)(contexts & 1u);
            ok = mbar_wait_short(bar(B_CEMPTY + cs), ((contexts >> 1) & 1u) ^ 1u, abort_word, ST_TIMEOUT_ATTENTION);
            if (!ok) break;
            ++contexts;
            ContextInfo<R> &info = sm.ctx[cs];
            if (lane == 0) {
                info.groups = c.to - c.from;
                info.rows = rows;
                info.first = c.from, info.sink = c.w.span.sink, info.from = c.w.span.from;
                info.pos_lo = c.w.start + a.by_group.div(c.row_tile * U);
                info.pos_hi = c.w.start + a.by_group.div(c.row_tile * U + rows - 1);
                info.slot = p.whole || (first_unit == c.unit0 && at >= c.real1) ? -1 : 2 * (int)blockIdx.x + (c.unit0 > begin ? 1 : 0);
            }
            __syncwarp();
            if (SHARED_FIRST && contexts == 1) {
                if (leader) {
                    sm.begin = {c.row_tile * U, c.head, c.w.row0, c.w.start};
                    mbar_arrive(bar(B_FIRST));
                }
                __syncwarp();
                if (!put_v()) break;
                continue;
            }
#pragma unroll 1
            for (int r = lane / QL; r < U; r += QROWS) {
                uint4 next[QI];
                if (r + QROWS < U) load_row<QL>(a, r + QROWS < rows, next, c.row_tile * U + r + QROWS, c.head, c.w.row0);
                split_row<QL>(a, sm, cs, r, r < rows, q, c.row_tile * U + r, c.head, c.w.row0, c.w.start);
                if (r + QROWS < U) {
#pragma unroll
                    for (int i = 0; i < QI; ++i) q[i] = next[i];
                }
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (leader) mbar_arrive(bar(B_CFULL + cs));
            if (!put_v()) break;
        }
        if (leader && !p.whole) p.part.join[blockIdx.x] = join;
        const int cs = (int)(contexts & 1u);
        if (ok && mbar_wait_short(bar(B_CEMPTY + cs), ((contexts >> 1) & 1u) ^ 1u, abort_word, ST_TIMEOUT_ATTENTION) && leader) {
            sm.ctx[cs].groups = 0;                            // the end
            mbar_arrive(bar(B_CFULL + cs));
            if (SHARED_FIRST && contexts == 0) mbar_arrive(bar(B_FIRST));
        }
    } else if (warp == PRODUCTS) {
        // ================================ products ==============================
        const bool leader = elect_one();
        constexpr uint32_t idesc_s = idesc_e4m3(128, N);
        constexpr uint32_t idesc_o = idesc_e4m3(128, NP) | kIdescBE5m2 | kIdescAMnMajor | kIdescBMnMajor;
        const uint32_t t_o = tmem + 2 * N;
        uint32_t t = 0, contexts = 0;
        bool ok = true;
        // O^T of tile u: `steps` of 32 tokens; the first tile of a context overwrites the accumulator once the last result has been read
        auto weigh = [&](uint32_t u, int steps, bool first) {
            const int s = (int)(u & 1u);
            if (!mbar_wait_short(bar(B_VFULL + s), (u >> 1) & 1u, abort_word, ST_TIMEOUT_ATTENTION)) return false;
            if (!mbar_wait_short(bar(B_PFULL), u & 1u, abort_word, ST_TIMEOUT_ATTENTION)) return false;
            if (first && !mbar_wait_short(bar(B_OFREE), ((contexts - 1) & 1u) ^ 1u, abort_word, ST_TIMEOUT_ATTENTION)) return false;
            tc_fence_after();
            if (leader) {
                const uint64_t ad = smem_desc_sw128_mn(smem_u32(sm.v[s]), TILE_BYTES), bd = smem_desc_mn(smem_u32(sm.p), 16 * SOFTMAX);
                for (int k = 0; k < steps; ++k)
                    umma_f8(t_o, ad + (uint64_t)((k * 4096) >> 4), bd + (uint64_t)((k * 512) >> 4), idesc_o, !first || k > 0 ? 1u : 0u);
                umma_commit(bar(B_PVDONE + s));
            }
            __syncwarp();
            return true;
        };
        while (ok) {
            const int cs = (int)(contexts & 1u);
            if (!mbar_wait_short(bar(B_CFULL + cs), (contexts >> 1) & 1u, abort_word, ST_TIMEOUT_ATTENTION)) break;
            const int groups_here = sm.ctx[cs].groups, n = (groups_here + TILE_GROUPS - 1) / TILE_GROUPS;
            if (n == 0) break;
            ++contexts;
            for (int j = 0; j <= n; ++j) {
                if (j < n) {
                    const int s = (int)(t & 1u);
                    // the score buffer is free: the weights of two tiles ago came after its last read, and their product was issued
                    if (!mbar_wait_short(bar(B_KFULL + s), (t >> 1) & 1u, abort_word, ST_TIMEOUT_ATTENTION)) { ok = false; break; }
                    tc_fence_after();
                    if (leader) {
                        const uint64_t ad = smem_desc_sw128(smem_u32(sm.k[s])), bd = smem_desc_sw128(smem_u32(sm.q[cs]));
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            umma_f8(tmem + (uint32_t)s * N, ad + (uint64_t)((k * 32) >> 4), bd + (uint64_t)((k * 32) >> 4), idesc_s, k > 0 ? 1u : 0u);
                        umma_commit(bar(B_KEMPTY + s));
                        umma_commit(bar(B_SFULL + s));
                        if (j == n - 1) umma_commit(bar(B_CEMPTY + cs));
                    }
                    __syncwarp();
                    ++t;
                }
                if (j >= 1) {
                    const int groups = min(TILE_GROUPS, groups_here - (j - 1) * TILE_GROUPS);
                    const uint32_t u = j < n ? t - 2 : t - 1;
                    if (!weigh(u, (groups + 1) / 2, j == 1)) { ok = false; break; }
                }
            }
        }
    } else {
        // ================================ softmax ===============================
        constexpr int V = U / SPLIT;
        const int tid = (int)threadIdx.x, me = tid % SOFTMAX;   // me: token of the tile, lane of tensor memory, dim of the result
        const int base = tid / SOFTMAX * V, quarter = warp % 4; // the first of this thread's V rows; its warp's place among those of the tokens
        const uint32_t t_lane = tmem + ((uint32_t)(quarter * 32) << 16);
        const uint32_t t_o = t_lane + 2 * N;
        if constexpr (SHARED_FIRST) {
            constexpr int QL = query_lanes(U);
            static_assert(U * QL <= WORKERS && U * QL % 32 == 0, "a row for QL lanes, whole warps");
            const bool ok = mbar_wait_short(bar(B_FIRST), 0u, abort_word, ST_TIMEOUT_ATTENTION);
            const bool any = sm.ctx[0].groups != 0;
            if (ok && any && tid < U * QL) {
                const int r = tid / QL;
                const bool exists = r < sm.ctx[0].rows;
                uint4 q[16 / QL];
                load_row<QL>(a, exists, q, sm.begin.row0 + r, sm.begin.head, sm.begin.first_token);
                split_row<QL>(a, sm, 0, r, exists, q, sm.begin.row0 + r, sm.begin.head, sm.begin.first_token, sm.begin.start);
                fence_proxy_async_smem();
            }
            if (!any_of_softmax<WORKERS>(!ok) && any && tid == 0) mbar_arrive(bar(B_CFULL));
        }
        uint32_t t = 0;
        for (uint32_t contexts = 0;; ++contexts) {
            const int cs = (int)(contexts & 1u);
            bool ok = mbar_wait_short(bar(B_CFULL + cs), (contexts >> 1) & 1u, abort_word, ST_TIMEOUT_ATTENTION);
            const ContextInfo<R> &c = sm.ctx[cs];
            const int n = (c.groups + TILE_GROUPS - 1) / TILE_GROUPS;
            const int pos_lo = c.pos_lo, pos_hi = c.pos_hi;
            float sum[V];
#pragma unroll
            for (int r = 0; r < V; ++r) sum[r] = 0.0f;
            if (tid < U) sm.row[tid] = make_float4(kNothing, kNothing, -kNothing, -kNothing);
            if (any_of_softmax<WORKERS>(!ok) || n == 0) break;
            for (int j = 0; j < n; ++j, ++t) {
                const int s = (int)(t & 1u);
                ok = mbar_wait_short(bar(B_SCALES + s), (t >> 1) & 1u, abort_word, ST_TIMEOUT_ATTENTION);
                const int in = c.first + j * TILE_GROUPS + me / kKv8Group;
                const int tok = (in < c.sink ? in : c.from + (in - c.sink)) * kKv8Group + me % kKv8Group;
                const bool there = me % kKv8Group < sm.tokens[s][me / kKv8Group];
                const float2 sc = sm.scales[s][me / kKv8Group];
                const float vs = lg2(sc.y);
                const bool all = there && tok <= pos_lo && (a.window == 0 || pos_hi - tok < a.window || tok < a.sinks);
                ok = ok && mbar_wait_short(bar(B_SFULL + s), (t >> 1) & 1u, abort_word, ST_TIMEOUT_ATTENTION);
                tc_fence_after();
                float x[V];
                uint32_t high[V], low[V];
                load_columns<V>(t_lane + (uint32_t)(s * N + base), high);
                load_columns<V>(t_lane + (uint32_t)(s * N + R + base), low);
                tmem_ld_wait();
#pragma unroll
                for (int r = 0; r < V; ++r) x[r] = fmaf(__uint_as_float(low[r]), kQLo, __uint_as_float(high[r])) * (c.qscale[base + r] * sc.x);
                if (!there) {
#pragma unroll
                    for (int r = 0; r < V; ++r) x[r] = -INFINITY;
                } else if (!all) {
                    // 0 <= p - tok < window as one comparison (a row that does not exist has the position -1)
                    const uint32_t reach = a.window == 0 || tok < a.sinks ? 0x80000000u : (uint32_t)a.window;
#pragma unroll
                    for (int r = 0; r < V; ++r)
                        if ((uint32_t)(c.pos[base + r] - tok) >= reach) x[r] = -INFINITY;
                }
                bool grown = !ok;
#pragma unroll
                for (int r = 0; r < V; ++r) {
                    const float2 top = *reinterpret_cast<const float2 *>(&sm.row[base + r].x);
                    grown = grown || x[r] > fminf(top.x, top.y - vs);
                }
                if (any_of_softmax<WORKERS>(grown)) {
#pragma unroll
                    for (int r = 0; r < V; ++r) {
                        const float m = redux_max(fmaxf(x[r], kNothing)), w = redux_max(fmaxf(x[r] + vs, kNothing));
                        if (lane == 0) *reinterpret_cast<float2 *>(sm.red[quarter][base + r]) = make_float2(m, w);
                    }
                    // the accumulator is expressed against the new W: the product before has to be complete
                    if (j > 0) ok = ok && mbar_wait_short(bar(B_PVDONE + (int)((t - 1) & 1u)), ((t - 1) >> 1) & 1u, abort_word, ST_TIMEOUT_ATTENTION);
                    if (any_of_softmax<WORKERS>(!ok)) { ok = false; break; }
                    if (tid < U) {
                        const float4 was = sm.row[tid];
                        const float m = fmaxf(fmaxf(fmaxf(sm.red[0][tid][0], sm.red[1][tid][0]), fmaxf(sm.red[2][tid][0], sm.red[3][tid][0])), -was.z);
                        const float w = fmaxf(fmaxf(fmaxf(sm.red[0][tid][1], sm.red[1][tid][1]), fmaxf(sm.red[2][tid][1], sm.red[3][tid][1])), kWeightBase - was.w);
                        sm.factor[tid][0] = ex2(-was.z - m);
                        sm.factor[tid][1] = ex2(kWeightBase - was.w - w);
                        sm.row[tid] = make_float4(m + kTop, w + kWeightTop, -m, kWeightBase - w);
                    }
                    (void)any_of_softmax<WORKERS>(false);
                    if (j > 0) {
#pragma unroll
                        for (int r = 0; r < V; ++r) sum[r] *= sm.factor[base + r][0];
                        tc_fence_after();
#pragma unroll 1
                        for (int part = 0; part < PARTS * U; part += U) {
                            uint32_t o[V];
                            load_columns<V>(t_o + (uint32_t)(part + base), o);
                            tmem_ld_wait();
#pragma unroll
                            for (int r = 0; r < V; ++r) o[r] = __float_as_uint(__uint_as_float(o[r]) * sm.factor[base + r][1]);
                            store_columns<V>(t_o + (uint32_t)(part + base), o);
                        }
                        tmem_st_wait();
                    }
                }
                uint32_t codes[PARTS][V / 4];                 // the token's weights
#pragma unroll
                for (int r = 0; r < V; r += 4) {
                    uint32_t part[PARTS][2];
#pragma unroll
                    for (int two = 0; two < 2; ++two) {
                        float w[2];
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const int i = r + 2 * two + e;
                            const float2 ref = *reinterpret_cast<const float2 *>(&sm.row[base + i].z);
                            sum[i] += ex2(x[i] + ref.x);
                            // a token that is not seen weighs 0 whatever its block's scale is
                            w[e] = !all && x[i] == -INFINITY ? 0.0f : ex2(x[i] + (vs + ref.y));
                        }
                        split_weights(w[0], w[1], part[0][two], part[1][two], part[2][two]);
                    }
#pragma unroll
                    for (int i = 0; i < PARTS; ++i) codes[i][r / 4] = __byte_perm(part[i][0], part[i][1], 0x7531);
                }
                // the weights of the tile before have been read
                ok = t == 0 || mbar_wait_short(bar(B_PVDONE + (s ^ 1)), ((t - 1) >> 1) & 1u, abort_word, ST_TIMEOUT_ATTENTION);
                // a token that does not exist weighs 0, but what lies in its place may be anything, and 0 * NaN is not 0
                if (__any_sync(0xFFFFFFFFu, !there)) {
                    ok = ok && mbar_wait_short(bar(B_VFULL + s), (t >> 1) & 1u, abort_word, ST_TIMEOUT_ATTENTION);
                    if (!there) {
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(smem_u32(sm.v[s]) + me * kKv8Dim + i * 16), "r"(0) : "memory");
                    }
                }
                if (!ok) *abort_word = ST_TIMEOUT_ATTENTION;  // said at the next vote
                const uint32_t to = smem_u32(sm.p) + me * 16;
                if constexpr (V == 4) {                       // 16 columns, the last four of which nobody reads
                    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %3};" ::"r"(to), "r"(codes[0][0]), "r"(codes[1][0]), "r"(codes[2][0]) : "memory");
                } else {
#pragma unroll
                    for (int i = 0; i < PARTS; ++i) {
#pragma unroll
                        for (int r = 0; r < V; r += V % 8 == 0 ? 8 : 4) {
                            const int at = i * U + base + r;
                            const uint32_t dst = to + (uint32_t)(at / 16 * (16 * SOFTMAX) + at % 16);
                            if constexpr (V % 8 == 0) asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(dst), "r"(codes[i][r / 4]), "r"(codes[i][r / 4 + 1]) : "memory");
                            else asm volatile("st.shared.b32 [%0], %1;" ::"r"(dst), "r"(codes[i][r / 4]) : "memory");
                        }
                    }
                }
                fence_proxy_async_smem();
                tc_fence_before();
                mbar_arrive_warp(bar(B_PFULL));
            }

            // ---- the result of these groups ----
            ok = ok && mbar_wait_short(bar(B_PVDONE + (int)((t - 1) & 1u)), ((t - 1) >> 1) & 1u, abort_word, ST_TIMEOUT_ATTENTION);
            // sums over the warp's 32 tokens: halves of the rows are exchanged until a lane has one, then the lanes that share it add up
            {
                constexpr int P2 = V <= 4 ? 4 : V <= 8 ? 8 : 16;
                float v[P2];
#pragma unroll
                for (int r = 0; r < P2; ++r) v[r] = r < V ? sum[r < V ? r : 0] : 0.0f;
                int held = P2;
#pragma unroll
                for (int d = 16; d > 0; d >>= 1) {
                    if (held > 1) {
                        held /= 2;
                        const bool upper = (lane & d) != 0;
#pragma unroll
                        for (int i = 0; i < P2 / 2; ++i)
                            if (i < held) {
                                const float give = upper ? v[i] : v[held + i], keep = upper ? v[held + i] : v[i];
                                v[i] = keep + __shfl_xor_sync(0xFFFFFFFFu, give, d);
                            }
                    } else {
                        v[0] += __shfl_xor_sync(0xFFFFFFFFu, v[0], d);
                    }
                }
                if ((lane & (32 / P2 - 1)) == 0 && lane / (32 / P2) < V) sm.red[quarter][base + lane / (32 / P2)][0] = v[0];
            }
            if (any_of_softmax<WORKERS>(!ok)) break;
            if (tid < c.rows) {
                const float l = (sm.red[0][tid][0] + sm.red[1][tid][0]) + (sm.red[2][tid][0] + sm.red[3][tid][0]);
                const float4 st = sm.row[tid];
                if (c.slot < 0) sm.factor[tid][0] = l == 0.0f ? 0.0f : ex2(st.z - st.w) / l;     // NaN stays NaN
                else p.part.stats[(size_t)c.slot * U + tid] = make_float4(-st.z, l, -st.w, 0.0f);
            }
            tc_fence_after();
            uint32_t high[V], mid[V], low[V];
            load_columns<V>(t_o + (uint32_t)base, high);
            load_columns<V>(t_o + (uint32_t)(U + base), mid);
            load_columns<V>(t_o + (uint32_t)(2 * U + base), low);
            tmem_ld_wait();
            tc_fence_before();
            mbar_arrive_warp(bar(B_OFREE));
            (void)any_of_softmax<WORKERS>(false);
            float *to = p.part.acc + (size_t)(c.slot < 0 ? 0 : c.slot) * U * kKv8Dim + me;
#pragma unroll
            for (int r = 0; r < V; ++r) {
                if (base + r >= c.rows) break;
                const float o = fmaf(__uint_as_float(low[r]), kPLo, fmaf(__uint_as_float(mid[r]), kPMid, __uint_as_float(high[r])));
                if (c.slot < 0) c.out[base + r][me] = __float2bfloat16(o * sm.factor[base + r][0]);
                else to[(base + r) * kKv8Dim] = o;
            }
            mbar_arrive_warp(bar(B_CEMPTY + cs));
            // the rows' state and factors are written again after the next context's first vote
        }
    }

    // ================================ teardown ==========================================
    tc_fence_before();
    __syncthreads();
    if (*abort_word != 0) {
        for (int i = 0; i < 64; ++i) __nanosleep(1000);      // let copies in flight land
        if (threadIdx.x == 0) atomicCAS(&g_kv8_status[0], 0, *abort_word);
    }
    if (warp == PRODUCTS) {
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

// Contexts that several pieces share: CTA (piece, row) joins that row of the context that begins in the piece, if there is one.  The parts
// are dealt out to the warps, every one joins its own, and the first joins those.
constexpr int JOIN_WARPS = 4;
__global__ void __launch_bounds__(JOIN_WARPS * 32) kv8_join_kernel(const __grid_constant__ Kv8Attend a, const Partial part, int rows) {
    __shared__ float4 stats[JOIN_WARPS], acc[JOIN_WARPS][kKv8Dim / 4];
    pdl_launch_dependents();
    pdl_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int piece = (int)blockIdx.x, r = (int)blockIdx.y;
    const JoinInfo info = part.join[piece];
    if (info.last < 0 || r >= info.rows) return;
    Joined j;
    const int parts = info.last - piece + 1;
#pragma unroll 4
    for (int i = warp; i < parts; i += JOIN_WARPS) {
        const size_t at = (size_t)(i == 0 ? info.slot : 2 * (piece + i)) * rows + r;
        j.add(part.stats[at], *reinterpret_cast<const float4 *>(part.acc + at * kKv8Dim + lane * 4));
    }
    if (warp != 0) {
        if (lane == 0) stats[warp] = make_float4(j.m, j.l, j.w, 0.0f);
        acc[warp][lane] = j.o;
    }
    __syncthreads();
    if (warp != 0) return;
    for (int w = 1; w < min(JOIN_WARPS, parts); ++w) j.add(stats[w], acc[w][lane]);
    const float inv = j.l == 0.0f ? 0.0f : ex2(j.w - j.m) / j.l;
    const int row = info.row0 + r, tok = a.by_group.div(row);
    *reinterpret_cast<uint2 *>(a.out + (long long)(info.first_token + tok) * a.ldo + (size_t)(info.head * a.group + row - tok * a.group) * kKv8Dim + lane * 4) =
        make_uint2(pack2(j.o.x * inv, j.o.y * inv), pack2(j.o.z * inv, j.o.w * inv));
}

constexpr int kSmemPerSm = 228 * 1024, kSmemReserved = 1024;       // of an SM; taken by the system from each CTA

template <int R, int U>
size_t smem_bytes(int num_seqs) { return sizeof(Smem<R, U>) + (size_t)num_seqs * sizeof(int); }
// CTAs per SM that the launch bounds and the shared memory allow
template <int R, int U>
int ctas_per_sm(int num_seqs) {
    const int fit = (int)(kSmemPerSm / (smem_bytes<R, U>(num_seqs) + kSmemReserved));
    return fit < 1 ? 1 : fit > max_ctas(R) ? max_ctas(R) : fit;
}

template <int R, int U>
bool launch_rows(Params &p, void *workspace, int num_seqs, cudaStream_t st, int &grid) {
    static PerDevice<bool> configured;
    const cudaError_t ready = once_per_device(configured, [] {
        const cudaError_t e = cudaFuncSetAttribute(kv8_attend_kernel<R, U>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem_bytes<R, U>(MAX_SEQS));
        if (e != cudaSuccess) return e;
        return cudaFuncSetAttribute(kv8_attend_kernel<R, U>, cudaFuncAttributePreferredSharedMemoryCarveout, (int)cudaSharedmemCarveoutMaxShared);
    });
    if (ready != cudaSuccess) return false;
    const int line = p.whole ? 0 : num_seqs;              // whole contexts need no table of the line
    grid = p.whole ? num_seqs * p.a.b.kv_heads : num_sms() * ctas_per_sm<R, U>(line);
    partial_bytes(grid, U, workspace, &p.part);
    return launch_chained(kv8_attend_kernel<R, U>, dim3(grid), dim3(threads(R)), smem_bytes<R, U>(line), st, p) == cudaSuccess;
}

}  // namespace

size_t kv8_attention_workspace_bytes() {
    size_t most = 0;
    for (int rows = 8; rows <= 32; rows += 8) {
        const size_t bytes = partial_bytes(num_sms() * max_ctas(rows), rows, nullptr, nullptr);
        if (bytes > most) most = bytes;
    }
    return most;
}

// Whole (sequence, kv head) pairs or pieces?  In cycles, from what the phases of the kernel take: a tile's chain 2200, the steps around a
// context 2600, an SM's share of HBM 1400 a tile; pieces need 2000 for the table of units and 5000 for the join.  The longest
// context stands for all, which flatters whole pairs where lengths are uneven, hence their limit of 8 tiles, or 16 if a window makes
// them even.  Measured, us, whole : pieces (sequences of one new token, four kv heads with four heads each, tokens):
//   1 x 250        7.0 : 8.1    1 x 900      13.9 : 9.1    16 x 450      9.5 : 11.7   16 x 900     14.2 : 13.1   64 x 450     11.3 : 13.8
//   64 x 900      18.1 : 20.1   64 x 2000    28.9 : 30.7*  128 x 900    31.5 : 29.6*  128 x 2000   55.2 : 51.2   256 x 450    28.4 : 31.5
//   64 x 500..2000  27.4 : 23.5   128 x 225..900  25.8 : 23.3*  128 x 500..2000  48.6 : 36.5  256 x 112..450  23.4 : 25.6  256 x 500..2000  67.3 : 61.8
// On the lines with a star the rule takes the slower side, by 6 to 11%: it takes the same for even and uneven lengths, which it cannot tell
// apart.  Other head layouts were not measured; the rule knows them by the number of contexts alone.
static bool deal_whole(const Kv8Attend &a, int max_len, int slots) {
    const long long contexts = (long long)a.b.num_seqs * a.b.kv_heads;
    long long tokens = max_len < a.b.max_tokens ? max_len : a.b.max_tokens;
    long long limit = 8;
    if (a.window > 0) {
        const long long most = (long long)a.window + a.sinks + 2 * kKv8Group;
        if (most < tokens) tokens = most, limit = 16;
    }
    const long long tiles = (tokens + SOFTMAX - 1) / SOFTMAX;
    const long long memory = contexts * tiles * 1400 / num_sms();
    const long long whole = (contexts + slots - 1) / slots * (2600 + tiles * 2200);
    const long long pieces = (contexts * tiles * 2200 + contexts * 2600) / slots + 2200 + 2600;
    return tiles <= limit && (whole > memory ? whole : memory) <= 7000 + (pieces > memory ? pieces : memory);
}

// Rows of a row tile of this kernel for so many query rows of a sequence.
static int tile_rows(long long want) {
    if (want <= 4) return 4;
    const long long tiles = (want + 31) / 32, each = (want + tiles - 1) / tiles;
    return (int)((each + 7) / 8 * 8);
}

// This kernel, or the one for many queries (128 rows of a (sequence, kv head) to a CTA, no splitting of long contexts)?  In cycles, two CTAs
// per SM.  This one: 17000 around it all, 10000 for a tile of 128 tokens and up to 32 rows; lengths are taken to be uneven, half of the
// longest on average, with a tile's worth for each context.  The other: 10000 for an item, and 2100 for 64 keys, 2700 when two
// items share an SM.  Measured, us, this one : the other (sequences x new tokens, four kv heads with four heads each, context):
//   64 x 8, 200..2000    51 : 49     256 x 8, 200..450   61 : 55     19 x 8, 40..4450   34 : 83     4 x 8, 8000     31 : 143
//   64 x 16, 200..2000   80 : 51     256 x 16, 200..450  119 : 59    19 x 12, 40..4450  45 : 82     2 x 16, 30000   56 : 519
//   1 x 16, 200          18 : 10     1 x 32, 200         32 : 11     19 x 24, 40..4450  67 : 83*    64 x 4, 200..2000  35 : 49
// Up to 16 rows it is always this one.  On the line with a star the rule takes the slower side; other head layouts were not measured.
// The choice is one for the whole batch: a prompt's piece takes the decode steps beside it along to the other kernel.
static bool few_rows(const Kv8Attend &a, long long want, int max_len) {
    if (a.b.num_seqs > MAX_SEQS) return false;
    // units are counted in 32 bits
    const long long groups = (long long)a.b.max_tokens / kKv8Group + 2 * TILE_GROUPS;
    const long long most = ((long long)a.b.total_new * a.group / tile_rows(want) + a.b.num_seqs) * a.b.kv_heads;
    if (most > 0x7FFFFFFFLL / groups) return false;
    if (want <= 16) return true;
    const long long contexts = (long long)a.b.num_seqs * a.b.kv_heads, slots = 2LL * num_sms();
    long long tokens = max_len < a.b.max_tokens ? max_len : a.b.max_tokens, few_tokens = tokens;
    if (a.window > 0) {
        const long long seen = (long long)a.window + a.sinks + 2 * kKv8Group;
        if (seen + 128 / a.group < tokens) tokens = seen + 128 / a.group;
        if (seen + want / a.group < few_tokens) few_tokens = seen + want / a.group;      // a row tile reads what any row of the sequence sees
    }
    const long long units = contexts * ((want + 31) / 32) * ((few_tokens + SOFTMAX - 1) / SOFTMAX + 2) / 2;
    const long long few = 17000 + (units + slots - 1) / slots * 10000;
    const long long items = contexts * ((want + 127) / 128), steps = (tokens + 63) / 64;
    const long long many = (items + slots - 1) / slots * (10000 + steps * (items > slots / 2 ? 2700 : 2100));
    return few <= many;
}

bool kv8_attention_launch(const Kv8Attend &a, int max_new, int max_len, void *workspace, cudaStream_t st, int &launches) {
    const long long want = (long long)max_new * a.group;
    if (!few_rows(a, want, max_len)) {
        launches = 1;
        return kv8_prefill_launch(a, st);
    }
    const int rows = tile_rows(want);
    Params p;
    memset(&p, 0, sizeof(p));
    const uint64_t pool_rows = (uint64_t)a.b.num_blocks * a.b.kv_heads * a.b.block_size;
    if (!make_u8_tmap_sw128(&p.tm_k, a.k_cache, kKv8Dim, pool_rows, kKv8Dim, kKv8Dim, kKv8Group)) return false;
    if (!make_u8_tmap_sw128(&p.tm_v, a.v_cache, kKv8Dim, pool_rows, kKv8Dim, kKv8Dim, kKv8Group)) return false;
    p.a = a;
    p.min_units = 4;
    p.whole = deal_whole(a, max_len, num_sms() * max_ctas(rows)) ? 1 : 0;
    int grid = 0;
    bool ok = false;
    switch (rows) {
        case 4: ok = launch_rows<8, 4>(p, workspace, a.b.num_seqs, st, grid); break;
        case 8: ok = launch_rows<8, 8>(p, workspace, a.b.num_seqs, st, grid); break;
        case 16: ok = launch_rows<16, 16>(p, workspace, a.b.num_seqs, st, grid); break;
        case 24: ok = launch_rows<24, 24>(p, workspace, a.b.num_seqs, st, grid); break;
        default: ok = launch_rows<32, 32>(p, workspace, a.b.num_seqs, st, grid); break;
    }
    if (!ok) return false;
    launches = 1;
    if (p.whole) return true;
    if (launch_chained(kv8_join_kernel, dim3((unsigned)grid, (unsigned)rows), dim3(JOIN_WARPS * 32), 0, st, a, p.part, rows) != cudaSuccess) return false;
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
    const int prefill = kv8_prefill_take_status();
    return code[0] != 0 ? code[0] : prefill;
}

}  // namespace glmasr
