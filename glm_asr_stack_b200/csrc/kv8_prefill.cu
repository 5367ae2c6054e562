// Attention of many queries per sequence over the 8-bit paged cache: prompts, and pieces of prompts behind what the cache holds.
//
// 128 rows (new token, query head of the group) of one (sequence, kv head) per work item, 64 keys per step:
//   S = Q K^T         e4m3 x e4m3 on tcgen05, K straight from the cache.  A query row is taken times a power of two that brings its largest
//                     element to 2^7 and split into two e4m3 numbers, q = hi + lo, both products into the same sums: exact for
//                     elements down to 2^-9 of the largest, off by 2^-17 of the largest below.  Two products of 8-bit operands
//                     cost what one of 16-bit operands does, and no key is converted.
//   p = 2^(x - m + 9) x = s * (row scale) * (K scale of the block of 16 keys), in one pass over the scores: m moves when a weight would be
//                     above 2^15, and only then is O touched.
//   O += P V          f16 x f16: weights have 11 bits down to 2^-23 of the largest, and are off by 2^-34 of it below, which a long tail of
//                     small weights can do with.  (At most 2^8 and from 2^0 on they lost tails: 2^-26 each came out as 0.)  V's codes become
//                     f16, times the scale of their block over the largest scale of the item so far (exact: a power of two),
//                     which O is expressed against.  Once the scales of an item's blocks, in whatever order they come, are more than 2^5
//                     apart (a block of zeros has the smallest one there is), small weights on large values may be what counts: from
//                     that step on P and V are bf16, 8 bits of any size.
// Bound: the two products are 2 x 128 x 64 x 128 multiply-adds a step, 512 cycles at the tensor cores' nominal rate, and the exponentials 512
// of the special-function units.  The softmax of a step is a chain of some 2000 cycles, so two CTAs share an SM, and a CTA's scores of
// the next step are computed under its softmax: tensor memory has two of S and one of O.  (128 keys per step with one S: 382 us
// where this took 345, two sequences of 2000 new tokens behind 5000: 320 to 330 now; 128 columns of S are all that O leaves of the half of
// tensor memory that a CTA has.  Two threads per row, eight warps of softmax: 386.)
//   warp 8      producer: the work items, K and V tiles (a TMA box of 2 KB per group of 16 keys), scales of each step; places in the pool are
//               looked up 8 steps ahead, which is worth 60 us there
//   warp 9      products; scores [0, 64) and [64, 128), output [128, 256) of tensor memory, P as f16 over the scores it was made from
//   warps 4-7   V of a step as f16 (or bf16)
//   warps 0-3   softmax: thread = row = lane of tensor memory; it also splits its row of queries and brings out its row of the output.  The
//               queries of the next item are asked for under its last softmax and split before its output goes out, so that the
//               products of the next item run meanwhile (25 prompts of 400 tokens: 61.5 us, 71 one after the other; 59 now)
// (warps 10 and 11 only give their registers to the softmax.)  The loops are kept rolled up: fully unrolled, the kernel was 92 KB of code
// and its softmax waited for instructions, 30 cycles a key instead of 21.
// The grid has a CTA for every work item there could be; those that run take over the items of those that have not started.
// The last tiles of a sequence, which see most keys, come first.
#include <math.h>

#include "kv8_attention.cuh"
#include "ptx.cuh"
#include "runtime.cuh"

namespace glmasr {

static __device__ int g_kv8_prefill_status[4];

namespace {

constexpr int QT = 128, KT = 64, THREADS = 384;
// Registers of a thread by warpgroup: two CTAs share an SM, 80 each at launch, and 128 + 56 + 56 = 3 x 80.
constexpr int REGS_SOFTMAX = 128, REGS_VALUES = 56, REGS_REST = 56;
constexpr int GROUPS = KT / kKv8Group, GROUP_BYTES = kKv8Group * kKv8Dim;
constexpr int TMEM_COLS = 256, COL_O = 128;
constexpr float kBase = 9.0f, kLazy = 6.0f;   // log2: weights at the reference, and how far above it before that moves (f16 ends below 2^16)
constexpr float kF16Range = 1.0f / 32.0f;     // smallest over largest V scale of an item's steps so far that f16 weights are taken for

static_assert(GROUPS == 4, "a step's K scales are read as one float4");
constexpr int STEPS = 4;                      // steps whose scales and lengths are kept

enum : int { B_QFULL = 0, B_OFREE, B_NEXT, B_KFULL, B_RFULL = B_KFULL + 2, B_REMPTY = B_RFULL + 2, B_VFULL = B_REMPTY + 2, B_SFULL = B_VFULL + 2,
             B_PFULL = B_SFULL + 2, B_INFO = B_PFULL + 2, B_INFOFREE = B_INFO + 2, B_STEP = B_INFOFREE + 2, B_PVDONE = B_STEP + STEPS, B_COUNT = B_PVDONE + STEPS };

struct ItemInfo {
    int rows;                                 // query rows that exist; 0: no more work
    int steps, head, row0, first_token;       // row0 + r counts (new token, head of the group) of the sequence
    int start;                                // position of the sequence's first new token
};
struct StepInfo {
    int tokens[GROUPS];                       // keys of each group of 16 that exist
    int key[GROUPS];                          // first position
    alignas(16) float ks[GROUPS];             // K scale
    float vmul[GROUPS];                       // V scale over vref
    float vref, vstep;                        // the largest V scale so far, and the one before over it
    int plain;                                // every row sees every key
    int wide;                                 // bf16
    uint32_t poisoned;                        // groups whose V scale is not a number
};
struct Smem {
    uint8_t q[2][QT * kKv8Dim];               // hi, lo; before that the row as it came, even and odd eights of its dims
    uint8_t k[2][KT * kKv8Dim], raw[2][KT * kKv8Dim];       // codes of K and V
    uint8_t v[2][2][KT * 128];                // f16, two boxes of 64 dims
    uint8_t stage[4][32 * 64];                // 32 columns of a warp's output rows on their way out
    ItemInfo item[2];
    StepInfo step[STEPS];
    uint4 next;
    unsigned long long bars[B_COUNT];
    uint32_t tmem;
    int abort;
};

struct Params {
    CUtensorMap tm_k, tm_v;
    Kv8Attend a;
    int tiles;                                // row tiles there could be, all sequences
};

constexpr uint32_t kIdescF16 = (1u << 4) | ((uint32_t)(kKv8Dim >> 3) << 17) | ((uint32_t)(QT >> 4) << 24) | kIdescBMnMajor;

__device__ __forceinline__ uint32_t pack2_f16(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&h);
}
// two codes (low or high half of a word) as f16
__device__ __forceinline__ uint32_t f16_codes(uint32_t w, bool high) {
    const uint16_t c = (uint16_t)(high ? w >> 16 : w);
    uint32_t r;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(c));
    return r;
}

// This lane's 128 output columns times f.
__device__ __forceinline__ void scale_columns(uint32_t t_o, float f) {
#pragma unroll 1
    for (int c = 0; c < 8; ++c) {
        uint32_t o[16];
        tmem_ld_x16(t_o + (uint32_t)c * 16, o);
        tmem_ld_wait();
#pragma unroll
        for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
        tmem_st_x16(t_o + (uint32_t)c * 16, o);
    }
}

template <int N>
__device__ __forceinline__ void more_registers() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void fewer_registers() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

__global__ void __launch_bounds__(THREADS, 2) kv8_prefill_kernel(const __grid_constant__ Params p) {
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    Smem &sm = *reinterpret_cast<Smem *>(smem_raw);
    const Kv8Attend &a = p.a;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    auto bar = [&](int i) { return smem_u32(&sm.bars[i]); };
    if ((smem_u32(smem_raw) & 1023u) != 0) {                  // the swizzled tiles need a 1024-byte aligned base
        if (threadIdx.x == 0) atomicCAS(&g_kv8_prefill_status[0], 0, ST_BAD_LAYOUT);
        return;
    }
    if (threadIdx.x == 0) {
        mbar_init(bar(B_QFULL), 4);
        mbar_init(bar(B_OFREE), 4);
        mbar_init(bar(B_NEXT), 1);
        for (int i = 0; i < 2; ++i) {
            mbar_init(bar(B_KFULL + i), 1);
            mbar_init(bar(B_RFULL + i), 1);
            mbar_init(bar(B_REMPTY + i), 4);
            mbar_init(bar(B_VFULL + i), 4);
            mbar_init(bar(B_SFULL + i), 1);
            mbar_init(bar(B_PFULL + i), 4);
            mbar_init(bar(B_INFO + i), 1);
            mbar_init(bar(B_INFOFREE + i), 4 + 4 + 1);
        }
        for (int i = 0; i < STEPS; ++i) {
            mbar_init(bar(B_STEP + i), 1);
            mbar_init(bar(B_PVDONE + i), 1);
        }
        sm.abort = 0;
        fence_mbar_init();
        tma_prefetch_desc(&p.tm_k);
        tma_prefetch_desc(&p.tm_v);
    }
    // as in the kernel for few queries: tensor memory after every earlier kernel, later ones when this one has it
    pdl_wait();
    if (warp == 9) {
        tmem_alloc(smem_u32(&sm.tmem), TMEM_COLS);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    pdl_launch_dependents();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t *>(&sm.tmem);
    volatile int *abort_word = &sm.abort;

    auto wait = [&](int i, uint32_t parity) { return mbar_wait_short(bar(i), parity & 1u, abort_word, ST_TIMEOUT_ATTENTION); };
    // the weighted sum of step t, the (t / STEPS)-th of its barrier, is done
    auto wait_sum = [&](uint32_t t) { return wait(B_PVDONE + (int)(t % STEPS), t / STEPS); };

    if (warp >= 8) {
        fewer_registers<REGS_REST>();           // the whole warpgroup, before its warps part
        if (warp == 8) {
            // ================================ producer ================================
            const bool leader = elect_one();
            const int *cu = a.b.cu_new;
            uint32_t t = 0, items = 0, answers = 0;               // steps, items and answers so far
            bool ok = true;
            int work = (int)blockIdx.x;
            int seq = -1, head = 0, len = 0, pos_lo = 0, pos_hi = 0;
            Kv8Span span = {0, 0, 0};
            // Lane l has the l-th of 32 groups, 8 steps: their places are looked up 8 steps before, and their scales are on their way
            // while the copies are asked for.
            int place = -1, place_ahead = -1, tokens = 0, key = 0;
            float ks = 0.0f, vs = 0.0f;
            auto place_of = [&](int g) {
                const long long row = g < span.count ? kv8_group_row(a.b, seq, head, span.group_of(g)) : -1;
                return row >= 0 ? (int)(row / kKv8Group) : -1;
            };
            for (bool first = true; ok; first = false) {
                if (!first) {                                     // the item after this one
                    if (leader) {
                        mbar_expect_tx(bar(B_NEXT), 16);
                        ask_cancelled_cta(smem_u32(&sm.next), bar(B_NEXT));
                    }
                    __syncwarp();
                }
                int next_seq = -1, next_head = 0, next_len = 0, next_lo = 0, next_hi = 0;
                Kv8Span next_span = {0, 0, 0};
                float vref = 0.0f;
                uint32_t vlow = 0x7F7FFFFFu;                      // the smallest V scale so far: bits of floats >= 0 are in their order
                bool wide = false, looked = false;
                int g = 0;
                place_ahead = place_of(lane);
                do {
                    if (g < span.count) {
                        if (g % 32 == 0) {
                            place = place_ahead;
                            key = g + lane < span.count ? span.group_of(g + lane) * kKv8Group : 0;
                            tokens = place >= 0 ? min(kKv8Group, len - key) : 0;
                            ks = place >= 0 ? a.k_scale[place] : 0.0f;
                            vs = place >= 0 ? a.v_scale[place] : 0.0f;
                            place_ahead = place_of(g + 32 + lane);
                        }
                        const int s = (int)(t & 1u), slot = lane % GROUPS;
                        const bool mine = lane / GROUPS == g % 32 / GROUPS, load = mine && place >= 0;
                        const uint32_t bytes = (uint32_t)__popc(__ballot_sync(0xFFFFFFFFu, load)) * GROUP_BYTES;
                        ok = wait(B_SFULL + s, (t >> 1) ^ 1u);       // the scores of the keys before, in their place, are there
                        if (!ok) break;
                        if (leader) mbar_expect_tx(bar(B_KFULL + s), bytes);
                        __syncwarp();
                        if (load) tma_load_2d(smem_u32(sm.k[s]) + slot * GROUP_BYTES, &p.tm_k, bar(B_KFULL + s), 0, place * kKv8Group);
                        ok = wait(B_REMPTY + s, (t >> 1) ^ 1u);
                        if (!ok) break;
                        if (leader) mbar_expect_tx(bar(B_RFULL + s), bytes);
                        __syncwarp();
                        if (load) tma_load_2d(smem_u32(sm.raw[s]) + slot * GROUP_BYTES, &p.tm_v, bar(B_RFULL + s), 0, place * kKv8Group);
                        const bool number = vs >= 0.0f && vs <= 3.4028234664e38f;
                        float most = number ? vs : 0.0f;
#pragma unroll
                        for (int d = 1; d < GROUPS; d <<= 1) most = fmaxf(most, __shfl_xor_sync(0xFFFFFFFFu, most, d));
                        most = fmaxf(vref, __shfl_sync(0xFFFFFFFFu, most, g % 32));
                        const float vmul = number && most > 0.0f ? vs / most : 0.0f;
                        const bool plain_here = tokens == kKv8Group && key + kKv8Group - 1 <= pos_lo &&
                                                (a.window == 0 || pos_hi - key < a.window || key + kKv8Group <= a.sinks);
                        vlow = min(vlow, __reduce_min_sync(0xFFFFFFFFu, mine && tokens > 0 && number ? __float_as_uint(vs) : 0x7F7FFFFFu));
                        wide = wide || __uint_as_float(vlow) < most * kF16Range;
                        const uint32_t poisoned = __ballot_sync(0xFFFFFFFFu, mine && !number) >> (g % 32);
                        const bool plain = !__any_sync(0xFFFFFFFFu, mine && !plain_here);
                        // the step whose place this is has been summed: softmax and V are done with it
                        if (t >= STEPS) ok = wait_sum(t - STEPS);
                        if (!ok) break;
                        StepInfo &st = sm.step[t % STEPS];
                        if (mine) {
                            st.tokens[slot] = tokens, st.key[slot] = key;
                            st.ks[slot] = ks, st.vmul[slot] = vmul;
                        }
                        if (lane == 0) {
                            st.vref = most;
                            st.vstep = most > 0.0f ? vref / most : 1.0f;
                            st.plain = plain ? 1 : 0;
                            st.wide = wide ? 1 : 0;
                            st.poisoned = poisoned;
                        }
                        __syncwarp();
                        if (leader) mbar_arrive(bar(B_STEP + (int)(t % STEPS)));
                        vref = most;
                        ++t;
                        g += GROUPS;
                    }
                    if (!looked && (g > GROUPS || g >= span.count)) {        // two steps are on their way: the next item, early enough for its queries
                        looked = true;
                        if (!first) {
                            ok = wait(B_NEXT, answers);
                            if (!ok) break;
                            ++answers;
                            work = cancelled_cta(smem_u32(&sm.next));
                            fence_proxy_async_smem();             // the answer has been read before the next one is written
                            __syncwarp();
                        }
                        ItemInfo info = {0, 0, 0, 0, 0, 0};       // the end
                        if (work >= 0) {
                            const int y0 = a.b.by_kv_heads.div(work), y = p.tiles - 1 - y0;
                            next_head = work - y0 * a.b.kv_heads;
                            // sequence s has the tiles from cu_new[s] * group / 128 + s on: a bound that needs no pass over the lengths
                            next_seq = warp_last_not_above(a.b.num_seqs, (long long)y, [&](int s) { return (((long long)cu[s] * a.group) >> 7) + s; });
                            if (next_seq >= 0) {
                                const int row0 = cu[next_seq], end = cu[next_seq + 1], n = row0 < 0 ? 0 : max(0, min(end, a.b.total_new) - row0);
                                const int tile = y - (int)(((long long)row0 * a.group) >> 7) - next_seq, rows = min(QT, n * a.group - tile * QT);
                                next_len = a.b.seq_lens[next_seq];
                                if (rows > 0) {
                                    const int start = next_len - (end - row0);
                                    next_lo = start + a.by_group.div(tile * QT), next_hi = start + a.by_group.div(tile * QT + rows - 1);
                                    next_span = kv8_span(a, next_len, next_lo, next_hi);
                                    info = {rows, (next_span.count + GROUPS - 1) / GROUPS, next_head, tile * QT, row0, start};
                                }
                            }
                        }
                        if (work < 0 || info.rows > 0) {
                            const int is = (int)(items & 1u);
                            ok = wait(B_INFOFREE + is, (items >> 1) ^ 1u);
                            if (!ok) break;
                            if (leader) {
                                sm.item[is] = info;
                                mbar_arrive(bar(B_INFO + is));
                            }
                            __syncwarp();
                            ++items;
                        }
                    }
                } while (g < span.count);
                if (work < 0) break;
                seq = next_seq, head = next_head, len = next_len, pos_lo = next_lo, pos_hi = next_hi, span = next_span;
            }
        } else if (warp == 9) {
            // ================================ products ================================
            const bool leader = elect_one();
            constexpr uint32_t idesc_s = idesc_e4m3(QT, KT);
            const uint32_t t_o = tmem + COL_O;
            uint32_t t = 0, items = 0, worked = 0;                // worked: items with any step
            bool ok = true;
            while (ok) {
                const int is = (int)(items & 1u);
                if (!wait(B_INFO + is, items >> 1)) break;
                const int rows = sm.item[is].rows, steps = sm.item[is].steps;
                if (rows == 0) break;
                ++items;
                __syncwarp();
                if (leader) mbar_arrive(bar(B_INFOFREE + is));
                if (steps == 0) continue;
                if (!wait(B_QFULL, worked)) break;
                // The scores of step j + 1 are asked for before the weights of step j are there; they take the place of the weights of j - 1.
                for (int j = -1; j < steps; ++j) {
                    if (j + 1 < steps) {
                        const uint32_t u = t + (uint32_t)(j + 1);
                        const int s = (int)(u & 1u);
                        ok = wait(B_KFULL + s, u >> 1) && (u < 2 || wait_sum(u - 2));
                        if (!ok) break;
                        tc_fence_after();
                        if (leader) {
                            const uint64_t bd = smem_desc_sw128(smem_u32(sm.k[s]));
#pragma unroll
                            for (int k = 0; k < 8; ++k)
                                umma_f8(tmem + (uint32_t)(s * KT), smem_desc_sw128(smem_u32(sm.q[k >> 2])) + (uint64_t)(((k & 3) * 32) >> 4), bd + (uint64_t)(((k & 3) * 32) >> 4), idesc_s, k > 0 ? 1u : 0u);
                            umma_commit(bar(B_SFULL + s));
                        }
                        __syncwarp();
                    }
                    if (j < 0) continue;
                    const uint32_t u = t + (uint32_t)j;
                    const int s = (int)(u & 1u);
                    ok = wait(B_VFULL + s, u >> 1) && wait(B_PFULL + s, u >> 1);
                    // the first weighted sum of an item overwrites the output of the item before
                    if (ok && j == 0) ok = wait(B_OFREE, worked ^ 1u);
                    if (!ok) break;
                    tc_fence_after();
                    const bool wide = sm.step[u % STEPS].wide != 0;
                    if (leader) {
                        const uint64_t bd = smem_desc_sw128_mn(smem_u32(sm.v[s][0]), KT * 128);
                        const uint32_t idesc_o = wide ? idesc_bf16(QT, kKv8Dim) | kIdescBMnMajor : kIdescF16;
#pragma unroll
                        for (int k = 0; k < KT / 16; ++k)
                            umma_bf16_ts(t_o, tmem + (uint32_t)(s * KT + k * 8), bd + (uint64_t)((k * 2048) >> 4), idesc_o, j > 0 || k > 0 ? 1u : 0u);
                        umma_commit(bar(B_PVDONE + (int)(u % STEPS)));
                    }
                    __syncwarp();
                }
                t += (uint32_t)steps;
                ++worked;
            }
        }
    } else if (warp >= 4) {
        // ================================ V ================================
        fewer_registers<REGS_VALUES>();
        // A thread has 16 dims of one key of each group.  Eight threads that access shared memory together have four chunks of a key a and
        // the same of key a ^ 5: eight different places among the 128 bytes of a row, of codes as well as of the result.
        const int pair = (threadIdx.x >> 4) & 7, a_key = (pair & 3) + (pair >> 2) * 8, in_group = (lane & 4) != 0 ? a_key ^ 5 : a_key;
        const int chunk = (lane & 3) + ((lane >> 3) & 1) * 4;
        const uint32_t src0 = smem_u32(sm.raw[0]) + (uint32_t)(in_group * kKv8Dim + ((chunk ^ (in_group & 7)) << 4));
        // the 16-byte chunks 2 (chunk % 4) and the next of the row, swizzled: they differ in the lowest bit
        const uint32_t dst0 = smem_u32(sm.v[0][chunk >> 2]) + (uint32_t)(in_group * 128 + ((((chunk & 3) * 2) ^ (in_group & 7)) << 4));
        uint32_t t = 0, items = 0;
        bool ok = true;
        while (ok) {
            const int is = (int)(items & 1u);
            if (!wait(B_INFO + is, items >> 1)) break;
            const int rows = sm.item[is].rows, steps = sm.item[is].steps;
            if (rows == 0) break;
            ++items;
            mbar_arrive_warp(bar(B_INFOFREE + is));
            for (int j = 0; j < steps; ++j, ++t) {
                const int s = (int)(t & 1u);
                const StepInfo &st = sm.step[t % STEPS];
                ok = wait(B_STEP + (int)(t % STEPS), t / STEPS) && wait(B_RFULL + s, t >> 1) && (t < 2 || wait_sum(t - 2));
                if (!ok) break;
                const bool wide = st.wide != 0;
                const uint32_t src = src0 + (uint32_t)s * sizeof(sm.raw[0]), dst = dst0 + (uint32_t)s * sizeof(sm.v[0]);
#pragma unroll 1
                for (int i = 0; i < GROUPS; ++i) {
                    uint32_t w[4], h[8];
                    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(src + i * GROUP_BYTES) : "memory");
                    const float mul = st.vmul[i];
                    if (in_group >= st.tokens[i]) w[0] = w[1] = w[2] = w[3] = 0u;         // behind the end may be anything: zeros instead
                    if (!wide) {
                        const __half2 m2 = __float2half2_rn(mul);
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            const uint32_t c = f16_codes(w[e >> 1], (e & 1) != 0);
                            const __half2 y = __hmul2(*reinterpret_cast<const __half2 *>(&c), m2);
                            h[e] = *reinterpret_cast<const uint32_t *>(&y);
                        }
                    } else {
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            const uint32_t c = f16_codes(w[e >> 1], (e & 1) != 0);
                            const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&c));
                            h[e] = pack2(f.x * mul, f.y * mul);
                        }
                    }
                    const uint32_t at = dst + i * (kKv8Group * 128);
                    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(h[0]), "r"(h[1]), "r"(h[2]), "r"(h[3]) : "memory");
                    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at ^ 16u), "r"(h[4]), "r"(h[5]), "r"(h[6]), "r"(h[7]) : "memory");
                }
                mbar_arrive_warp(bar(B_REMPTY + s));
                fence_proxy_async_smem();
                mbar_arrive_warp(bar(B_VFULL + s));
            }
        }
    } else {
        // ================================ softmax ================================
        more_registers<REGS_SOFTMAX>();
        const int me = warp * 32 + lane;                      // row of the tile, lane of tensor memory
        const uint32_t t_row = tmem + ((uint32_t)(warp * 32) << 16), t_o = t_row + COL_O;
        uint32_t t = 0, items = 0;
        ItemInfo info, next;
        // The next item, and this warp's rows of its queries on their way to where the present ones are done with: 16 lanes have a row.
        auto look_ahead = [&]() {
            const int is = (int)(items & 1u);
            if (!wait(B_INFO + is, items >> 1)) return false;
            next = sm.item[is];
            ++items;
            if (next.rows == 0) return true;
            mbar_arrive_warp(bar(B_INFOFREE + is));
            if (next.steps == 0) return true;
            const int part = lane & 15;
#pragma unroll 4
            for (int i = 0; i < 32; i += 2) {
                const int r = warp * 32 + i + (lane >> 4), row = min(r, next.rows - 1) + next.row0, tok = a.by_group.div(row);
                cp_async16_zfill(smem_u32(sm.q[part & 1]) + swizzled(r, (part >> 1) * 16),
                        a.query + (long long)(next.first_token + tok) * a.ldq + (size_t)(next.head * a.group + row - tok * a.group) * kKv8Dim + part * 8, r < next.rows);
            }
            cp_async_commit();
            return true;
        };
        // Queries of the next item: 2^shift brings the largest element to [2^7, 2^8) (one below 2^-119 less far); a row that is not finite
        // gets NaN scores by its scale.  16 dims of this thread's row are split into the 32 bytes they came in.
        float next_qs = 0.0f;
        auto split_queries = [&]() {
            if (next.rows == 0 || next.steps == 0) return;
            cp_async_wait<0>();
            __syncwarp();
            uint32_t big = 0u;
#pragma unroll 2
            for (int i = 0; i < 16; ++i) {
                const uint4 q = *reinterpret_cast<const uint4 *>(sm.q[i & 1] + swizzled(me, (i >> 1) * 16));
                big = __vmaxu2(big, __vmaxu2(__vmaxu2(q.x & 0x7FFF7FFFu, q.y & 0x7FFF7FFFu), __vmaxu2(q.z & 0x7FFF7FFFu, q.w & 0x7FFF7FFFu)));
            }
            big = max(big >> 16, big & 0xFFFFu);
            const int expo = (int)(big >> 7), shift = expo == 255 ? 0 : min(7 + 127 - expo, 126);
            const float up = pow2(shift);
            next_qs = expo == 255 ? __int_as_float(0x7FFFFFFF) : a.scale_log2 * pow2(-shift);
#pragma unroll 1
            for (int c = 0; c < 8; ++c) {
                uint4 *first = reinterpret_cast<uint4 *>(sm.q[0] + swizzled(me, c * 16)), *second = reinterpret_cast<uint4 *>(sm.q[1] + swizzled(me, c * 16));
                const uint4 q0 = *first, q1 = *second;
                const uint32_t w[8] = {q0.x, q0.y, q0.z, q0.w, q1.x, q1.y, q1.z, q1.w};
                uint32_t hi[4] = {0u, 0u, 0u, 0u}, lo[4] = {0u, 0u, 0u, 0u};
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    float x0 = __uint_as_float(w[e] << 16) * up, x1 = __uint_as_float(w[e] & 0xFFFF0000u) * up;
                    hi[e >> 1] |= e4m3_split(x0, x1) << (16 * (e & 1));
                    lo[e >> 1] |= e4m3x2(x0, x1) << (16 * (e & 1));
                }
                *first = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                *second = make_uint4(lo[0], lo[1], lo[2], lo[3]);
            }
            fence_proxy_async_smem();
            mbar_arrive_warp(bar(B_QFULL));
        };
        bool ok = look_ahead();
        if (ok) split_queries();
        while (ok && next.rows > 0) {
            info = next;
            const int row = info.row0 + me, tok = a.by_group.div(row);
            const int pos = me < info.rows ? info.start + tok : -1;
            const float qs = next_qs;
            float m = kNothing, l = 0.0f, vref = 1.0f;
            if (info.steps == 0) ok = look_ahead();
            for (int j = 0; j < info.steps; ++j, ++t) {
                const int s = (int)(t & 1u);
                ok = wait(B_STEP + (int)(t % STEPS), t / STEPS) && wait(B_SFULL + s, t >> 1);
                if (!ok) break;
                tc_fence_after();
                const StepInfo &st = sm.step[t % STEPS];
                const uint32_t t_s = t_row + (uint32_t)(s * KT);
                uint32_t y[2][32];
                tmem_ld_x32(t_s, y[0]);
                tmem_ld_x32(t_s + 32, y[1]);
                const float4 ks = *reinterpret_cast<const float4 *>(st.ks);
                float f[GROUPS] = {qs * ks.x, qs * ks.y, qs * ks.z, qs * ks.w};
                const bool wide = st.wide != 0;
                float factor = j > 0 ? st.vstep : 1.0f;
                vref = st.vref;
                tmem_ld_wait();
                if (j == info.steps - 1) {                        // the last scores: the queries are done with
                    ok = look_ahead();
                    if (!ok) break;
                }
                if (st.plain == 0) {
                    // scores times their scales here, -inf for keys that this row does not see
#pragma unroll
                    for (int g = 0; g < GROUPS; ++g) {
                        const int k0 = st.key[g];
                        uint32_t seen = (1u << max(0, min(st.tokens[g], pos - k0 + 1))) - 1u;       // bit i: key i of the group
                        if (a.window > 0) {
                            const uint32_t gone = (1u << max(0, min(kKv8Group, pos - a.window + 1 - k0))) - 1u, first = (1u << max(0, min(kKv8Group, a.sinks - k0))) - 1u;
                            seen &= ~gone | first;
                        }
                        if ((st.poisoned >> g & 1u) != 0u && seen != 0u) l = __int_as_float(0x7FFFFFFF);
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            uint32_t &z = y[g >> 1][16 * (g & 1) + e];
                            z = (seen >> e & 1u) != 0u ? __float_as_uint(__uint_as_float(z) * f[g]) : 0xFF800000u;
                        }
                        f[g] = 1.0f;
                    }
                } else if (st.poisoned != 0u) {
                    l = __int_as_float(0x7FFFFFFF);
                }
                float high = kNothing;
#pragma unroll
                for (int g = 0; g < GROUPS; ++g) {
                    const uint32_t *z = &y[g >> 1][16 * (g & 1)];
                    float t0 = max3(__uint_as_float(z[0]), __uint_as_float(z[1]), __uint_as_float(z[2]));
                    float t1 = max3(__uint_as_float(z[3]), __uint_as_float(z[4]), __uint_as_float(z[5]));
#pragma unroll
                    for (int e = 6; e < 14; e += 4) {
                        t0 = max3(t0, __uint_as_float(z[e]), __uint_as_float(z[e + 1]));
                        t1 = max3(t1, __uint_as_float(z[e + 2]), __uint_as_float(z[e + 3]));
                    }
                    high = fmaxf(high, max3(t0, t1, fmaxf(__uint_as_float(z[14]), __uint_as_float(z[15]))) * f[g]);
                }
                float alpha = 1.0f;
                if (high > m + kLazy) {
                    alpha = ex2(m - high);
                    m = high;
                }
                // the output under the present references, once the sum of the step before is done
                factor *= alpha;
                l *= alpha;
                if (j > 0 && __any_sync(0xFFFFFFFFu, factor != 1.0f)) {
                    ok = wait_sum(t - 1);
                    if (!ok) break;
                    tc_fence_after();
                    scale_columns(t_o, factor);
                }
                unsigned long long sum2[2] = {pack_f32x2(0.0f, 0.0f), pack_f32x2(0.0f, 0.0f)};
                const unsigned long long neg_m2 = pack_f32x2(kBase - m, kBase - m);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    uint32_t w[16];
#pragma unroll
                    for (int e = 0; e < 32; e += 2) {
                        const unsigned long long f2 = pack_f32x2(f[2 * h + (e >> 4)], f[2 * h + (e >> 4)]);
                        float y0, y1;
                        unpack_f32x2(fma_f32x2(pack_f32x2(__uint_as_float(y[h][e]), __uint_as_float(y[h][e + 1])), f2, neg_m2), y0, y1);
                        const float p0 = ex2(y0), p1 = ex2(y1);
                        sum2[e >> 4] = add_f32x2(sum2[e >> 4], pack_f32x2(p0, p1));
                        w[e >> 1] = wide ? pack2(p0, p1) : pack2_f16(p0, p1);
                    }
                    tmem_st_x16(t_s + (uint32_t)(h * 16), w);     // over scores that have been read
                }
                float s0, s1;
                unpack_f32x2(add_f32x2(sum2[0], sum2[1]), s0, s1);
                l += s0 + s1;
                tmem_st_wait();
                tc_fence_before();
                mbar_arrive_warp(bar(B_PFULL + s));
            }
            if (!ok) break;
            split_queries();                                      // so that the next item's scores come while this one's output goes
            if (info.steps > 0) {
                ok = wait_sum(t - 1);
                if (!ok) break;
                tc_fence_after();
            }
            const float inv = l == 0.0f ? 0.0f : vref / l;    // a row that sees nothing; NaN stays NaN
            // 32 columns at a time through shared memory: four lanes then have a row's 64 bytes
            uint8_t *stage = sm.stage[warp];
            const int mine = lane >> 2, part = lane & 3;
            __nv_bfloat16 *out[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int r = info.row0 + warp * 32 + i * 8 + mine, tk = a.by_group.div(r);
                out[i] = a.out + (long long)(info.first_token + tk) * a.ldo + (size_t)(info.head * a.group + r - tk * a.group) * kKv8Dim + part * 8;
            }
#pragma unroll 1
            for (int c = 0; c < 4; ++c) {
                uint32_t o[32];
                if (info.steps > 0) {
                    tmem_ld_x32(t_o + (uint32_t)c * 32, o);
                    tmem_ld_wait();
                } else {
#pragma unroll
                    for (int e = 0; e < 32; ++e) o[e] = 0u;
                }
                __syncwarp();                                 // the columns before have been read
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    *reinterpret_cast<uint4 *>(stage + lane * 64 + ((e ^ (lane >> 1)) & 3) * 16) =
                        make_uint4(pack2(__uint_as_float(o[8 * e]) * inv, __uint_as_float(o[8 * e + 1]) * inv), pack2(__uint_as_float(o[8 * e + 2]) * inv, __uint_as_float(o[8 * e + 3]) * inv),
                                   pack2(__uint_as_float(o[8 * e + 4]) * inv, __uint_as_float(o[8 * e + 5]) * inv), pack2(__uint_as_float(o[8 * e + 6]) * inv, __uint_as_float(o[8 * e + 7]) * inv));
                __syncwarp();
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int r = i * 8 + mine;
                    if (warp * 32 + r < info.rows) *reinterpret_cast<uint4 *>(out[i] + c * 32) = *reinterpret_cast<const uint4 *>(stage + r * 64 + ((part ^ (r >> 1)) & 3) * 16);
                }
            }
            if (info.steps > 0) {
                tc_fence_before();
                mbar_arrive_warp(bar(B_OFREE));
            }
        }
        cp_async_wait<0>();
    }

    // ================================ teardown ==========================================
    tc_fence_before();
    __syncthreads();
    if (*abort_word != 0) {
        for (int i = 0; i < 64; ++i) __nanosleep(1000);      // let copies in flight land
        if (threadIdx.x == 0) atomicCAS(&g_kv8_prefill_status[0], 0, *abort_word);
    }
    if (warp == 9) {
        __syncwarp();
        tmem_dealloc(tmem, TMEM_COLS);
    }
}

}  // namespace

bool kv8_prefill_launch(const Kv8Attend &a, cudaStream_t st) {
    static PerDevice<bool> configured;
    const cudaError_t ready = once_per_device(configured, [] {
        const cudaError_t e = cudaFuncSetAttribute(kv8_prefill_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(Smem));
        if (e != cudaSuccess) return e;
        return cudaFuncSetAttribute(kv8_prefill_kernel, cudaFuncAttributePreferredSharedMemoryCarveout, (int)cudaSharedmemCarveoutMaxShared);
    });
    if (ready != cudaSuccess) return false;
    Params p;
    memset(&p, 0, sizeof(p));
    if (!make_u8_tmap_sw128(&p.tm_k, a.k_cache, kKv8Dim, (uint64_t)a.b.num_blocks * a.b.kv_heads * a.b.block_size, kKv8Dim, kKv8Dim, kKv8Group)) return false;
    if (!make_u8_tmap_sw128(&p.tm_v, a.v_cache, kKv8Dim, (uint64_t)a.b.num_blocks * a.b.kv_heads * a.b.block_size, kKv8Dim, kKv8Dim, kKv8Group)) return false;
    p.a = a;
    const long long tiles = ((long long)a.b.total_new * a.group >> 7) + a.b.num_seqs;
    if (tiles * a.b.kv_heads > 0x7FFFFFFFLL) return false;
    p.tiles = (int)tiles;
    return launch_chained(kv8_prefill_kernel, dim3((unsigned)(tiles * a.b.kv_heads)), dim3(THREADS), sizeof(Smem), st, p) == cudaSuccess;
}

int kv8_prefill_take_status() {
    int code[4] = {0, 0, 0, 0};
    if (cudaMemcpyFromSymbol(code, g_kv8_prefill_status, sizeof(code)) != cudaSuccess) return -1;
    if (code[0] != 0) {
        const int zero[4] = {0, 0, 0, 0};
        (void)cudaMemcpyToSymbol(g_kv8_prefill_status, zero, sizeof(zero));
    }
    return code[0];
}

}  // namespace glmasr
