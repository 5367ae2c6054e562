// C entry points of the 8-bit paged cache: argument checks, then the launches (kv8_append.cu, kv8_attention.cu).
#include <math.h>

#include "../../include/glmasr_fp4.h"
#include "kv8_attention.cuh"
#include "runtime.cuh"

using namespace glmasr;

// two copies to the host and their module's load, which a program without this cache should not pay for
static PerDevice<bool> g_attention_used;
int glmasr::kv8_status() {
    const bool *used = g_attention_used.here();
    return used != nullptr && *used ? kv8_take_status() : 0;
}

namespace {

bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }

// The shape of cache and batch; what a kernel could not index safely is refused here.
bool make_batch(Kv8Batch &b, const glmasr_kv8_cache *c, const int *block_tables, int max_blocks, const int *seq_lens, const int *cu_new,
                int num_seqs, int total_new, int q_heads) {
    if (c == nullptr || c->k == nullptr || c->v == nullptr || c->k_scale == nullptr || c->v_scale == nullptr) return false;
    if (!aligned16(c->k) || !aligned16(c->v) || ((uintptr_t)c->k_scale & 3) != 0 || ((uintptr_t)c->v_scale & 3) != 0) return false;
    if (c->head_dim != kKv8Dim || c->kv_heads <= 0 || c->num_blocks <= 0 || c->block_size <= 0 || c->block_size % kKv8Group != 0) return false;
    if ((long long)c->num_blocks * c->kv_heads > 0x7FFFFFFFLL / c->block_size) return false;      // rows of codes are numbered in 32 bits
    if (num_seqs < 0 || total_new < 0 || max_blocks <= 0 || q_heads < 0) return false;
    if ((num_seqs > 0 && total_new > 0) && (block_tables == nullptr || seq_lens == nullptr || cu_new == nullptr)) return false;
    if ((((uintptr_t)block_tables | (uintptr_t)seq_lens | (uintptr_t)cu_new) & 3) != 0) return false;
    b.by_kv_heads = FastDiv(c->kv_heads);
    b.by_page = FastDiv(c->block_size / kKv8Group);
    b.block_tables = block_tables;
    b.seq_lens = seq_lens;
    b.cu_new = cu_new;
    b.num_seqs = num_seqs;
    b.max_blocks = max_blocks;
    b.num_blocks = c->num_blocks;
    b.block_size = c->block_size;
    b.kv_heads = c->kv_heads;
    b.q_heads = q_heads;
    b.total_new = total_new;
    const long long tokens = (long long)max_blocks * c->block_size;
    b.max_tokens = tokens > 0x7FFFFFF0LL ? 0x7FFFFFF0 : (int)tokens;
    return true;
}

// rows of `heads` heads of 128 at a pitch of ld elements, read and written 16 bytes at a time
bool rows_ok(const void *p, long long ld, int heads, int rows) {
    return p != nullptr && aligned16(p) && ld % 8 == 0 && (rows <= 1 || ld >= (long long)heads * kKv8Dim);
}

// Whether two sets of `rows` rows (of heads_a and heads_b heads) have an element in common.  At one pitch, rows i of the one and j of the other are
// (b - a) + (j - i) * pitch apart, of which only the two next to zero matter; rows of different pitches count as one piece each.
bool rows_overlap(const void *a, long long lda, int heads_a, const void *b, long long ldb, int heads_b, int rows) {
    const long long wa = (long long)heads_a * kKv8Dim, wb = (long long)heads_b * kKv8Dim;
    const long long apart = ((long long)(uintptr_t)b - (long long)(uintptr_t)a) / 2;          // elements; both are 16-byte aligned
    if (rows <= 1) lda = ldb = 0;
    if (apart >= (rows - 1) * lda + wa || -apart >= (rows - 1) * ldb + wb) return false;
    if (lda != ldb || rows <= 1) return true;
    long long j = -apart / lda;                               // apart + j * lda is the first that is not below zero
    if (apart + j * lda < 0) ++j;
    return (j < rows && -j < rows && apart + j * lda < wa) || (j - 1 < rows && 1 - j < rows && -(apart + (j - 1) * lda) < wb);
}

}  // namespace

extern "C" int glmasr_kv8_append(const glmasr_kv8_cache *cache, const uint16_t *key, long long ldk, const uint16_t *value, long long ldv,
                                 const uint16_t *query, long long ldq, uint16_t *query_out, long long ldqo, int q_heads,
                                 const int *block_tables, int max_blocks, const int *seq_lens, const int *cu_new, int num_seqs,
                                 int total_new, double theta) {
    Kv8Batch b;
    if (!make_batch(b, cache, block_tables, max_blocks, seq_lens, cu_new, num_seqs, total_new, query != nullptr ? q_heads : 0)) return -1;
    if (!isfinite(theta) || theta < 0.0 || (query != nullptr && q_heads <= 0) || (query == nullptr) != (query_out == nullptr)) return -1;
    if (num_seqs == 0 || total_new == 0) return 0;
    if (!rows_ok(key, ldk, b.kv_heads, total_new) || !rows_ok(value, ldv, b.kv_heads, total_new)) return -1;
    if (query != nullptr) {
        if (!rows_ok(query, ldq, q_heads, total_new) || !rows_ok(query_out, ldqo, q_heads, total_new)) return -1;
        const bool in_place = query_out == query && (ldqo == ldq || total_new == 1);
        if (!in_place && rows_overlap(query_out, ldqo, q_heads, query, ldq, q_heads, total_new)) return -1;
        if (rows_overlap(query_out, ldqo, q_heads, key, ldk, b.kv_heads, total_new) || rows_overlap(query_out, ldqo, q_heads, value, ldv, b.kv_heads, total_new)) return -1;
    }
    if (!kv8_append_launch(cache->k, cache->v, cache->k_scale, cache->v_scale, (const __nv_bfloat16 *)key, ldk, (const __nv_bfloat16 *)value, ldv,
                           (const __nv_bfloat16 *)query, ldq, (__nv_bfloat16 *)query_out, ldqo, b, theta, current_stream())) {
        (void)cudaGetLastError();
        return -1;
    }
    note_launches(1);
    return 0;
}

extern "C" long long glmasr_kv8_attention_workspace(void) {
    if (g_attention_used.here() != nullptr) return (long long)kv8_attention_workspace_bytes();
    (void)cudaGetLastError();                                 // no device: what asks for its size would end the process
    return 0;
}

extern "C" int glmasr_kv8_attention(uint16_t *out, long long ldo, const uint16_t *query, long long ldq, const glmasr_kv8_cache *cache,
                                    const int *block_tables, int max_blocks, const int *seq_lens, const int *cu_new, int num_seqs,
                                    int total_new, int q_heads, int max_new, int max_len, int window, int sinks, float scale,
                                    void *workspace, long long workspace_bytes) {
    Kv8Attend a;
    if (!make_batch(a.b, cache, block_tables, max_blocks, seq_lens, cu_new, num_seqs, total_new, q_heads)) return -1;
    if (q_heads <= 0 || q_heads % a.b.kv_heads != 0 || window < 0 || sinks < 0 || max_new < 0 || max_len < 0 || !(scale >= 0.0f) || !isfinite(scale)) return -1;
    if (num_seqs == 0 || total_new == 0) return 0;
    if (!rows_ok(query, ldq, q_heads, total_new) || !rows_ok(out, ldo, q_heads, total_new)) return -1;
    if (rows_overlap(out, ldo, q_heads, query, ldq, q_heads, total_new)) return -1;
    bool *used = g_attention_used.here();
    if (used == nullptr) (void)cudaGetLastError();
    if (used == nullptr || workspace == nullptr || !aligned16(workspace) || workspace_bytes < (long long)kv8_attention_workspace_bytes()) return -1;
    a.k_cache = cache->k, a.v_cache = cache->v;
    a.k_scale = cache->k_scale, a.v_scale = cache->v_scale;
    a.query = (const __nv_bfloat16 *)query;
    a.out = (__nv_bfloat16 *)out;
    a.ldq = ldq, a.ldo = ldo;
    if ((long long)total_new * q_heads > 0x7FFFFF00LL) return -1;                // rows are numbered in 32 bits
    a.group = q_heads / a.b.kv_heads;
    a.by_group = FastDiv(a.group);
    a.window = window >= a.b.max_tokens ? 0 : window;              // one that reaches past the table leaves nothing out
    a.sinks = sinks < a.b.max_tokens ? sinks : a.b.max_tokens;
    a.scale_log2 = scale * 1.4426950408889634f;
    int launches = 0;
    *used = true;
    if (!kv8_attention_launch(a, max_new, max_len, workspace, current_stream(), launches)) {
        (void)cudaGetLastError();
        return -1;
    }
    note_launches(launches);
    return 0;
}
