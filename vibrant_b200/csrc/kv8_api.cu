// kv8_api.cu -- extern "C" entry points of the rotary positions and the 8-bit
// paged KV cache (declared in include/vkq.h): argument checks, then a launch.
#include <cmath>
#include <cstdint>

#include "../../include/vkq.h"
#include "act.cuh"
#include "vkq_internal.h"

using namespace vkq;

namespace vkq {

static bool misaligned(const void *p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) != 0; }

static int check_dtype(int dtype, const char *who) {
    if (act_bytes(dtype)) return VKQ_OK;
    set_error("%s: unsupported dtype %d (expected VKQ_F32, VKQ_F16 or VKQ_BF16)", who, dtype);
    return VKQ_ERR_UNSUPPORTED;
}

static int check_cache(const vkq_kv8_cache *c, int64_t layer, const char *who) {
    if (!c || !c->k || !c->v || !c->k_scale || !c->v_scale) {
        set_error("%s: null cache or pool pointer", who);
        return VKQ_ERR_INVALID_ARGUMENT;
    }
    if (c->format != VKQ_KV8_INT8 && c->format != VKQ_KV8_E4M3) {
        set_error("%s: unsupported format %d", who, c->format);
        return VKQ_ERR_UNSUPPORTED;
    }
    if (c->head_dim != 64 && c->head_dim != 128) {
        set_error("%s serves head_dim 64 or 128 (got %d)", who, c->head_dim);
        return VKQ_ERR_UNSUPPORTED;
    }
    if (c->page_size <= 0 || c->page_size > 4096 || c->page_size % VKQ_KV8_BLOCK || c->kv_heads <= 0 ||
        c->kv_heads > 65535 || c->layers <= 0 || c->layers > (1 << 20) || c->num_pages <= 0 ||
        c->num_pages > INT32_MAX || layer < 0 || layer >= c->layers) {
        set_error("%s: page_size %d (a multiple of 16, at most 4096), kv_heads %d, num_pages %lld or layer %lld of %lld "
                  "is out of range",
                  who, c->page_size, c->kv_heads, (long long)c->num_pages, (long long)layer, (long long)c->layers);
        return VKQ_ERR_INVALID_ARGUMENT;
    }
    if (misaligned(c->k, 16) || misaligned(c->v, 16) || misaligned(c->k_scale, 4) || misaligned(c->v_scale, 4)) {
        set_error("%s: the pool's codes must be 16-byte and its scales 4-byte aligned", who);
        return VKQ_ERR_MISALIGNED;
    }
    return VKQ_OK;
}

static int check_batch(const vkq_kv8_cache *c, const vkq_kv8_batch *b, const char *who) {
    if (!b || !b->table || !b->lens) {
        set_error("%s: null batch, table or lens", who);
        return VKQ_ERR_INVALID_ARGUMENT;
    }
    // lengths and positions are int32 on the device
    if (b->rows <= 0 || b->rows > INT32_MAX || b->max_pages <= 0 || b->max_pages > INT32_MAX || b->batch <= 0 ||
        b->batch > 65535 || b->tokens < 0 || b->tokens > INT32_MAX / 2 || b->max_tokens <= 0 ||
        b->max_tokens > INT32_MAX / 2 || b->max_len < 0 || b->max_len > INT32_MAX / 2) {
        set_error("%s: rows %lld, max_pages %lld, batch %lld, tokens %lld, max_tokens %lld or max_len %lld is out of range",
                  who, (long long)b->rows, (long long)b->max_pages, (long long)b->batch, (long long)b->tokens,
                  (long long)b->max_tokens, (long long)b->max_len);
        return VKQ_ERR_INVALID_ARGUMENT;
    }
    if (b->max_len > b->max_pages * (int64_t)c->page_size || (!b->slots && b->batch > b->rows) ||
        (!b->cu_tokens && b->tokens < b->batch)) {
        set_error("%s: max_len %lld does not fit %lld pages of %d, or the batch of %lld its rows or tokens", who,
                  (long long)b->max_len, (long long)b->max_pages, c->page_size, (long long)b->batch);
        return VKQ_ERR_INVALID_ARGUMENT;
    }
    if (misaligned(b->table, 4) || misaligned(b->lens, 4) || misaligned(b->slots, 4) || misaligned(b->cu_tokens, 4)) {
        set_error("%s: the batch's arrays must be 4-byte aligned", who);
        return VKQ_ERR_MISALIGNED;
    }
    return VKQ_OK;
}

static int check_heads(const vkq_kv8_cache *c, const vkq_kv8_batch *b, int64_t heads, const char *who) {
    if (heads <= 0 || heads % c->kv_heads || heads > 65535 || b->max_tokens * (heads / c->kv_heads) > INT32_MAX / 2) {
        set_error("%s: %lld heads are no multiple of %d KV heads, or too many", who, (long long)heads, c->kv_heads);
        return VKQ_ERR_INVALID_ARGUMENT;
    }
    return VKQ_OK;
}

// Whether two of the heads at token * a + head * b, of D values each, share
// values (a, b >= D where there is more than one token or head): only a token
// more and heads less can meet.
static bool heads_meet(int64_t tokens, int64_t a, int64_t heads, int64_t b, int64_t D) {
    if (tokens == 1 || heads == 1 || (a - D) / b >= heads - 1 || (b - D) / a >= tokens - 1) return false;
    if (tokens > heads) return heads_meet(heads, b, tokens, a, D);
    for (int64_t d = 1; d < tokens; d++) {  // tokens * heads is bounded: at most 2^20
        const int64_t k = d * a / b;        // the heads just below and above d tokens on
        if (k >= 1 && k < heads && d * a - k * b < D) return true;
        if (k + 1 < heads && (k + 1) * b - d * a < D) return true;
    }
    return false;
}

// Rows of `heads` heads a token: the stride holds them, the elements are aligned.
static int check_rows(const void *p, int64_t token_stride, int64_t width, int dtype, const char *who, const char *name) {
    if (!p) {
        set_error("%s: null %s", who, name);
        return VKQ_ERR_INVALID_ARGUMENT;
    }
    if (token_stride < width || token_stride > (int64_t(1) << 40)) {
        set_error("%s: token stride %lld of %s is below its %lld values, or too large", who, (long long)token_stride, name,
                  (long long)width);
        return VKQ_ERR_INVALID_ARGUMENT;
    }
    if (misaligned(p, (uintptr_t)act_bytes(dtype))) {
        set_error("%s: %s is not aligned to its elements", who, name);
        return VKQ_ERR_MISALIGNED;
    }
    return VKQ_OK;
}

static int check_seqs(const vkq_kv8_cache *c, const vkq_kv8_seqs *q, const void *ws, size_t ws_bytes, const char *who) {
    if (!q || !q->table || !q->lens || !q->refs || q->rows <= 0 || q->rows > INT32_MAX || q->max_pages <= 0 ||
        q->max_pages > INT32_MAX || q->max_pages * (int64_t)c->page_size > INT32_MAX / 2) {
        set_error("%s: null bookkeeping array, or rows or max_pages out of range (max_pages * page_size below 2^30)", who);
        return VKQ_ERR_INVALID_ARGUMENT;
    }
    if (misaligned(q->table, 4) || misaligned(q->lens, 4) || misaligned(q->refs, 4)) {
        set_error("%s: the bookkeeping arrays must be 4-byte aligned", who);
        return VKQ_ERR_MISALIGNED;
    }
    if (!ws || misaligned(ws, 16) || ws_bytes < kv8_pages_workspace(*c, *q)) {
        set_error("%s: workspace of %zu bytes, 16-byte aligned, needed (got %zu)", who, kv8_pages_workspace(*c, *q),
                  ws ? ws_bytes : (size_t)0);
        return VKQ_ERR_WORKSPACE;
    }
    return VKQ_OK;
}

static int check_list(const vkq_kv8_seqs *q, const int32_t *a, const int32_t *b, const int32_t *done, int64_t n,
                      const char *who) {
    if (!a || !b || n <= 0 || n > q->rows || misaligned(a, 4) || misaligned(b, 4) || misaligned(done, 4)) {
        set_error("%s: null or misaligned list, or its length %lld is not within 1 .. %lld rows", who, (long long)n,
                  (long long)q->rows);
        return VKQ_ERR_INVALID_ARGUMENT;
    }
    return VKQ_OK;
}

}  // namespace vkq

extern "C" {

int vkq_rotary(int device, int dtype, const void *x, int64_t x_token_stride, int64_t x_head_stride, void *out,
               int64_t out_token_stride, int64_t out_head_stride, const float *cos_table, const float *sin_table,
               const int32_t *positions, int64_t tokens, int64_t heads, int64_t head_dim, int64_t rot_dim,
               int64_t max_seq, int layout, int inverse, void *stream) {
    int st = enter(device);
    if (st) return st;
    if ((st = check_dtype(dtype, "vkq_rotary"))) return st;
    const int64_t most = int64_t(1) << 40;
    if (!x || !out || !cos_table || !sin_table || !positions || tokens <= 0 || tokens > INT32_MAX || heads <= 0 ||
        heads > INT32_MAX || head_dim <= 0 || head_dim > 65536 || rot_dim <= 0 || rot_dim % 2 != 0 ||
        rot_dim > head_dim || max_seq <= 0 || tokens * heads > most / head_dim ||
        (layout != VKQ_ROPE_INTERLEAVED && layout != VKQ_ROPE_HALF)) {
        set_error("invalid arguments to vkq_rotary (rot_dim even and at most head_dim, every count positive)");
        return VKQ_ERR_INVALID_ARGUMENT;
    }
    if (x_token_stride < 0 || x_token_stride > most || x_head_stride < 0 || x_head_stride > most ||
        out_token_stride < 0 || out_token_stride > most || out_head_stride < 0 || out_head_stride > most ||
        (heads > 1 && out_head_stride < head_dim) || (tokens > 1 && out_token_stride < head_dim) ||
        heads_meet(tokens, out_token_stride, heads, out_head_stride, head_dim)) {
        set_error("vkq_rotary: strides must not be negative, and the output's heads must not overlap");
        return VKQ_ERR_INVALID_ARGUMENT;
    }
    const uintptr_t size = (uintptr_t)act_bytes(dtype);
    if (misaligned(x, size) || misaligned(out, size) || misaligned(cos_table, 4) || misaligned(sin_table, 4) ||
        misaligned(positions, 4)) {
        set_error("vkq_rotary needs buffers aligned to their elements");
        return VKQ_ERR_MISALIGNED;
    }
    RotaryArgs a{dtype,  x,         x_token_stride, x_head_stride, out,      out_token_stride, out_head_stride, cos_table,
                 sin_table, positions, tokens,         heads,         head_dim, rot_dim,          max_seq,         layout,
                 inverse};
    return check_launch(rotary(a, (cudaStream_t)stream, device), "rotary");
}

int vkq_rotary_tables_f32(int device, float *cos_table, float *sin_table, int64_t max_seq, int64_t rot_dim, double base,
                          int scaling, double factor, int64_t orig_len, double beta_fast, double beta_slow,
                          double attn_factor, void *stream) {
    int st = enter(device);
    if (st) return st;
    if (scaling < VKQ_ROPE_SCALE_NONE || scaling > VKQ_ROPE_SCALE_YARN) {
        set_error("vkq_rotary_tables_f32: unknown scaling %d", scaling);
        return VKQ_ERR_UNSUPPORTED;
    }
    if (!cos_table || !sin_table || max_seq <= 0 || rot_dim <= 0 || rot_dim % 2 != 0 || rot_dim > 65536 ||
        max_seq > (int64_t(1) << 40) / rot_dim || !(base > 1.0) || !std::isfinite(base) ||
        (scaling != VKQ_ROPE_SCALE_NONE && (!(factor >= 1.0) || !std::isfinite(factor))) ||
        (scaling == VKQ_ROPE_SCALE_NTK && rot_dim < 4) ||
        (scaling == VKQ_ROPE_SCALE_YARN && (orig_len <= 0 || !(beta_slow > 0.0) || !(beta_fast > beta_slow) ||
                                            !std::isfinite(beta_fast) || !(attn_factor >= 0.0) || !std::isfinite(attn_factor)))) {
        set_error("invalid arguments to vkq_rotary_tables_f32");
        return VKQ_ERR_INVALID_ARGUMENT;
    }
    if (misaligned(cos_table, 4) || misaligned(sin_table, 4)) {
        set_error("vkq_rotary_tables_f32 needs 4-byte aligned tables");
        return VKQ_ERR_MISALIGNED;
    }
    return check_launch(rotary_tables(cos_table, sin_table, max_seq, rot_dim, base, scaling, factor, orig_len, beta_fast,
                                      beta_slow, attn_factor, (cudaStream_t)stream, device),
                        "rotary tables");
}

int vkq_kv8_append(int device, const vkq_kv8_cache *cache, int64_t layer, const vkq_kv8_batch *batch, int dtype,
                   const void *k, int64_t k_token_stride, const void *v, int64_t v_token_stride, const void *q,
                   int64_t q_token_stride, void *q_out, int64_t q_out_token_stride, int64_t heads,
                   const float *cos_table, const float *sin_table, int64_t max_seq, int64_t rot_dim, int layout,
                   void *stream) {
    const char *who = "vkq_kv8_append";
    int st = enter(device);
    if (st) return st;
    if ((st = check_dtype(dtype, who))) return st;
    if ((st = check_cache(cache, layer, who))) return st;
    if ((st = check_batch(cache, batch, who))) return st;
    const int64_t width = (int64_t)cache->kv_heads * cache->head_dim;
    if ((st = check_rows(k, k_token_stride, width, dtype, who, "k"))) return st;
    if ((st = check_rows(v, v_token_stride, width, dtype, who, "v"))) return st;
    if (!cos_table != !sin_table || (q && !cos_table)) {
        set_error("%s: both tables or neither, and both to rotate q", who);
        return VKQ_ERR_INVALID_ARGUMENT;
    }
    if (cos_table) {
        if (max_seq <= 0 || rot_dim <= 0 || rot_dim % 2 || rot_dim > cache->head_dim ||
            (layout != VKQ_ROPE_INTERLEAVED && layout != VKQ_ROPE_HALF)) {
            set_error("%s: max_seq, rot_dim (even, at most head_dim) or layout is out of range", who);
            return VKQ_ERR_INVALID_ARGUMENT;
        }
        if (misaligned(cos_table, 4) || misaligned(sin_table, 4)) {
            set_error("%s needs 4-byte aligned tables", who);
            return VKQ_ERR_MISALIGNED;
        }
    }
    if (q) {
        if ((st = check_heads(cache, batch, heads, who))) return st;
        const int64_t qw = heads * cache->head_dim;
        if ((st = check_rows(q, q_token_stride, qw, dtype, who, "q"))) return st;
        if ((st = check_rows(q_out, q_out_token_stride, qw, dtype, who, "q_out"))) return st;
        if (q == q_out && q_token_stride != q_out_token_stride) {
            set_error("%s: q_out is q with another stride", who);
            return VKQ_ERR_INVALID_ARGUMENT;
        }
    }
    if (batch->tokens == 0) return VKQ_OK;
    if (kv8_append_ctas(*cache, *batch, q != nullptr) > INT32_MAX) {
        set_error("%s: batch of %lld sequences of up to %lld tokens is too large for one call", who,
                  (long long)batch->batch, (long long)batch->max_tokens);
        return VKQ_ERR_UNSUPPORTED;
    }
    Kv8AppendArgs a{dtype,     k,         v,       q,       k_token_stride, v_token_stride, q_token_stride, q_out, q_out_token_stride,
                    heads, cos_table, sin_table, max_seq, rot_dim, layout};
    return check_launch(kv8_append(*cache, layer, *batch, a, (cudaStream_t)stream, device), "KV cache append");
}

int vkq_kv8_read(int device, const vkq_kv8_cache *cache, int64_t layer, const vkq_kv8_batch *batch, const int32_t *seq,
                 const int32_t *pos, int64_t n, int dtype, void *k_out, void *v_out, void *stream) {
    const char *who = "vkq_kv8_read";
    int st = enter(device);
    if (st) return st;
    if ((st = check_dtype(dtype, who))) return st;
    if ((st = check_cache(cache, layer, who))) return st;
    if ((st = check_batch(cache, batch, who))) return st;
    if (!seq || !pos || n <= 0 || n > INT32_MAX || (!k_out && !v_out)) {
        set_error("%s: null list or outputs, or a count of %lld", who, (long long)n);
        return VKQ_ERR_INVALID_ARGUMENT;
    }
    if (misaligned(seq, 4) || misaligned(pos, 4) || misaligned(k_out, 16) || misaligned(v_out, 16)) {
        set_error("%s: the lists must be 4-byte and the outputs 16-byte aligned", who);
        return VKQ_ERR_MISALIGNED;
    }
    return check_launch(kv8_read(*cache, layer, *batch, seq, pos, n, dtype, k_out, v_out, (cudaStream_t)stream),
                        "KV cache read");
}

static int check_attention(const vkq_kv8_cache *cache, int64_t layer, const vkq_kv8_batch *batch, int dtype, int64_t heads,
                           int causal, int64_t window, const char *who) {
    int st;
    if ((st = check_dtype(dtype, who))) return st;
    if ((st = check_cache(cache, layer, who))) return st;
    if ((st = check_batch(cache, batch, who))) return st;
    if ((st = check_heads(cache, batch, heads, who))) return st;
    if (window < 0 || window > INT32_MAX / 2 || (window > 0 && !causal)) {
        set_error("%s: window %lld is out of range, or given without causal", who, (long long)window);
        return VKQ_ERR_INVALID_ARGUMENT;
    }
    return VKQ_OK;
}

// The workspace's size, or an error for bounds whose launch no grid holds.
static int attention_workspace(const vkq_kv8_cache *cache, const vkq_kv8_batch *batch, int dtype, int64_t heads, int causal,
                               int64_t window, int device, const char *who, size_t *bytes) {
    int64_t ctas = 0;
    *bytes = kv8_attention_workspace(*cache, *batch, dtype, heads, causal, window, device, &ctas);
    if (ctas <= INT32_MAX) return VKQ_OK;
    set_error("%s: batch of %lld sequences of up to %lld tokens and %lld heads is too large for one call", who,
              (long long)batch->batch, (long long)batch->max_tokens, (long long)heads);
    return VKQ_ERR_UNSUPPORTED;
}

int vkq_kv8_attention_workspace_bytes(int device, const vkq_kv8_cache *cache, const vkq_kv8_batch *batch, int dtype,
                                      int64_t heads, int causal, int64_t window, size_t *bytes) {
    int st = enter(device);
    if (st) return st;
    const char *who = "vkq_kv8_attention_workspace_bytes";
    if ((st = check_attention(cache, 0, batch, dtype, heads, causal, window, who))) return st;
    if (!bytes) {
        set_error("%s: null bytes", who);
        return VKQ_ERR_INVALID_ARGUMENT;
    }
    return attention_workspace(cache, batch, dtype, heads, causal, window, device, who, bytes);
}

int vkq_kv8_attention(int device, const vkq_kv8_cache *cache, int64_t layer, const vkq_kv8_batch *batch, int dtype,
                      const void *q, int64_t q_token_stride, void *out, int64_t out_token_stride, int64_t heads,
                      float scale, int causal, int64_t window, void *workspace, size_t workspace_bytes, void *stream) {
    const char *who = "vkq_kv8_attention";
    int st = enter(device);
    if (st) return st;
    if ((st = check_attention(cache, layer, batch, dtype, heads, causal, window, who))) return st;
    const int64_t width = heads * cache->head_dim;
    if ((st = check_rows(q, q_token_stride, width, dtype, who, "q"))) return st;
    if ((st = check_rows(out, out_token_stride, width, dtype, who, "out"))) return st;
    if (!(scale > 0.f) || !std::isfinite(scale)) {
        set_error("%s: scale must be positive and finite", who);
        return VKQ_ERR_INVALID_ARGUMENT;
    }
    if (batch->tokens == 0) return VKQ_OK;
    size_t need = 0;
    if ((st = attention_workspace(cache, batch, dtype, heads, causal, window, device, who, &need))) return st;
    if (!workspace || misaligned(workspace, 16) || workspace_bytes < need) {
        set_error("%s: workspace of %zu bytes, 16-byte aligned, needed (got %zu)", who, need,
                  workspace ? workspace_bytes : (size_t)0);
        return VKQ_ERR_WORKSPACE;
    }
    Kv8AttentionArgs a{dtype, q, q_token_stride, out, out_token_stride, heads, scale, causal != 0, window, workspace};
    return check_launch(kv8_attention(*cache, layer, *batch, a, (cudaStream_t)stream, device), "KV cache attention");
}

int vkq_kv8_pages_workspace_bytes(const vkq_kv8_cache *cache, const vkq_kv8_seqs *seqs, size_t *bytes) {
    if (!cache || !seqs || !bytes || cache->num_pages <= 0 || cache->num_pages > INT32_MAX || seqs->rows <= 0 ||
        seqs->rows > INT32_MAX) {
        set_error("invalid arguments to vkq_kv8_pages_workspace_bytes");
        return VKQ_ERR_INVALID_ARGUMENT;
    }
    *bytes = kv8_pages_workspace(*cache, *seqs);
    return VKQ_OK;
}

int vkq_kv8_extend(int device, const vkq_kv8_cache *cache, const vkq_kv8_seqs *seqs, const int32_t *slots,
                   const int32_t *add, int64_t n, int32_t *done, void *workspace, size_t workspace_bytes, void *stream) {
    const char *who = "vkq_kv8_extend";
    int st = enter(device);
    if (st) return st;
    if ((st = check_cache(cache, 0, who))) return st;
    if ((st = check_seqs(cache, seqs, workspace, workspace_bytes, who))) return st;
    if ((st = check_list(seqs, slots, add, done, n, who))) return st;
    return check_launch(kv8_extend(*cache, *seqs, slots, add, n, done, workspace, (cudaStream_t)stream), "KV pages extend");
}

int vkq_kv8_fork(int device, const vkq_kv8_cache *cache, const vkq_kv8_seqs *seqs, const int32_t *src, const int32_t *dst,
                 int64_t n, int32_t *done, void *workspace, size_t workspace_bytes, void *stream) {
    const char *who = "vkq_kv8_fork";
    int st = enter(device);
    if (st) return st;
    if ((st = check_cache(cache, 0, who))) return st;
    if ((st = check_seqs(cache, seqs, workspace, workspace_bytes, who))) return st;
    if ((st = check_list(seqs, src, dst, done, n, who))) return st;
    return check_launch(kv8_fork(*cache, *seqs, src, dst, n, done, workspace, (cudaStream_t)stream, device),
                        "KV pages fork");
}

int vkq_kv8_free(int device, const vkq_kv8_cache *cache, const vkq_kv8_seqs *seqs, const int32_t *slots, int64_t n,
                 int32_t *done, void *workspace, size_t workspace_bytes, void *stream) {
    const char *who = "vkq_kv8_free";
    int st = enter(device);
    if (st) return st;
    if ((st = check_cache(cache, 0, who))) return st;
    if ((st = check_seqs(cache, seqs, workspace, workspace_bytes, who))) return st;
    if ((st = check_list(seqs, slots, slots, done, n, who))) return st;
    return check_launch(kv8_free(*cache, *seqs, slots, n, done, workspace, (cudaStream_t)stream), "KV pages free");
}

int vkq_kv8_compact(int device, const vkq_kv8_cache *cache, const vkq_kv8_seqs *seqs, int32_t *used, void *workspace,
                    size_t workspace_bytes, void *stream) {
    const char *who = "vkq_kv8_compact";
    int st = enter(device);
    if (st) return st;
    if ((st = check_cache(cache, 0, who))) return st;
    if ((st = check_seqs(cache, seqs, workspace, workspace_bytes, who))) return st;
    if (misaligned(used, 4)) {
        set_error("%s: used must be 4-byte aligned", who);
        return VKQ_ERR_MISALIGNED;
    }
    return check_launch(kv8_compact(*cache, *seqs, used, workspace, (cudaStream_t)stream, device), "KV pages compact");
}

int vkq_kv8_copy_pages(int device, const vkq_kv8_cache *cache, const int32_t *src, const int32_t *dst, int64_t n,
                       void *stream) {
    const char *who = "vkq_kv8_copy_pages";
    int st = enter(device);
    if (st) return st;
    if ((st = check_cache(cache, 0, who))) return st;
    if (!src || !dst || n <= 0 || n > cache->num_pages || misaligned(src, 4) || misaligned(dst, 4)) {
        set_error("%s: null or misaligned list, or its length %lld is not within 1 .. %lld pages", who, (long long)n,
                  (long long)cache->num_pages);
        return VKQ_ERR_INVALID_ARGUMENT;
    }
    return check_launch(kv8_copy_pages(*cache, src, dst, n, (cudaStream_t)stream, device), "KV pages copy");
}

}  // extern "C"
