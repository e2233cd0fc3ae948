// extern "C" entry points of the serving operators: argument checks and
// workspaces.  Kernels in serve_rope.hip, serve_decode.hip, serve_prompt.hip and
// serve_sample.hip.
#include "kernels.h"
#include "serving.h"

namespace {

constexpr int kMaxSeq = 8192;
constexpr int kMaxVocab = 1 << 21;

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

int check_heads(const char* fn, int n_head, int n_head_kv, int head_dim) {
  if (n_head <= 0 || n_head_kv <= 0 || n_head % n_head_kv)
    return gm_fail_arg("%s: n_head=%d must be a positive multiple of n_head_kv=%d", fn, n_head, n_head_kv);
  if (head_dim != 64 && head_dim != 128 && head_dim != 256)
    return gm_fail_arg("%s: head_dim=%d must be 64, 128 or 256", fn, head_dim);
  if ((int64_t)n_head * head_dim > 1 << 24) return gm_fail_arg("%s: n_head=%d too large", fn, n_head);
  return GM_OK;
}

// A cache's pages and the tables into them: row numbers and positions are int32.
int check_pages(const char* fn, int n_pages, int page_size, int table_width, int64_t table_stride, int n_seq) {
  if (n_pages <= 0 || page_size <= 0) return gm_fail_arg("%s: n_pages and page_size must be positive", fn);
  if ((int64_t)n_pages * page_size > 0x7fffffff) return gm_fail_arg("%s: more than 2^31 - 1 cache rows", fn);
  if (table_width < 0 || table_stride < table_width)
    return gm_fail_arg("%s: table_stride must be at least table_width, which must not be negative", fn);
  if (((int64_t)table_width * page_size + 31) / 32 * n_seq > 0x7fffffff)
    return gm_fail_arg("%s: n_seq x table_width x page_size above 2^36 positions", fn);
  return GM_OK;
}

int check_paged(const gm_paged_attn_args* a) {
  const char* fn = "gm_paged_attention";
  if (!a) return gm_fail_arg("%s: NULL arguments", fn);
  if (int rc = check_heads(fn, a->n_head, a->n_head_kv, a->head_dim)) return rc;
  if (a->n_seq < 0 || a->n_seq > kMaxSeq) return gm_fail_arg("%s: n_seq=%d must be 0 .. %d", fn, a->n_seq, kMaxSeq);
  if (int rc = check_pages(fn, a->n_pages, a->page_size, a->table_width, a->table_stride, a->n_seq)) return rc;
  if (!gm_is_t16(a->cache_type)) return gm_fail_arg("%s: cache_type %d must be F16 or BF16", fn, a->cache_type);
  if (a->q_type != GM_QTYPE_F32 && a->q_type != a->cache_type)
    return gm_fail_arg("%s: q_type %d must be F32 or the cache's type", fn, a->q_type);
  if (!(a->scale > 0.f) || a->scale > 3e38f) return gm_fail_arg("%s: scale must be positive and finite", fn);
  if ((int64_t)a->n_seq * a->n_head > 0x7fffffff) return gm_fail_arg("%s: n_seq x n_head too large", fn);
  return GM_OK;
}

int check_sample(const gm_sample_args* a) {
  if (!a) return gm_fail_arg("gm_sample: NULL arguments");
  if (a->n_row < 0 || a->n_row > 65535) return gm_fail_arg("gm_sample: n_row=%d must be 0 .. 65535", a->n_row);
  if (a->vocab <= 0 || a->vocab > kMaxVocab)
    return gm_fail_arg("gm_sample: vocab=%d must be 1 .. %d", a->vocab, kMaxVocab);
  if (!gm_is_elem(a->type)) return gm_fail_arg("gm_sample: type %d must be F32, F16 or BF16", a->type);
  if (a->row_stride < 0) return gm_fail_arg("gm_sample: negative row_stride");
  return GM_OK;
}

hipStream_t as_stream(void* s) { return reinterpret_cast<hipStream_t>(s); }

}  // namespace

extern "C" {

int gm_rope_append(const gm_rope_append_args* a, void* stream) {
  const char* fn = "gm_rope_append";
  if (!a) return gm_fail_arg("%s: NULL arguments", fn);
  if (int rc = check_heads(fn, a->n_head, a->n_head_kv, a->head_dim)) return rc;
  if (a->T < 0 || a->n_axes < 1) return gm_fail_arg("%s: negative T or no axis", fn);
  if (a->rope_dim < 0 || a->rope_dim % 2 || a->rope_dim > a->head_dim)
    return gm_fail_arg("%s: rope_dim=%d must be even and 0 .. head_dim=%d", fn, a->rope_dim, a->head_dim);
  if (!gm_is_elem(a->in_type)) return gm_fail_arg("%s: in_type %d must be F32, F16 or BF16", fn, a->in_type);
  if (!gm_is_t16(a->cache_type)) return gm_fail_arg("%s: cache_type %d must be F16 or BF16", fn, a->cache_type);
  if (!gm_is_elem(a->out_type)) return gm_fail_arg("%s: out_type %d must be F32, F16 or BF16", fn, a->out_type);
  if (!(a->eps >= 0.f)) return gm_fail_arg("%s: eps must be >= 0", fn);
  if (a->n_rows < 0 || a->n_rows > 0x7fffffff) return gm_fail_arg("%s: n_rows must be 0 .. 2^31 - 1", fn);
  if (a->T == 0) return GM_OK;
  if (!a->q || !a->k || !a->v || !a->positions || !a->q_out || !a->slots || (a->rope_dim && !a->inv_freq) ||
      (a->n_rows && (!a->k_pages || !a->v_pages)))
    return gm_fail_arg("%s: NULL pointer", fn);
  if (!aligned16(a->q_out) || !aligned16(a->k_pages) || !aligned16(a->v_pages))
    return gm_fail_arg("%s: q_out, k_pages and v_pages must be 16-byte aligned", fn);
  return gm_rope_append_run(a, as_stream(stream));
}

size_t gm_paged_attention_workspace_bytes(const gm_paged_attn_args* a) {
  return check_paged(a) ? 0 : gm_paged_attn_ws(a);
}

int gm_paged_attention(const gm_paged_attn_args* a, void* ws, size_t ws_bytes, void* stream) {
  const char* fn = "gm_paged_attention";
  if (int rc = check_paged(a)) return rc;
  if (a->n_seq == 0) return GM_OK;
  if (!a->q || !a->k_pages || !a->v_pages || (a->table_width && !a->block_table) || !a->lengths || !a->out || !ws)
    return gm_fail_arg("%s: NULL pointer", fn);
  if (!aligned16(a->k_pages) || !aligned16(a->v_pages) || !aligned16(a->out))
    return gm_fail_arg("%s: k_pages, v_pages and out must be 16-byte aligned", fn);
  if (a->gate && !gm_is_elem(a->gate_type))
    return gm_fail_arg("%s: gate_type %d must be F32, F16 or BF16", fn, a->gate_type);
  const size_t need = gm_paged_attn_ws(a);
  if (ws_bytes < need) return gm_fail_arg("%s: workspace %zu bytes < %zu needed", fn, ws_bytes, need), GM_EWORKSPACE;
  if (reinterpret_cast<uintptr_t>(ws) % 256) return gm_fail_arg("%s: workspace must be 256-byte aligned", fn);
  return gm_paged_attn_run(a, static_cast<uint8_t*>(ws), as_stream(stream));
}

int gm_prompt_attention(const gm_prompt_attn_args* a, void* stream) {
  const char* fn = "gm_prompt_attention";
  if (!a) return gm_fail_arg("%s: NULL arguments", fn);
  if (int rc = check_heads(fn, a->n_head, a->n_head_kv, a->head_dim)) return rc;
  if (a->n_q < 0 || a->n_k < 0) return gm_fail_arg("%s: negative n_q or n_k", fn);
  if (a->n_seq < 0 || a->n_seq > kMaxSeq) return gm_fail_arg("%s: n_seq=%d must be 0 .. %d", fn, a->n_seq, kMaxSeq);
  if ((int64_t)a->n_q * a->n_head > 0x7fffff00) return gm_fail_arg("%s: n_q x n_head above 2^31", fn);
  if (!gm_is_t16(a->type)) return gm_fail_arg("%s: type %d must be F16 or BF16", fn, a->type);
  if (!(a->scale > 0.f) || a->scale > 3e38f) return gm_fail_arg("%s: scale must be positive and finite", fn);
  if (a->block_table || a->lengths) {
    if (!a->block_table || !a->lengths || a->cu_k)
      return gm_fail_arg("%s: keys are packed (cu_k) or in pages (block_table and lengths)", fn);
    if (int rc = check_pages(fn, a->n_pages, a->page_size, a->table_width, a->table_stride, a->n_seq)) return rc;
  }
  if (a->n_q == 0 || a->n_seq == 0) return GM_OK;
  if (!a->q || !a->k || !a->v || !a->cu_q || (!a->block_table && !a->cu_k) || !a->out)
    return gm_fail_arg("%s: NULL pointer", fn);
  if (!a->block_table && (!gm_rows_aligned(a->k, a->type, a->k_stride_t, a->k_stride_h) ||
                          !gm_rows_aligned(a->v, a->type, a->v_stride_t, a->v_stride_h)))
    return gm_fail_arg("%s: rows of k and v must be 16-byte aligned", fn);
  if (!aligned16(a->k) || !aligned16(a->v) || !aligned16(a->out))
    return gm_fail_arg("%s: k, v and out must be 16-byte aligned", fn);
  if (a->gate && !gm_is_elem(a->gate_type))
    return gm_fail_arg("%s: gate_type %d must be F32, F16 or BF16", fn, a->gate_type);
  return gm_prompt_attn_run(a, as_stream(stream));
}

size_t gm_sample_workspace_bytes(const gm_sample_args* a) { return check_sample(a) ? 0 : gm_sample_ws(a); }

int gm_sample(const gm_sample_args* a, void* ws, size_t ws_bytes, void* stream) {
  if (int rc = check_sample(a)) return rc;
  if (a->n_row == 0) return GM_OK;
  if (!a->logits || !a->u || !a->ids || !ws) return gm_fail_arg("gm_sample: NULL pointer");
  if (reinterpret_cast<uintptr_t>(a->logits) % gm_elem_bytes(a->type))
    return gm_fail_arg("gm_sample: logits must be aligned to their type");
  const size_t need = gm_sample_ws(a);
  if (ws_bytes < need) return gm_fail_arg("gm_sample: workspace %zu bytes < %zu needed", ws_bytes, need), GM_EWORKSPACE;
  if (reinterpret_cast<uintptr_t>(ws) % 256) return gm_fail_arg("gm_sample: workspace must be 256-byte aligned");
  return gm_sample_run(a, static_cast<uint8_t*>(ws), as_stream(stream));
}

}  // extern "C"
