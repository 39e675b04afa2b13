// extern "C" entry points of the paged serving step: argument checks, then
// the launches of pages.cu, kv4.cu, kv4_attention.cu and sample_rows.cu.
#include <string>

#include "serve.cuh"

using namespace ifx;

namespace {

cudaStream_t S(void *s) { return reinterpret_cast<cudaStream_t>(s); }

bool aligned(const void *p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

ifx_status bad(const char *what) { return fail(IFX_ERR_INVALID_ARGUMENT, what); }

constexpr size_t kIntMax = 0x7fffffff;
constexpr size_t kMaxPoolPages = kIntMax / kKv4PageRows;  // slots are int32

ifx_status check_pool(size_t n_seqs, size_t most, size_t max_pages, size_t n_pages, const char *name) {
  const std::string n(name);
  if (n_seqs > most) return fail(IFX_ERR_INVALID_ARGUMENT, n + ": more than " + std::to_string(most) + " sequences");
  if (max_pages > kMaxPoolPages || n_pages > kMaxPoolPages)
    return fail(IFX_ERR_INVALID_ARGUMENT, n + ": too many pages for 32-bit slots");
  return IFX_OK;
}

ifx_status check_kv4(int type, size_t n_pages, size_t G, size_t hd, const char *name) {
  const std::string n(name);
  if (type != IFX_TYPE_F32 && type != IFX_TYPE_F16)
    return fail(IFX_ERR_UNSUPPORTED, n + ": rows are F32 or F16");
  if (!kv4_head_dim_ok(hd))
    return fail(IFX_ERR_UNSUPPORTED, n + ": head_dim must be a multiple of 32, at most 256");
  if (!G || G > 1024) return fail(IFX_ERR_SHAPE, n + ": 1 to 1024 kv heads");
  if (n_pages > kMaxPoolPages) return fail(IFX_ERR_INVALID_ARGUMENT, n + ": too many pages for 32-bit slots");
  return IFX_OK;
}

size_t type_size(int type) { return type == IFX_TYPE_F16 ? 2 : 4; }

}  // namespace

extern "C" {

ifx_status ifx_op_pages_extend(const int32_t *lens, const int32_t *add, size_t n_seqs, int32_t *table,
                               size_t max_pages, const int32_t *free_pages, size_t n_pages,
                               const int32_t *n_free, size_t max_tokens, int32_t *lens_out,
                               int32_t *n_free_out, int32_t *q_start, int32_t *slots, int32_t *positions,
                               int32_t *seqs, int32_t *status, void *stream) {
  if (!n_free || !n_free_out || !q_start || !status || (n_seqs && (!lens || !add || !lens_out)) ||
      (n_seqs && max_pages && !table) || (n_pages && !free_pages) || (max_tokens && !slots))
    return bad("pages_extend: null");
  if (lens_out == lens && n_seqs) return bad("pages_extend: lens_out is lens");
  if (n_free_out == n_free) return bad("pages_extend: n_free_out is n_free");
  IFX_TRY(check_pool(n_seqs, kMaxServeSeqs, max_pages, n_pages, "pages_extend"));
  if (max_tokens > kIntMax) return bad("pages_extend: max_tokens above 2^31 - 1");
  PagesExtendArgs a{lens, add, (int)n_seqs, table, (int)max_pages, free_pages, (int)n_pages, n_free,
                    (int64_t)max_tokens, lens_out, n_free_out, q_start, slots, positions, seqs, status};
  return op_pages_extend(a, S(stream));
}

ifx_status ifx_op_pages_release(const int32_t *done, const int32_t *lens, size_t n_seqs, const int32_t *table,
                                size_t max_pages, int32_t *free_pages, size_t n_pages, const int32_t *n_free,
                                int32_t *lens_out, int32_t *n_free_out, void *stream) {
  if (!n_free || !n_free_out || (n_seqs && (!done || !lens || !lens_out)) || (n_seqs && max_pages && !table) ||
      (n_pages && !free_pages))
    return bad("pages_release: null");
  if (lens_out == lens && n_seqs) return bad("pages_release: lens_out is lens");
  if (n_free_out == n_free) return bad("pages_release: n_free_out is n_free");
  IFX_TRY(check_pool(n_seqs, kMaxServeSeqs, max_pages, n_pages, "pages_release"));
  PagesReleaseArgs a{done, lens, (int)n_seqs, table, (int)max_pages, free_pages, (int)n_pages, n_free, lens_out, n_free_out};
  return op_pages_release(a, S(stream));
}

size_t ifx_kv4_page_bytes(size_t n_kv_heads, size_t head_dim) {
  if (!n_kv_heads || n_kv_heads > 1024 || !kv4_head_dim_ok(head_dim)) return 0;
  return kv4_page_bytes(n_kv_heads, head_dim);
}

ifx_status ifx_op_kv4_store(int type, const void *k, size_t k_stride, const void *v, size_t v_stride,
                            const int32_t *slots, size_t n, void *pages, size_t n_pages, size_t n_kv_heads,
                            size_t head_dim, void *stream) {
  IFX_TRY(check_kv4(type, n_pages, n_kv_heads, head_dim, "kv4_store"));
  if (!n) return IFX_OK;
  if (!k || !v || !slots || (n_pages && !pages)) return bad("kv4_store: null");
  const size_t w = n_kv_heads * head_dim, ts = type_size(type);
  if (k_stride < w || v_stride < w) return fail(IFX_ERR_SHAPE, "kv4_store: rows overlap");
  if (!aligned(k, 16) || !aligned(v, 16) || !aligned(pages, 16) || k_stride * ts % 16 || v_stride * ts % 16)
    return bad("kv4_store: rows and pages must be 16-byte aligned");
  if (n > kIntMax) return bad("kv4_store: more than 2^31 - 1 rows");
  Kv4RowsArgs a{k, v, nullptr, nullptr, type, (int64_t)n, (int64_t)k_stride, (int64_t)v_stride, slots,
                static_cast<uint8_t *>(pages), (int64_t)n_pages, (int)n_kv_heads, (int)head_dim};
  return op_kv4_store(a, S(stream));
}

ifx_status ifx_op_kv4_load(int type, const void *pages, size_t n_pages, size_t n_kv_heads, size_t head_dim,
                           const int32_t *slots, size_t n, void *k, void *v, void *stream) {
  IFX_TRY(check_kv4(type, n_pages, n_kv_heads, head_dim, "kv4_load"));
  if (!n) return IFX_OK;
  if (!k || !v || !slots || (n_pages && !pages)) return bad("kv4_load: null");
  if (!aligned(k, 16) || !aligned(v, 16) || !aligned(pages, 16))
    return bad("kv4_load: rows and pages must be 16-byte aligned");
  if (n > kIntMax) return bad("kv4_load: more than 2^31 - 1 rows");
  Kv4RowsArgs a{nullptr, nullptr, k, v, type, (int64_t)n, 0, 0, slots,
                static_cast<uint8_t *>(const_cast<void *>(pages)), (int64_t)n_pages, (int)n_kv_heads, (int)head_dim};
  return op_kv4_load(a, S(stream));
}

size_t ifx_kv4_attention_workspace(size_t n_heads, size_t n_kv_heads, size_t head_dim) {
  if (!n_kv_heads || n_kv_heads > 1024 || n_heads > 65536 || n_heads % n_kv_heads || !kv4_head_dim_ok(head_dim)) return 0;
  return kv4_attention_ws((int)n_heads, (int)n_kv_heads, (int)head_dim);
}

ifx_status ifx_op_kv4_attention(int type, const void *q, size_t q_stride, size_t rows, const void *pages,
                                size_t n_pages, const int32_t *table, size_t max_pages, const int32_t *kv_len,
                                const int32_t *q_start, size_t n_seqs, size_t n_heads, size_t n_kv_heads,
                                size_t head_dim, float scale, size_t window, void *out, size_t out_stride,
                                int zero_rest, void *ws, size_t ws_bytes, void *stream) {
  IFX_TRY(check_kv4(type, n_pages, n_kv_heads, head_dim, "kv4_attention"));
  if (!n_heads || n_heads > 65536 || n_heads % n_kv_heads)
    return fail(IFX_ERR_SHAPE, "kv4_attention: query heads must be a multiple of the kv heads");
  if (!q_start && rows != n_seqs) return fail(IFX_ERR_SHAPE, "kv4_attention: one row per sequence without q_start");
  if (!rows || (!n_seqs && !zero_rest)) return IFX_OK;
  if (!q || !out || (n_seqs && (!kv_len || (max_pages && !table))) || (n_pages && !pages)) return bad("kv4_attention: null");
  const size_t w = n_heads * head_dim, ts = type_size(type);
  if (q_stride < w || out_stride < w) return fail(IFX_ERR_SHAPE, "kv4_attention: rows overlap");
  if (!aligned(q, 16) || !aligned(out, 16) || !aligned(pages, 16) || q_stride * ts % 16 || out_stride * ts % 16)
    return bad("kv4_attention: rows and pages must be 16-byte aligned");
  IFX_TRY(check_pool(n_seqs, kMaxAttnSeqs, max_pages, n_pages, "kv4_attention"));
  if (rows > kIntMax || rows * n_heads > kIntMax) return bad("kv4_attention: too many rows");
  if (!(scale == scale) || scale - scale != 0.f) return bad("kv4_attention: scale is not finite");
  if (ws_bytes < kv4_attention_ws((int)n_heads, (int)n_kv_heads, (int)head_dim) || (ws_bytes && (!ws || !aligned(ws, 256))))
    return bad("kv4_attention: workspace too small or not 256-byte aligned");
  if (!n_seqs) {
    IFX_CUDA(cudaMemset2DAsync(out, out_stride * ts, 0, w * ts, rows, S(stream)));
    return IFX_OK;
  }
  // a window that no sequence outgrows is none (and differences with one stay within 32 bits)
  const int seen = window >= max_pages * kKv4PageRows ? 0 : (int)window;
  Kv4AttnArgs a{q, out, type, (int64_t)q_stride, (int64_t)out_stride, (int64_t)rows,
                static_cast<const uint8_t *>(pages), (int64_t)n_pages, table, kv_len, q_start, (int)max_pages,
                (int)n_seqs, (int)n_heads, (int)n_kv_heads, (int)head_dim,
                seen, scale, ws, zero_rest != 0 && q_start};
  return op_kv4_attention(a, S(stream));
}

ifx_status ifx_op_sample_rows(const float *logits, size_t stride, size_t rows, size_t n, const float *u,
                              const float *temperature, const int32_t *top_k, const float *top_p,
                              const float *min_p, int32_t *token, float *logprob, void *stream) {
  if (!n) return fail(IFX_ERR_SHAPE, "sample_rows: empty logits");
  if (n > IFX_SAMPLE_ROWS_MAX) return bad("sample_rows: more than IFX_SAMPLE_ROWS_MAX logits in a row");
  if (stride < n) return fail(IFX_ERR_SHAPE, "sample_rows: rows overlap");
  if (!rows) return IFX_OK;
  if (rows > (size_t)kIntMax / 32) return bad("sample_rows: too many rows");
  if (!logits || !u || !token) return bad("sample_rows: null");
  SampleRowsArgs a{logits, (int64_t)rows, (int64_t)n, (int64_t)stride, u, temperature, top_k, top_p, min_p, token, logprob};
  return op_sample_rows(a, S(stream));
}

}  // extern "C"
