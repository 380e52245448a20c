// paged_host.cc -- C entry points of the paged KV cache (rpgc_paged_*, rpgc_paged8_*,
// rpgc_attention_prompt): every check of the arguments, then the launch.  The
// kernels read lengths, tables and page ids on the device and bound them there.
#include <cmath>
#include <cstdarg>
#include <cstdint>
#include <cstdio>
#include <exception>
#include <string>

#include "../../include/rpgc.h"
#include "kernels.h"

namespace rpgc {
void set_last_error(const char* msg);  // engine.cu
}

namespace {

using rpgc::PagedAttnArgs;
using rpgc::PagedSeqs;
using rpgc::PagedView;

struct Failure {
  int code;
  std::string msg;
};

[[noreturn]] void fail(int code, const char* fmt, ...) __attribute__((format(printf, 2, 3)));
[[noreturn]] void fail(int code, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  std::vsnprintf(buf, sizeof buf, fmt, ap);
  va_end(ap);
  throw Failure{code, buf};
}

template <typename T, typename F>
T guard(F&& f) {
  try {
    rpgc::set_last_error("");
    return f();
  } catch (const Failure& e) {
    rpgc::set_last_error(e.msg.c_str());
    return e.code;
  } catch (const std::exception& e) {
    rpgc::set_last_error(e.what());
    return RPGC_E_CUDA;
  } catch (...) {
    rpgc::set_last_error("unknown exception");
    return RPGC_E_CUDA;
  }
}

void check(cudaError_t e, const char* what) {
  if (e != cudaSuccess)
    fail(e == cudaErrorInvalidValue ? RPGC_E_ARG : e == cudaErrorMemoryAllocation ? RPGC_E_OOM : RPGC_E_CUDA, "%s: %s", what,
         cudaGetErrorString(e));
}

void need_ptr(const void* p, const char* what) {
  if (!p) fail(RPGC_E_ARG, "%s is NULL", what);
  if (reinterpret_cast<uintptr_t>(p) & 15) fail(RPGC_E_ARG, "%s must be 16-byte aligned", what);
}

void need_words(const void* p, const char* what) {
  if (reinterpret_cast<uintptr_t>(p) & 3) fail(RPGC_E_ARG, "%s must be 4-byte aligned", what);
}

// A stride in elements of `size` bytes: not negative, a multiple of 16
// bytes, and small enough that no product with a count overflows.
void need_stride(int64_t st, int size, const char* what) {
  if (st < 0 || st % (16 / size) || st > (int64_t(1) << 40))
    fail(RPGC_E_ARG, "%s: stride %lld must be a multiple of %d elements, not negative", what, (long long)st, 16 / size);
}

void need_heads(int32_t n_heads, int32_t n_kv, int32_t hd) {
  if (hd != 64 && hd != 128) fail(RPGC_E_ARG, "head_dim %d: 64 and 128 are supported", hd);
  if (n_kv <= 0 || n_kv > 4096) fail(RPGC_E_ARG, "n_kv_heads %d out of range", n_kv);
  if (n_heads <= 0 || n_heads % n_kv || n_heads / n_kv > 16)
    fail(RPGC_E_ARG, "n_heads %d must be 1 to 16 times n_kv_heads %d", n_heads, n_kv);
}

void need_16bit(uint32_t type, const char* what) {
  if (type != RPGC_F16 && type != RPGC_BF16) fail(RPGC_E_ARG, "%s: type %u is neither RPGC_F16 nor RPGC_BF16", what, type);
}

// size: bytes of a value
template <typename KV>
PagedView view_of(const KV* kv, int size = 2) {
  if (!kv) fail(RPGC_E_ARG, "kv is NULL");
  need_ptr(kv->k, "kv->k");
  need_ptr(kv->v, "kv->v");
  need_16bit(kv->type, "kv");
  if (kv->n_pages <= 0) fail(RPGC_E_ARG, "n_pages %d must be positive", kv->n_pages);
  int shift = 4;
  while (shift < 8 && (1 << shift) != kv->page_size) ++shift;
  if ((1 << shift) != kv->page_size) fail(RPGC_E_ARG, "page_size %d: 16, 32, 64, 128 and 256 are supported", kv->page_size);
  static const char* const names[3] = {"kv page", "kv position", "kv head"};
  for (int i = 0; i < 3; ++i) {
    need_stride(kv->k_stride[i], size, names[i]);
    need_stride(kv->v_stride[i], size, names[i]);
  }
  PagedView v{};
  v.k = kv->k;
  v.v = kv->v;
  v.k_page = kv->k_stride[0], v.k_pos = kv->k_stride[1], v.k_head = kv->k_stride[2];
  v.v_page = kv->v_stride[0], v.v_pos = kv->v_stride[1], v.v_head = kv->v_stride[2];
  v.n_pages = kv->n_pages;
  v.page_shift = shift;
  v.n_kv = kv->n_kv_heads;
  v.hd = kv->head_dim;
  v.bf16 = kv->type == RPGC_BF16;
  return v;
}

// View of an 8-bit cache, and its scales' strides.
PagedView view8_of(const rpgc_paged_kv8* kv, int64_t* sc_page, int64_t* sc_head) {
  const PagedView v = view_of(kv, 1);
  need_ptr(kv->scales, "kv->scales");
  need_stride(kv->scale_stride[0], 4, "scale page");
  need_stride(kv->scale_stride[1], 4, "scale head");
  *sc_page = kv->scale_stride[0];
  *sc_head = kv->scale_stride[1];
  return v;
}

void need_counts(int32_t n_seqs, int64_t n_tokens) {
  if (n_seqs < 0 || n_seqs > (1 << 20)) fail(RPGC_E_ARG, "n_seqs %d out of range", n_seqs);
  if (n_tokens < 0 || n_tokens > (1 << 24)) fail(RPGC_E_ARG, "n_tokens %lld out of range", (long long)n_tokens);
}

void need_table(int64_t stride, int32_t max_pages) {
  if (max_pages <= 0 || max_pages > (1 << 26)) fail(RPGC_E_ARG, "max_pages %d out of range", max_pages);
  // (0: one row that all sequences share; the kernels only read the table)
  if ((stride && stride < max_pages) || stride > (int64_t(1) << 40))
    fail(RPGC_E_ARG, "table_stride %lld must be 0 or at least max_pages %d", (long long)stride, max_pages);
}

PagedSeqs seqs_of(const rpgc_paged_batch* b) {
  if (!b) fail(RPGC_E_ARG, "batch is NULL");
  need_counts(b->n_seqs, b->n_tokens);
  need_table(b->table_stride, b->max_pages);
  if (b->n_seqs > 0 && (!b->block_table || !b->kv_lens)) fail(RPGC_E_ARG, "block_table or kv_lens is NULL");
  if (!b->cu_q && b->n_tokens != b->n_seqs)
    fail(RPGC_E_ARG, "without cu_q there is one token per sequence: n_tokens %lld, n_seqs %d", (long long)b->n_tokens, b->n_seqs);
  need_words(b->block_table, "block_table");
  need_words(b->kv_lens, "kv_lens");
  need_words(b->cu_q, "cu_q");
  need_words(b->status, "status");
  PagedSeqs s{};
  s.table = b->block_table;
  s.table_stride = b->table_stride;
  s.max_pages = b->max_pages;
  s.n_seqs = b->n_seqs;
  s.kv_lens = b->kv_lens;
  s.cu = b->cu_q;
  s.n_tokens = b->n_tokens;
  s.status = b->status;
  return s;
}

void need_attn(const void* q, const int64_t* q_stride, float scale, const void* out) {
  need_ptr(q, "q");
  need_ptr(out, "out");
  if (!q_stride) fail(RPGC_E_ARG, "q_stride is NULL");
  need_stride(q_stride[0], 2, "q token");
  need_stride(q_stride[1], 2, "q head");
  if (!(scale > 0.0f) || !std::isfinite(scale)) fail(RPGC_E_ARG, "scale must be finite and positive");
}

PagedAttnArgs attn_of(const rpgc_paged_kv* kv, const rpgc_paged_batch* b, const void* q, const int64_t* q_stride,
                      int32_t n_heads, float scale, void* out) {
  PagedAttnArgs a{};
  a.kv = view_of(kv);
  a.b = seqs_of(b);
  need_heads(n_heads, a.kv.n_kv, a.kv.hd);
  if (a.b.n_seqs == 0 || a.b.n_tokens == 0) return a;
  need_attn(q, q_stride, scale, out);
  a.q = q;
  a.q_tok = q_stride[0];
  a.q_head = q_stride[1];
  a.n_heads = n_heads;
  a.scale = scale;
  a.out = out;
  return a;
}

cudaStream_t as_stream(void* s) { return static_cast<cudaStream_t>(s); }

// The rest of an append call: `a` has the cache and the batch.
int append(rpgc::PagedAppendArgs a, uint32_t in_type, const void* q, const int64_t* q_stride, int32_t n_heads, const void* k,
           const int64_t* k_stride, const void* v, const int64_t* v_stride, const float* q_norm, const float* k_norm, float eps,
           const float* rope, int64_t rope_rows, void* q_out, void* stream) {
  if (in_type != RPGC_F32) need_16bit(in_type, "append's input");
  if ((q == nullptr) != (q_out == nullptr)) fail(RPGC_E_ARG, "q and q_out go together");
  need_heads(q ? n_heads : a.kv.n_kv, a.kv.n_kv, a.kv.hd);
  if ((q_norm == nullptr) != (k_norm == nullptr) && q) fail(RPGC_E_ARG, "q_norm and k_norm go together");
  if ((q_norm || k_norm) && !(eps >= 0.0f && std::isfinite(eps))) fail(RPGC_E_ARG, "eps must be finite and not negative");
  if (rope && rope_rows <= 0) fail(RPGC_E_ARG, "rope_rows must be positive");
  if (a.b.n_seqs == 0 || a.b.n_tokens == 0) return RPGC_OK;
  const int size = in_type == RPGC_F32 ? 4 : 2;
  auto rows = [&](const void* p, const int64_t* st, const char* what, int64_t* tok, int64_t* head) {
    need_ptr(p, what);
    if (!st) fail(RPGC_E_ARG, "%s's strides are NULL", what);
    need_stride(st[0], size, what);
    need_stride(st[1], size, what);
    *tok = st[0];
    *head = st[1];
  };
  if (q) {
    rows(q, q_stride, "q", &a.q_tok, &a.q_head);
    need_ptr(q_out, "q_out");
  }
  rows(k, k_stride, "k", &a.k_tok, &a.k_head);
  rows(v, v_stride, "v", &a.v_tok, &a.v_head);
  if (q_norm) need_ptr(q_norm, "q_norm");
  if (k_norm) need_ptr(k_norm, "k_norm");
  if (rope) need_ptr(rope, "rope");
  a.in_type = in_type;
  a.q = q, a.k = k, a.v = v;
  a.n_heads = q ? n_heads : 0;
  a.q_norm = q_norm, a.k_norm = k_norm;
  a.eps = eps;
  a.rope = rope;
  a.rope_rows = rope_rows;
  a.q_out = q_out;
  check(rpgc::paged_append_launch(a, as_stream(stream)), "paged append");
  return RPGC_OK;
}

// A call of single-token attention with a prefix, over 8-bit pages, or both: `a` has the cache.
int own_decode(rpgc::PagedOwnArgs a, const rpgc_paged_batch* b, const rpgc_paged_prefix* prefix, const void* q,
               const int64_t* q_stride, int32_t n_heads, float scale, void* out, void* workspace, int64_t workspace_bytes,
               void* stream) {
  a.b = seqs_of(b);
  need_heads(n_heads, a.kv.n_kv, a.kv.hd);
  if (a.b.cu) fail(RPGC_E_ARG, "decode takes one new token per sequence: cu_q must be NULL");
  if (prefix) {
    a.pre.kv = view_of(prefix->kv);
    if (a.pre.kv.n_kv != a.kv.n_kv || a.pre.kv.hd != a.kv.hd || a.pre.kv.bf16 != a.kv.bf16)
      fail(RPGC_E_ARG, "the prefix's kv heads, head_dim and type must be the cache's");
    need_table(prefix->table_stride, prefix->max_pages);
    if (prefix->n_groups < 0 || prefix->n_groups > (1 << 20)) fail(RPGC_E_ARG, "n_groups %d out of range", prefix->n_groups);
    if (prefix->n_groups > 0 && (!prefix->block_table || !prefix->lens || !prefix->cu_seqs))
      fail(RPGC_E_ARG, "the prefix's block_table, lens or cu_seqs is NULL");
    need_words(prefix->block_table, "the prefix's block_table");
    need_words(prefix->lens, "the prefix's lens");
    need_words(prefix->cu_seqs, "the prefix's cu_seqs");
    a.pre.table = prefix->block_table;
    a.pre.table_stride = prefix->table_stride;
    a.pre.max_pages = prefix->max_pages;
    a.pre.n_groups = prefix->n_groups;
    a.pre.lens = prefix->lens;
    a.pre.cu = prefix->cu_seqs;
  }
  if (!a.b.n_seqs) return RPGC_OK;
  need_attn(q, q_stride, scale, out);
  need_ptr(workspace, "workspace");
  const int64_t need = prefix ? rpgc::paged_prefix_workspace(a.b.n_seqs, n_heads, a.kv.n_kv, a.kv.hd) : rpgc::paged_decode_workspace(a.kv, n_heads);
  if (workspace_bytes < need)
    fail(RPGC_E_ARG, "workspace of %lld bytes: %lld are needed", (long long)workspace_bytes, (long long)need);
  a.q = q;
  a.q_tok = q_stride[0];
  a.q_head = q_stride[1];
  a.n_heads = n_heads;
  a.scale = scale;
  a.out = out;
  a.workspace = workspace;
  if (!a.pre.n_groups) {
    check(a.scales ? rpgc::paged8_decode_launch(a, as_stream(stream)) : rpgc::paged_decode_launch(a, as_stream(stream)),
          "paged decode attention");
    return RPGC_OK;
  }
  check(rpgc::paged_prefix_decode_launch(a, as_stream(stream)), "paged decode attention");
  return RPGC_OK;
}

}  // namespace

extern "C" {

int rpgc_paged_append(const rpgc_paged_kv* kv, const rpgc_paged_batch* b, uint32_t in_type, const void* q,
                      const int64_t* q_stride, int32_t n_heads, const void* k, const int64_t* k_stride, const void* v,
                      const int64_t* v_stride, const float* q_norm, const float* k_norm, float eps, const float* rope,
                      int64_t rope_rows, void* q_out, void* stream) {
  return guard<int>([&] {
    rpgc::PagedAppendArgs a{};
    a.kv = view_of(kv);
    a.b = seqs_of(b);
    return append(a, in_type, q, q_stride, n_heads, k, k_stride, v, v_stride, q_norm, k_norm, eps, rope, rope_rows, q_out, stream);
  });
}

int rpgc_paged_status(int32_t* bits) {
  return guard<int>([&] {
    if (!bits) fail(RPGC_E_ARG, "bits is NULL");
    *bits = 0;
    check(rpgc::paged_append_status(bits), "append's status");
    check(rpgc::paged_decode_status(bits), "single-token attention's status");
    check(rpgc::prompt_attn_status(bits), "prompt attention's status");
    check(rpgc::paged8_decode_status(bits), "single-token attention's status");
    check(rpgc::paged_decode_prefix_status(bits), "single-token attention's status");
    check(rpgc::paged8_decode_prefix_status(bits), "single-token attention's status");
    check(rpgc::paged_decode_through_status(bits), "single-token attention's status");
    check(rpgc::paged_prefix_status(bits), "the prefix's status");
    check(rpgc::paged_read_status(bits), "read's status");
    return RPGC_OK;
  });
}

int64_t rpgc_paged_decode_workspace(const rpgc_paged_kv* kv, int32_t n_seqs, int32_t n_heads) {
  return guard<int64_t>([&]() -> int64_t {
    const PagedView v = view_of(kv);
    need_counts(n_seqs, 0);
    need_heads(n_heads, v.n_kv, v.hd);
    return rpgc::paged_decode_workspace(v, n_heads);
  });
}

int rpgc_paged_attention_decode(const rpgc_paged_kv* kv, const rpgc_paged_batch* b, const void* q, const int64_t* q_stride,
                                int32_t n_heads, float scale, void* out, void* workspace, int64_t workspace_bytes,
                                void* stream) {
  return guard<int>([&] {
    PagedAttnArgs a = attn_of(kv, b, q, q_stride, n_heads, scale, out);
    if (a.b.cu) fail(RPGC_E_ARG, "decode takes one new token per sequence: cu_q must be NULL");
    if (!a.b.n_seqs) return RPGC_OK;
    need_ptr(workspace, "workspace");
    const int64_t need = rpgc::paged_decode_workspace(a.kv, n_heads);
    if (workspace_bytes < need)
      fail(RPGC_E_ARG, "workspace of %lld bytes: %lld are needed", (long long)workspace_bytes, (long long)need);
    a.workspace = workspace;
    check(rpgc::paged_decode_launch(a, as_stream(stream)), "paged decode attention");
    return RPGC_OK;
  });
}

int rpgc_paged_attention_prompt(const rpgc_paged_kv* kv, const rpgc_paged_batch* b, const void* q, const int64_t* q_stride,
                                int32_t n_heads, float scale, void* out, void* stream) {
  return guard<int>([&] {
    const PagedAttnArgs a = attn_of(kv, b, q, q_stride, n_heads, scale, out);
    if (!a.q) return RPGC_OK;
    check(rpgc::prompt_attn_launch(a, as_stream(stream)), "paged prompt attention");
    return RPGC_OK;
  });
}

int rpgc_attention_prompt(uint32_t type, const void* q, const int64_t* q_stride, const void* k, const int64_t* k_stride,
                          const void* v, const int64_t* v_stride, const int32_t* cu, int32_t n_seqs, int64_t n_tokens,
                          int32_t n_heads, int32_t n_kv_heads, int32_t head_dim, float scale, void* out, int32_t* status,
                          void* stream) {
  return guard<int>([&] {
    need_16bit(type, "attention");
    need_heads(n_heads, n_kv_heads, head_dim);
    need_counts(n_seqs, n_tokens);
    if (n_seqs == 0 || n_tokens == 0) return RPGC_OK;
    if (!cu) fail(RPGC_E_ARG, "cu is NULL");
    need_words(cu, "cu");
    need_words(status, "status");
    need_attn(q, q_stride, scale, out);
    need_ptr(k, "k");
    need_ptr(v, "v");
    if (!k_stride || !v_stride) fail(RPGC_E_ARG, "k_stride or v_stride is NULL");
    for (int i = 0; i < 2; ++i) {
      need_stride(k_stride[i], 2, "k");
      need_stride(v_stride[i], 2, "v");
    }
    PagedAttnArgs a{};
    a.kv.k = k, a.kv.v = v;
    a.kv.k_pos = k_stride[0], a.kv.k_head = k_stride[1];
    a.kv.v_pos = v_stride[0], a.kv.v_head = v_stride[1];
    a.kv.n_kv = n_kv_heads;
    a.kv.hd = head_dim;
    a.kv.bf16 = type == RPGC_BF16;
    a.b.n_seqs = n_seqs;
    a.b.cu = cu;
    a.b.n_tokens = n_tokens;
    a.b.status = status;
    a.q = q;
    a.q_tok = q_stride[0], a.q_head = q_stride[1];
    a.n_heads = n_heads;
    a.scale = scale;
    a.out = out;
    check(rpgc::prompt_attn_launch(a, as_stream(stream)), "prompt attention");
    return RPGC_OK;
  });
}

int rpgc_paged8_append(const rpgc_paged_kv8* kv, const rpgc_paged_batch* b, uint32_t in_type, const void* q,
                       const int64_t* q_stride, int32_t n_heads, const void* k, const int64_t* k_stride, const void* v,
                       const int64_t* v_stride, const float* q_norm, const float* k_norm, float eps, const float* rope,
                       int64_t rope_rows, void* q_out, void* stream) {
  return guard<int>([&] {
    rpgc::PagedAppendArgs a{};
    a.kv = view8_of(kv, &a.sc_page, &a.sc_head);
    a.scales = kv->scales;
    a.b = seqs_of(b);
    return append(a, in_type, q, q_stride, n_heads, k, k_stride, v, v_stride, q_norm, k_norm, eps, rope, rope_rows, q_out, stream);
  });
}

int rpgc_paged8_read(const rpgc_paged_kv8* kv, const rpgc_paged_batch* b, const rpgc_paged_kv* to, const int32_t* to_table,
                     int64_t to_table_stride, int32_t to_max_pages, void* stream) {
  return guard<int>([&] {
    rpgc::PagedReadArgs a{};
    a.kv = view8_of(kv, &a.sc_page, &a.sc_head);
    need_heads(a.kv.n_kv, a.kv.n_kv, a.kv.hd);
    a.scales = kv->scales;
    a.b = seqs_of(b);
    a.to = view_of(to);
    if (a.to.n_kv != a.kv.n_kv || a.to.hd != a.kv.hd) fail(RPGC_E_ARG, "to's kv heads and head_dim must be the cache's");
    need_table(to_table_stride, to_max_pages);
    if (!a.b.n_seqs) return RPGC_OK;
    if (!to_table) fail(RPGC_E_ARG, "to_table is NULL");
    need_words(to_table, "to_table");
    a.to_table = to_table;
    a.to_stride = to_table_stride;
    a.to_max = to_max_pages;
    check(rpgc::paged_read_launch(a, as_stream(stream)), "paged read");
    return RPGC_OK;
  });
}

int64_t rpgc_paged_prefix_workspace(int32_t n_seqs, int32_t n_heads, int32_t n_kv_heads, int32_t head_dim) {
  return guard<int64_t>([&]() -> int64_t {
    need_counts(n_seqs, 0);
    need_heads(n_heads, n_kv_heads, head_dim);
    return rpgc::paged_prefix_workspace(n_seqs, n_heads, n_kv_heads, head_dim);
  });
}

int rpgc_paged_attention_decode_prefix(const rpgc_paged_kv* kv, const rpgc_paged_batch* b, const rpgc_paged_prefix* prefix,
                                       const void* q, const int64_t* q_stride, int32_t n_heads, float scale, void* out,
                                       void* workspace, int64_t workspace_bytes, void* stream) {
  return guard<int>([&] {
    rpgc::PagedOwnArgs a{};
    a.kv = view_of(kv);
    if (!prefix) fail(RPGC_E_ARG, "prefix is NULL");
    return own_decode(a, b, prefix, q, q_stride, n_heads, scale, out, workspace, workspace_bytes, stream);
  });
}

int64_t rpgc_paged8_decode_workspace(const rpgc_paged_kv8* kv, int32_t n_seqs, int32_t n_heads) {
  return guard<int64_t>([&]() -> int64_t {
    int64_t st[2];
    const PagedView v = view8_of(kv, st, st + 1);
    need_counts(n_seqs, 0);
    need_heads(n_heads, v.n_kv, v.hd);
    return rpgc::paged_decode_workspace(v, n_heads);
  });
}

int rpgc_paged8_attention_decode(const rpgc_paged_kv8* kv, const rpgc_paged_batch* b, const rpgc_paged_prefix* prefix,
                                 const void* q, const int64_t* q_stride, int32_t n_heads, float scale, void* out,
                                 void* workspace, int64_t workspace_bytes, void* stream) {
  return guard<int>([&] {
    rpgc::PagedOwnArgs a{};
    a.kv = view8_of(kv, &a.sc_page, &a.sc_head);
    a.scales = kv->scales;
    return own_decode(a, b, prefix, q, q_stride, n_heads, scale, out, workspace, workspace_bytes, stream);
  });
}

}  // extern "C"
