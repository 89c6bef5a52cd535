// C entries of the operators over a paged key-value cache: argument checks,
// parameter blocks, launches.  Every check that needs no device comes before
// the first CUDA call, and nothing throws across the C boundary.
#include <cuda_runtime.h>

#include <new>
#include <string>

#include "../../include/cljxla_b200.h"
#include "common.h"
#include "paged.h"

namespace cljxla {
namespace {

template <class F>
int entry(const char* name, char* err, size_t cap, F&& f) {
  int code = E_INTERNAL;
  const char* what = "unknown failure";
  try {
    try {
      f();
      return 0;
    } catch (const Error& e) {
      code = e.code;
      if (err && cap) snprintf(err, cap, "%s: %s", name, e.what());
      return code;
    } catch (const std::bad_alloc&) {
      code = E_OOM;
      what = "host out of memory";
    }
    if (err && cap) snprintf(err, cap, "%s: %s", name, what);
    return code;
  } catch (...) {
    if (err && cap) snprintf(err, cap, "%s: unknown failure", name);
    return E_INTERNAL;
  }
}

void need(bool ok, const char* msg) {
  if (!ok) fail(E_INVALID, msg);
}

int element_type(int32_t dtype) {
  switch (dtype) {
    case PJRT_Buffer_Type_F32: return KDT_F32;
    case PJRT_Buffer_Type_F16: return KDT_F16;
    case PJRT_Buffer_Type_BF16: return KDT_BF16;
    default: fail(E_INVALID, "dtype must be F32, F16 or BF16");
  }
}

int64_t element_size(int dt) { return dt == KDT_F32 ? 4 : 2; }

// every extent that takes part in address arithmetic stays below this, and every
// stride below 2^40 elements: no product of an index that memory can hold and its
// stride comes near 64 bits
constexpr int64_t kMaxCount = 1 << 30;
constexpr int64_t kMaxStride = (int64_t)1 << 40;

void need_stride(int64_t stride, const char* msg) { need(stride >= 0 && stride <= kMaxStride, msg); }

bool vec16(const void* p) { return ((uintptr_t)p & 15) == 0; }
template <class... P>
bool aligned(int64_t bytes, const P*... p) {  // 2 or 4; a null pointer is
  return (((uintptr_t)p | ...) & (uintptr_t)(bytes - 1)) == 0;
}
void need_words(const PagedView& c) {
  need(aligned(4, c.table, c.lens, c.starts), "page_table, seq_lens and starts must be aligned to their type");
}
// strides of dimensions with one entry are never used
bool vec16(int64_t extent, int64_t stride_bytes) { return extent <= 1 || stride_bytes % 16 == 0; }

PagedView view_of(const CLJXLA_PagedKV* kv, int64_t tokens, const int32_t* starts, bool write) {
  need(kv != nullptr, "null cache");
  need(kv->struct_size >= sizeof(CLJXLA_PagedKV), "cache struct_size is too small");
  const int64_t es = element_size(element_type(kv->dtype));
  need(kv->head_dim == 32 || kv->head_dim == 64 || kv->head_dim == 128 || kv->head_dim == 256,
       "head_dim must be 32, 64, 128 or 256");
  need(kv->kv_heads >= 1 && kv->kv_heads <= 65535, "kv_heads out of range");
  need(kv->page_size >= 1 && kv->page_size <= kMaxCount, "page_size out of range");
  need(kv->num_pages >= 0 && kv->num_pages <= kMaxCount, "num_pages out of range");
  need(kv->num_seqs >= 0 && kv->num_seqs <= (1 << 20), "num_seqs out of range");
  need(kv->pages_per_seq >= 0 && kv->pages_per_seq <= kMaxCount &&
           kv->pages_per_seq * kv->page_size <= kMaxCount,
       "pages_per_seq * page_size must be at most 2^30");
  need(kv->num_seqs <= 1 || (kv->page_table_stride >= kv->pages_per_seq && kv->page_table_stride <= kMaxStride),
       "page_table rows overlap");
  need_stride(kv->k_page_stride, "k_page_stride out of range");
  need_stride(kv->k_head_stride, "k_head_stride out of range");
  need_stride(kv->k_row_stride, "k_row_stride out of range");
  need_stride(kv->v_page_stride, "v_page_stride out of range");
  need_stride(kv->v_head_stride, "v_head_stride out of range");
  need_stride(kv->v_row_stride, "v_row_stride out of range");
  if (write)
    need((kv->num_pages <= 1 || (kv->k_page_stride > 0 && kv->v_page_stride > 0)) &&
             (kv->kv_heads <= 1 || (kv->k_head_stride > 0 && kv->v_head_stride > 0)) &&
             (kv->page_size <= 1 || (kv->k_row_stride > 0 && kv->v_row_stride > 0)),
         "pages that are written need strides of their own (no broadcast)");
  need(tokens >= 0 && tokens <= kMaxCount, "tokens out of range");
  if (tokens > 0 && kv->num_seqs > 0) {
    need(kv->seq_lens != nullptr, "null seq_lens");
    need(kv->page_table != nullptr || kv->pages_per_seq == 0, "null page_table");
    need((kv->k_pages && kv->v_pages) || kv->num_pages == 0, "null pages");
    if (!starts) need(tokens % kv->num_seqs == 0, "without starts, tokens must be a multiple of num_seqs");
  }
  need(vec16(kv->k_pages) && vec16(kv->v_pages) && vec16(kv->num_pages, kv->k_page_stride * es) &&
           vec16(kv->num_pages, kv->v_page_stride * es) && vec16(kv->kv_heads, kv->k_head_stride * es) &&
           vec16(kv->kv_heads, kv->v_head_stride * es) && vec16(kv->page_size, kv->k_row_stride * es) &&
           vec16(kv->page_size, kv->v_row_stride * es),
       "K / V pages must have 16-byte aligned rows");
  PagedView c{};
  c.k = (char*)kv->k_pages;
  c.v = (char*)kv->v_pages;
  c.k_page = kv->k_page_stride * es;
  c.k_head = kv->k_head_stride * es;
  c.k_row = kv->k_row_stride * es;
  c.v_page = kv->v_page_stride * es;
  c.v_head = kv->v_head_stride * es;
  c.v_row = kv->v_row_stride * es;
  c.table = kv->page_table;
  c.table_stride = kv->page_table_stride;
  c.lens = kv->seq_lens;
  c.starts = starts;
  c.num_pages = (int32_t)kv->num_pages;
  c.page_size = (int32_t)kv->page_size;
  c.pages_per_seq = (int32_t)kv->pages_per_seq;
  c.page_shift = -1;
  for (int i = 0; i <= 30; ++i)
    if (kv->page_size == (int64_t)1 << i) c.page_shift = i;
  c.nkv = (int32_t)kv->kv_heads;
  c.num_seqs = (int32_t)kv->num_seqs;
  c.tokens = (int32_t)tokens;
  c.each = kv->num_seqs > 0 ? (int32_t)(tokens / kv->num_seqs) : 0;
  return c;
}

int64_t attention_workspace(const PagedAttnParams& p) {
  return p.dt == KDT_F32 ? paged_attention_workspace_f32(p)
                         : (p.dt == KDT_F16 ? paged_attention_workspace_f16(p) : paged_attention_workspace_bf16(p));
}

bool nothing_to_do(const PagedView& c) { return c.tokens == 0 || c.num_seqs == 0; }
// nor where no row of a sequence is computed
bool nothing_to_do(const PagedAttnParams& p) { return nothing_to_do(p.c) || p.max_rows == 0; }

PagedAttnParams attention_params(const CLJXLA_PagedKV* kv, const CLJXLA_PagedAttentionArgs* a, bool pointers) {
  need(a != nullptr, "null arguments");
  need(a->struct_size >= sizeof(CLJXLA_PagedAttentionArgs), "arguments' struct_size is too small");
  PagedAttnParams p{};
  CLJXLA_PagedKV sizes;
  if (!pointers && kv && kv->struct_size >= sizeof(CLJXLA_PagedKV)) {  // sizes alone: any pointer will do
    sizes = *kv;
    alignas(16) static char some[16];
    sizes.k_pages = sizes.v_pages = some;
    sizes.page_table = sizes.seq_lens = (const int32_t*)some;
    kv = &sizes;
  }
  p.c = view_of(kv, a->tokens, a->starts, false);
  p.dt = element_type(kv->dtype);
  p.hd = (int32_t)kv->head_dim;
  need(a->q_heads >= 1 && a->q_heads <= 65535 && a->q_heads % kv->kv_heads == 0,
       "q_heads must be a multiple of kv_heads");
  p.group = (int32_t)(a->q_heads / kv->kv_heads);
  need(p.group <= 32768, "q_heads is more than 32768 times kv_heads");
  const int out_dt = element_type(a->out_dtype);
  need(out_dt == p.dt || out_dt == KDT_F32, "out_dtype must be the pages' type or F32");
  p.out_f32 = out_dt == KDT_F32;
  need(a->max_tokens >= 0 && a->max_tokens <= kMaxCount, "max_tokens out of range");
  p.max_rows = (int32_t)(a->starts ? a->max_tokens : p.c.each);
  if (!a->starts) need(a->max_tokens >= p.c.each, "max_tokens is below tokens / num_seqs");
  if (p.max_rows > p.c.tokens) p.max_rows = p.c.tokens;
  need((int64_t)p.max_rows * p.group <= kMaxCount, "max_tokens * query heads per KV head out of range");
  need(a->scale == a->scale && a->softcap == a->softcap && a->softcap >= 0.f && a->softcap - a->softcap == 0.f &&
           a->scale - a->scale == 0.f,
       "scale must be finite, softcap finite and not negative");
  p.scale = a->scale;
  p.softcap = a->softcap;
  const float per_cap = p.softcap > 0.f ? p.scale / p.softcap : 0.f;
  need(per_cap - per_cap == 0.f, "scale / softcap must be finite");
  p.window = a->window < 0 ? -1 : (a->window > kMaxCount ? kMaxCount : a->window);
  const int64_t es = element_size(p.dt), eo = element_size(out_dt);
  need_stride(a->q_token_stride, "q_token_stride out of range");
  need_stride(a->q_head_stride, "q_head_stride out of range");
  need_stride(a->out_token_stride, "out_token_stride out of range");
  need_stride(a->out_head_stride, "out_head_stride out of range");
  p.q_tok = a->q_token_stride * es;
  p.q_head = a->q_head_stride * es;
  p.o_tok = a->out_token_stride * eo;
  p.o_head = a->out_head_stride * eo;
  need(vec16(a->tokens, p.q_tok) && vec16(a->q_heads, p.q_head), "q must have 16-byte aligned rows");
  need(vec16(a->tokens, p.o_tok) && vec16(a->q_heads, p.o_head), "out must have 16-byte aligned rows");
  need((a->tokens <= 1 || p.o_tok > 0) && (a->q_heads <= 1 || p.o_head > 0), "out must not be a broadcast");
  if (pointers && !nothing_to_do(p)) {
    need_words(p.c);
    need(a->q && a->out, "null q or out");
    need(vec16(a->q), "q must have 16-byte aligned rows");
    need(vec16(a->out), "out must have 16-byte aligned rows");
    need(vec16(a->workspace), "workspace must be 16-byte aligned");
  }
  p.q = (const char*)a->q;
  p.out = (char*)a->out;
  return p;
}

VerifyParams verify_params(const CLJXLA_VerifyDraftArgs* a) {
  need(a != nullptr, "null arguments");
  need(a->struct_size >= sizeof(CLJXLA_VerifyDraftArgs), "arguments' struct_size is too small");
  VerifyParams p{};
  p.dt = element_type(a->dtype);
  const int64_t es = element_size(p.dt);
  need(a->tokens >= 0 && a->tokens <= (1 << 24), "tokens out of range");
  need(a->num_seqs >= 0 && a->num_seqs <= (1 << 20), "num_seqs out of range");
  need(a->vocab >= 1 && a->vocab <= kMaxCount, "vocab out of range");
  need(a->max_tokens >= 1 && a->max_tokens <= 128, "max_tokens must be 1 to 128");
  if (!a->starts && a->num_seqs > 0) {
    need(a->tokens % a->num_seqs == 0, "without starts, tokens must be a multiple of num_seqs");
    need(a->tokens / a->num_seqs <= a->max_tokens, "max_tokens is below tokens / num_seqs");
  }
  need(a->tokens <= 1 || (a->target_stride >= a->vocab && a->target_stride <= kMaxStride), "target rows overlap");
  need(!a->draft || a->greedy || a->tokens <= 1 || (a->draft_stride >= a->vocab && a->draft_stride <= kMaxStride),
       "draft rows overlap");
  need(a->greedy || a->num_seqs <= 1 || (a->race_stride >= a->vocab && a->race_stride <= kMaxStride),
       "race rows overlap");
  auto usable = [](float t) {  // its reciprocal times log2(e) is finite too
    const float c = 1.5f / t;
    return t > 0.f && t - t == 0.f && c - c == 0.f;
  };
  need(usable(a->temperature), "temperature must be positive and finite, and not next to zero");
  need(!a->draft || a->greedy || usable(a->draft_temperature),
       "draft_temperature must be positive and finite, and not next to zero");
  p.target = (const char*)a->target;
  p.draft = a->greedy ? nullptr : (const char*)a->draft;  // a greedy decision needs no distribution
  p.tokens_in = a->tokens_in;
  p.starts = a->starts;
  p.uniform = a->uniform;
  p.race = a->race;
  p.target_stride = a->target_stride * es;
  p.draft_stride = a->draft_stride * es;
  p.race_stride = a->race_stride;
  p.vocab = a->vocab;
  p.tokens = (int32_t)a->tokens;
  p.num_seqs = (int32_t)a->num_seqs;
  p.max_tokens = (int32_t)a->max_tokens;
  p.each = a->num_seqs > 0 ? (int32_t)(a->tokens / a->num_seqs) : 0;
  p.greedy = a->greedy != 0;
  p.inv_t = 1.f / a->temperature;
  p.inv_td = p.draft ? 1.f / a->draft_temperature : 1.f;
  p.tokens_out = a->tokens_out;
  p.accepted = a->accepted;
  p.logprobs = a->logprobs;
  p.seq_lens = a->seq_lens;
  p.new_lens = a->new_lens;
  return p;
}

}  // namespace
}  // namespace cljxla

using namespace cljxla;

extern "C" CLJXLA_EXPORT int cljxla_b200_paged_append(const CLJXLA_PagedKV* kv, const CLJXLA_PagedAppendArgs* a,
                                                      void* stream, char* err, size_t errcap) {
  return entry("paged_append", err, errcap, [&] {
    need(a != nullptr, "null arguments");
    need(a->struct_size >= sizeof(CLJXLA_PagedAppendArgs), "arguments' struct_size is too small");
    PagedAppendParams p{};
    p.c = view_of(kv, a->tokens, a->starts, true);
    p.dt = element_type(kv->dtype);
    const int64_t es = element_size(p.dt);
    p.hd = (int32_t)kv->head_dim;
    need(a->rotary_dim >= 0 && a->rotary_dim <= kv->head_dim && a->rotary_dim % 2 == 0,
         "rotary_dim must be even and at most head_dim");
    need(a->rotary_dim == 0 || a->inv_freq, "null inv_freq");
    need(a->rope_scale - a->rope_scale == 0.f, "rope_scale must be finite");
    need(!a->q == !a->q_out, "q and q_out go together");
    need(!a->q || (a->q_heads >= 1 && a->q_heads <= 65535), "q_heads out of range");
    need_stride(a->k_token_stride, "k_token_stride out of range");
    need_stride(a->k_head_stride, "k_head_stride out of range");
    need_stride(a->v_token_stride, "v_token_stride out of range");
    need_stride(a->v_head_stride, "v_head_stride out of range");
    if (a->q) {
      need_stride(a->q_token_stride, "q_token_stride out of range");
      need_stride(a->q_head_stride, "q_head_stride out of range");
      need_stride(a->q_out_token_stride, "q_out_token_stride out of range");
      need_stride(a->q_out_head_stride, "q_out_head_stride out of range");
      need((a->tokens <= 1 || a->q_out_token_stride > 0) && (a->q_heads <= 1 || a->q_out_head_stride > 0),
           "q_out must not be a broadcast");
      need(a->q_out != (void*)a->q ||
               ((a->tokens <= 1 || a->q_out_token_stride == a->q_token_stride) &&
                (a->q_heads <= 1 || a->q_out_head_stride == a->q_head_stride)),
           "q_out in place of q needs the strides of q");
    }
    if (nothing_to_do(p.c)) return;
    need(a->k && a->v, "null k or v");
    need_words(p.c);
    need(aligned(4, a->inv_freq), "inv_freq must be aligned to its type");
    need(aligned(es, a->k, a->v, a->q, (const void*)a->q_out), "k, v, q and q_out must be aligned to their type");
    p.ks = (const char*)a->k;
    p.vs = (const char*)a->v;
    p.qs = (const char*)a->q;
    p.qo = (char*)a->q_out;
    p.ks_tok = a->k_token_stride * es;
    p.ks_head = a->k_head_stride * es;
    p.vs_tok = a->v_token_stride * es;
    p.vs_head = a->v_head_stride * es;
    p.nq = a->q ? (int32_t)a->q_heads : 0;
    if (a->q) {
      p.qs_tok = a->q_token_stride * es;
      p.qs_head = a->q_head_stride * es;
      p.qo_tok = a->q_out_token_stride * es;
      p.qo_head = a->q_out_head_stride * es;
    }
    p.inv_freq = a->inv_freq;
    p.rotary = (int32_t)a->rotary_dim;
    p.interleaved = a->interleaved != 0;
    p.rope_scale = a->rope_scale;
    const int64_t lot = (p.interleaved ? p.rotary : p.rotary / 2) * es;
    p.vec = lot % 16 == 0 && vec16(p.ks) && vec16(p.vs) && vec16(p.qs) && vec16(p.qo) &&
            vec16(a->tokens, p.ks_tok) && vec16(a->tokens, p.vs_tok) && vec16(a->tokens, p.qs_tok) &&
            vec16(a->tokens, p.qo_tok) && vec16(p.c.nkv, p.ks_head) && vec16(p.c.nkv, p.vs_head) &&
            vec16(p.nq, p.qs_head) && vec16(p.nq, p.qo_head);
    launch_paged_append(p, (cudaStream_t)stream);
  });
}

extern "C" CLJXLA_EXPORT int cljxla_b200_paged_attention_workspace(const CLJXLA_PagedKV* kv,
                                                                   const CLJXLA_PagedAttentionArgs* a, int64_t* bytes,
                                                                   char* err, size_t errcap) {
  return entry("paged_attention_workspace", err, errcap, [&] {
    need(bytes != nullptr, "null bytes");
    const PagedAttnParams p = attention_params(kv, a, false);
    *bytes = nothing_to_do(p) ? 0 : attention_workspace(p);
  });
}

extern "C" CLJXLA_EXPORT int cljxla_b200_paged_attention(const CLJXLA_PagedKV* kv, const CLJXLA_PagedAttentionArgs* a,
                                                         void* stream, char* err, size_t errcap) {
  return entry("paged_attention", err, errcap, [&] {
    PagedAttnParams p = attention_params(kv, a, true);
    if (nothing_to_do(p)) return;
    const int64_t want = attention_workspace(p);
    if (want > 0 && (!a->workspace || a->workspace_bytes < want))
      fail(E_INVALID, "workspace of " + std::to_string(a->workspace ? a->workspace_bytes : 0) + " bytes, " +
                          std::to_string(want) + " needed");
    p.part = (float*)a->workspace;
    if (p.dt == KDT_F32) launch_paged_attention_f32(p, (cudaStream_t)stream);
    else if (p.dt == KDT_F16) launch_paged_attention_f16(p, (cudaStream_t)stream);
    else launch_paged_attention_bf16(p, (cudaStream_t)stream);
  });
}

extern "C" CLJXLA_EXPORT int cljxla_b200_verify_draft_workspace(const CLJXLA_VerifyDraftArgs* a, int64_t* bytes,
                                                                char* err, size_t errcap) {
  return entry("verify_draft_workspace", err, errcap, [&] {
    need(bytes != nullptr, "null bytes");
    VerifyParams p = verify_params(a);
    *bytes = 0;
    if (p.num_seqs == 0) return;
    p.splits = verify_splits(p.tokens, p.vocab, p.draft != nullptr);
    *bytes = verify_workspace(p);
  });
}

extern "C" CLJXLA_EXPORT int cljxla_b200_verify_draft(const CLJXLA_VerifyDraftArgs* a, void* stream, char* err,
                                                      size_t errcap) {
  return entry("verify_draft", err, errcap, [&] {
    VerifyParams p = verify_params(a);
    if (p.num_seqs == 0) return;
    need(a->tokens_out && a->accepted, "null tokens_out or accepted");
    need(!a->new_lens || a->seq_lens, "new_lens needs seq_lens");
    need(p.tokens == 0 || (a->target && a->tokens_in), "null target or tokens_in");
    need(p.tokens == 0 || a->greedy || (a->uniform && a->race), "null uniform or race");
    const int64_t es = element_size(p.dt);
    need(aligned(es, a->target, p.draft), "logits must be aligned to their type");
    need(aligned(4, a->tokens_in, a->starts, p.greedy ? nullptr : a->uniform, p.greedy ? nullptr : a->race),
         "tokens_in, starts, uniform and race must be aligned to their type");
    need(aligned(4, a->tokens_out, a->accepted, a->logprobs, a->new_lens, a->new_lens ? a->seq_lens : nullptr),
         "tokens_out, accepted, logprobs, seq_lens and new_lens must be aligned to their type");
    p.splits = verify_splits(p.tokens, p.vocab, p.draft != nullptr);
    const int64_t want = verify_workspace(p);
    if (want > 0 && (!a->workspace || a->workspace_bytes < want))
      fail(E_INVALID, "workspace of " + std::to_string(a->workspace ? a->workspace_bytes : 0) + " bytes, " +
                          std::to_string(want) + " needed");
    need(vec16(a->workspace), "workspace must be 16-byte aligned");
    p.part = (float*)a->workspace;
    launch_verify(p, (cudaStream_t)stream);
  });
}
