// Operators over a paged key-value cache (include/cljxla_b200.h, "paged
// key-value cache"): parameter blocks and the device-side view they share.
#pragma once

#include <cstdint>
#include <cuda_runtime.h>

#include "kernels.h"

namespace cljxla {

// The step's packed rows and the cache they live in.  Strides are bytes.
struct PagedView {
  char *k, *v;
  int64_t k_page, k_head, k_row, v_page, v_head, v_row;
  const int32_t* table;
  const int32_t* lens;
  const int32_t* starts;  // null: `each` rows per sequence
  int64_t table_stride;   // entries
  int32_t num_pages, page_size, pages_per_seq, nkv, num_seqs, tokens, each;
  int32_t page_shift;  // log2(page_size), or -1
};

struct PagedAppendParams {
  PagedView c;
  const char *ks, *vs, *qs;
  char* qo;
  int64_t ks_tok, ks_head, vs_tok, vs_head, qs_tok, qs_head, qo_tok, qo_head;  // bytes
  const float* inv_freq;
  int32_t nq, hd, rotary, interleaved, vec, dt;  // vec: whole 16-byte vectors
  int32_t tok, lot_bits;  // set at the launch: rows of a CTA, log2 of the threads of a head
  float rope_scale;
};

struct PagedAttnParams {
  PagedView c;
  const char* q;
  char* out;
  int64_t q_tok, q_head, o_tok, o_head;  // bytes
  int32_t group, hd, dt, out_f32, max_rows, pad_;  // max_rows: rows of a sequence at most
  int64_t window;  // < 0: none
  float scale, softcap;
  // set at the launch: the factor from q.k to the argument of 2^x (with a cap:
  // of tanh), log2(e) * softcap
  float mul, cap2;
  float* part;  // per CTA: two slots of rows and their (max, sum)
  uint32_t group_mul;  // 2^32 / group rounded up (0: group 1), set at the launch
};

struct VerifyParams {
  const char *target, *draft;
  const int32_t* tokens_in;
  const int32_t* starts;
  const float *uniform, *race;
  int64_t target_stride, draft_stride;  // bytes
  int64_t race_stride;                  // elements
  int64_t vocab;
  int32_t tokens, num_seqs, max_tokens, each, dt, greedy, splits, pad_;
  float inv_t, inv_td;
  int32_t *tokens_out, *accepted;
  float* logprobs;
  const int32_t* seq_lens;
  int32_t* new_lens;
  float* part;  // [2][tokens][splits] (max, sum) pairs, then [tokens][splits] argmax indices
};

void launch_paged_append(const PagedAppendParams& p, cudaStream_t s);
// by element type (one translation unit each)
void launch_paged_attention_bf16(const PagedAttnParams& p, cudaStream_t s);
void launch_paged_attention_f16(const PagedAttnParams& p, cudaStream_t s);
void launch_paged_attention_f32(const PagedAttnParams& p, cudaStream_t s);
int64_t paged_attention_workspace_bf16(const PagedAttnParams& p);
int64_t paged_attention_workspace_f16(const PagedAttnParams& p);
int64_t paged_attention_workspace_f32(const PagedAttnParams& p);
void launch_verify(const VerifyParams& p, cudaStream_t s);
int verify_splits(int64_t tokens, int64_t vocab, bool draft);
int64_t verify_workspace(const VerifyParams& p);

#ifdef __CUDACC__
// First row and row count of sequence b, whatever `starts` holds.
__device__ __forceinline__ void seq_rows(const PagedView& c, int b, int& first, int& count) {
  if (!c.starts) {
    first = b * c.each;
    count = c.each;
    return;
  }
  const int lo = min(max(c.starts[b], 0), c.tokens), hi = min(max(c.starts[b + 1], 0), c.tokens);
  first = lo;
  count = max(hi - lo, 0);
}

// Positions of sequence b, which may be more than its table holds (the host
// checks that capacity fits 30 bits).
__device__ __forceinline__ int seq_len(const PagedView& c, int b) { return min(max(c.lens[b], 0), 1 << 30); }
__device__ __forceinline__ int capacity(const PagedView& c) { return c.pages_per_seq * c.page_size; }

// The page of position `pos` of sequence b, or -1 where the table names none.
__device__ __forceinline__ int page_of(const PagedView& c, int b, int pos) {
  if ((unsigned)pos >= (unsigned)capacity(c)) return -1;
  const int page = c.table[(int64_t)b * c.table_stride + pos / c.page_size];
  return (unsigned)page < (unsigned)c.num_pages ? page : -1;
}

// The sequence that owns packed row `t`, or -1: the last b with starts[b] <= t,
// found 32 ways at a time by a whole warp.
__device__ __forceinline__ int seq_of_row(const int32_t* starts, int num_seqs, int each, int t) {
  if (!starts) {
    const int b = t / each;
    return b < num_seqs ? b : -1;
  }
  const int lane = threadIdx.x & 31;
  int lo = -1, hi = num_seqs;  // invariant: starts[lo] <= t (or lo = -1), starts[hi] > t (or hi = num_seqs)
  while (hi - lo > 1) {
    const int step = (hi - lo + 31) / 32;
    const int at = lo + 1 + lane * step;  // candidates lo + 1, lo + 1 + step, ...
    const bool le = at < hi && starts[at] <= t;
    const int n = __popc(__ballot_sync(0xffffffffu, le));  // ascending: the first n hold
    const int base = lo;
    if (n == 0) {
      hi = lo + 1;
    } else {
      lo = base + 1 + (n - 1) * step;
      hi = min(hi, lo + step);
    }
  }
  if (lo < 0 || t >= starts[lo + 1]) return -1;
  return lo;
}
#endif

}  // namespace cljxla
