/*
 * cljxla_b200.h - C ABI of libcljxla_b200.so, the B200 (sm_100a) executor
 * that clj-xla loads in place of its PJRT CPU plugin.
 *
 * The boundary is the PJRT C API.  clj-xla's host binds exactly one symbol,
 * GetPjrtApi (src/clj_xla/pjrt.clj:201-206 looks it up, :207 reads 984 bytes
 * of the returned table), and then calls these table slots: Error_Destroy /
 * Error_Message (pjrt.clj:63-82), Plugin_Initialize (:211-215),
 * Plugin_Attributes (:116-146), Event_Await / Event_Destroy (:420-433,
 * :508-522, :548-562), Client_Create (:261-275), Client_PlatformName
 * (:277-291), Client_AddressableDevices (:293-308), Client_Compile with format
 * "mlir" (:310-340), Client_BufferFromHostBuffer (:342-434),
 * LoadedExecutable_Execute (:454-525), Buffer_Destroy (:436-452) and
 * Buffer_ToHostBuffer (:527-611).  Struct layouts: pjrt_abi.h.
 *
 * The cljxla_b200_* functions are additions with no counterpart in the
 * reference; they expose counters and profiling for tests and benchmarks.
 */
#ifndef CLJXLA_B200_H_
#define CLJXLA_B200_H_

#include <stddef.h>
#include <stdint.h>

#include "pjrt_abi.h"

#if defined(__GNUC__)
#define CLJXLA_EXPORT __attribute__((visibility("default")))
#else
#define CLJXLA_EXPORT
#endif

#ifdef __cplusplus
extern "C" {
#endif

/* Replaces the plugin entry point of xla_cpu_pjrt / jax_cuda12_pjrt that
 * clj-xla resolves at pjrt.clj:201-206. */
CLJXLA_EXPORT const PJRT_Api* GetPjrtApi(void);

/* Number of device kernels launched by executions so far (all executables). */
CLJXLA_EXPORT int64_t cljxla_b200_kernel_launches(void);

/* Number of LoadedExecutable_Execute calls completed so far. */
CLJXLA_EXPORT int64_t cljxla_b200_executions(void);

/* Per-kernel CUDA-event timing of subsequent executions (eager launches). */
CLJXLA_EXPORT void cljxla_b200_profile_enable(int on);

/* Writes the accumulated profile as JSON into out[cap]; returns the size needed. */
CLJXLA_EXPORT size_t cljxla_b200_profile_dump(char* out, size_t cap);

/* info[0..n): launches, scratch bytes, graph nodes, live nodes, fused
 * elementwise groups, constant bytes, launches whose compiled (NVRTC) form
 * failed so that an interpreting kernel runs instead, attention launches whose
 * causal / sliding-window mask is computed in the kernel instead of read.
 * Returns 0 on success. */
CLJXLA_EXPORT int cljxla_b200_plan_info(const PJRT_LoadedExecutable* exec, int64_t* info, int n);

/* Parses and plans MLIR text on the host only (no device needed).  `fuse`
 * holds flags: bit 0 enables fusion and the fast kernels, bit 1 plans
 * KV-cache updates in place.  info as above; returns 0 or a PJRT_Error_Code
 * with the message in err[errcap]. */
CLJXLA_EXPORT int cljxla_b200_plan_text(const char* text, size_t len, int fuse, int64_t* info, int n, char* err,
                                        size_t errcap);

/* Host-only check of the compiled fused kernels: plans the MLIR text (flags
 * as cljxla_b200_plan_text), generates the source of every fused elementwise
 * and row kernel and compiles each distinct one with NVRTC for sm_100a (no
 * device needed).  *kernels receives the number of generated kernels.
 * Returns the number that failed to compile (first log in err), -1 when
 * NVRTC is not available, -2 when planning failed. */
CLJXLA_EXPORT int cljxla_b200_jit_check(const char* text, size_t len, int flags, int* kernels, char* err,
                                        size_t errcap);

/* Programs this process found in (hits) or added to (misses) the on-disk
 * cache of compiled fused kernels.  The cache is keyed like clj-xla's compile
 * cache (src/clj_xla/compile.clj:13-24: SHA-256 of the program text), here of
 * each generated kernel's source with the NVRTC version and options, and
 * lives in CLJXLA_B200_CACHE_DIR (else $XDG_CACHE_HOME/cljxla_b200, else
 * $HOME/.cache/cljxla_b200; "0" turns it off).  No counterpart in the
 * reference, whose compile cache is in memory only. */
CLJXLA_EXPORT void cljxla_b200_jit_cache_stats(int64_t* hits, int64_t* misses);

/* Tensor parallelism (no counterpart in the reference, which runs on one
 * device).  A graph with "stablehlo.all_reduce" ops is one rank's shard of a
 * model; its client is created with the named values tp_size (int64),
 * tp_rank (int64) and tp_nccl_id (string): the hex id this function returns on
 * one rank (256 characters + NUL into out[cap]), passed to every rank by the
 * host.  Returns 0 or a PJRT_Error_Code (9: NCCL could not be loaded). */
CLJXLA_EXPORT int cljxla_b200_nccl_unique_id(char* out, size_t cap);

/* One-shot all-reduce over NVLink peer memory for tensor-parallel clients (no
 * counterpart in the reference).  Once every rank of a group has called
 * cljxla_b200_p2p_export (a CUDA IPC handle of a new exchange buffer with two
 * phases of one slot_bytes slot per rank, as hex: 128 characters + NUL into
 * out[cap]) and then cljxla_b200_p2p_import with all ranks' handles
 * concatenated in rank order, every all_reduce of at most slot_bytes (f32 or
 * bf16, 16-byte multiple) runs as one kernel per rank that stores its operand
 * into every rank's buffer, waits (bounded, about 16 s) for the others and
 * sums in rank order; larger ones stay on NCCL.  A wait that runs out makes
 * the client's next execution fail.  `client` is the PJRT_Client*. */
CLJXLA_EXPORT int cljxla_b200_p2p_export(void* client, int64_t slot_bytes, char* out, size_t cap);
CLJXLA_EXPORT int cljxla_b200_p2p_import(void* client, const char* handles, size_t len);

/* The cudaStream_t a client launches on (for event timing by the caller). */
CLJXLA_EXPORT void* cljxla_b200_stream(const PJRT_Client* client);

/* Device address backing a buffer. */
CLJXLA_EXPORT void* cljxla_b200_buffer_device_pointer(const PJRT_Buffer* buffer);

/* Size of the fixed device scratch used by cljxla_b200_attention_decode_static. */
#define CLJXLA_STATIC_ATTN_SCRATCH_BYTES (1u << 20)

/* Decode attention of one layer that allocates no device memory.  No
 * counterpart in the reference: it is the split-KV kernel an executable uses
 * for the printed attention block (attention.clj:343-365), callable directly
 * by hosts that cannot allocate at that point (all free memory already handed
 * to a KV pool, allocator callbacks, code that must not grow the memory pool).
 *
 *   q        bf16 [batch, q_heads, 1, head_dim]          (device)
 *   k_cache  bf16 [batch, kv_heads, positions, head_dim] (device, head_dim/16-byte aligned)
 *   v_cache  bf16 [batch, kv_heads, positions, head_dim] (device, same alignment)
 *   mask     f32  [positions] additive mask shared by every batch row and head (device)
 *   out      f32  [batch, q_heads, 1, head_dim]          (device)
 *
 * scores = bf16(bf16(q.k) * bf16(scale)) + mask, softmax in f32, out = p.v:
 * the printed graph's op order and roundings.  A position whose mask value is
 * at or below -5000 is skipped: it contributes weight 0, which is what the
 * formula gives for the -10000 causal mask whenever some position of the row
 * is unmasked.  A row whose every position is at or below -5000 therefore
 * yields zeros (the formula would give the uniform average, or NaN for -inf).
 * Failures (bad sizes, a failed launch) are returned, never thrown.  head_dim in {32,64,128,256},
 * q_heads a multiple of kv_heads with at most 8 per KV head.  Work is enqueued
 * on `stream` (a cudaStream_t; NULL = legacy default stream) of the calling
 * thread's current device.
 *
 * Partial results live in one file-scope device array per device of
 * CLJXLA_STATIC_ATTN_SCRATCH_BYTES; calls needing more
 * (splits * batch * q_heads * (head_dim + 2) * 4 bytes) are rejected before
 * anything runs.  Nothing in it has to start at zero.  Calls that may overlap
 * on the device race on the scratch.  The first call on each device looks up
 * the scratch address (and may load the module): make it before any stream
 * capture.  Returns 0, or a PJRT_Error_Code with the message in err[errcap]. */
CLJXLA_EXPORT int cljxla_b200_attention_decode_static(const void* q, const void* k_cache, const void* v_cache,
                                                      const float* mask, void* out, int64_t batch, int64_t q_heads,
                                                      int64_t kv_heads, int64_t positions, int64_t head_dim,
                                                      float scale, void* stream, char* err, size_t errcap);

/* ------------------------------------------------- paged key-value cache
 * Serving over a paged cache, for hosts that own device memory themselves (as
 * with cljxla_b200_attention_decode_static).  No counterpart in the
 * reference, whose paged cache is a design note only
 * (docs/xla/paged_attention_vram.md:38-94).  One step of a serving loop is
 *
 *   paged_append     new K / V rows into their pages, K and Q rotated on the way
 *   paged_attention  the step's queries over each sequence's pages
 *   verify_draft     the drafted tokens among them accepted or replaced
 *
 * A step's tokens are packed rows: sequence b has rows starts[b] ..
 * starts[b + 1] - 1, and seq_lens[b] counts its positions, those rows
 * included, so row starts[b] + i is position seq_lens[b] - count + i.  Position
 * j lives in row j % page_size of page page_table[b][j / page_size], for every
 * KV head.  Rows at or behind starts[num_seqs] belong to nobody: nothing is
 * written for them, so a captured graph may carry padding.
 *
 * Every pointer below is a device pointer unless it says otherwise.  starts,
 * seq_lens and page_table are read by the kernels when they run, so a captured
 * graph follows their contents.  What the host cannot see is bounded in the
 * kernels: seq_lens is clamped to [0, 2^30], starts to [0, tokens], and a page
 * number outside [0, num_pages) is a page that is not there, as is every page
 * past pages_per_seq (a longer length keeps its rows' positions): append leaves
 * such rows out, attention leaves such positions out (so a sliding-window layer
 * may give pages back and mark them -1).
 *
 * Work is enqueued on `stream` (a cudaStream_t; NULL = legacy default stream)
 * of the calling thread's current device, without synchronising and without
 * allocating device memory.  The argument structs are read before the call returns.
 * struct_size is sizeof the struct.  Functions return 0, or a PJRT_Error_Code
 * with the message in err[errcap]; a refused call has enqueued nothing. */
typedef struct CLJXLA_PagedKV {
  size_t struct_size;
  void* k_pages; /* [num_pages, kv_heads, page_size, head_dim], strides below */
  void* v_pages;
  int64_t k_page_stride, k_head_stride, k_row_stride; /* in elements, >= 0; head_dim is contiguous */
  int64_t v_page_stride, v_head_stride, v_row_stride;
  int64_t num_pages, kv_heads, page_size, head_dim;   /* head_dim 32, 64, 128 or 256 */
  const int32_t* page_table; /* [num_seqs, pages_per_seq], row stride below */
  const int32_t* seq_lens;   /* [num_seqs] */
  int64_t num_seqs, pages_per_seq, page_table_stride;
  int32_t dtype; /* PJRT_Buffer_Type F32, F16 or BF16: of the pages, and of q, k and v */
  int32_t reserved;
} CLJXLA_PagedKV;

typedef struct CLJXLA_PagedAppendArgs {
  size_t struct_size;
  const void* k; /* [tokens, kv_heads, head_dim], strides in elements, head_dim contiguous */
  const void* v;
  const void* q; /* [tokens, q_heads, head_dim], or NULL: no queries */
  void* q_out;   /* the rotated queries; may be q itself (same strides) */
  int64_t tokens, q_heads;
  int64_t k_token_stride, k_head_stride, v_token_stride, v_head_stride;
  int64_t q_token_stride, q_head_stride, q_out_token_stride, q_out_head_stride;
  const int32_t* starts;  /* [num_seqs + 1], ascending; NULL: tokens / num_seqs rows each */
  const float* inv_freq;  /* [rotary_dim / 2] angle per position of each pair; NULL with rotary_dim 0 */
  int64_t rotary_dim;     /* even, <= head_dim: elements past it are copied */
  int32_t interleaved;    /* pairs (2i, 2i + 1) instead of (i, i + rotary_dim / 2) */
  float rope_scale;       /* factor on cos and sin (1 for none) */
} CLJXLA_PagedAppendArgs;

/* Rotates K and Q rows by their positions and writes K and V into the pages:
 * (x1, x2) -> rope_scale * (x1 cos a - x2 sin a, x2 cos a + x1 sin a) with a =
 * position * inv_freq[i] (the angle reduced in 64 bits), computed in f32 and
 * rounded once.  Two rows of one call must not share a (page, row): which of
 * them stays is not defined.  K and V pages must be 16-byte aligned rows; k, v, q
 * and q_out may begin at any element, but 16-byte aligned ones with rotary_dim / 2
 * (interleaved: rotary_dim) a multiple of 16 bytes are two to three times as fast. */
CLJXLA_EXPORT int cljxla_b200_paged_append(const CLJXLA_PagedKV* kv, const CLJXLA_PagedAppendArgs* args, void* stream,
                                           char* err, size_t errcap);

typedef struct CLJXLA_PagedAttentionArgs {
  size_t struct_size;
  const void* q; /* [tokens, q_heads, head_dim], strides in elements, 16-byte aligned rows */
  void* out;     /* same shape, out_dtype, 16-byte aligned rows */
  int64_t tokens, q_heads; /* q_heads a multiple of kv_heads */
  int64_t q_token_stride, q_head_stride, out_token_stride, out_head_stride;
  const int32_t* starts; /* [num_seqs + 1], ascending; NULL: tokens / num_seqs rows each */
  int64_t max_tokens;    /* upper bound of a sequence's rows (rows past it are not computed).  Row tiles are
                            chosen for it, so give a tight one: 64 sequences of one row and 2048 positions take
                            165 us with 1, 419 with 64 */
  int64_t window;        /* >= 0: a row sees its own position and `window` before it; < 0: all */
  float scale, softcap;  /* score = softcap * tanh(scale * q.k / softcap), or scale * q.k with softcap 0 */
  int32_t out_dtype;     /* the pages' type, or F32 */
  int32_t reserved;
  void* workspace;       /* of cljxla_b200_paged_attention_workspace bytes, 16-byte aligned; needs no
                            initialisation; calls that may overlap need one each */
  int64_t workspace_bytes;
} CLJXLA_PagedAttentionArgs;

/* Row r at position p of its sequence: out = sum_j w_j v_j / sum_j w_j over the
 * positions j <= p (and j >= p - window) of the sequence's pages, w_j =
 * exp(score_j - max).  A row that sees no position is zero, as is one whose scores
 * are all -inf.  What a row does not see (later drafts, evicted pages, page tails)
 * may hold anything, NaN and infinities included; an infinity in a value that it
 * does see makes the result infinite or NaN.  K and V pages must be 16-byte aligned
 * rows. */
CLJXLA_EXPORT int cljxla_b200_paged_attention(const CLJXLA_PagedKV* kv, const CLJXLA_PagedAttentionArgs* args,
                                              void* stream, char* err, size_t errcap);

/* Bytes of workspace the call above needs on the current device (0: none;
 * pointers are not looked at).  Depends on the sizes, not on the contents. */
CLJXLA_EXPORT int cljxla_b200_paged_attention_workspace(const CLJXLA_PagedKV* kv,
                                                        const CLJXLA_PagedAttentionArgs* args, int64_t* bytes,
                                                        char* err, size_t errcap);

typedef struct CLJXLA_VerifyDraftArgs {
  size_t struct_size;
  const void* target; /* [tokens, vocab] logits: row r is the distribution of the token behind row r */
  const void* draft;  /* [tokens, vocab] logits row r + 1's token was drawn from; NULL: the guesses have no
                         distribution (each counts as certain). A sequence's last row is not read: the
                         buffer may end before it */
  const int32_t* tokens_in; /* [tokens] the tokens the rows were fed: rows past a sequence's first are drafts */
  const int32_t* starts;    /* [num_seqs + 1], ascending; NULL: tokens / num_seqs rows each */
  const float* uniform;     /* [tokens] in [0, 1): row r decides on row r + 1's token; NULL when greedy */
  const float* race;        /* [num_seqs, vocab] positive, exponentially distributed; NULL when greedy */
  int64_t tokens, num_seqs, vocab, max_tokens; /* max_tokens: upper bound of a sequence's rows, at most 128
                                                  (drafts past it count as rejected) */
  int64_t target_stride, draft_stride, race_stride; /* elements from row to row */
  float temperature, draft_temperature; /* logits are divided by these, > 0 */
  int32_t dtype;  /* of target and draft: F32, F16 or BF16 */
  int32_t greedy;
  int32_t* tokens_out; /* [num_seqs, max_tokens]: accepted drafts, then the target's own token, then -1 */
  int32_t* accepted;   /* [num_seqs]: accepted drafts */
  float* logprobs;     /* [num_seqs, max_tokens] log p of each token in tokens_out (0 behind them), or NULL */
  const int32_t* seq_lens; /* [num_seqs], or NULL with new_lens */
  int32_t* new_lens;       /* seq_lens less the rejected drafts; may be seq_lens itself */
  void* workspace;         /* of cljxla_b200_verify_draft_workspace bytes, 16-byte aligned; as above */
  int64_t workspace_bytes;
} CLJXLA_VerifyDraftArgs;

/* With p = softmax(target / temperature) and q = softmax(draft /
 * draft_temperature), a sequence's drafts x are accepted in order while
 * uniform * q(x) < p(x).  The token behind the accepted ones is argmax_v
 * w_v / race_v, a draw from w / sum w: w = max(p - q, 0) at a rejection (p
 * without x where draft is NULL; p where that leaves nothing), p behind the last
 * draft.  greedy: x is accepted while it is the argmax, and the argmax follows.
 * Ties go to the lowest index.  A draft outside [0, vocab) is rejected.  Logits
 * may be -inf (probability 0) or any finite value.  p and q are held in f32: in w
 * one below 2^-126 is 0, and a difference below 2^-22 of them is rounding (drafts
 * drawn from q meet such a w less than once in 2^22).  A NaN is never an argmax, and
 * leaves a sampled row without a token; a row without a finite maximum gives token -1. A
 * sequence without rows gives 0 accepted, -1 throughout and its length. */
CLJXLA_EXPORT int cljxla_b200_verify_draft(const CLJXLA_VerifyDraftArgs* args, void* stream, char* err,
                                           size_t errcap);
CLJXLA_EXPORT int cljxla_b200_verify_draft_workspace(const CLJXLA_VerifyDraftArgs* args, int64_t* bytes, char* err,
                                                     size_t errcap);

#ifdef __cplusplus
}
#endif

#endif /* CLJXLA_B200_H_ */
