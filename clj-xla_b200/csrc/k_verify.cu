// Verification of drafted tokens against the target's logits.
//
// With p = softmax(l / T) and q = softmax(d / T'), drafts x are accepted in
// order while u q(x) < p(x); the token behind them is argmax_v w_v / e_v, w =
// max(p - q, 0) at a rejection and p behind the last draft.  Greedily: x is
// accepted while it is argmax l, and argmax l follows.
//
// What bounds it: the logits are read once for a maximum and a sum of
// exponentials per row (HBM), and the one row of each sequence that decides is
// read again for the race (L2 for what is left there, HBM for e).  Two kernels:
// * verify_rows_kernel, one CTA per (row, slice of the vocabulary): running
//   maximum, sum and, greedily, the argmax, 16-byte loads, four in flight a thread;
// * verify_pick_kernel, one cluster of CTAs per sequence: every CTA joins the
//   rows' slices and finds the accepted count for itself (a few values), races
//   over its slice of the one deciding row, and the first CTA takes the best
//   of the cluster through distributed shared memory.  A single sequence so still
//   has eight SMs, and no CTA waits for another launch.
// Measured (B200): 102 rows of 262144 bf16 logits with drafts 39 us, of which the
// first kernel 22 (4.1 TB/s; its issue slots are 64 % busy) and the race 11; greedily
// 161 rows of 256000 22 us; five rows of 50257 in f32 10 us.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <type_traits>

#include "common.h"
#include "paged.h"

namespace cljxla {
namespace {

namespace cg = cooperative_groups;

constexpr int VD_THREADS = 256, VD_PICK_THREADS = 512;
constexpr int VD_MAX_ROWS = 128;    // of a sequence
constexpr int VD_MAX_SPLITS = 32;   // slices of a row: a warp joins them
constexpr int VD_CLUSTER = 8;
constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float vd_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float vd_f(__half v) { return __half2float(v); }
__device__ __forceinline__ float vd_f(float v) { return v; }
__device__ __forceinline__ float vd_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// the values of a 16-byte vector
template <typename T>
__device__ __forceinline__ void vd_unpack(const uint4& v, float* x) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 4) {
      x[i] = __uint_as_float(w[i]);
    } else if constexpr (std::is_same<T, __half>::value) {
      const float2 f = __half22float2(*(const __half2*)&w[i]);
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    } else {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
}

// Statistics of a set of logits: the maximum m, the sum of 2^(x c - R) with the
// reference R = m c as it rounds (the same R wherever m is the same, so its
// rounding cancels in every quotient and one FMA gives each exponent), and the
// lowest index of the maximum.  Of nothing, or of -inf alone: (-inf, 0, -1).  A
// NaN is no maximum and makes the sum one.
//
// R is kept within 2^24, so that it is finite and its rounding at most half a bit.
// Parts whose maximum is lower (finite masks) so have sums next to zero or zero, as
// they should beside any other; a whole row beyond that (logits near the ends of f32
// or bf16, or next to no temperature) is "far": its sum is made again from x - m.
struct Stat {
  float m, s;
  int i;
};
constexpr float kFar = 16777216.f;
__device__ __forceinline__ float vd_ref(float m, float c) { return fminf(fmaxf(__fmul_rn(m, c), -kFar), kFar); }
__device__ __forceinline__ bool vd_far(float m, float c) { return fabsf(m * c) > kFar && m > -INFINITY; }
// base-2 logarithm of the weight of x in a row with maximum m (NaN for x = m = +inf)
__device__ __forceinline__ float vd_power(float x, float m, float c) {
  return vd_far(m, c) ? (x - m) * c : fmaf(x, c, -vd_ref(m, c));
}
// one logit more
__device__ __forceinline__ void vd_take(Stat& a, float f, int v, float c) {
  const float s = vd_ex2(fmaf(f, c, -vd_ref(f, c)));
  if (f > a.m) {
    a.s *= vd_ex2(vd_ref(a.m, c) - vd_ref(f, c));
    a.m = f;
    a.i = v;
    a.s += s;
  } else {
    a.s += s * vd_ex2(f == f ? vd_ref(f, c) - vd_ref(a.m, c) : 0.f);
    if (f == a.m && f > -INFINITY) a.i = min(a.i, v);
  }
}
// The lanes' parts: their maximum, the sums brought to it and added, the lowest index.
__device__ __forceinline__ void vd_join_warp(Stat& a, float c) {
  float M = a.m;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
  a.s *= vd_ex2(vd_ref(a.m, c) - vd_ref(M, c));  // at most 1
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) a.s += __shfl_xor_sync(0xffffffffu, a.s, o);
  a.i = (int)__reduce_min_sync(0xffffffffu, a.m == M ? (unsigned)a.i : 0xffffffffu);  // none: -1, the largest
  a.m = M;
}

// the largest of a 16-byte vector's values (NaN aside)
template <typename T>
__device__ __forceinline__ float vd_top(const uint4& v) {
  if constexpr (sizeof(T) == 4) {
    return fmaxf(fmaxf(__uint_as_float(v.x), __uint_as_float(v.y)), fmaxf(__uint_as_float(v.z), __uint_as_float(v.w)));
  } else if constexpr (std::is_same<T, __half>::value) {
    const __half2 t = __hmax2(__hmax2(*(const __half2*)&v.x, *(const __half2*)&v.y),
                              __hmax2(*(const __half2*)&v.z, *(const __half2*)&v.w));
    return __half2float(__hmax(__low2half(t), __high2half(t)));
  } else {
    const __nv_bfloat162 t = __hmax2(__hmax2(*(const __nv_bfloat162*)&v.x, *(const __nv_bfloat162*)&v.y),
                                     __hmax2(*(const __nv_bfloat162*)&v.z, *(const __nv_bfloat162*)&v.w));
    return __bfloat162float(__hmax(__low2bfloat16(t), __high2bfloat16(t)));
  }
}

// First row, rows that are looked at and rows of sequence b.
__device__ __forceinline__ void vd_rows(const VerifyParams& P, int b, int& first, int& count, int& all) {
  if (!P.starts) {
    first = b * P.each;
    count = P.each;
  } else {
    const int lo = min(max(P.starts[b], 0), P.tokens), hi = min(max(P.starts[b + 1], 0), P.tokens);
    first = lo;
    count = max(hi - lo, 0);
  }
  all = count;
  count = min(count, P.max_tokens);
}

// workspace: [2][tokens][splits] (max, sum) pairs, then [tokens][splits] indices
__device__ __forceinline__ float2* vd_part(const VerifyParams& P, int which, int row) {
  return (float2*)P.part + ((int64_t)which * P.tokens + row) * P.splits;
}
__device__ __forceinline__ int* vd_index(const VerifyParams& P, int row) {
  return (int*)((float2*)P.part + (int64_t)2 * P.tokens * P.splits) + (int64_t)row * P.splits;
}

template <typename T, bool GREEDY>
__global__ void __launch_bounds__(VD_THREADS) verify_rows_kernel(const __grid_constant__ VerifyParams P) {
  constexpr int V = 16 / sizeof(T), U = 4;
  pdl_enter();
  const int split = blockIdx.y, row = blockIdx.x, which = blockIdx.z, tid = threadIdx.x;
  const T* const x = (const T*)((which ? P.draft : P.target) + row * (which ? P.draft_stride : P.target_stride));
  const float c = (which ? P.inv_td : P.inv_t) * kLog2e;
  // elements in front of the first 16-byte boundary, whole vectors, and the rest
  const int64_t head = min((int64_t)((16 - ((uintptr_t)x & 15)) & 15) / (int64_t)sizeof(T), P.vocab);
  const int64_t vecs = (P.vocab - head) / V;
  const int64_t lo = vecs * split / P.splits, hi = vecs * (split + 1) / P.splits;
  const uint4* const xv = (const uint4*)(x + head);
  // U vectors ahead of the ones in work, the target's first while the row's sequence is
  // looked up.  A sequence's last row of the draft need not be there: not before.
  uint4 ahead[U];
  auto fetch = [&](int64_t at) {
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (at + u * VD_THREADS < hi) ahead[u] = xv[at + u * VD_THREADS];
  };
  if (!which) fetch(lo + tid);
  const int b = seq_of_row(P.starts, P.num_seqs, P.each, row);
  if (b < 0) return;
  int first, count, all;
  vd_rows(P, b, first, count, all);
  if (row - first >= count - which) return;  // not looked at; the draft of a sequence's last row is none
  if (which) fetch(lo + tid);
  Stat a{-INFINITY, 0.f, -1};
  if (split == 0 && tid < head) vd_take(a, vd_f(x[tid]), tid, c);
  float ref = vd_ref(a.m, c);
  for (int64_t at = lo + tid; at < hi; at += U * VD_THREADS) {
    uint4 raw[U];
#pragma unroll
    for (int u = 0; u < U; ++u) raw[u] = ahead[u];
    fetch(at + U * VD_THREADS);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (at + u * VD_THREADS >= hi) break;
      const float top = vd_top<T>(raw[u]);
      float f[V];
      vd_unpack<T>(raw[u], f);
      if (top > a.m) {
        if (GREEDY) {  // later vectors have higher indices: the first of the larger values stays
#pragma unroll
          for (int i = V - 1; i >= 0; --i)
            if (f[i] == top) a.i = (int)(head + (at + u * VD_THREADS) * V + i);
        }
        const float R = vd_ref(top, c);
        a.s *= vd_ex2(ref - R);
        a.m = top;
        ref = R;
      }
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < V; ++i) sum += vd_ex2(fmaf(f[i], c, -ref));
      a.s += sum;
    }
  }
  const int64_t rest = head + vecs * V + tid;
  if (split == P.splits - 1 && rest < P.vocab) vd_take(a, vd_f(x[rest]), (int)rest, c);
  __shared__ Stat s_warp[VD_THREADS / 32];
  vd_join_warp(a, c);
  if ((tid & 31) == 0) s_warp[tid >> 5] = a;
  __syncthreads();
  if (tid >= 32) return;
  a = tid < VD_THREADS / 32 ? s_warp[tid] : Stat{-INFINITY, 0.f, -1};
  vd_join_warp(a, c);
  if (tid) return;
  vd_part(P, which, row)[split] = make_float2(a.m, a.s);
  if (GREEDY) vd_index(P, row)[split] = a.i;
}

// The race's best so far: the larger w / e, compared by cross products (a
// reciprocal per token would cost a third of the exponentials again), or the
// lower index of equal ones.  Nothing yet: (0, 1, 0, -1).
struct Best {
  float w, e, l;  // l: the token's logit
  int i;
};
__device__ __forceinline__ void vd_best(Best& a, const Best& b) {
  const float x = b.w * a.e, y = a.w * b.e;
  if (b.i >= 0 && (a.i < 0 || x > y || (x == y && b.i < a.i))) a = b;
}
__device__ __forceinline__ void vd_best_warp(Best& a) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    Best b;
    b.w = __shfl_xor_sync(0xffffffffu, a.w, o);
    b.e = __shfl_xor_sync(0xffffffffu, a.e, o);
    b.l = __shfl_xor_sync(0xffffffffu, a.l, o);
    b.i = __shfl_xor_sync(0xffffffffu, a.i, o);
    vd_best(a, b);
  }
}

// The sum of a far row's weights, by all threads of a CTA; the same in each.
template <typename T>
__device__ __noinline__ float vd_far_sum(const T* x, int64_t vocab, float m, float c, float* s_far) {
  float sum = 0.f;
#pragma unroll 8
  for (int64_t v = threadIdx.x; v < vocab; v += VD_PICK_THREADS) sum += vd_ex2((vd_f(x[v]) - m) * c);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  __syncthreads();  // what a call before left there is read
  if ((threadIdx.x & 31) == 0) s_far[threadIdx.x >> 5] = sum;
  __syncthreads();
  sum = 0.f;
  for (int w = 0; w < VD_PICK_THREADS / 32; ++w) sum += s_far[w];
  return sum;
}

template <typename T>
__global__ void __launch_bounds__(VD_PICK_THREADS, 2) verify_pick_kernel(const __grid_constant__ VerifyParams P) {
  constexpr int THREADS = VD_PICK_THREADS, WARPS = THREADS / 32;
  constexpr int V = 16 / sizeof(T);  // elements a thread takes at a time
  __shared__ float s_max[2][VD_MAX_ROWS], s_sum[2][VD_MAX_ROWS];
  __shared__ int s_arg[VD_MAX_ROWS], s_taken;
  __shared__ Best s_best[WARPS], s_mine[2];
  __shared__ float s_far[WARPS];
  cg::cluster_group cluster = cg::this_cluster();
  const int ctas = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int b = blockIdx.x / ctas, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t lots = (P.vocab + V - 1) / V, lo = lots * rank / ctas, hi = lots * (rank + 1) / ctas;
  // what comes from the caller's tensors is fetched before the wait: the kernel
  // that this one overlaps has itself waited for whatever wrote them
  int first, count, all;
  vd_rows(P, b, first, count, all);
  if (tid == 0) s_taken = max(count - 1, 0);
  const float c = P.inv_t * kLog2e, cd = P.inv_td * kLog2e;
  auto target = [&](int r) { return (const T*)(P.target + (first + r) * P.target_stride); };
  auto draft = [&](int r) { return (const T*)(P.draft + (first + r) * P.draft_stride); };
  // thread r's draft, with its logits and random number
  int x = -1;
  bool valid = false;
  float lx = 0.f, dx = 0.f, ux = 0.f;
  if (tid < count - 1) {
    x = P.tokens_in[first + tid + 1];
    valid = x >= 0 && x < P.vocab;
    if (valid) {
      lx = vd_f(target(tid)[x]);
      if (P.draft) dx = vd_f(draft(tid)[x]);
    }
    if (!P.greedy) ux = P.uniform[first + tid];
  }
  pdl_enter();
  // the rows' slices, joined
  bool far = false;
  for (int i = warp; i < 2 * count; i += WARPS) {
    const int which = i >= count, r = which ? i - count : i;
    if (which && (!P.draft || r == count - 1)) continue;
    Stat a{-INFINITY, 0.f, -1};
    if (lane < P.splits) {
      const float2 ms = vd_part(P, which, first + r)[lane];
      a.m = ms.x;
      a.s = ms.y;
      if (P.greedy) a.i = vd_index(P, first + r)[lane];
    }
    vd_join_warp(a, which ? cd : c);
    far = far || vd_far(a.m, which ? cd : c);
    if (lane == 0) {
      s_max[which][r] = a.m;
      s_sum[which][r] = a.s;
      if (!which) s_arg[r] = a.m - a.m == 0.f ? a.i : -1;
    }
  }
  far = __syncthreads_or(far);
  for (int i = 0; far && i < 2 * count; ++i) {
    const int which = i >= count, r = which ? i - count : i;
    if (which && (!P.draft || r == count - 1)) break;
    const float m = s_max[which][r], k = which ? cd : c;
    if (vd_far(m, k)) s_sum[which][r] = vd_far_sum<T>(which ? draft(r) : target(r), P.vocab, m, k, s_far);
  }
  auto logp = [&](float l, int r) { return (vd_power(l, s_max[0][r], c) - log2f(s_sum[0][r])) * 0.6931471805599453f; };
  if (tid < count - 1) {
    bool good = valid;
    if (good && P.greedy) good = x == s_arg[tid];
    if (good && !P.greedy) {
      // in logarithms: both sides may lie far below the smallest float
      float lq = 0.f;
      if (P.draft) lq = vd_power(dx, s_max[1][tid], cd) - log2f(s_sum[1][tid]);
      good = log2f(ux) + lq < vd_power(lx, s_max[0][tid], c) - log2f(s_sum[0][tid]);
    }
    if (!good) atomicMin(&s_taken, tid);
  }
  __syncthreads();
  const int taken = s_taken;
  int token = -1;
  float token_l = 0.f;
  if (P.greedy) {
    if (count > 0) token = s_arg[taken];
  } else if (count > 0) {
    const bool rejected = taken < count - 1;
    bool residual = rejected && P.draft;
    int out = rejected && !P.draft ? P.tokens_in[first + taken + 1] : -1;
    const T* const l = target(taken);
    const T* const d = residual ? draft(taken) : l;
    const float* const e = P.race + b * P.race_stride;
    const float ref = vd_ref(s_max[0][taken], c), inv = 1.f / s_sum[0][taken];
    const float refd = residual ? vd_ref(s_max[1][taken], cd) : 0.f, invd = residual ? 1.f / s_sum[1][taken] : 0.f;
    const bool aligned = (((uintptr_t)e | (uintptr_t)l | (uintptr_t)d) & 15) == 0;
    // the race for w; once more for p in the rare case that w is nothing
    for (int pass = 0; pass < 2 && token < 0; ++pass) {
      Best best{0.f, 1.f, 0.f, -1};
      auto enter = [&](float w, float lv, float ev, int64_t v) {
        if (w * best.e > best.w * ev && (int)v != out) best = {w, ev, lv, (int)v};  // a thread's indices ascend
      };
      auto race = [&](float lv, float dv, float ev, int64_t v) {
        float w = vd_ex2(fmaf(lv, c, -ref)) * inv;
        if (residual) w -= vd_ex2(fmaf(dv, cd, -refd)) * invd;
        enter(w, lv, ev, v);
      };
      const int64_t end = min(hi * V, P.vocab);
      if (vd_far(s_max[0][taken], c) || (residual && vd_far(s_max[1][taken], cd))) {
        for (int64_t v = lo * V + tid; v < end; v += THREADS) {
          float w = vd_ex2(vd_power(vd_f(l[v]), s_max[0][taken], c)) * inv;
          if (residual) w -= vd_ex2(vd_power(vd_f(d[v]), s_max[1][taken], cd)) * invd;
          enter(w, vd_f(l[v]), e[v], v);
        }
      } else if (aligned) {
        uint4 la, da = {}, ln, dn = {};
        float4 ea[V / 4], en[V / 4];
        auto fetch = [&](int64_t at) {  // one lot ahead of the one in work
          const int64_t v = at * V;
          if (at >= hi || v + V > P.vocab) return;
          ln = *(const uint4*)(l + v);
          if (residual) dn = *(const uint4*)(d + v);
#pragma unroll
          for (int i = 0; i < V / 4; ++i) en[i] = *(const float4*)(e + v + 4 * i);
        };
        fetch(lo + tid);
        for (int64_t at = lo + tid; at < hi; at += THREADS) {
          const int64_t v = at * V;
          if (v + V > P.vocab) {  // the vocabulary's last elements
            for (int64_t k = v; k < P.vocab; ++k) race(vd_f(l[k]), vd_f(d[k]), e[k], k);
            break;
          }
          la = ln;
          da = dn;
#pragma unroll
          for (int i = 0; i < V / 4; ++i) ea[i] = en[i];
          fetch(at + THREADS);
          float lv[V], dv[V];
          vd_unpack<T>(la, lv);
          vd_unpack<T>(da, dv);
#pragma unroll
          for (int i = 0; i < V; ++i) {
            const float4& f = ea[i / 4];
            race(lv[i], dv[i], i % 4 == 0 ? f.x : i % 4 == 1 ? f.y : i % 4 == 2 ? f.z : f.w, v + i);
          }
        }
      } else {
        // rows that start anywhere: element by element, a warp's loads side by side
#pragma unroll 8
        for (int64_t v = lo * V + tid; v < end; v += THREADS) race(vd_f(l[v]), residual ? vd_f(d[v]) : 0.f, e[v], v);
      }
      vd_best_warp(best);
      if (lane == 0) s_best[warp] = best;
      __syncthreads();
      if (warp == 0) {
        Best a = lane < WARPS ? s_best[lane] : Best{0.f, 1.f, 0.f, -1};
        vd_best_warp(a);
        if (lane == 0) s_mine[pass] = a;
      }
      cluster.sync();  // the CTAs' best are there
      Best a{0.f, 1.f, 0.f, -1};
      if (lane < ctas) a = *cluster.map_shared_rank(&s_mine[pass], lane);
      vd_best_warp(a);
      token = a.i;  // the same in every thread of the cluster
      token_l = a.l;
      residual = false;
      out = -1;
    }
    cluster.barrier_arrive();
  }
  if (rank == 0) {
    if (tid < P.max_tokens) {  // at most VD_MAX_ROWS
      const int t = tid < taken ? x : tid == taken && count > 0 ? token : -1;
      P.tokens_out[(int64_t)b * P.max_tokens + tid] = t;
      if (P.logprobs) {
        if (tid == taken && t >= 0) lx = P.greedy ? s_max[0][taken] : token_l;
        P.logprobs[(int64_t)b * P.max_tokens + tid] = t < 0 ? 0.f : logp(lx, tid);
      }
    }
    if (tid == 0) {
      P.accepted[b] = taken;
      if (P.new_lens) P.new_lens[b] = P.seq_lens[b] - max(all - 1 - taken, 0);
    }
  }
  if (!P.greedy && count > 0) cluster.barrier_wait();  // no CTA leaves while its best is read
}

template <typename T>
void launch_t(const VerifyParams& p, cudaStream_t s) {
  if (p.tokens > 0) {
    const dim3 grid((unsigned)p.tokens, (unsigned)p.splits, p.draft ? 2 : 1);
    if (p.greedy) launch_k(verify_rows_kernel<T, true>, grid, VD_THREADS, 0, s, 1, p);
    else launch_k(verify_rows_kernel<T, false>, grid, VD_THREADS, 0, s, 1, p);
  }
  // a cluster races as wide as the vocabulary gives every thread a few vectors
  int ctas = 1;
  while (!p.greedy && ctas < VD_CLUSTER && p.vocab > (int64_t)ctas * VD_PICK_THREADS * 8) ctas *= 2;
  launch_k(verify_pick_kernel<T>, dim3((unsigned)(p.num_seqs * ctas)), VD_PICK_THREADS, 0, s, ctas, p);
}

}  // namespace

// Slices of a row: up to eight CTAs per SM over all rows, none below eight logits
// (one 16-bit vector or two of f32) a thread.
int verify_splits(int64_t tokens, int64_t vocab, bool draft) {
  const int64_t rows = std::max<int64_t>(tokens * (draft ? 2 : 1), 1);
  const int64_t want = std::max<int64_t>(8 * (int64_t)device_sm_count() / rows, 1);
  const int64_t most = std::max<int64_t>(vocab / (VD_THREADS * 8), 1);
  return (int)std::min<int64_t>(std::min(want, most), VD_MAX_SPLITS);
}

int64_t verify_workspace(const VerifyParams& p) { return (int64_t)p.tokens * p.splits * (2 * 8 + 4); }

void launch_verify(const VerifyParams& p, cudaStream_t s) {
  if (p.dt == KDT_F32) launch_t<float>(p, s);
  else if (p.dt == KDT_F16) launch_t<__half>(p, s);
  else launch_t<__nv_bfloat16>(p, s);
}

}  // namespace cljxla
