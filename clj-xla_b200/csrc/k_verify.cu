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

constexpr int VD_THREADS = 256;
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

// Statistics of a set of logits: maximum, sum of 2^((x - max) c), and the lowest
// index of the maximum.  Of nothing, or of -inf alone: (-inf, 0, -1).  A NaN
// is no maximum and makes the sum one.
struct Stat {
  float m, s;
  int i;
};
__device__ __forceinline__ void vd_join(Stat& a, const Stat& b, float c) {
  const float M = fmaxf(a.m, b.m), base = M == -INFINITY ? 0.f : M;
  if (b.i >= 0 && (a.i < 0 || b.m > a.m || (b.m == a.m && b.i < a.i))) a.i = b.i;
  a.s = a.s * vd_ex2((a.m - base) * c) + b.s * vd_ex2((b.m - base) * c);
  a.m = M;
}
__device__ __forceinline__ void vd_join_warp(Stat& a, float c) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    Stat b;
    b.m = __shfl_xor_sync(0xffffffffu, a.m, o);
    b.s = __shfl_xor_sync(0xffffffffu, a.s, o);
    b.i = __shfl_xor_sync(0xffffffffu, a.i, o);
    vd_join(a, b, c);
  }
}

__device__ __forceinline__ void vd_rows(const VerifyParams& P, int b, int& first, int& count) {
  if (!P.starts) {
    first = b * P.each;
    count = P.each;
  } else {
    const int lo = min(max(P.starts[b], 0), P.tokens), hi = min(max(P.starts[b + 1], 0), P.tokens);
    first = lo;
    count = max(hi - lo, 0);
  }
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
  const int b = seq_of_row(P.starts, P.num_seqs, P.each, row);
  if (b < 0) return;
  int first, count;
  vd_rows(P, b, first, count);
  if (row - first >= count - which) return;  // not looked at; the draft of a sequence's last row is none
  const T* const x = (const T*)((which ? P.draft : P.target) + row * (which ? P.draft_stride : P.target_stride));
  const float c = (which ? P.inv_td : P.inv_t) * kLog2e;
  Stat a{-INFINITY, 0.f, -1};
  auto take = [&](float f, int64_t v) {
    Stat one{f, f == -INFINITY ? 0.f : f == f ? 1.f : f, f > -INFINITY ? (int)v : -1};
    if (!(f == f)) one.m = -INFINITY;
    vd_join(a, one, c);
  };
  // elements in front of the first 16-byte boundary, whole vectors, and the rest
  const int64_t head = min((int64_t)((16 - ((uintptr_t)x & 15)) & 15) / (int64_t)sizeof(T), P.vocab);
  const int64_t vecs = (P.vocab - head) / V;
  if (split == 0 && tid < head) take(vd_f(x[tid]), tid);
  const int64_t lo = vecs * split / P.splits, hi = vecs * (split + 1) / P.splits;
  const uint4* const xv = (const uint4*)(x + head);
  for (int64_t at = lo + tid; at < hi; at += U * VD_THREADS) {
    uint4 raw[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (at + u * VD_THREADS < hi) raw[u] = xv[at + u * VD_THREADS];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (at + u * VD_THREADS >= hi) break;
      float f[V];
      vd_unpack<T>(raw[u], f);
      float top = f[0];
#pragma unroll
      for (int i = 1; i < V; ++i) top = fmaxf(top, f[i]);
      if (top > a.m) {
        if (GREEDY) {  // later vectors have higher indices: the first of the larger values stays
#pragma unroll
          for (int i = V - 1; i >= 0; --i)
            if (f[i] == top) a.i = (int)(head + (at + u * VD_THREADS) * V + i);
        }
        a.s *= vd_ex2((a.m - top) * c);
        a.m = top;
      }
      const float base = a.m == -INFINITY ? 0.f : a.m;
#pragma unroll
      for (int i = 0; i < V; ++i) a.s += vd_ex2((f[i] - base) * c);
    }
  }
  if (split == P.splits - 1 && tid < P.vocab - head - vecs * V) take(vd_f(x[head + vecs * V + tid]), head + vecs * V + tid);
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

// a token with a positive weight: the larger key, or the lower index of equal ones
struct Best {
  float key;
  int i;
};
__device__ __forceinline__ void vd_best(Best& a, const Best& b) {
  if (b.i >= 0 && (a.i < 0 || b.key > a.key || (b.key == a.key && b.i < a.i))) a = b;
}
__device__ __forceinline__ void vd_best_warp(Best& a) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    Best b;
    b.key = __shfl_xor_sync(0xffffffffu, a.key, o);
    b.i = __shfl_xor_sync(0xffffffffu, a.i, o);
    vd_best(a, b);
  }
}

template <typename T>
__global__ void __launch_bounds__(VD_THREADS) verify_pick_kernel(const __grid_constant__ VerifyParams P) {
  constexpr int V = 4;  // elements a thread takes at a time
  __shared__ float s_max[2][VD_MAX_ROWS], s_sum[2][VD_MAX_ROWS];
  __shared__ int s_arg[VD_MAX_ROWS], s_taken;
  __shared__ Best s_best[2][VD_THREADS / 32], s_mine[2];
  cg::cluster_group cluster = cg::this_cluster();
  const int ctas = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int b = blockIdx.x / ctas, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  pdl_enter();
  int first, count;
  vd_rows(P, b, first, count);
  if (tid == 0) s_taken = max(count - 1, 0);
  const float c = P.inv_t * kLog2e, cd = P.inv_td * kLog2e;
  // the rows' slices, joined
  for (int i = warp; i < 2 * count; i += VD_THREADS / 32) {
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
    if (lane == 0) {
      s_max[which][r] = a.m;
      s_sum[which][r] = a.s;
      if (!which) s_arg[r] = a.m - a.m == 0.f ? a.i : -1;
    }
  }
  __syncthreads();
  auto target = [&](int r) { return (const T*)(P.target + (first + r) * P.target_stride); };
  auto draft = [&](int r) { return (const T*)(P.draft + (first + r) * P.draft_stride); };
  auto logp = [&](int r, int x) { return (vd_f(target(r)[x]) - s_max[0][r]) * P.inv_t - logf(s_sum[0][r]); };
  if (tid < count - 1) {
    const int x = P.tokens_in[first + tid + 1];
    bool good = x >= 0 && x < P.vocab;
    if (good && P.greedy) good = x == s_arg[tid];
    if (good && !P.greedy) {
      // in logarithms: both sides may lie far below the smallest float
      float lq = 0.f;
      if (P.draft) lq = (vd_f(draft(tid)[x]) - s_max[1][tid]) * P.inv_td - logf(s_sum[1][tid]);
      good = logf(P.uniform[first + tid]) + lq < logp(tid, x);
    }
    if (!good) atomicMin(&s_taken, tid);
  }
  __syncthreads();
  const int taken = s_taken;
  int token = -1;
  if (P.greedy) {
    if (count > 0) token = s_arg[taken];
  } else {
    if (count > 0) {
      const bool rejected = taken < count - 1, residual = rejected && P.draft;
      const int out = rejected && !P.draft ? P.tokens_in[first + taken + 1] : -1;
      const T *const l = target(taken), *const d = residual ? draft(taken) : l;
      const float* const e = P.race + b * P.race_stride;
      const float m = s_max[0][taken], inv = 1.f / s_sum[0][taken];
      const float md = s_max[1][taken], invd = 1.f / s_sum[1][taken];
      Best best[2] = {{0.f, -1}, {0.f, -1}};  // of w, and of p for where w is nothing
      auto race = [&](float lv, float dv, float ev, int64_t v) {
        const float p = vd_ex2((lv - m) * c) * inv;
        const float w = residual ? p - vd_ex2((dv - md) * cd) * invd : v == out ? 0.f : p;
        if (w > 0.f) vd_best(best[0], {w / ev, (int)v});
        else if (best[0].i < 0 && p > 0.f) vd_best(best[1], {p / ev, (int)v});
      };
      const bool aligned = (((uintptr_t)e | (uintptr_t)l * (4 / sizeof(T)) | (uintptr_t)d * (4 / sizeof(T))) & 15) == 0;
      const int64_t lots = (P.vocab + V - 1) / V, lo = lots * rank / ctas, hi = lots * (rank + 1) / ctas;
#pragma unroll 2
      for (int64_t at = lo + tid; at < hi; at += VD_THREADS) {
        const int64_t v = at * V;
        float lv[V], dv[V], ev[V];
        if (aligned && v + V <= P.vocab) {
          const float4 f = *(const float4*)(e + v);
          ev[0] = f.x; ev[1] = f.y; ev[2] = f.z; ev[3] = f.w;
          if constexpr (sizeof(T) == 4) {
            vd_unpack<T>(*(const uint4*)(l + v), lv);
            if (residual) vd_unpack<T>(*(const uint4*)(d + v), dv);
          } else {
            float t[8];
            const uint2 w = *(const uint2*)(l + v);
            uint2 w2 = w;
            if (residual) w2 = *(const uint2*)(d + v);
            vd_unpack<T>(make_uint4(w.x, w.y, w2.x, w2.y), t);
#pragma unroll
            for (int i = 0; i < V; ++i) {
              lv[i] = t[i];
              dv[i] = t[V + i];
            }
          }
        } else {
#pragma unroll
          for (int i = 0; i < V; ++i) {
            const bool in = v + i < P.vocab;
            lv[i] = in ? vd_f(l[v + i]) : -INFINITY;
            dv[i] = in && residual ? vd_f(d[v + i]) : -INFINITY;
            ev[i] = in ? e[v + i] : 1.f;
          }
        }
#pragma unroll
        for (int i = 0; i < V; ++i) race(lv[i], dv[i], ev[i], v + i);
      }
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        vd_best_warp(best[k]);
        if (lane == 0) s_best[k][warp] = best[k];
      }
      __syncthreads();
      if (warp == 0) {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          Best a = lane < VD_THREADS / 32 ? s_best[k][lane] : Best{0.f, -1};
          vd_best_warp(a);
          if (lane == 0) s_mine[k] = a;
        }
      }
    }
    cluster.sync();  // the CTAs' best are there
    if (rank == 0 && count > 0) {
      Best a[2] = {{0.f, -1}, {0.f, -1}};
      for (int r = 0; r < ctas; ++r) {
        const Best* const other = cluster.map_shared_rank(s_mine, r);
        vd_best(a[0], other[0]);
        vd_best(a[1], other[1]);
      }
      token = a[0].i >= 0 ? a[0].i : a[1].i;
    }
    cluster.sync();  // and read
  }
  if (rank) return;
  for (int i = tid; i < P.max_tokens; i += VD_THREADS) {
    const int x = i < taken ? P.tokens_in[first + i + 1] : (i == taken && count > 0 ? token : -1);
    P.tokens_out[(int64_t)b * P.max_tokens + i] = x;
    if (P.logprobs) P.logprobs[(int64_t)b * P.max_tokens + i] = x < 0 ? 0.f : logp(i, x);
  }
  if (tid == 0) {
    P.accepted[b] = taken;
    if (P.new_lens) P.new_lens[b] = P.seq_lens[b] - max(count - 1 - taken, 0);
  }
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
  while (!p.greedy && ctas < VD_CLUSTER && p.vocab > (int64_t)ctas * VD_THREADS * 16) ctas *= 2;
  launch_k(verify_pick_kernel<T>, dim3((unsigned)(p.num_seqs * ctas)), VD_THREADS, 0, s, ctas, p);
}

}  // namespace

// Slices of a row: four CTAs' worth per SM over all rows, none below two
// vectors a thread.
int verify_splits(int64_t tokens, int64_t vocab, bool draft) {
  const int64_t rows = std::max<int64_t>(tokens * (draft ? 2 : 1), 1);
  const int64_t want = (4 * (int64_t)device_sm_count() + rows - 1) / rows;
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
