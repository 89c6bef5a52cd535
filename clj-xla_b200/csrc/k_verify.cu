// Verification of drafted tokens against the target's logits.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "common.h"
#include "paged.h"

namespace cljxla {
namespace {

constexpr int VD_THREADS = 256;
constexpr int VD_MAX_ROWS = 128;

__device__ __forceinline__ float vd_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float vd_f(__half v) { return __half2float(v); }
__device__ __forceinline__ float vd_f(float v) { return v; }

// (max, sum of exp((x - max) / T)) pairs; an empty or all -inf part is (-inf, 0)
__device__ __forceinline__ void vd_join(float& m, float& s, float m2, float s2, float inv_t) {
  const float M = fmaxf(m, m2);
  if (M == -INFINITY) {
    s += s2;  // 0, or the NaN of a NaN logit
    return;
  }
  s = s * expf((m - M) * inv_t) + s2 * expf((m2 - M) * inv_t);
  m = M;
}

// the larger value, or the lower index of equal ones (index -1: none yet)
__device__ __forceinline__ void vd_best(float& v, int& i, float v2, int i2) {
  if (i2 >= 0 && (i < 0 || v2 > v || (v2 == v && i2 < i))) {
    v = v2;
    i = i2;
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

// Maximum, sum and (greedy) argmax of each row of the target, and of the draft.
template <typename T>
__global__ void __launch_bounds__(VD_THREADS) verify_rows_kernel(const __grid_constant__ VerifyParams P) {
  pdl_enter();
  const int row = blockIdx.x, which = blockIdx.y;
  const int b = seq_of_row(P.starts, P.num_seqs, P.each, row);
  if (b < 0) return;
  const T* x = (const T*)((which ? P.draft : P.target) + row * (which ? P.draft_stride : P.target_stride));
  const float inv_t = which ? P.inv_td : P.inv_t;
  float m = -INFINITY, s = 0.f;
  int arg = -1;
  for (int64_t v = threadIdx.x; v < P.vocab; v += VD_THREADS) {
    const float f = vd_f(x[v]);
    if (f > m) arg = (int)v;
    if (f != -INFINITY) vd_join(m, s, f, 1.f, inv_t);
  }
  float best = m;
  __shared__ float sm[VD_THREADS], ss[VD_THREADS];
  __shared__ int si[VD_THREADS];
  sm[threadIdx.x] = m;
  ss[threadIdx.x] = s;
  si[threadIdx.x] = arg;
  __syncthreads();
  if (threadIdx.x) return;
  for (int i = 1; i < VD_THREADS; ++i) {
    vd_best(best, arg, sm[i], si[i]);
    vd_join(m, s, sm[i], ss[i], inv_t);
  }
  float* part = P.part + ((int64_t)which * P.tokens + row) * 2;
  part[0] = m;
  part[1] = s;
  if (!which) ((int32_t*)(P.part + (int64_t)4 * P.tokens))[row] = arg;
}

// One CTA per sequence: what is accepted, and the token behind it.
template <typename T>
__global__ void __launch_bounds__(VD_THREADS) verify_pick_kernel(const __grid_constant__ VerifyParams P) {
  pdl_enter();
  const int b = blockIdx.x;
  int first, count;
  vd_rows(P, b, first, count);
  __shared__ int s_taken;
  __shared__ float sv[2][VD_THREADS];
  __shared__ int si[2][VD_THREADS];
  const int32_t* arg = (const int32_t*)(P.part + (int64_t)4 * P.tokens);
  auto logit = [&](int row, int64_t v) { return vd_f(((const T*)(P.target + row * P.target_stride))[v]); };
  auto prob = [&](int row, int64_t v) {
    const float* part = P.part + (int64_t)row * 2;
    const float f = logit(row, v);
    return f == -INFINITY ? 0.f : expf((f - part[0]) * P.inv_t) / part[1];
  };
  auto dprob = [&](int row, int64_t v) {
    const float* part = P.part + ((int64_t)P.tokens + row) * 2;
    const float f = vd_f(((const T*)(P.draft + row * P.draft_stride))[v]);
    return f == -INFINITY ? 0.f : expf((f - part[0]) * P.inv_td) / part[1];
  };
  auto logp = [&](int row, int64_t v) {
    const float* part = P.part + (int64_t)row * 2;
    return (logit(row, v) - part[0]) * P.inv_t - logf(part[1]);
  };
  auto dlogp = [&](int row, int64_t v) {
    const float* part = P.part + ((int64_t)P.tokens + row) * 2;
    return (vd_f(((const T*)(P.draft + row * P.draft_stride))[v]) - part[0]) * P.inv_td - logf(part[1]);
  };
  if (threadIdx.x == 0) {
    int n = 0;
    for (; n < count - 1; ++n) {
      const int row = first + n, x = P.tokens_in[row + 1];
      if (x < 0 || x >= P.vocab) break;
      // in logarithms: both sides may lie far below the smallest float
      const bool good = P.greedy ? x == arg[row]
                                 : logf(P.uniform[row]) + (P.draft ? dlogp(row, x) : 0.f) < logp(row, x);
      if (!good) break;
    }
    s_taken = n;
  }
  __syncthreads();
  const int taken = s_taken, row = first + taken;
  int token = -1;
  if (count > 0 && P.greedy) token = arg[row];
  if (count > 0 && !P.greedy) {
    const bool rejected = taken < count - 1;
    const int out = rejected && !P.draft ? P.tokens_in[row + 1] : -1;
    float best[2] = {0.f, 0.f};
    int at[2] = {-1, -1};  // of the residual, of the target itself
    for (int64_t v = threadIdx.x; v < P.vocab; v += VD_THREADS) {
      const float p = prob(row, v), e = P.race[b * P.race_stride + v];
      const float w = rejected && P.draft ? p - dprob(row, v) : (v == out ? 0.f : p);
      if (w > 0.f) vd_best(best[0], at[0], w / e, (int)v);
      if (p > 0.f) vd_best(best[1], at[1], p / e, (int)v);
    }
    for (int k = 0; k < 2; ++k) {
      sv[k][threadIdx.x] = best[k];
      si[k][threadIdx.x] = at[k];
    }
    __syncthreads();
    if (threadIdx.x == 0) {
      for (int i = 1; i < VD_THREADS; ++i)
        for (int k = 0; k < 2; ++k) vd_best(best[k], at[k], sv[k][i], si[k][i]);
      token = at[0] >= 0 ? at[0] : at[1];
    }
  }
  if (threadIdx.x) return;
  for (int i = 0; i < P.max_tokens; ++i) {
    const int x = i < taken ? P.tokens_in[first + i + 1] : (i == taken && count > 0 ? token : -1);
    P.tokens_out[(int64_t)b * P.max_tokens + i] = x;
    if (P.logprobs) P.logprobs[(int64_t)b * P.max_tokens + i] = x < 0 ? 0.f : logp(first + i, x);
  }
  P.accepted[b] = taken;
  if (P.new_lens) P.new_lens[b] = P.seq_lens[b] - max(count - 1 - taken, 0);
}

template <typename T>
void launch_t(const VerifyParams& p, cudaStream_t s) {
  if (p.tokens > 0)
    launch_k(verify_rows_kernel<T>, dim3((unsigned)p.tokens, p.draft ? 2 : 1), VD_THREADS, 0, s, 1, p);
  launch_k(verify_pick_kernel<T>, dim3((unsigned)p.num_seqs), VD_THREADS, 0, s, 1, p);
}

}  // namespace

int verify_splits(int64_t, int64_t, bool) { return 1; }

int64_t verify_workspace(const VerifyParams& p) { return (int64_t)p.tokens * 5 * 4; }

void launch_verify(const VerifyParams& p, cudaStream_t s) {
  if (p.dt == KDT_F32) launch_t<float>(p, s);
  else if (p.dt == KDT_F16) launch_t<__half>(p, s);
  else launch_t<__nv_bfloat16>(p, s);
}

}  // namespace cljxla
