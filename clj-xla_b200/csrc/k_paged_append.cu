// New keys and values into a paged cache, K and Q rotated by their positions.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.h"
#include "paged.h"

namespace cljxla {
namespace {

constexpr int PA_THREADS = 256;

__device__ __forceinline__ float pa_load(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ float pa_load(const __half* p) { return __half2float(*p); }
__device__ __forceinline__ float pa_load(const float* p) { return *p; }
__device__ __forceinline__ void pa_store(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
__device__ __forceinline__ void pa_store(__half* p, float v) { *p = __float2half_rn(v); }
__device__ __forceinline__ void pa_store(float* p, float v) { *p = v; }

// One CTA per packed row, a thread per pair or element.
template <typename T>
__global__ void __launch_bounds__(PA_THREADS) paged_append_kernel(const __grid_constant__ PagedAppendParams P) {
  pdl_enter();
  const PagedView& c = P.c;
  const int t = blockIdx.x;
  const int b = seq_of_row(c.starts, c.num_seqs, c.each, t);
  if (b < 0) return;
  int first, count;
  seq_rows(c, b, first, count);
  const int pos = seq_len(c, b) - count + (t - first);
  const int page = page_of(c, b, pos);
  const int row = page >= 0 ? pos % c.page_size : 0;
  const int half = P.rotary / 2;
  const int per = half + (P.hd - P.rotary);  // work items of a head: its pairs, then its copied elements
  for (int i = threadIdx.x; i < (P.nq + c.nkv) * per; i += PA_THREADS) {
    const int head = i / per, w = i % per;
    const bool is_q = head < P.nq;
    if (!is_q && page < 0) continue;
    const T* src = (const T*)(is_q ? P.qs + t * P.qs_tok + head * P.qs_head
                                   : P.ks + t * P.ks_tok + (head - P.nq) * P.ks_head);
    T* dst = (T*)(is_q ? P.qo + t * P.qo_tok + head * P.qo_head
                       : c.k + page * c.k_page + (head - P.nq) * c.k_head + row * c.k_row);
    if (w >= half) {
      const int e = P.rotary + (w - half);
      dst[e] = src[e];
      continue;
    }
    const int e1 = P.interleaved ? 2 * w : w, e2 = P.interleaved ? 2 * w + 1 : w + half;
    const double turns = (double)pos * (double)P.inv_freq[w] * 0.15915494309189535;
    float sn, cs;
    sincospif((float)(2.0 * (turns - rint(turns))), &sn, &cs);
    sn *= P.rope_scale;
    cs *= P.rope_scale;
    const float x1 = pa_load(src + e1), x2 = pa_load(src + e2);
    pa_store(dst + e1, x1 * cs - x2 * sn);
    pa_store(dst + e2, x2 * cs + x1 * sn);
  }
  if (page < 0) return;
  for (int i = threadIdx.x; i < c.nkv * P.hd; i += PA_THREADS) {
    const int head = i / P.hd, e = i % P.hd;
    ((T*)(c.v + page * c.v_page + head * c.v_head + row * c.v_row))[e] =
        ((const T*)(P.vs + t * P.vs_tok + head * P.vs_head))[e];
  }
}

}  // namespace

void launch_paged_append(const PagedAppendParams& p, cudaStream_t s) {
  const dim3 grid((unsigned)p.c.tokens);
  if (p.dt == KDT_F32) launch_k(paged_append_kernel<float>, grid, PA_THREADS, 0, s, 1, p);
  else if (p.dt == KDT_F16) launch_k(paged_append_kernel<__half>, grid, PA_THREADS, 0, s, 1, p);
  else launch_k(paged_append_kernel<__nv_bfloat16>, grid, PA_THREADS, 0, s, 1, p);
}

}  // namespace cljxla
