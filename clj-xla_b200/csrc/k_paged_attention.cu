// Attention of a step's queries over the pages of their sequences.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.h"
#include "paged.h"

namespace cljxla {
namespace {

__device__ __forceinline__ float at_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float at_f(__half v) { return __half2float(v); }
__device__ __forceinline__ float at_f(float v) { return v; }
__device__ __forceinline__ void at_store(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
__device__ __forceinline__ void at_store(__half* p, float v) { *p = __float2half_rn(v); }
__device__ __forceinline__ void at_store(float* p, float v) { *p = v; }

// One CTA of four warps per (row, query head): each warp takes every fourth
// position with a running maximum and sum, and the four are joined.
template <typename T, int HD>
__global__ void __launch_bounds__(128) paged_attn_kernel(const __grid_constant__ PagedAttnParams P) {
  pdl_enter();
  constexpr int E = HD / 32;
  const PagedView& c = P.c;
  const int t = blockIdx.x, h = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int b = seq_of_row(c.starts, c.num_seqs, c.each, t);
  if (b < 0) return;
  int first, count;
  seq_rows(c, b, first, count);
  if (t - first >= P.max_rows) return;
  const int pos = seq_len(c, b) - count + (t - first);
  int64_t lo = P.window < 0 ? 0 : (int64_t)pos - P.window;
  if (lo < 0) lo = 0;
  float q[E], acc[E], m = -INFINITY, l = 0.f;
  const T* qp = (const T*)(P.q + t * P.q_tok + h * P.q_head);
#pragma unroll
  for (int e = 0; e < E; ++e) {
    q[e] = at_f(qp[e * 32 + lane]);
    acc[e] = 0.f;
  }
  const int kvh = h / P.group;
  const int hi = min(pos, capacity(c) - 1);
  for (int64_t j = lo + warp; j <= hi; j += 4) {
    const int page = page_of(c, b, (int)j);
    if (page < 0) continue;
    const int r = (int)j % c.page_size;
    const T* kp = (const T*)(c.k + page * c.k_page + kvh * c.k_head + r * c.k_row);
    const T* vp = (const T*)(c.v + page * c.v_page + kvh * c.v_head + r * c.v_row);
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) s += q[e] * at_f(kp[e * 32 + lane]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    s *= P.scale;
    if (P.softcap > 0.f) s = P.softcap * tanhf(s / P.softcap);
    const float mn = fmaxf(m, s);
    const float base = mn == -INFINITY ? 0.f : mn;
    const float a = __expf(m - base), w = __expf(s - base);
    l = l * a + w;
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = acc[e] * a + w * at_f(vp[e * 32 + lane]);
    m = mn;
  }
  __shared__ float sm[4], sl[4], so[4][HD];
  if (lane == 0) {
    sm[warp] = m;
    sl[warp] = l;
  }
#pragma unroll
  for (int e = 0; e < E; ++e) so[warp][e * 32 + lane] = acc[e];
  __syncthreads();
  float M = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
  if (M == -INFINITY) M = 0.f;
  float a[4], L = 0.f;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    a[w] = __expf(sm[w] - M);
    L += sl[w] * a[w];
  }
  for (int d = threadIdx.x; d < HD; d += 128) {
    float o = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) o += a[w] * so[w][d];
    o = L > 0.f ? o / L : (L == 0.f ? 0.f : L);  // a NaN sum stays NaN
    char* op = P.out + t * P.o_tok + h * P.o_head;
    if (P.out_f32) ((float*)op)[d] = o;
    else at_store((T*)op + d, o);
  }
}

template <typename T>
void launch_t(const PagedAttnParams& p, cudaStream_t s) {
  const dim3 grid((unsigned)p.c.tokens, (unsigned)(p.c.nkv * p.group));
  switch (p.hd) {
    case 32: launch_k(paged_attn_kernel<T, 32>, grid, 128, 0, s, 1, p); break;
    case 64: launch_k(paged_attn_kernel<T, 64>, grid, 128, 0, s, 1, p); break;
    case 128: launch_k(paged_attn_kernel<T, 128>, grid, 128, 0, s, 1, p); break;
    default: launch_k(paged_attn_kernel<T, 256>, grid, 128, 0, s, 1, p); break;
  }
}

}  // namespace

int64_t paged_attention_workspace(const PagedAttnParams&) { return 0; }

void launch_paged_attention(const PagedAttnParams& p, cudaStream_t s) {
  if (p.dt == KDT_F32) launch_t<float>(p, s);
  else if (p.dt == KDT_F16) launch_t<__half>(p, s);
  else launch_t<__nv_bfloat16>(p, s);
}

}  // namespace cljxla
