// New keys and values into a paged cache, K and Q rotated by their positions.
//
// (x1, x2) -> scale * (x1 cos a - x2 sin a, x2 cos a + x1 sin a), a = position *
// inv_freq[i], for pairs (i, i + n) or (2 i, 2 i + 1), n = rotary_dim / 2; one
// f32 evaluation and one rounding.  The angle is taken in turns and reduced in
// 64 bits (a far position times a frequency has few exact f32 digits left of
// the point), so cos and sin see at most half a turn.
//
// What bounds it: every element is read and written once, so HBM bandwidth for
// prompts and the chain starts -> length -> page -> store for a decode step.
// Angles cost more than the copies they turn: a CTA takes TOK rows (4 of a long
// prompt, 1 of a decode step, where rows are few and CTAs share a row's heads
// instead), computes their cos and sin once in shared memory for all heads, and
// each thread has its pairs of all the CTA's rows in flight for one head after another.
// Measured (B200): 4968 f16 rows of 16 + 16 heads of 256 31 to 33 us (24.8 at the copy
// rate); one element off a 16-byte boundary 74, with a rotated part of 60 elements 102.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <type_traits>

#include "common.h"
#include "paged.h"

namespace cljxla {
namespace {

constexpr int PA_THREADS = 256;
constexpr int PA_TOK = 4;

// A lot: the V elements of one access (16 bytes, or one element), as they lie in
// memory: what is only copied keeps its bits.
template <typename T, bool VEC>
struct Lot {
  static constexpr int V = VEC ? 16 / (int)sizeof(T) : 1;
  union {
    uint4 raw;
    T e[VEC ? V : 1];
  };
  __device__ __forceinline__ Lot() {}
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (VEC) raw = *(const uint4*)p;
    else e[0] = *p;
  }
  __device__ __forceinline__ void store(T* p) const {
    if constexpr (VEC) *(uint4*)p = raw;
    else *p = e[0];
  }
  __device__ __forceinline__ float get(int i) const { return (float)e[i]; }
  __device__ __forceinline__ void set(int i, float x) {
    if constexpr (sizeof(T) == 4) e[i] = x;
    else if constexpr (std::is_same<T, __half>::value) e[i] = __float2half_rn(x);
    else e[i] = __float2bfloat16_rn(x);
  }
};

__device__ __forceinline__ void turn_pair(float x, float y, float cs, float sn, float& a, float& b) {
  a = x * cs - y * sn;
  b = y * cs + x * sn;
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(PA_THREADS, 3) paged_append_kernel(const __grid_constant__ PagedAppendParams P) {
  constexpr int V = Lot<T, VEC>::V;
  __shared__ int s_pos[PA_TOK];
  __shared__ char *s_k[PA_TOK], *s_v[PA_TOK];  // where the row goes; null: its page is not there
  __shared__ bool s_live[PA_TOK];              // the row is some sequence's
  __shared__ __align__(16) float s_cos[PA_TOK * 128], s_sin[PA_TOK * 128];
  const PagedView& c = P.c;
  const int tid = threadIdx.x, warp = tid >> 5, half = P.rotary / 2;
  const int t0 = blockIdx.x * P.tok, n = min(P.tok, c.tokens - t0);
  // a head's lots: pairs of lots (interleaved: lots of pairs; by elements: pairs), then lots that are copied
  const bool whole = P.interleaved && VEC;  // a lot holds both elements of its pairs
  const int turning = whole ? P.rotary / V : half / V, lots = turning + (P.hd - P.rotary) / V;
  const int lot = tid & ((1 << P.lot_bits) - 1), lane0 = tid >> P.lot_bits, lanes = PA_THREADS >> P.lot_bits;
  const int heads = P.nq + c.nkv, step = lanes * gridDim.y;
  const bool turn = lot < turning;
  const int e1 = !turn ? P.rotary + (lot - turning) * V : whole ? lot * V : P.interleaved ? 2 * lot : lot * V;
  const int e2 = P.interleaved ? 2 * lot + 1 : half + lot * V;
  const bool two = turn && !whole;
  const int angle = whole ? lot * (V / 2) : lot * V;
  pdl_enter();
  // The next head of the CTA's rows: their loads are in flight together, the
  // first ones while the rows' pages and angles are found.
  Lot<T, VEC> a[PA_TOK], b[PA_TOK];
  int h = blockIdx.y * lanes + lane0;
  auto fetch = [&]() {
    if (lot >= lots || h >= heads) return;
    const bool is_q = h < P.nq;
    const char* const src = is_q ? P.qs + t0 * P.qs_tok + h * P.qs_head : P.ks + t0 * P.ks_tok + (h - P.nq) * P.ks_head;
    const int64_t src_tok = is_q ? P.qs_tok : P.ks_tok;
#pragma unroll
    for (int k = 0; k < PA_TOK; ++k) {
      if (k >= n) break;
      a[k].load((const T*)(src + k * src_tok) + e1);
      if (two) b[k].load((const T*)(src + k * src_tok) + e2);
    }
  };
  fetch();
  if (warp < n) {
    const int t = t0 + warp, b = seq_of_row(c.starts, c.num_seqs, c.each, t);
    int pos = 0, page = -1;
    if (b >= 0) {
      int first, count;
      seq_rows(c, b, first, count);
      pos = seq_len(c, b) - count + (t - first);
      page = page_of(c, b, pos);
    }
    if ((tid & 31) == 0) {
      const int row = page < 0 ? 0 : c.page_shift >= 0 ? pos & (c.page_size - 1) : pos % c.page_size;
      s_pos[warp] = pos;
      s_live[warp] = b >= 0;
      s_k[warp] = page < 0 ? nullptr : c.k + page * c.k_page + row * c.k_row;
      s_v[warp] = page < 0 ? nullptr : c.v + page * c.v_page + row * c.v_row;
    }
  }
  __syncthreads();
  for (int i = tid; i < n * half; i += PA_THREADS) {
    const int k = i / half;
    const double turns = (double)s_pos[k] * ((double)P.inv_freq[i - k * half] * 0.15915494309189535);
    float sn, cs;
    sincospif(2.f * (float)(turns - rint(turns)), &sn, &cs);
    s_cos[k * 128 + i - k * half] = cs * P.rope_scale;
    s_sin[k * 128 + i - k * half] = sn * P.rope_scale;
  }
  __syncthreads();

  for (; lot < lots && h < heads;) {
    const bool is_q = h < P.nq;
#pragma unroll
    for (int k = 0; k < PA_TOK; ++k) {
      if (k >= n || !s_live[k] || (!is_q && !s_k[k])) continue;
      T* const dst = (T*)(is_q ? P.qo + (t0 + k) * P.qo_tok + h * P.qo_head : s_k[k] + (h - P.nq) * c.k_head);
      if (two) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          float x, y;
          turn_pair(a[k].get(i), b[k].get(i), s_cos[k * 128 + angle + i], s_sin[k * 128 + angle + i], x, y);
          a[k].set(i, x);
          b[k].set(i, y);
        }
        b[k].store(dst + e2);
      } else if (turn) {
#pragma unroll
        for (int i = 0; i + 1 < V; i += 2) {
          float x, y;
          turn_pair(a[k].get(i), a[k].get(i + 1), s_cos[k * 128 + angle + i / 2], s_sin[k * 128 + angle + i / 2], x, y);
          a[k].set(i, x);
          a[k].set(i + 1, y);
        }
      }
      a[k].store(dst + e1);
    }
    h += step;
    fetch();
  }
  const int vlots = P.hd / V, all = c.nkv * vlots;
  for (int i = blockIdx.y * PA_THREADS + tid; i < all; i += PA_THREADS * gridDim.y) {
    const int h = i / vlots, e = (i - h * vlots) * V;
    const char* const src = P.vs + t0 * P.vs_tok + h * P.vs_head;
    Lot<T, VEC> a[PA_TOK];
#pragma unroll
    for (int k = 0; k < PA_TOK; ++k)
      if (k < n && s_v[k]) a[k].load((const T*)(src + k * P.vs_tok) + e);
#pragma unroll
    for (int k = 0; k < PA_TOK; ++k)
      if (k < n && s_v[k]) a[k].store((T*)(s_v[k] + h * c.v_head) + e);
  }
}

template <typename T>
void launch_t(PagedAppendParams p, cudaStream_t s) {
  const int v = p.vec ? 16 / (int)sizeof(T) : 1;
  const int turning = p.vec && p.interleaved ? p.rotary / v : p.rotary / 2 / v;
  const int lots = std::max(turning + (p.hd - p.rotary) / v, 1);
  p.lot_bits = 0;
  while ((1 << p.lot_bits) < lots) ++p.lot_bits;  // at most 256 lots: a head's elements
  // Rows of a long prompt four to a CTA, so that angles are computed once for
  // many heads; where that would leave SMs without work, one row to a CTA, and
  // the heads of few rows over several.
  const int sms = device_sm_count();
  p.tok = p.c.tokens >= 2 * PA_TOK * sms ? PA_TOK : 1;
  const int rows = (p.c.tokens + p.tok - 1) / p.tok;
  const int lanes = PA_THREADS >> p.lot_bits;
  const int passes = std::max((p.nq + p.c.nkv + lanes - 1) / lanes, 1);
  const int share = std::min(passes, std::max(1, 2 * sms / rows));
  const dim3 grid((unsigned)rows, (unsigned)share);
  if (p.vec) launch_k(paged_append_kernel<T, true>, grid, PA_THREADS, 0, s, 1, p);
  else launch_k(paged_append_kernel<T, false>, grid, PA_THREADS, 0, s, 1, p);
}

}  // namespace

void launch_paged_append(const PagedAppendParams& p, cudaStream_t s) {
  if (p.dt == KDT_F32) launch_t<float>(p, s);
  else if (p.dt == KDT_F16) launch_t<__half>(p, s);
  else launch_t<__nv_bfloat16>(p, s);
}

}  // namespace cljxla
