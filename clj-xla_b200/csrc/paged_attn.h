// Attention of a step's queries over the pages of their sequences.
//
// For each row at position p of its sequence and each query head,
//   out = sum_j w_j v_j / sum_j w_j,  w_j = 2^(s_j - m),  s_j = log2(e) * score_j,
// over the positions j the row sees, in one pass with the running maximum m
// and sum (a new maximum m' scales what is there by 2^(m - m')).
//
// What bounds it: each visible K and V row is read once from HBM for
// 4 * head_dim FLOPs per query row, at most 64 rows to a byte pair, so the
// bound is HBM bandwidth as long as enough copies are in flight.
//
// Split.  A segment is (sequence, KV head, up to ROWS query rows of that head's
// group), a row of tiles of its positions.  All tiles of the call, laid end to
// end, are cut into one equal range per CTA, whatever the sequences' lengths: one long context fills the GPU as well as many ragged ones do.  Each
// CTA finds its range itself from seq_lens (a scan over the sequences), so a
// captured graph follows the lengths.  A segment that lies within one CTA is
// finished there; a cut one leaves (m, sum, unnormalised row) partials that
// paged_attn_join_kernel, launched as a programmatic dependent, adds up in
// range order: no atomics, the same bits every time.
//
// Tile.  64 positions (32 in f32) of K and V rows go through a ring of stages.
// Warp 4 is the producer: it walks the schedule, looks the pages of a tile up
// one tile ahead, and gathers the rows with 16-byte cp.async (any page size, any
// strides; positions nobody sees are filled with zeros and not read).  Warps 0
// to 3 score 16 (8) positions each on mma.sync, share row maxima and weights
// through shared memory, and each adds P.V for a quarter of head_dim, so the
// accumulators stay small and no warp holds partials.  Stages change hands over
// named barriers.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <type_traits>

#include "common.h"
#include "paged.h"

namespace cljxla {
namespace {

constexpr int AT_CONSUMERS = 128, AT_THREADS = AT_CONSUMERS + 32, AT_JOIN_THREADS = 128;
constexpr int kAttnMaxCtas = 1024;  // SMs times CTAs on one, at most

// ------------------------------------------------------------------ layout
template <typename T, int HD, int MT>
struct Tile {
  static constexpr int ES = sizeof(T);
  static constexpr int TP = ES == 2 ? 64 : 32;  // positions of a tile
  static constexpr int WP = TP / 4;             // positions a warp scores
  static constexpr int ROWS = MT * 16;
  static constexpr int RB = HD * ES;            // bytes of a row
  static constexpr int CPR = RB / 16;           // 16-byte chunks of a row
  static constexpr int KB = TP * RB;
  static constexpr int QB = ROWS * RB;
  static constexpr int STAGE = 2 * KB + QB;     // K, V, and the queries of a segment that starts here
  // weights as two 16-bit parts or one f32: in the tile's K rows once they are scored, if they fit
  static constexpr int PB = ROWS * TP * 4;
  static constexpr bool P_IN_K = PB <= KB;
  static constexpr int fixed(int nst) { return (P_IN_K ? 0 : PB) + 2 * 4 * ROWS * 4 + nst * 64 + 64 + TP * 16; }
  static constexpr int fit(int ctas) {  // stages that fit with this many CTAs on an SM (228 KB, 1 KB each reserved)
    int n = 0;
    while (n < 4 && fixed(n + 1) + (n + 1) * STAGE <= 233472 / ctas - 1024) ++n;
    return n;
  }
  static constexpr int pick() {
    int ctas = HD >= 256 ? 1 : HD == 128 ? 2 : 3;
    while (ctas > 1 && fit(ctas) < 3) --ctas;
    return ctas;
  }
  static constexpr int CTAS = pick();
  static constexpr int NST = fit(CTAS);
  static constexpr int SMEM = fixed(NST) + NST * STAGE;
  static_assert(NST >= 2, "a ring needs two stages");
};

// chunk c of row r sits at chunk swz(c, r): the eight rows that a matrix load
// or a column of threads touches fall on different banks
template <int CPR>
__device__ __forceinline__ int swz(int c, int r) {
  if constexpr (CPR >= 8) return c ^ (r & 7);
  else return c ^ ((r >> 1) & (CPR - 1));  // 64-byte rows: two to a bank line
}
// f32 V rows are read by 4 positions x 8 columns
template <typename T, int CPR>
__device__ __forceinline__ int swz_v(int c, int r) {
  if constexpr (sizeof(T) == 4) return c ^ ((r & 3) << 1);
  else return swz<CPR>(c, r);
}

// -------------------------------------------------------------- primitives
__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void cp16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes));  // ordered by the commit, not among themselves
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
template <int N>
__device__ __forceinline__ void bar_sync(int id) {
  asm volatile("bar.sync %0, %1;" ::"r"(id), "n"(N) : "memory");
}
template <int N>
__device__ __forceinline__ void bar_arrive(int id) {
  asm volatile("bar.arrive %0, %1;" ::"r"(id), "n"(N) : "memory");
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t* r) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t addr, uint32_t* r) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm2t(uint32_t addr, uint32_t* r) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x2.trans.shared.b16 {%0,%1}, [%2];"
               : "=r"(r[0]), "=r"(r[1]) : "r"(addr) : "memory");
}
template <typename T>
__device__ __forceinline__ void mma16(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __half>::value)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_tf32(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// x = hi + lo to 22 bits: three tf32 products then lose about 2^-21 of an f32 one
__device__ __forceinline__ void split_tf32(float x, uint32_t& hi, uint32_t& lo) {
  asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(hi) : "f"(x));
  asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(lo) : "f"(x - __uint_as_float(hi)));
}
__device__ __forceinline__ void mma_f32(float* c, const uint32_t* ah, const uint32_t* al, float b0, float b1) {
  uint32_t h0, l0, h1, l1;
  split_tf32(b0, h0, l0);
  split_tf32(b1, h1, l1);
  mma_tf32(c, al, h0, h1);
  mma_tf32(c, ah, l0, l1);
  mma_tf32(c, ah, h0, h1);
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (std::is_same<T, __half>::value) {
    const __half2 v = __floats2half2_rn(a, b);
    return *(const uint32_t*)&v;
  } else {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *(const uint32_t*)&v;
  }
}
template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t v) {
  if constexpr (std::is_same<T, __half>::value) return __half22float2(*(const __half2*)&v);
  else return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
}
// tanh: from 2^x where that is accurate (1 - 2 / (1 + e^2y) is off by about
// 2^-23), from its series where that would cancel (|y| < 0.1: the next term is
// below 2^-32 of the result)
__device__ __forceinline__ float tanh_f(float y) {
  const float big = 1.f - __fdividef(2.f, 1.f + ex2(y * 2.8853900817779268f));
  const float z = y * y;
  const float small = y * fmaf(z, fmaf(z, fmaf(z, -17.f / 315.f, 2.f / 15.f), -1.f / 3.f), 1.f);
  return fabsf(y) < 0.1f ? small : big;
}
// whether either 16-bit value is an infinity or NaN
template <typename T>
__device__ __forceinline__ bool odd2(uint32_t v) {
  constexpr uint32_t e = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
  return (v & e) == e || ((v >> 16) & e) == e;
}
template <typename T>
__device__ __forceinline__ bool odd_chunk(const uint4& v) {
  if constexpr (sizeof(T) == 2) {
    return odd2<T>(v.x) || odd2<T>(v.y) || odd2<T>(v.z) || odd2<T>(v.w);
  } else {
    constexpr uint32_t e = 0x7f800000u;
    return (v.x & e) == e || (v.y & e) == e || (v.z & e) == e || (v.w & e) == e;
  }
}

// --------------------------------------------------------------- schedule
// A tile: positions [pos0, pos0 + npos) of segment (b, head, rows row0 ..).
struct TileDesc {
  int head, row0, pos0, npos, flags, qslot, first, count, p0;  // p0: position of the sequence's first row
  uint32_t mask[2];  // positions whose page is there
};
enum { T_FIRST = 1, T_LAST = 2, T_FROM0 = 4, T_TOEND = 8, T_FULL = 16, T_END = 32 };  // T_END: the CTA's last tile

// One sequence's share of the schedule.
struct SeqPlan {
  int first, count, rows, p0, lo, hi, units, tiles;  // rows: computed ones; tiles: row tiles
  __device__ __forceinline__ void load(const PagedAttnParams& P, int b, int tile, int row_tile) {
    int n;
    seq_rows(P.c, b, first, n);
    count = min(n, P.max_rows);
    rows = count * P.group;
    tiles = (rows + row_tile - 1) / row_tile;
    p0 = seq_len(P.c, b) - n;
    lo = P.window < 0 ? 0 : (int)max((int64_t)p0 - P.window, (int64_t)0);
    hi = min(p0 + count, capacity(P.c));
    units = max((hi - lo + tile - 1) / tile, 1);
  }
  __device__ __forceinline__ int64_t cost(int nkv) const { return (int64_t)units * nkv * tiles; }
};

template <typename T, int HD, int MT>
__global__ void __launch_bounds__(AT_THREADS, Tile<T, HD, MT>::CTAS)
    paged_attn_kernel(const __grid_constant__ PagedAttnParams P) {
  using L = Tile<T, HD, MT>;
  constexpr int TP = L::TP, WP = L::WP, ROWS = L::ROWS, RB = L::RB, CPR = L::CPR, NST = L::NST;
  constexpr int NT = HD / 32;  // 8-column output tiles of a warp
  extern __shared__ __align__(1024) unsigned char smem[];
  unsigned char* const ring = smem;
  unsigned char* const p_own = smem + NST * L::STAGE;
  float* const wmax = (float*)(p_own + (L::P_IN_K ? 0 : L::PB));  // [4][ROWS]
  float* const wsum = wmax + 4 * ROWS;
  TileDesc* const desc = (TileDesc*)(wsum + 4 * ROWS);  // [NST], 64 bytes each
  int64_t* const sh = (int64_t*)((unsigned char*)desc + NST * 64);
  longlong2* const offs = (longlong2*)(sh + 8);  // [TP] the producer's K and V row offsets

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const PagedView& c = P.c;
  pdl_enter();

  // ---- this CTA's range of tiles
  int64_t left, total = 0, ctas;
  {
    SeqPlan sp;
    const int per = (c.num_seqs + AT_THREADS - 1) / AT_THREADS;
    const int b0 = min(tid * per, c.num_seqs), b1 = min(b0 + per, c.num_seqs);
    int64_t mine = 0;
    for (int i = b0; i < b1; ++i) {
      sp.load(P, i, TP, ROWS);
      mine += sp.cost(c.nkv);
    }
    int64_t incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    if (lane == 31) sh[warp] = incl;
    __syncthreads();
    for (int w = 0; w < AT_THREADS / 32; ++w) {
      if (w < warp) incl += sh[w];
      total += sh[w];
    }
    ctas = min((int64_t)gridDim.x, total);
    if ((int64_t)blockIdx.x >= ctas) {
      if (tid == 0 && P.meta) P.meta[blockIdx.x * 4] = 0;
      return;
    }
    const int64_t beg = total * blockIdx.x / ctas, end = total * (blockIdx.x + 1) / ctas;
    left = end - beg;
    __syncthreads();
    if (tid == 0) {
      sh[0] = sh[1] = 0;
      if (P.meta) P.meta[blockIdx.x * 4] = 0;  // no segment that starts here is cut, so far
    }
    __syncthreads();
    int64_t excl = incl - mine;
    if (beg >= excl && beg < incl) {
      for (int i = b0; i < b1; ++i) {
        sp.load(P, i, TP, ROWS);
        if (beg < excl + sp.cost(c.nkv)) {
          sh[0] = i;
          sh[1] = beg - excl;
          break;
        }
        excl += sp.cost(c.nkv);
      }
    }
    __syncthreads();
  }

  // Stage hand-over: full[s] (producer arrives, consumers wait), empty[s] the other way round.
  constexpr int FULL = 2, EMPTY = FULL + NST, INNER = 1;

  if (warp == AT_CONSUMERS / 32) {
    // ================================================================ producer
    int b = (int)sh[0];  // cursor: sequence, segment of it (head, row tile), tile of that
    SeqPlan sp;
    sp.load(P, b, TP, ROWS);
    const int64_t off = sh[1];
    if (off >= sp.cost(c.nkv)) left = 0;  // lengths that change under the kernel: stay in bounds
    int seg = (int)(off / sp.units), at = (int)(off % sp.units), qslot = -1;
    bool fresh = true;  // the next tile is the first of its piece
    bool piece0 = false;  // whether the piece starts its segment
    TileDesc nd;
    int page[TP / 32], in_page[TP / 32];
    auto next = [&]() -> bool {  // the cursor's next tile into nd; starts its page lookup
      if (left == 0) return false;
      if (at >= sp.units) {
        at = 0;
        if (++seg >= c.nkv * sp.tiles) {
          seg = 0;
          do {
            if (++b >= c.num_seqs) {
              left = 0;
              return false;
            }
            sp.load(P, b, TP, ROWS);
          } while (sp.tiles == 0);
        }
        fresh = true;
      }
      if (fresh) {
        qslot = qslot + 1 == NST ? 0 : qslot + 1;
        piece0 = at == 0;
      }
      nd.head = sp.tiles == 1 ? seg : seg / sp.tiles;
      nd.row0 = (seg - nd.head * sp.tiles) * ROWS;
      nd.pos0 = sp.lo + at * TP;
      nd.npos = max(min(TP, sp.hi - nd.pos0), 0);
      nd.qslot = qslot;
      nd.first = sp.first;
      nd.count = sp.count;
      nd.p0 = sp.p0;
      nd.flags = (fresh ? T_FIRST : 0) | (piece0 ? T_FROM0 : 0);
      ++at;
      --left;
      if (at == sp.units) nd.flags |= T_LAST | T_TOEND;
      if (left == 0) {
        nd.flags |= T_LAST;
        if (piece0 && at < sp.units && lane == 0) {
          // the range ends inside a segment that starts here: its last tile belongs to CTA `to`
          const int64_t end = total * (blockIdx.x + 1) / ctas;
          const int64_t to = ((end + (sp.units - at)) * ctas - 1) / total;
          int32_t* meta = P.meta + blockIdx.x * 4;
          meta[0] = (int32_t)(min(to, ctas - 1) - blockIdx.x + 1);
          meta[1] = b;
          meta[2] = nd.head;
          meta[3] = nd.row0;
        }
      }
      // every row sees every position, were all pages there
      if (nd.npos == TP && nd.pos0 + TP - 1 <= nd.p0 && (P.window < 0 || nd.pos0 >= nd.p0 + nd.count - 1 - P.window))
        nd.flags |= T_FULL;
      fresh = false;
#pragma unroll
      for (int i = 0; i < TP / 32; ++i) {
        const int j = nd.pos0 + i * 32 + lane;
        page[i] = -1;
        in_page[i] = 0;
        if (i * 32 + lane < nd.npos) {
          const int slot = j / c.page_size;
          page[i] = c.table[(int64_t)b * c.table_stride + slot];
          in_page[i] = j - slot * c.page_size;
        }
      }
      return true;
    };

    constexpr int LANES = CPR < 32 ? CPR : 32;  // lanes of a row
    constexpr int RPI = 32 / LANES;             // rows of one warp-wide copy
    constexpr int CPL = CPR / LANES;            // chunks of a row for a lane
    const int my_row = lane / LANES, my_chunk = lane % LANES;
    int tile = 0;
    bool have = next();
    if (!have) {  // only if lengths change under the kernel: a tile of nothing ends the consumers
      if (lane == 0) *(TileDesc*)desc = TileDesc{0, 0, 0, 0, T_FIRST | T_END, 0, 0, 0, 0, {0u, 0u}};
      bar_arrive<AT_THREADS>(FULL);
      return;
    }
    while (have) {
      // tell the consumers of the oldest tile in flight before waiting for a free stage
      if (tile >= NST - 1) {
        cp_wait<NST - 2>();
        bar_arrive<AT_THREADS>(FULL + (tile + 1) % NST);
      }
      const int slot = tile % NST;
      if (tile >= NST) bar_sync<AT_THREADS>(EMPTY + slot);
      __syncwarp();  // offs of the tile before are read
#pragma unroll
      for (int i = 0; i < TP / 32; ++i) {
        const bool ok = (unsigned)page[i] < (unsigned)c.num_pages;
        longlong2 o;
        o.x = ok ? page[i] * c.k_page + nd.head * c.k_head + in_page[i] * c.k_row : -1;
        o.y = ok ? page[i] * c.v_page + nd.head * c.v_head + in_page[i] * c.v_row : -1;
        offs[i * 32 + lane] = o;
        nd.mask[i] = __ballot_sync(0xffffffffu, ok);
      }
      if (lane == 0) *(TileDesc*)((char*)desc + slot * 64) = nd;
      __syncwarp();
      const uint32_t kd = smem_u32(ring + slot * L::STAGE), vd = kd + L::KB;
      // eight rows' offsets are fetched before their copies are issued: the warp's
      // time goes to issue, not to the latency of each row's address
      constexpr int BATCH = 8;
      static_assert(TP % (BATCH * RPI) == 0, "whole batches");
#pragma unroll 1
      for (int r0 = 0; r0 < TP; r0 += BATCH * RPI) {
        longlong2 o[BATCH];
#pragma unroll
        for (int i = 0; i < BATCH; ++i) o[i] = offs[r0 + i * RPI + my_row];
#pragma unroll
        for (int i = 0; i < BATCH; ++i) {
          const int r = r0 + i * RPI + my_row, rr = i * RPI + my_row;  // r0 is a multiple of 8: equal swizzles
          const int size = o[i].x >= 0 ? 16 : 0;
          const char* kp = (size ? c.k + o[i].x : P.q) + my_chunk * 16;
          const char* vp = (size ? c.v + o[i].y : P.q) + my_chunk * 16;
#pragma unroll
          for (int e = 0; e < CPL; ++e) {
            const int ch = my_chunk + e * LANES;
            cp16(kd + r * RB + swz<CPR>(ch, rr) * 16, kp + (size ? e * LANES * 16 : 0), size);
            cp16(vd + r * RB + swz_v<T, CPR>(ch, rr) * 16, vp + (size ? e * LANES * 16 : 0), size);
          }
        }
      }
      if (nd.flags & T_FIRST) {
        const uint32_t qd = smem_u32(ring + qslot * L::STAGE + 2 * L::KB);
        for (int r0 = 0; r0 < ROWS; r0 += RPI) {
          const int r = r0 + my_row, row = nd.row0 + r;
          const bool ok = row < nd.count * P.group;
          const int qi = row / P.group;
          const char* src = ok ? P.q + (int64_t)(nd.first + qi) * P.q_tok +
                                     (int64_t)(nd.head * P.group + row - qi * P.group) * P.q_head
                               : P.q;
#pragma unroll
          for (int e = 0; e < CPL; ++e) {
            const int ch = my_chunk + e * LANES;
            cp16(qd + r * RB + swz<CPR>(ch, r) * 16, src + (ok ? ch * 16 : 0), ok ? 16 : 0);
          }
        }
      }
      cp_commit();
      have = next();
      if (!have && lane == 0) ((TileDesc*)((char*)desc + slot * 64))->flags |= T_END;
      ++tile;
    }
    // the tiles still in flight
#pragma unroll
    for (int k = NST - 2; k >= 0; --k) {
      if (tile - 1 - k < 0) continue;
      if (k == 0) cp_wait<0>();
      else if (k == 1) cp_wait<1>();
      else cp_wait<2>();
      bar_arrive<AT_THREADS>(FULL + (tile - 1 - k) % NST);
    }
    for (int k = max(tile - NST, 0); k < tile - 1; ++k) bar_sync<AT_THREADS>(EMPTY + k % NST);  // no arrival is left over
    return;
  }

  // ================================================================ consumers
  float acc[MT][NT][4], m[MT][2], l[MT][2];
  const int g = lane >> 2, t4 = lane & 3;
  for (int tile = 0;; ++tile) {
    const int slot = tile % NST;
    bar_sync<AT_THREADS>(FULL + slot);
    const TileDesc d = *(const TileDesc*)((char*)desc + slot * 64);
    unsigned char* const stage = ring + slot * L::STAGE;
    const uint32_t ks = smem_u32(stage), vs = ks + L::KB, qs = smem_u32(ring + d.qslot * L::STAGE + 2 * L::KB);
    unsigned char* const pw = L::P_IN_K ? stage : p_own;
    const uint64_t vis = TP == 64 ? (uint64_t)d.mask[1] << 32 | d.mask[0] : d.mask[0];
    const bool plain = (d.flags & T_FULL) && vis == (TP == 64 ? ~0ull : 0xffffffffull);
    if (d.flags & T_FIRST) {
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        m[i][0] = m[i][1] = -INFINITY;
        l[i][0] = l[i][1] = 0.f;
#pragma unroll
        for (int n = 0; n < NT; ++n) acc[i][n][0] = acc[i][n][1] = acc[i][n][2] = acc[i][n][3] = 0.f;
      }
    }

    // ---- scores of this warp's WP positions
    constexpr int SN = WP / 8;
    float s[MT][SN][4];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int n = 0; n < SN; ++n) s[i][n][0] = s[i][n][1] = s[i][n][2] = s[i][n][3] = 0.f;
    if constexpr (L::ES == 2) {
      // chunk 2 k + (0 or 1) of a row: its swizzled address differs from chunk
      // 0 or 1's by an exclusive or with 32 k
      const int kr = warp * WP + (lane >> 4) * 8 + (lane & 7), qr = lane & 15;
      const uint32_t ka = ks + kr * RB + swz<CPR>((lane >> 3) & 1, kr) * 16;
      const uint32_t qa = qs + qr * RB + swz<CPR>(lane >> 4, qr) * 16;
      float s2[SN][4];  // one row tile: even and odd steps apart, to halve the chain of dependent products
      if constexpr (MT == 1) {
#pragma unroll
        for (int n = 0; n < SN; ++n) s2[n][0] = s2[n][1] = s2[n][2] = s2[n][3] = 0.f;
      }
#pragma unroll
      for (int k = 0; k < HD / 16; ++k) {
        uint32_t kb[4];
        ldsm4(ka ^ (k * 32), kb);
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          uint32_t a[4];
          ldsm4((qa ^ (k * 32)) + i * 16 * RB, a);
          float(*t)[4] = MT == 1 && (k & 1) ? s2 : s[i];
          mma16<T>(t[0], a, kb[0], kb[1]);
          mma16<T>(t[SN - 1], a, kb[2], kb[3]);
        }
      }
      if constexpr (MT == 1) {
#pragma unroll
        for (int n = 0; n < SN; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[0][n][e] += s2[n][e];
      }
    } else {
      const int kr = warp * WP + g;
      const float* kp = (const float*)(stage + kr * RB);
      const float* qp = (const float*)(ring + d.qslot * L::STAGE + 2 * L::KB);
#pragma unroll 4
      for (int k = 0; k < HD / 8; ++k) {
        const float b0 = kp[swz<CPR>(2 * k, kr) * 4 + t4], b1 = kp[swz<CPR>(2 * k + 1, kr) * 4 + t4];
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          uint32_t ah[4], al[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int r = i * 16 + g + (e & 1) * 8;
            split_tf32(qp[r * HD + swz<CPR>(2 * k + (e >> 1), r) * 4 + t4], ah[e], al[e]);
          }
          mma_f32(s[i][0], ah, al, b0, b1);
        }
      }
    }
    // base-2 scores; positions a row does not see: -inf
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int n = 0; n < SN; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float x = s[i][n][e] * P.mul;
          if (P.softcap > 0.f) x = P.cap2 * tanh_f(x);
          s[i][n][e] = x;
        }
    int jhi[MT][2], jlo[MT][2];  // positions of this tile each of the thread's rows sees
    if (!plain) {
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const int row = d.row0 + i * 16 + g + r * 8;
          const int q = d.p0 + row / P.group;  // this row's position
          jhi[i][r] = row < d.count * P.group ? q - d.pos0 : -1;
          jlo[i][r] = P.window < 0 ? 0 : (int)max((int64_t)q - P.window - d.pos0, (int64_t)0);
        }
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int n = 0; n < SN; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int j = warp * WP + n * 8 + t4 * 2 + (e & 1);
            if (!(j <= jhi[i][e >> 1] && j >= jlo[i][e >> 1] && (vis >> j & 1u))) s[i][n][e] = -INFINITY;
          }
    }
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        float x = fmaxf(s[i][0][2 * r], s[i][0][2 * r + 1]);
        if (SN > 1) x = fmaxf(x, fmaxf(s[i][SN - 1][2 * r], s[i][SN - 1][2 * r + 1]));
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
        if (t4 == 0) wmax[warp * ROWS + i * 16 + r * 8 + g] = x;
      }
    bar_sync<AT_CONSUMERS>(INNER);  // maxima are there, and K is read: its rows may take the weights

    float alpha[MT][2];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int row = i * 16 + r * 8 + g;
        float x = m[i][r];
#pragma unroll
        for (int w = 0; w < 4; ++w) x = fmaxf(x, wmax[w * ROWS + row]);
        const float base = x == -INFINITY ? 0.f : x;
        alpha[i][r] = ex2(m[i][r] - base);
        m[i][r] = x;
        float sum = 0.f;
#pragma unroll
        for (int n = 0; n < SN; ++n) {
          const float p0 = ex2(s[i][n][2 * r] - base), p1 = ex2(s[i][n][2 * r + 1] - base);
          sum += p0 + p1;
          if constexpr (L::ES == 2) {
            // hi + lo keep 16 bits (f16: 22) of a weight, so the product with V
            // is good for an f32 output
            const uint32_t hi = pack2<T>(p0, p1);
            const float2 h = unpack2<T>(hi);
            const uint32_t lo = pack2<T>(p0 - h.x, p1 - h.y);
            unsigned char* at16 = pw + row * (TP * 2) + (((warp * SN + n) ^ (row & 7)) * 16) + t4 * 4;
            *(uint32_t*)at16 = hi;
            *(uint32_t*)(at16 + ROWS * TP * 2) = lo;
          } else {
            unsigned char* at32 = pw + row * (TP * 4) + (((warp * 2 + (t4 >> 1)) ^ (row & 7)) * 16) + (t4 & 1) * 8;
            *(float2*)at32 = make_float2(p0, p1);
          }
        }
        l[i][r] = l[i][r] * alpha[i][r] + sum;
      }
    bar_sync<AT_CONSUMERS>(INNER);  // weights are there

    // ---- P.V for this warp's quarter of head_dim
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        acc[i][n][0] *= alpha[i][0];
        acc[i][n][1] *= alpha[i][0];
        acc[i][n][2] *= alpha[i][1];
        acc[i][n][3] *= alpha[i][1];
      }
    // A position that some rows see and others do not may hold an infinity or
    // NaN, which a weight of zero does not keep out of a matrix product.  Tiles
    // with row-dependent masks look for such values first; with one of them in
    // this warp's columns the products are made one by one, for the rows that
    // do see the position.
    bool odd = false;
    if (!plain && d.count > 1) {
      constexpr int W = RB / 64;  // 16-byte chunks of a row in a quarter of it
#pragma unroll 1
      for (int i = lane; i < TP * W; i += 32) {
        const int j = i / W;
        const uint4 v = *(const uint4*)(stage + L::KB + j * RB + swz_v<T, CPR>(warp * W + i % W, j) * 16);
        odd = odd || odd_chunk<T>(v);
      }
      odd = __any_sync(0xffffffffu, odd);
    }
    if (odd) {
#pragma unroll 1
      for (int j = 0; j < TP; ++j) {
        if (!(vis >> j & 1u)) continue;
        float p[MT][2];
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const int row = i * 16 + r * 8 + g;
            if constexpr (L::ES == 2) {
              const unsigned char* at16 = pw + row * (TP * 2) + (((j >> 3) ^ (row & 7)) * 16) + (j & 7) * 2;
              p[i][r] = (float)*(const T*)at16 + (float)*(const T*)(at16 + ROWS * TP * 2);
            } else {
              p[i][r] = *(const float*)(pw + row * (TP * 4) + (((j >> 2) ^ (row & 7)) * 16) + (j & 3) * 4);
            }
          }
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int col = warp * (HD / 4) + n * 8 + t4 * 2 + e;
            constexpr int PC = 16 / L::ES;  // elements of a chunk
            const float v = (float)((const T*)(stage + L::KB + j * RB + swz_v<T, CPR>(col / PC, j) * 16))[col % PC];
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
              for (int r = 0; r < 2; ++r)
                if (j <= jhi[i][r] && j >= jlo[i][r]) acc[i][n][2 * r + e] += p[i][r] * v;
          }
      }
    } else if constexpr (L::ES == 2) {
      const int pr = lane & 15;
      const uint32_t pa = smem_u32(pw) + pr * (TP * 2) + (((lane >> 4) ^ (pr & 7)) * 16);
      const uint32_t va = vs + pr * RB + swz_v<T, CPR>(warp * NT + (NT > 1 ? lane >> 4 : 0), pr) * 16;
#pragma unroll
      for (int k = 0; k < TP / 16; ++k) {
        uint32_t ph[MT][4], pl[MT][4];
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          ldsm4((pa ^ (k * 32)) + i * 16 * TP * 2, ph[i]);
          ldsm4((pa ^ (k * 32)) + (ROWS + i * 16) * TP * 2, pl[i]);
        }
#pragma unroll
        for (int n = 0; n < NT; n += 2) {
          uint32_t vb[4];
          if constexpr (NT == 1) ldsm2t(va + k * 16 * RB, vb);
          else ldsm4t((va ^ (n * 16)) + k * 16 * RB, vb);
#pragma unroll
          for (int i = 0; i < MT; ++i) {
            mma16<T>(acc[i][n], ph[i], vb[0], vb[1]);
            if constexpr (NT > 1) mma16<T>(acc[i][n + 1], ph[i], vb[2], vb[3]);
            mma16<T>(acc[i][n], pl[i], vb[0], vb[1]);
            if constexpr (NT > 1) mma16<T>(acc[i][n + 1], pl[i], vb[2], vb[3]);
          }
        }
      }
    } else {
#pragma unroll
      for (int k = 0; k < TP / 8; ++k) {
        uint32_t ph[MT][4], pl[MT][4];
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int r = i * 16 + g + (e & 1) * 8;
            split_tf32(*(const float*)(pw + r * (TP * 4) + (((2 * k + (e >> 1)) ^ (r & 7)) * 16) + t4 * 4), ph[i][e], pl[i][e]);
          }
        const int r0 = k * 8 + t4, r1 = r0 + 4;
        const float* v0p = (const float*)(stage + L::KB + r0 * RB);
        const float* v1p = (const float*)(stage + L::KB + r1 * RB);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const int col = warp * (HD / 4) + n * 8 + g;
          const float b0 = v0p[swz_v<T, CPR>(col / 4, r0) * 4 + col % 4], b1 = v1p[swz_v<T, CPR>(col / 4, r1) * 4 + col % 4];
#pragma unroll
          for (int i = 0; i < MT; ++i) mma_f32(acc[i][n], ph[i], pl[i], b0, b1);
        }
      }
    }
    if (!(d.flags & T_END)) bar_arrive<AT_THREADS>(EMPTY + slot);

    // ---- the piece ends: the rows, or partials of them
    if (d.flags & T_LAST) {
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          float x = l[i][r];
          x += __shfl_xor_sync(0xffffffffu, x, 1);
          x += __shfl_xor_sync(0xffffffffu, x, 2);
          if (t4 == 0) wsum[warp * ROWS + i * 16 + r * 8 + g] = x;
        }
      bar_sync<AT_CONSUMERS>(INNER);
      const bool from0 = d.flags & T_FROM0, whole = from0 && (d.flags & T_TOEND);
      float* const part = P.part + ((int64_t)blockIdx.x * 2 + (from0 ? 1 : 0)) * (ROWS * (HD + 2));
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const int in_tile = i * 16 + r * 8 + g, row = d.row0 + in_tile;
          if (row >= d.count * P.group) continue;
          const float sum = wsum[in_tile] + wsum[ROWS + in_tile] + wsum[2 * ROWS + in_tile] + wsum[3 * ROWS + in_tile];
          if (whole) {
            const float inv = sum == 0.f ? 0.f : 1.f / sum;  // no position seen: zeros; a NaN stays one
            const int qi = row / P.group;
            char* o = P.out + (int64_t)(d.first + qi) * P.o_tok +
                      (int64_t)(d.head * P.group + row - qi * P.group) * P.o_head;
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              const int col = warp * (HD / 4) + n * 8 + t4 * 2;
              const float x = acc[i][n][2 * r] * inv, y = acc[i][n][2 * r + 1] * inv;
              if (L::ES == 4 || P.out_f32) *(float2*)(o + col * 4) = make_float2(x, y);
              else if constexpr (L::ES == 2) *(uint32_t*)(o + col * 2) = pack2<T>(x, y);
            }
          } else {
#pragma unroll
            for (int n = 0; n < NT; ++n)
              *(float2*)(part + in_tile * HD + warp * (HD / 4) + n * 8 + t4 * 2) =
                  make_float2(acc[i][n][2 * r], acc[i][n][2 * r + 1]);
            if (warp == 0 && t4 == 0) *(float2*)(part + ROWS * HD + in_tile * 2) = make_float2(m[i][r], sum);
          }
        }
    }
    if (d.flags & T_END) break;
  }
}

// Adds up the partials of the segment that starts in CTA blockIdx.x and is cut
// by its end: one row of it per blockIdx.y.
template <typename T, int HD, int ROWS>
__global__ void __launch_bounds__(AT_JOIN_THREADS) paged_attn_join_kernel(const __grid_constant__ PagedAttnParams P) {
  constexpr int LANES = HD / 4, GROUPS = AT_JOIN_THREADS / LANES;
  __shared__ float weight[kAttnMaxCtas];
  __shared__ float red[2][4];
  __shared__ float4 sums[GROUPS][LANES];
  pdl_enter();
  const int tid = threadIdx.x, r = blockIdx.y;
  const int32_t* meta = P.meta + blockIdx.x * 4;
  const int n = min(meta[0], (int)(gridDim.x - blockIdx.x));
  if (n < 1) return;
  int first, count;
  seq_rows(P.c, meta[1], first, count);
  const int row = meta[3] + r;
  if (row >= min(count, P.max_rows) * P.group) return;
  // partial i: slot 1 of this CTA, then slot 0 of the ones behind it
  auto part = [&](int i) { return P.part + ((int64_t)(blockIdx.x + i) * 2 + (i == 0)) * (ROWS * (HD + 2)); };
  float m = -INFINITY;
  for (int i = tid; i < n; i += AT_JOIN_THREADS) m = fmaxf(m, part(i)[ROWS * HD + r * 2]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  if ((tid & 31) == 0) red[0][tid >> 5] = m;
  __syncthreads();
  m = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
  const float base = m == -INFINITY ? 0.f : m;
  float l = 0.f;
  for (int i = tid; i < n; i += AT_JOIN_THREADS) {
    const float2 ml = *(const float2*)(part(i) + ROWS * HD + r * 2);
    const float w = ex2(ml.x - base);
    weight[i] = w;
    l += w * ml.y;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
  if ((tid & 31) == 0) red[1][tid >> 5] = l;
  __syncthreads();
  l = (red[1][0] + red[1][1]) + (red[1][2] + red[1][3]);
  const int lane = tid % LANES, grp = tid / LANES;
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int i = grp; i < n; i += GROUPS) {
    const float4 v = *(const float4*)(part(i) + r * HD + lane * 4);
    const float w = weight[i];
    a.x += w * v.x;
    a.y += w * v.y;
    a.z += w * v.z;
    a.w += w * v.w;
  }
  sums[grp][lane] = a;
  __syncthreads();
  if (grp) return;
#pragma unroll
  for (int i = 1; i < GROUPS; ++i) {
    const float4 v = sums[i][lane];
    a.x += v.x;
    a.y += v.y;
    a.z += v.z;
    a.w += v.w;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  char* o = P.out + (int64_t)(first + row / P.group) * P.o_tok + (int64_t)(meta[2] * P.group + row % P.group) * P.o_head;
  if (sizeof(T) == 4 || P.out_f32) {
    ((float4*)o)[lane] = make_float4(a.x * inv, a.y * inv, a.z * inv, a.w * inv);
  } else if constexpr (sizeof(T) == 2) {
    ((uint2*)o)[lane] = make_uint2(pack2<T>(a.x * inv, a.y * inv), pack2<T>(a.z * inv, a.w * inv));
  }
}

// ------------------------------------------------------------------- host
// Row tiles of 16, 32 or 64 rows: the smallest that holds a sequence's rows for
// one KV head (more rows than 64 take several tiles, each reading K and V
// again, from L2).  f32 rows of 256 stop at 32: two stages of more do not fit.
template <typename T, int HD>
constexpr int max_mt() {
  return sizeof(T) == 4 && HD == 256 ? 2 : 4;
}
template <typename T, int HD>
int pick_mt(const PagedAttnParams& p) {
  const int64_t rows = (int64_t)p.max_rows * p.group;
  return rows <= 16 ? 1 : (rows <= 32 || max_mt<T, HD>() == 2 ? 2 : 4);
}

// One tile at most in any segment: none is cut, and nothing needs joining.
template <typename T, int HD, int MT>
bool uncut(const PagedAttnParams& p) {
  int64_t span = (int64_t)p.c.pages_per_seq * p.c.page_size;
  if (p.window >= 0) span = std::min(span, p.window + p.max_rows);
  return span <= Tile<T, HD, MT>::TP;
}

template <typename T, int HD, int MT>
int64_t workspace_mt(const PagedAttnParams& p) {
  if (uncut<T, HD, MT>(p)) return 0;
  const int64_t ctas = (int64_t)device_sm_count() * Tile<T, HD, MT>::CTAS;
  return ctas * (2 * MT * 16 * (HD + 2) * 4 + 16);
}

template <typename T, int HD, int MT>
void launch_mt(PagedAttnParams p, cudaStream_t s) {
  using L = Tile<T, HD, MT>;
  const int ctas = device_sm_count() * L::CTAS;
  check(ctas <= kAttnMaxCtas, E_INTERNAL, "more SMs than the attention join holds");
  const bool cut = !uncut<T, HD, MT>(p);
  p.mul = p.softcap > 0.f ? p.scale / p.softcap : p.scale * 1.4426950408889634f;
  p.cap2 = p.softcap * 1.4426950408889634f;
  p.meta = cut ? (int32_t*)(p.part + (int64_t)ctas * 2 * L::ROWS * (HD + 2)) : nullptr;
  ensure_smem_optin((const void*)paged_attn_kernel<T, HD, MT>, L::SMEM);
  launch_k(paged_attn_kernel<T, HD, MT>, dim3(ctas), AT_THREADS, L::SMEM, s, 1, p);
  if (cut) {
    const int rows = (int)std::min<int64_t>((int64_t)p.max_rows * p.group, L::ROWS);
    launch_k(paged_attn_join_kernel<T, HD, L::ROWS>, dim3(ctas, rows), AT_JOIN_THREADS, 0, s, 1, p);
  }
}

template <typename T, int HD, class F>
auto with_mt(const PagedAttnParams& p, F f) {
  switch (pick_mt<T, HD>(p)) {
    case 1: return f(std::integral_constant<int, 1>());
    case 2: return f(std::integral_constant<int, 2>());
    default: return f(std::integral_constant<int, max_mt<T, HD>()>());
  }
}
template <typename T, class F>
auto with_hd(const PagedAttnParams& p, F f) {
  switch (p.hd) {
    case 32: return with_mt<T, 32>(p, [&](auto mt) { return f(std::integral_constant<int, 32>(), mt); });
    case 64: return with_mt<T, 64>(p, [&](auto mt) { return f(std::integral_constant<int, 64>(), mt); });
    case 128: return with_mt<T, 128>(p, [&](auto mt) { return f(std::integral_constant<int, 128>(), mt); });
    default: return with_mt<T, 256>(p, [&](auto mt) { return f(std::integral_constant<int, 256>(), mt); });
  }
}

template <typename T>
int64_t attention_workspace_of(const PagedAttnParams& p) {
  return with_hd<T>(p, [&](auto hd, auto mt) { return workspace_mt<T, decltype(hd)::value, decltype(mt)::value>(p); });
}
template <typename T>
void launch_attention_of(const PagedAttnParams& p, cudaStream_t s) {
  with_hd<T>(p, [&](auto hd, auto mt) { launch_mt<T, decltype(hd)::value, decltype(mt)::value>(p, s); });
}

}  // namespace
}  // namespace cljxla
