// Attention of a step's queries over the pages of their sequences.
//
// For each row at position p of its sequence and each query head,
//   out = sum_j w_j v_j / sum_j w_j,  w_j = 2^(s_j - m),  s_j = log2(e) * score_j,
// over the positions j the row sees, in one pass with the running maximum m
// and sum (a new maximum m' scales what is there by 2^(m - m')).
//
// What bounds it: each visible K and V row is read once from HBM for
// 4 * head_dim FLOPs per query row.  A decode step's 1 to 16 rows are bound by
// HBM bandwidth as long as enough copies are in flight; from about 32 rows per KV
// head on the tensor and issue slots of the consumer warps are.
//
// Split.  A segment is (sequence, KV head, up to ROWS query rows of that head's
// group), a row of tiles of its positions.  All tiles of the call, laid end to
// end, are cut into one equal range per CTA, whatever the sequences' lengths: one
// long context fills the GPU as well as many ragged ones do.  Each CTA finds its
// range itself from seq_lens (a scan over the sequences), so a captured graph
// follows the lengths.  A segment that lies within one CTA is finished there; a cut
// one leaves (m, sum, unnormalised row) partials that paged_attn_join_kernel,
// launched as a programmatic dependent, adds up in range order: no atomics, the
// same bits every time.
//
// Tile.  64 positions (32 for f32 rows of 256) of K and V rows go through a ring
// of stages.  Behind the four consumer warps, a scheduler warp walks the schedule
// and looks the pages of a tile up ahead, and two copier warps (one warp issues
// copies for about 3 TB/s over the GPU) gather its K and V rows with 16-byte
// cp.async (any page size, any strides; positions nobody sees are filled with zeros
// and not read).  Products run on mma.sync with the positions (scores) and the
// columns (P.V) as its 16 rows and 8 query rows as its columns: a decode step has
// few query rows, so this wastes the least.  Each consumer warp scores 16
// positions, row maxima and weights are shared through shared memory, and each
// warp adds P.V for its part of head_dim, so the accumulators stay small and no
// warp holds partials.  Stages change hands over named barriers.
//
// Measured (B200, device time): 1.07 GB of bf16 pages in one sequence 160 us (6.7
// TB/s, the copy rate), 32 sequences of 2 to 8447 positions at head_dim 256 28 us
// (4.3 TB/s; 9 us of that are the first tile's three dependent reads and the join),
// 256 sequences of 1 to 601 positions 49 us (4.3 TB/s).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <type_traits>

#include "common.h"
#include "paged.h"

namespace cljxla {
namespace {

constexpr int AT_CONSUMERS = 128, AT_JOIN_THREADS = 128;

// ------------------------------------------------------------------ layout
// floats of a slot of partials: rows, then their (max, sum), to whole 16 bytes
constexpr int slot_floats(int rows, int hd) { return (rows * (hd + 2) + 3) & ~3; }

template <typename T, int HD, int NR>
struct Tile {
  static constexpr int ES = sizeof(T);
  static constexpr int RB = HD * ES;            // bytes of a row
  static constexpr int TP = RB > 512 ? 32 : 64; // positions of a tile
  static constexpr bool SIMT = NR < 0;          // f32 and up to 4 rows: products on the FMA units, -NR rows
  static constexpr int ROWS = SIMT ? -NR : NR * 8;  // query rows
  static constexpr int CPR = RB / 16;           // 16-byte chunks of a row
  static constexpr int KB = TP * RB;
  static constexpr int QB = ROWS * RB;
  static constexpr int STAGE = 2 * KB + QB;     // K, V, and the queries of a segment that starts here
  // weights as two (bf16: three) 16-bit parts or one f32: in the tile's K rows once
  // they are scored, if they fit (SIMT: they do, and this is the warps' rows at a
  // piece's end)
  static constexpr int PARTS = std::is_same<T, __nv_bfloat16>::value ? 3 : 2;
  static constexpr int PB = SIMT ? 4 * ROWS * HD * 4 : ROWS * TP * (ES == 2 ? 2 * PARTS : 4);
  static constexpr bool P_IN_K = !SIMT && PB <= KB;
  static constexpr int fixed(int nst) { return (P_IN_K ? 0 : PB) + 2 * 4 * ROWS * 4 + nst * 64 + 160 + 4 * TP * 8; }
  static constexpr int fit(int ctas) {  // stages that fit with this many CTAs on an SM (228 KB, 1 KB each reserved)
    int n = 0;
    while (n < 4 && fixed(n + 1) + (n + 1) * STAGE <= 233472 / ctas - 1024) ++n;
    return n;
  }
  static constexpr int pick() {
    int ctas = KB > 16384 ? 1 : 2;
    while (ctas > 1 && fit(ctas) < 3) --ctas;
    return ctas;
  }
  static constexpr int CTAS = pick();
  static constexpr int NST = fit(CTAS);
  static constexpr int SMEM = fixed(NST) + NST * STAGE;
  static constexpr int THREADS = AT_CONSUMERS + 96;  // and a scheduler, a copier of K and one of V
  static_assert(NST >= 2, "a ring needs two stages");
  // Named barriers.  Stage hand-over: full[s] (copiers arrive, consumers wait),
  // empty[s] (consumers arrive, the scheduler waits); ahead: scheduler and copiers
  // among themselves; inner: the consumers.
  static constexpr int INNER = 1, AHEAD = 2, FULL = 3, EMPTY = FULL + NST;
  static constexpr int FULL_THREADS = AT_CONSUMERS + 64, EMPTY_THREADS = AT_CONSUMERS + 32, AHEAD_THREADS = 96;
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
  // ordered by the commit, not among themselves
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes));
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
__device__ __forceinline__ void stsm2t(uint32_t addr, uint32_t r0, uint32_t r1) {
  asm volatile("stmatrix.sync.aligned.m8n8.x2.trans.shared.b16 [%0], {%1,%2};" ::"r"(addr), "r"(r0), "r"(r1)
               : "memory");
}
__device__ __forceinline__ void stsm4t(uint32_t addr, uint32_t r0, uint32_t r1, uint32_t r2, uint32_t r3) {
  asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(r0), "r"(r1),
               "r"(r2), "r"(r3)
               : "memory");
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
__device__ __forceinline__ void mma_f32(float* c, const uint32_t* ah, const uint32_t* al, const uint32_t* bh,
                                        const uint32_t* bl) {
  mma_tf32(c, al, bh[0], bh[1]);
  mma_tf32(c, ah, bl[0], bl[1]);
  mma_tf32(c, ah, bh[0], bh[1]);
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
// tanh.  Below 1: Lambert's continued fraction y / (1 + y^2 / (3 + y^2 / (5 + ...)))
// to its sixth level, as a quotient (the rest is below 2^-27 of it there); from
// 1 on 1 - 2 / (1 + e^2y), which would cancel for small y: a capped score times the
// cap must keep its relative precision.
__device__ __forceinline__ float tanh_f(float y) {
  const float z = y * y;
  const float num = fmaf(z, fmaf(z, 21.f, 1260.f), 10395.f);
  const float den = fmaf(z, fmaf(z, z + 210.f, 4725.f), 10395.f);
  const float low = y * __fdividef(num, den);
  const float high = 1.f - __fdividef(2.f, 1.f + ex2(y * 2.8853900817779268f));
  return fabsf(y) < 1.f ? low : high;
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
// Its rows are `nrows` rows from head g0 of the group at the sequence's row q0 on.
struct TileDesc {
  int head, q0, g0, nrows, pos0, npos, flags, qslot, first, count, p0;  // p0: position of the sequence's first row
  uint32_t mask[2];  // positions whose page is there
};
enum { T_FIRST = 1, T_LAST = 2, T_FROM0 = 4, T_TOEND = 8, T_FULL = 16, T_END = 32 };  // T_END: the CTA's last tile

// One sequence's share of the schedule.
struct SeqPlan {
  int first, count, rows, p0, lo, hi, units, tiles;  // rows: computed ones; units: position tiles; tiles: row tiles
  __device__ __forceinline__ void make(const PagedAttnParams& P, int begin, int n, int len, int tile, int row_tile) {
    first = begin;
    count = min(n, P.max_rows);
    rows = count * P.group;
    tiles = (rows + row_tile - 1) / row_tile;
    p0 = len - n;
    lo = P.window < 0 ? 0 : (int)max((int64_t)p0 - P.window, (int64_t)0);
    hi = min(p0 + count, capacity(P.c));
    units = max((hi - lo + tile - 1) / tile, 1);
  }
  __device__ __forceinline__ void load(const PagedAttnParams& P, int b, int tile, int row_tile) {
    int begin, n;
    seq_rows(P.c, b, begin, n);
    make(P, begin, n, seq_len(P.c, b), tile, row_tile);
  }
  __device__ __forceinline__ int64_t segments(int nkv) const { return (int64_t)nkv * tiles; }
};

__device__ __forceinline__ int64_t div_small(int64_t a, int64_t b) {  // a >= 0, b > 0
  return (((uint64_t)a | (uint64_t)b) >> 32) == 0 ? (int64_t)((uint32_t)a / (uint32_t)b) : a / b;
}

// How the call's `total` slots are cut: the first `more` CTAs have each + 1 of
// them, the others each.  Where CTAs have several tiles each, a tile is two slots
// (`scale`) and every segment has one more in front (`extra`) for what its
// beginning and end cost (queries in, rows out: 0.5 to 0.7 us, a tile 1 to 1.4), or
// CTAs with many short segments would be the last; else a tile is one slot.  A tile
// belongs to the CTA that has its first slot.
struct Cut {
  int64_t total, each, more, ctas;
  int extra, scale;
  __device__ __forceinline__ void make(int64_t tiles, int64_t segments) {
    extra = tiles > 2 * (int64_t)gridDim.x ? 1 : 0;
    scale = 1 + extra;
    total = scale * tiles + extra * segments;
    ctas = min((int64_t)gridDim.x, total);
    each = ctas ? div_small(total, ctas) : 0;
    more = total - each * ctas;
  }
  __device__ __forceinline__ int64_t begin(int64_t cta) const { return each * cta + min(cta, more); }
  __device__ __forceinline__ int64_t owner(int64_t slot) const {
    const int64_t edge = more * (each + 1);
    return slot < edge ? div_small(slot, each + 1) : more + div_small(slot - edge, each);
  }
  __device__ __forceinline__ int64_t slots(int64_t units) const { return scale * units + extra; }  // of a segment
};

// Cuts the call's slots and finds the sequence that holds the one `pick` names
// (of the cut), and its place there: sh[8], sh[9] (-1: none was found, which takes
// lengths that change under the kernel).  By all THREADS threads of a CTA; the
// results are for use after the next barrier.
template <int THREADS, int TP, int ROWS, class F>
__device__ __forceinline__ Cut locate(const PagedAttnParams& P, int64_t* sh, F pick) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const PagedView& c = P.c;
  const int per = (c.num_seqs + THREADS - 1) / THREADS;
  const int b0 = min(tid * per, c.num_seqs), b1 = min(b0 + per, c.num_seqs);
  SeqPlan sp;
  int64_t tiles = 0, segments = 0;  // of this thread's sequences
  for (int i = b0; i < b1; ++i) {
    sp.load(P, i, TP, ROWS);
    segments += sp.segments(c.nkv);
    tiles += sp.segments(c.nkv) * sp.units;
  }
  int64_t tiles_to = tiles, segments_to = segments;  // up to and with them
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t t = __shfl_up_sync(0xffffffffu, tiles_to, o), s = __shfl_up_sync(0xffffffffu, segments_to, o);
    if (lane >= o) {
      tiles_to += t;
      segments_to += s;
    }
  }
  if (lane == 31) {
    sh[warp] = tiles_to;
    sh[10 + warp] = segments_to;
  }
  if (tid == 0) {
    sh[8] = 0;
    sh[9] = -1;
  }
  __syncthreads();
  int64_t all_tiles = 0, all_segments = 0;
  for (int w = 0; w < THREADS / 32; ++w) {
    if (w < warp) {
      tiles_to += sh[w];
      segments_to += sh[10 + w];
    }
    all_tiles += sh[w];
    all_segments += sh[10 + w];
  }
  Cut cut;
  cut.make(all_tiles, all_segments);
  const int64_t want = pick(cut);
  const int64_t incl = cut.scale * tiles_to + cut.extra * segments_to;
  int64_t excl = incl - cut.scale * tiles - cut.extra * segments;
  if (want >= excl && want < incl) {
    for (int i = b0; i < b1; ++i) {
      if (per > 1) sp.load(P, i, TP, ROWS);
      const int64_t slots = sp.segments(c.nkv) * cut.slots(sp.units);
      if (want < excl + slots) {
        sh[8] = i;
        sh[9] = want - excl;
        break;
      }
      excl += slots;
    }
  }
  return cut;
}

// x / group for x below 64 + group
__device__ __forceinline__ int div_group(const PagedAttnParams& P, int x) {
  return P.group_mul ? (int)__umulhi((uint32_t)x, P.group_mul) : x;
}

// The positions of tile `d` that its query row `r` sees: [jlo, jhi].
__device__ __forceinline__ void row_view(const PagedAttnParams& P, const TileDesc& d, int r, int& jlo, int& jhi) {
  const int pos = d.p0 + d.q0 + div_group(P, r + d.g0);  // the row's own position
  jhi = r < d.nrows ? pos - d.pos0 : -1;
  jlo = P.window < 0 ? 0 : (int)max((int64_t)pos - P.window - d.pos0, (int64_t)0);
}

// The consumer warps on mma.sync.
template <typename T, int HD, int NR>
__device__ __forceinline__ void consume_mma(const PagedAttnParams& P, unsigned char* const ring,
                                            unsigned char* const p_own, float* const wmax, float* const wsum,
                                            const TileDesc* const desc, const int warp, const int lane) {
  using L = Tile<T, HD, NR>;
  constexpr int TP = L::TP, ROWS = L::ROWS, RB = L::RB, CPR = L::CPR, NST = L::NST;
  constexpr int INNER = L::INNER, FULL = L::FULL, EMPTY = L::EMPTY;
  constexpr int FULL_THREADS = L::FULL_THREADS, EMPTY_THREADS = L::EMPTY_THREADS;
  constexpr int SCORERS = TP / 16;                  // warps that score 16 positions each
  constexpr int CW = HD >= 64 ? HD / 4 : 16;        // columns of P.V of a warp
  constexpr int MT = CW / 16, ADDERS = HD / CW;     // their 16-column tiles; warps that have some
  constexpr int PROW = TP * (L::ES == 2 ? 2 : 4);   // bytes of a row of weights
  constexpr int QK = HD / 32;                       // steps of 32 of head_dim
  float acc[MT][NR][4], m[NR][2], l[NR][2];
  constexpr bool Q_REGS = L::ES == 2 && (NR == 1 || (NR == 2 && L::CTAS == 1));
  uint32_t qf[Q_REGS ? QK : 1][Q_REGS ? NR : 1][4];  // the queries, where they fit registers
  const bool third = L::PARTS == 3 && P.out_f32;    // a third part of the weights
  // f16 has no exponents to spare: its weights are taken relative to the tile's own
  // maximum, 2^15 times as large (`beta` brings the tile's sums to the running maximum,
  // the 2^15 cancels in the quotient).  Relative to the running one, a dominant position
  // (2^25 times the others) would leave the others' weights no bits.
  constexpr bool HALF = std::is_same<T, __half>::value;
  // this thread's positions and columns: g, g + 8; its rows: 2 t4, 2 t4 + 1
  const int g = lane >> 2, t4 = lane & 3;
  for (int tile = 0;; ++tile) {
    const int slot = tile % NST;
    bar_sync<FULL_THREADS>(FULL + slot);
    const TileDesc d = *(const TileDesc*)((char*)desc + slot * 64);
    unsigned char* const stage = ring + slot * L::STAGE;
    unsigned char* const queries = ring + d.qslot * L::STAGE + 2 * L::KB;
    const uint32_t ks = smem_u32(stage), vs = ks + L::KB, qs = smem_u32(queries);
    unsigned char* const pw = L::P_IN_K ? stage : p_own;
    const uint64_t vis = TP == 64 ? (uint64_t)d.mask[1] << 32 | d.mask[0] : d.mask[0];
    const bool plain = (d.flags & T_FULL) && vis == (TP == 64 ? ~0ull : 0xffffffffull);
    // 8 query rows x 32 of head_dim: the second operands of two steps
    const uint32_t qa = qs + (lane & 7) * RB + swz<CPR>(lane >> 3, lane & 7) * 16;
    if (d.flags & T_FIRST) {
#pragma unroll
      for (int n = 0; n < NR; ++n) {
        m[n][0] = m[n][1] = -INFINITY;
        l[n][0] = l[n][1] = 0.f;
#pragma unroll
        for (int i = 0; i < MT; ++i) acc[i][n][0] = acc[i][n][1] = acc[i][n][2] = acc[i][n][3] = 0.f;
      }
      if constexpr (Q_REGS) {
#pragma unroll
        for (int j = 0; j < QK; ++j)
#pragma unroll
          for (int n = 0; n < NR; ++n) ldsm4((qa ^ (j * 64)) + n * 8 * RB, qf[j][n]);
      }
    }

    // ---- scores: s[n][e] is of position g + 8 (e / 2) of the warp's 16 and row 8 n + 2 t4 + e % 2
    float s[NR][4];
    if (SCORERS == 4 || warp < SCORERS) {
#pragma unroll
      for (int n = 0; n < NR; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
      if (warp * 16 >= d.npos) {
        // nothing of the tile reaches this warp's positions: all are masked below
      } else if constexpr (L::ES == 2) {
        // chunk 2 k + (0 or 1) of a row: its swizzled address differs from chunk
        // 0 or 1's by an exclusive or with 32 k
        const int kr = warp * 16 + (lane & 15);
        const uint32_t ka = ks + kr * RB + swz<CPR>(lane >> 4, kr) * 16;
        // one row tile: every other step apart, to halve the chain of dependent products
        float s2[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < QK; ++j) {
          uint32_t k0[4], k1[4];
          ldsm4(ka ^ (j * 64), k0);
          ldsm4(ka ^ (j * 64 + 32), k1);
#pragma unroll
          for (int n = 0; n < NR; ++n) {
            uint32_t q[4];
            if constexpr (Q_REGS) {
#pragma unroll
              for (int e = 0; e < 4; ++e) q[e] = qf[j][n][e];
            } else {
              ldsm4((qa ^ (j * 64)) + n * 8 * RB, q);
            }
            mma16<T>(s[n], k0, q[0], q[1]);
            mma16<T>(NR == 1 ? s2 : s[n], k1, q[2], q[3]);
          }
        }
        if constexpr (NR == 1) {
#pragma unroll
          for (int e = 0; e < 4; ++e) s[0][e] += s2[e];
        }
      } else {
        const int kr = warp * 16 + g;  // and kr + 8: the same swizzle
        const float* const kp = (const float*)(stage + kr * RB);
        const float* const qp = (const float*)(queries + g * RB);
        // four steps' sums apart, the small products from the large, and added with
        // rounding: the tensor cores cut sums off, which 96 times in one chain costs
        // 3e-6 of a score
#pragma unroll 1
        for (int k4 = 0; k4 < HD / 8; k4 += 4) {
          float big[NR][4], small[NR][4];
#pragma unroll
          for (int n = 0; n < NR; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) big[n][e] = small[n][e] = 0.f;
#pragma unroll
          for (int k = k4; k < k4 + 4; ++k) {
            const int c0 = swz<CPR>(2 * k, g) * 4 + t4, c1 = swz<CPR>(2 * k + 1, g) * 4 + t4;
            uint32_t ah[4], al[4];
            split_tf32(kp[c0], ah[0], al[0]);
            split_tf32(kp[c0 + 8 * HD], ah[1], al[1]);
            split_tf32(kp[c1], ah[2], al[2]);
            split_tf32(kp[c1 + 8 * HD], ah[3], al[3]);
#pragma unroll
            for (int n = 0; n < NR; ++n) {
              uint32_t bh[2], bl[2];
              split_tf32(qp[c0 + n * 8 * HD], bh[0], bl[0]);
              split_tf32(qp[c1 + n * 8 * HD], bh[1], bl[1]);
              mma_tf32(small[n], al, bh[0], bh[1]);
              mma_tf32(small[n], ah, bl[0], bl[1]);
              mma_tf32(big[n], ah, bh[0], bh[1]);
            }
          }
#pragma unroll
          for (int n = 0; n < NR; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[n][e] += big[n][e] + small[n][e];
        }
      }
      // base-2 scores
#pragma unroll
      for (int n = 0; n < NR; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[n][e] *= P.mul;
      if (P.softcap > 0.f) {
#pragma unroll
        for (int n = 0; n < NR; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[n][e] = P.cap2 * tanh_f(s[n][e]);
      }
      if (!plain) {  // positions a row does not see: -inf
#pragma unroll
        for (int n = 0; n < NR; ++n)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            int jlo, jhi;
            row_view(P, d, n * 8 + 2 * t4 + r, jlo, jhi);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int j = warp * 16 + g + h * 8;
              if (j < jlo || j > jhi || !(vis >> j & 1u)) s[n][h * 2 + r] = -INFINITY;
            }
          }
      }
#pragma unroll
      for (int n = 0; n < NR; ++n) {
        float2 x = make_float2(fmaxf(s[n][0], s[n][2]), fmaxf(s[n][1], s[n][3]));
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) {
          x.x = fmaxf(x.x, __shfl_xor_sync(0xffffffffu, x.x, o));
          x.y = fmaxf(x.y, __shfl_xor_sync(0xffffffffu, x.y, o));
        }
        if (g == 0) *(float2*)(wmax + warp * ROWS + n * 8 + 2 * t4) = x;
      }
    }
    bar_sync<AT_CONSUMERS>(INNER);  // maxima are there, and K is read: its rows may take the weights

    float alpha[NR][2], beta[HALF ? NR : 1][2];
#pragma unroll
    for (int n = 0; n < NR; ++n) {
      float2 top = make_float2(-INFINITY, -INFINITY);  // the tile's
#pragma unroll
      for (int w = 0; w < SCORERS; ++w) {
        const float2 y = *(const float2*)(wmax + w * ROWS + n * 8 + 2 * t4);
        top.x = fmaxf(top.x, y.x);
        top.y = fmaxf(top.y, y.y);
      }
      const float2 x = make_float2(fmaxf(m[n][0], top.x), fmaxf(m[n][1], top.y));
      float b0 = x.x == -INFINITY ? 0.f : x.x, b1 = x.y == -INFINITY ? 0.f : x.y;
      alpha[n][0] = ex2(m[n][0] - b0);
      alpha[n][1] = ex2(m[n][1] - b1);
      m[n][0] = x.x;
      m[n][1] = x.y;
      if constexpr (HALF) {
        beta[n][0] = ex2(top.x - b0);
        beta[n][1] = ex2(top.y - b1);
        b0 = top.x == -INFINITY ? 0.f : top.x;
        b1 = top.y == -INFINITY ? 0.f : top.y;
      }
      if (SCORERS == 4 || warp < SCORERS) {
        auto weight = [](float x, float b) {
          if constexpr (HALF) return ex2(x - b + 15.f);  // added last: scores of 2^30 have steps above 15
          else return ex2(x - b);
        };
        const float p0 = weight(s[n][0], b0), p1 = weight(s[n][1], b1), p2 = weight(s[n][2], b0), p3 = weight(s[n][3], b1);
        l[n][0] = fmaf(l[n][0], alpha[n][0], HALF ? beta[HALF ? n : 0][0] * (p0 + p2) : p0 + p2);
        l[n][1] = fmaf(l[n][1], alpha[n][1], HALF ? beta[HALF ? n : 0][1] * (p1 + p3) : p1 + p3);
        if constexpr (L::ES == 2) {
          // Parts of a weight, each what the ones before leave.  f16: two keep 22 bits, or
          // all above 2^-40 of the tile's largest.  bf16: two keep 16, enough for its own
          // outputs; an f32 one takes a third.
          const uint32_t h0 = pack2<T>(p0, p1), h1 = pack2<T>(p2, p3);
          const float2 f0 = unpack2<T>(h0), f1 = unpack2<T>(h1);
          const float q0 = p0 - f0.x, q1 = p1 - f0.y, q2 = p2 - f1.x, q3 = p3 - f1.y;
          const uint32_t l0 = pack2<T>(q0, q1), l1 = pack2<T>(q2, q3);
          const int row = n * 8 + (lane & 7), ch = warp * 2 + (lane >> 3 & 1);
          const uint32_t to = smem_u32(pw) + row * PROW + ((ch ^ (row & 7)) * 16);
          stsm4t(to + (lane >> 4) * (ROWS * PROW), h0, h1, l0, l1);
          if (third) {
            const float2 g0 = unpack2<T>(l0), g1 = unpack2<T>(l1);
            stsm2t(to + 2 * ROWS * PROW, pack2<T>(q0 - g0.x, q1 - g0.y), pack2<T>(q2 - g1.x, q3 - g1.y));
          }
        } else {
          const float p[4] = {p0, p1, p2, p3};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int row = n * 8 + 2 * t4 + (e & 1), j = warp * 16 + g + (e >> 1) * 8;
            *(float*)(pw + row * PROW + (((j >> 2) ^ (row & 7)) * 16) + (j & 3) * 4) = p[e];
          }
        }
      }
    }
    bar_sync<AT_CONSUMERS>(INNER);  // weights are there

    // ---- P.V: acc[i][n][e] is of column g + 8 (e / 2) of the warp's i-th 16 and row 8 n + 2 t4 + e % 2
    if (ADDERS == 4 || warp < ADDERS) {
      // A position that some rows see and others do not may hold an infinity or
      // NaN, which a weight of zero does not keep out of a matrix product.  Tiles
      // with row-dependent masks look for such values first; with one of them in
      // this warp's columns the products are made one by one, for the rows that
      // do see the position.
      bool odd = false;
      if (!plain && d.count > 1) {
        constexpr int W = CW * L::ES / 16;  // 16-byte chunks of a row that are this warp's
        auto look = [&](int from, int upto) {
#pragma unroll 1
          for (int i = max(from, 0) * W + lane; i < min(upto, d.npos) * W; i += 32) {
            const int j = i / W;
            const uint4 v = *(const uint4*)(stage + L::KB + j * RB + swz_v<T, CPR>(warp * W + i % W, j) * 16);
            odd = odd || odd_chunk<T>(v);
          }
        };
        const int own = d.p0 - d.pos0;  // the first row's position; the later ones see further, and less far back
        if (P.window >= 0) look(0, (int)max((int64_t)own + d.count - 1 - P.window, (int64_t)0));
        look(own + 1, own + d.count);
        odd = __any_sync(0xffffffffu, odd);
      }
      if (odd) {
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int n = 0; n < NR; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[i][n][e] *= alpha[n][e & 1];
#pragma unroll 1
        for (int j = 0; j < TP; ++j) {
          if (!(vis >> j & 1u)) continue;
#pragma unroll
          for (int n = 0; n < NR; ++n)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              const int row = n * 8 + 2 * t4 + r;
              int jlo, jhi;
              row_view(P, d, row, jlo, jhi);
              if (j < jlo || j > jhi) continue;
              float p;
              if constexpr (L::ES == 2) {
                const unsigned char* at16 = pw + row * PROW + (((j >> 3) ^ (row & 7)) * 16) + (j & 7) * 2;
                p = (float)*(const T*)at16 + (float)*(const T*)(at16 + ROWS * PROW);
                if (third) p += (float)*(const T*)(at16 + 2 * ROWS * PROW);
              } else {
                p = *(const float*)(pw + row * PROW + (((j >> 2) ^ (row & 7)) * 16) + (j & 3) * 4);
              }
              if constexpr (HALF) p *= beta[n][r];
#pragma unroll
              for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                  constexpr int PC = 16 / L::ES;  // elements of a chunk
                  const int col = warp * CW + i * 16 + g + h * 8;
                  acc[i][n][h * 2 + r] +=
                      p * (float)((const T*)(stage + L::KB + j * RB + swz_v<T, CPR>(col / PC, j) * 16))[col % PC];
                }
            }
        }
      } else {
        // A tile's sum is made apart and added with one rounding: the tensor cores
        // cut their sums off, and over a long context that adds up to 10^-5 of the result.
        constexpr int IB = MT * NR <= 8 ? MT : 1;  // 16-column tiles at a time, as registers allow
        const uint32_t pa = smem_u32(pw) + (lane & 7) * PROW + (((lane >> 3) ^ (lane & 7)) * 16);
        const int vr = (lane >> 4) * 8 + (lane & 7);
        const uint32_t va = vs + vr * RB + swz_v<T, CPR>(warp * (CW / 8) + (lane >> 3 & 1), vr) * 16;
#pragma unroll
        for (int i0 = 0; i0 < MT; i0 += IB) {
          float t[IB][NR][4];
#pragma unroll
          for (int i = 0; i < IB; ++i)
#pragma unroll
            for (int n = 0; n < NR; ++n) t[i][n][0] = t[i][n][1] = t[i][n][2] = t[i][n][3] = 0.f;
          if constexpr (L::ES == 2) {
#pragma unroll
            for (int j = 0; j < TP / 32; ++j) {
              if (j * 32 >= d.npos) break;  // rows from here on were not copied
              uint32_t ph[NR][4], pl[NR][4], pt[L::PARTS == 3 ? NR : 1][4];
#pragma unroll
              for (int n = 0; n < NR; ++n) {
                ldsm4((pa ^ (j * 64)) + n * 8 * PROW, ph[n]);
                ldsm4((pa ^ (j * 64)) + (ROWS + n * 8) * PROW, pl[n]);
                if constexpr (L::PARTS == 3)
                  if (third) ldsm4((pa ^ (j * 64)) + (2 * ROWS + n * 8) * PROW, pt[n]);
              }
#pragma unroll
              for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int i = 0; i < IB; ++i) {
                  uint32_t v[4];
                  ldsm4t((va ^ ((i0 + i) * 32)) + (j * 32 + h * 16) * RB, v);
#pragma unroll
                  for (int n = 0; n < NR; ++n)
                    mma16<T>(t[i][n], v, ph[n][2 * h], ph[n][2 * h + 1]);
#pragma unroll
                  for (int n = 0; n < NR; ++n)
                    mma16<T>(t[i][n], v, pl[n][2 * h], pl[n][2 * h + 1]);
                  if constexpr (L::PARTS == 3) {
                    if (third) {
#pragma unroll
                      for (int n = 0; n < NR; ++n)
                        mma16<T>(t[i][n], v, pt[n][2 * h], pt[n][2 * h + 1]);
                    }
                  }
                }
            }
          } else {
#pragma unroll 2
            for (int k = 0; k * 8 < d.npos; ++k) {
              uint32_t bh[NR][2], bl[NR][2];
#pragma unroll
              for (int n = 0; n < NR; ++n)
#pragma unroll
                for (int h = 0; h < 2; ++h)
                  split_tf32(*(const float*)(pw + (n * 8 + g) * PROW + (((2 * k + h) ^ g) * 16) + t4 * 4), bh[n][h],
                             bl[n][h]);
              const int r0 = k * 8 + t4;  // and r0 + 4: the same swizzle
              const float* const vp = (const float*)(stage + L::KB + r0 * RB);
#pragma unroll
              for (int i = 0; i < IB; ++i) {
                const int col = warp * CW + (i0 + i) * 16 + g;
                const int c0 = swz_v<T, CPR>(col / 4, r0) * 4 + col % 4;
                const int c1 = swz_v<T, CPR>(col / 4 + 2, r0) * 4 + col % 4;
                uint32_t ah[4], al[4];
                split_tf32(vp[c0], ah[0], al[0]);
                split_tf32(vp[c1], ah[1], al[1]);
                split_tf32(vp[c0 + 4 * HD], ah[2], al[2]);
                split_tf32(vp[c1 + 4 * HD], ah[3], al[3]);
#pragma unroll
                for (int n = 0; n < NR; ++n)
                  mma_f32(t[i][n], ah, al, bh[n], bl[n]);
              }
            }
          }
#pragma unroll
          for (int i = 0; i < IB; ++i)
#pragma unroll
            for (int n = 0; n < NR; ++n)
#pragma unroll
              for (int e = 0; e < 4; ++e)
                acc[i0 + i][n][e] = fmaf(acc[i0 + i][n][e], alpha[n][e & 1],
                                         HALF ? t[i][n][e] * beta[HALF ? n : 0][e & 1] : t[i][n][e]);
        }
      }
    }
    if (!(d.flags & T_END)) bar_arrive<EMPTY_THREADS>(EMPTY + slot);

    // ---- the piece ends: the rows, or partials of them
    if (d.flags & T_LAST) {
      if (SCORERS == 4 || warp < SCORERS) {
#pragma unroll
        for (int n = 0; n < NR; ++n) {
          float2 x = make_float2(l[n][0], l[n][1]);
#pragma unroll
          for (int o = 4; o < 32; o <<= 1) {
            x.x += __shfl_xor_sync(0xffffffffu, x.x, o);
            x.y += __shfl_xor_sync(0xffffffffu, x.y, o);
          }
          if (g == 0) *(float2*)(wsum + warp * ROWS + n * 8 + 2 * t4) = x;
        }
      }
      bar_sync<AT_CONSUMERS>(INNER);
      const bool from0 = d.flags & T_FROM0, whole = from0 && (d.flags & T_TOEND);
      float* const part = P.part + ((int64_t)blockIdx.x * 2 + (from0 ? 1 : 0)) * slot_floats(ROWS, HD);
      // neighbours in g swap a row, so that a thread has two columns of one row to
      // store: row 8 n + 2 t4 + g % 2, columns g - g % 2 and the next
      const int odd_g = g & 1;
#pragma unroll
      for (int n = 0; n < NR; ++n) {
        const int in_tile = n * 8 + 2 * t4 + odd_g;
        const bool mine = in_tile < d.nrows;
        float sum = 0.f;
#pragma unroll
        for (int w = 0; w < SCORERS; ++w) sum += wsum[w * ROWS + in_tile];
        if (mine && !whole && warp == 0 && g < 2)
          *(float2*)(part + ROWS * HD + in_tile * 2) = make_float2(odd_g ? m[n][1] : m[n][0], sum);
        if (ADDERS < 4 && warp >= ADDERS) continue;
        // no position seen: zeros; a NaN stays one
        const float scale = !whole ? 1.f : sum == 0.f ? 0.f : __fdividef(1.f, sum);
        const int dq = div_group(P, in_tile + d.g0);
        const bool wide = !whole || L::ES == 4 || P.out_f32;
        char* const o = whole ? P.out + (int64_t)(d.first + d.q0 + dq) * P.o_tok +
                                    (int64_t)(d.head * P.group + in_tile + d.g0 - dq * P.group) * P.o_head
                              : (char*)(part + in_tile * HD);
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float a0 = acc[i][n][h * 2], a1 = acc[i][n][h * 2 + 1];
            const float keep = odd_g ? a1 : a0, give = odd_g ? a0 : a1;
            const float got = __shfl_xor_sync(0xffffffffu, give, 4);
            const float x = (odd_g ? got : keep) * scale, y = (odd_g ? keep : got) * scale;
            const int col = warp * CW + i * 16 + h * 8 + g - odd_g;
            if (!mine) continue;
            if (wide) *(float2*)(o + col * 4) = make_float2(x, y);
            else if constexpr (L::ES == 2) *(uint32_t*)(o + col * 2) = pack2<T>(x, y);
          }
      }
    }
    if (d.flags & T_END) break;
  }
}

// The consumer warps for f32 and up to four query rows, on the FMA units: a warp
// has a quarter of a tile's positions to itself, scores (a lane per position and
// part of head_dim) and weighs them and adds its own P.V (a lane per four columns), and
// the four warps meet only at the end of a piece.  tf32 products in three terms
// cost about 1000 instructions a warp and tile whatever the rows, this about 130 per row
// and 100.
template <int HD, int NR>
__device__ __forceinline__ void consume_simt(const PagedAttnParams& P, unsigned char* const ring,
                                             unsigned char* const p_own, float* const wmax, float* const wsum,
                                             const TileDesc* const desc, const int warp, const int lane) {
  using L = Tile<float, HD, NR>;
  constexpr int TP = L::TP, ROWS = L::ROWS, RB = L::RB, CPR = L::CPR, NST = L::NST;
  constexpr int WP = TP / 4, HS = 32 / WP;                       // positions of a warp, lanes of a position
  // lanes of a V row, rows at a time, chunks of a lane
  constexpr int VL = CPR < 32 ? CPR : 32, VG = 32 / VL, VC = CPR / VL;
  const int pos = lane % WP, part = lane / WP, vl = lane % VL, vg = lane / VL;
  float4 acc[ROWS][VC];
  float m[ROWS], l[ROWS];
  for (int tile = 0;; ++tile) {
    const int slot = tile % NST;
    bar_sync<L::FULL_THREADS>(L::FULL + slot);
    const TileDesc d = *(const TileDesc*)((char*)desc + slot * 64);
    unsigned char* const stage = ring + slot * L::STAGE;
    const unsigned char* const queries = ring + d.qslot * L::STAGE + 2 * L::KB;
    const uint64_t vis = TP == 64 ? (uint64_t)d.mask[1] << 32 | d.mask[0] : d.mask[0];
    const bool plain = (d.flags & T_FULL) && vis == (TP == 64 ? ~0ull : 0xffffffffull);
    const int mine = min(max(d.npos - warp * WP, 0), WP);  // positions of this warp
    const int j = warp * WP + pos;
    if (d.flags & T_FIRST) {
#pragma unroll
      for (int r = 0; r < ROWS; ++r) {
        m[r] = -INFINITY;
        l[r] = 0.f;
#pragma unroll
        for (int i = 0; i < VC; ++i) acc[r][i] = make_float4(0.f, 0.f, 0.f, 0.f);
      }
    }
    if (mine > 0) {
      float4 s4[ROWS];
#pragma unroll
      for (int r = 0; r < ROWS; ++r) s4[r] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
      for (int ch = part; ch < CPR; ch += HS) {
        const float4 k = *(const float4*)(stage + j * RB + swz<CPR>(ch, j) * 16);
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
          const float4 q = *(const float4*)(queries + r * RB + swz<CPR>(ch, r) * 16);
          s4[r].x += q.x * k.x;
          s4[r].y += q.y * k.y;
          s4[r].z += q.z * k.z;
          s4[r].w += q.w * k.w;
        }
      }
      __syncwarp();  // this warp's K rows are read: the first takes its weights
      float* const pw = (float*)(stage + warp * WP * RB);
      bool part_seen = false;  // whether some row sees a position that another does not
#pragma unroll
      for (int r = 0; r < ROWS; ++r) {
        float s = (s4[r].x + s4[r].y) + (s4[r].z + s4[r].w);
#pragma unroll
        for (int o = WP; o < 32; o <<= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        s *= P.mul;
        if (P.softcap > 0.f) s = P.cap2 * tanh_f(s);
        bool see = true;
        if (!plain) {
          int jlo, jhi;
          row_view(P, d, r, jlo, jhi);
          see = j >= jlo && j <= jhi && (vis >> j & 1u);
          if (!see) s = -INFINITY;
          part_seen = d.count > 1;
        }
        float top = fmaxf(m[r], s);
#pragma unroll
        for (int o = WP / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        const float base = top == -INFINITY ? 0.f : top;
        const float alpha = ex2(m[r] - base), p = ex2(s - base);
        m[r] = top;
        l[r] = l[r] * alpha + (part == 0 ? p : 0.f);
        if (part == 0) pw[r * WP + pos] = see ? p : part_seen ? -1.f : 0.f;
#pragma unroll
        for (int i = 0; i < VC; ++i) {
          acc[r][i].x *= alpha;
          acc[r][i].y *= alpha;
          acc[r][i].z *= alpha;
          acc[r][i].w *= alpha;
        }
      }
      __syncwarp();
      auto add = [&](auto careful) {
#pragma unroll 4
        for (int i0 = 0; i0 < WP; i0 += VG) {
          const int jj = i0 + vg, row = warp * WP + jj;
          if (i0 >= mine) break;  // rows from here on may not have been copied
          float w[ROWS];
#pragma unroll
          for (int r = 0; r < ROWS; ++r) w[r] = jj < mine ? pw[r * WP + jj] : 0.f;
#pragma unroll
          for (int i = 0; i < VC; ++i) {
            float4 v = *(const float4*)(stage + L::KB + row * RB + swz_v<float, CPR>(vl + i * VL, row) * 16);
            if (VG > 1 && jj >= mine) v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int r = 0; r < ROWS; ++r) {
              if (decltype(careful)::value && w[r] == -1.f) continue;  // not seen: whatever it holds stays out
              acc[r][i].x += w[r] * v.x;
              acc[r][i].y += w[r] * v.y;
              acc[r][i].z += w[r] * v.z;
              acc[r][i].w += w[r] * v.w;
            }
          }
        }
      };
      if (part_seen) add(std::true_type());
      else add(std::false_type());
    }
    if (!(d.flags & T_END)) bar_arrive<L::EMPTY_THREADS>(L::EMPTY + slot);

    // ---- the piece ends: the warps' rows together, or partials of them
    if (d.flags & T_LAST) {
#pragma unroll
      for (int r = 0; r < ROWS; ++r) {
#pragma unroll
        for (int o = WP / 2; o > 0; o >>= 1) l[r] += __shfl_xor_sync(0xffffffffu, l[r], o);
        if (lane == 0) {
          wmax[warp * ROWS + r] = m[r];
          wsum[warp * ROWS + r] = l[r];
        }
      }
      bar_sync<AT_CONSUMERS>(L::INNER);
      float top[ROWS], sum[ROWS];
      float4* const rows4 = (float4*)p_own;  // [warp][row][chunk]
#pragma unroll
      for (int r = 0; r < ROWS; ++r) {
        top[r] = fmaxf(fmaxf(wmax[r], wmax[ROWS + r]), fmaxf(wmax[2 * ROWS + r], wmax[3 * ROWS + r]));
        const float base = top[r] == -INFINITY ? 0.f : top[r];
        sum[r] = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) sum[r] += wsum[w * ROWS + r] * ex2(wmax[w * ROWS + r] - base);
        const float f = ex2(m[r] - base);
#pragma unroll
        for (int i = 0; i < VC; ++i) {
          float4 a = acc[r][i];
#pragma unroll
          for (int o = VL; o < 32; o <<= 1) {
            a.x += __shfl_xor_sync(0xffffffffu, a.x, o);
            a.y += __shfl_xor_sync(0xffffffffu, a.y, o);
            a.z += __shfl_xor_sync(0xffffffffu, a.z, o);
            a.w += __shfl_xor_sync(0xffffffffu, a.w, o);
          }
          if (vg == 0) rows4[(warp * ROWS + r) * CPR + vl + i * VL] = make_float4(a.x * f, a.y * f, a.z * f, a.w * f);
        }
      }
      bar_sync<AT_CONSUMERS>(L::INNER);
      const bool from0 = d.flags & T_FROM0, whole = from0 && (d.flags & T_TOEND);
      float* const part_out = P.part + ((int64_t)blockIdx.x * 2 + (from0 ? 1 : 0)) * slot_floats(ROWS, HD);
#pragma unroll
      for (int r = 0; r < ROWS; ++r) {
        if (r >= d.nrows) break;
        if (!whole && warp == 0 && lane == 0) *(float2*)(part_out + ROWS * HD + r * 2) = make_float2(top[r], sum[r]);
        const float scale = !whole ? 1.f : sum[r] == 0.f ? 0.f : __fdividef(1.f, sum[r]);  // no position seen: zeros
        const int dq = div_group(P, r + d.g0);
        float4* const o = whole ? (float4*)(P.out + (int64_t)(d.first + d.q0 + dq) * P.o_tok +
                                            (int64_t)(d.head * P.group + r + d.g0 - dq * P.group) * P.o_head)
                                : (float4*)(part_out + r * HD);
        for (int ch = warp * 32 + lane; ch < CPR; ch += AT_CONSUMERS) {
          const float4 a = rows4[r * CPR + ch], b = rows4[(ROWS + r) * CPR + ch], c = rows4[(2 * ROWS + r) * CPR + ch],
                       e = rows4[(3 * ROWS + r) * CPR + ch];
          o[ch] = make_float4(((a.x + b.x) + (c.x + e.x)) * scale, ((a.y + b.y) + (c.y + e.y)) * scale,
                              ((a.z + b.z) + (c.z + e.z)) * scale, ((a.w + b.w) + (c.w + e.w)) * scale);
        }
      }
    }
    if (d.flags & T_END) break;
  }
}

template <typename T, int HD, int NR>
__global__ void __launch_bounds__(Tile<T, HD, NR>::THREADS, Tile<T, HD, NR>::CTAS)
    paged_attn_kernel(const __grid_constant__ PagedAttnParams P) {
  using L = Tile<T, HD, NR>;
  constexpr int TP = L::TP, ROWS = L::ROWS, RB = L::RB, CPR = L::CPR, NST = L::NST, AT_THREADS = L::THREADS;
  extern __shared__ __align__(1024) unsigned char smem[];
  unsigned char* const ring = smem;
  unsigned char* const p_own = smem + NST * L::STAGE;
  float* const wmax = (float*)(p_own + (L::P_IN_K ? 0 : L::PB));  // [4][ROWS]
  float* const wsum = wmax + 4 * ROWS;
  TileDesc* const desc = (TileDesc*)(wsum + 4 * ROWS);  // [NST], 64 bytes each
  int64_t* const sh = (int64_t*)((unsigned char*)desc + NST * 64);
  const char** const rows = (const char**)(sh + 20);  // [2][K, V][TP] addresses of a tile's rows (null: not there)

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const PagedView& c = P.c;
  pdl_enter();

  // ---- this CTA's range of tiles
  const Cut cut = locate<AT_THREADS, TP, ROWS>(P, sh, [](const Cut& k) { return k.begin(blockIdx.x); });
  if ((int64_t)blockIdx.x >= cut.ctas) return;
  int64_t left = cut.begin(blockIdx.x + 1) - cut.begin(blockIdx.x);
  __syncthreads();

  constexpr int AHEAD = L::AHEAD, FULL = L::FULL, EMPTY = L::EMPTY;
  constexpr int FULL_THREADS = L::FULL_THREADS, EMPTY_THREADS = L::EMPTY_THREADS, AHEAD_THREADS = L::AHEAD_THREADS;
  constexpr int LANES = CPR < 32 ? CPR : 32;  // lanes of a row
  constexpr int RPI = 32 / LANES;             // rows of one warp-wide copy
  constexpr int CPL = CPR / LANES;            // chunks of a row for a lane
  const int my_row = lane / LANES, my_chunk = lane % LANES;
  volatile int* const plan = (volatile int*)(sh + 18);  // [2] rows to copy of a tile, + ALL_THERE, or DONE
  constexpr int ALL_THERE = 256, DONE = -1, NOTHING = -2;
  // Copiers: before the next tile is waited for, the oldest one in flight is handed
  // to the consumers.
  auto hand_over = [&](int tile) {
    if (tile >= NST - 1) {
      cp_wait<NST - 2>();
      bar_arrive<FULL_THREADS>(FULL + (tile + 1) % NST);
    }
  };
  auto drain = [&](int tiles) {  // what is left of that after `tiles` tiles
    for (int k = NST - 3; k >= 0; --k) {
      if (tiles - 1 - k < 0) continue;
      if (k == 0) cp_wait<0>();
      else cp_wait<1>();
      bar_arrive<FULL_THREADS>(FULL + (tiles - 1 - k) % NST);
    }
  };

  if (warp > AT_CONSUMERS / 32) {
    // ========================================== copiers: K rows; V rows and queries
    const bool is_v = warp == AT_CONSUMERS / 32 + 2;
    for (int tile = 0;; ++tile) {
      hand_over(tile);
      bar_sync<AHEAD_THREADS>(AHEAD);  // the tile's rows are listed and its stage is free, or all is done
      const int what = plan[tile & 1];
      if (what < 0) {
        if (what == NOTHING) bar_arrive<FULL_THREADS>(FULL);
        drain(tile);
        return;
      }
      const uint32_t dst = smem_u32(ring + (tile % NST) * L::STAGE) + (is_v ? L::KB : 0);
      const char* const* const of = rows + ((tile & 1) * 2 + is_v) * TP;
      // eight rows' addresses are fetched before their copies are issued: the
      // warp's time goes to issue, not to the latency of each row's address
      constexpr int BATCH = 8;
      static_assert(TP % (BATCH * RPI) == 0, "whole batches");
      auto copy = [&](auto all, auto swizzle) {
        const int n = what & 255;
#pragma unroll 1
        for (int r0 = 0; r0 < n; r0 += BATCH * RPI) {
          const char* o[BATCH];
#pragma unroll
          for (int i = 0; i < BATCH; ++i) o[i] = of[r0 + i * RPI + my_row];
#pragma unroll
          for (int i = 0; i < BATCH; ++i) {
            const int rr = i * RPI + my_row;  // r0 is a multiple of 8: equal swizzles
            const bool ok = decltype(all)::value || o[i] != nullptr;
#pragma unroll
            for (int e = 0; e < CPL; ++e) {
              const int ch = my_chunk + e * LANES;
              cp16(dst + (r0 + rr) * RB + swizzle(ch, rr) * 16, ok ? o[i] + ch * 16 : P.q, ok ? 16 : 0);
            }
          }
        }
      };
      auto k_swz = [](int ch, int r) { return swz<CPR>(ch, r); };
      auto v_swz = [](int ch, int r) { return swz_v<T, CPR>(ch, r); };
      if constexpr (L::ES == 2) {  // the same for both
        if (what & ALL_THERE) copy(std::true_type(), k_swz);
        else copy(std::false_type(), k_swz);
      } else if (is_v) {
        copy(std::false_type(), v_swz);
      } else {
        copy(std::false_type(), k_swz);
      }
      if (is_v) {
        const TileDesc& d = *(const TileDesc*)((char*)desc + (tile % NST) * 64);
        if (d.flags & T_FIRST) {  // rows past nrows stay what they are: nothing of them is kept
          const uint32_t qd = smem_u32(ring + d.qslot * L::STAGE + 2 * L::KB);
          const char* const base = P.q + (int64_t)(d.first + d.q0) * P.q_tok + (int64_t)(d.head * P.group) * P.q_head;
          for (int r = my_row; r < d.nrows; r += RPI) {
            const int dq = div_group(P, r + d.g0);
            const char* const src = base + dq * P.q_tok + (r + d.g0 - dq * P.group) * P.q_head;
#pragma unroll
            for (int e = 0; e < CPL; ++e) {
              const int ch = my_chunk + e * LANES;
              cp16(qd + r * RB + swz<CPR>(ch, r) * 16, src + ch * 16, 16);
            }
          }
        }
      }
      cp_commit();
    }
  }
  if (warp == AT_CONSUMERS / 32) {
    // =============================================================== scheduler
    // Two tiles are on their way: one whose pages are known by now, one whose page
    // numbers have just been asked for; and the sequence behind the cursor's.
    struct Look {
      TileDesc d;
      int page[TP / 32], in_page[TP / 32];
    };
    int b = (int)sh[8];  // cursor: sequence, segment of it (head, row tile), tile of that
    SeqPlan sp;
    sp.load(P, b, TP, ROWS);
    const int64_t off = sh[9];
    if (off < 0 || off >= sp.segments(c.nkv) * cut.slots(sp.units)) left = 0;  // lengths that change under the kernel
    int seg = 0, at = 0, qslot = -1;
    if (left) {
      seg = (int)div_small(off, cut.slots(sp.units));
      const int64_t in = off - seg * cut.slots(sp.units) - cut.extra;  // -1: the slot in front
      at = in < 0 ? -1 : (int)in / cut.scale;
      if (in > 0 && in % cut.scale) {  // the middle of a tile that the CTA before has
        ++at;
        --left;
      }
    }
    int head = sp.tiles ? seg / sp.tiles : 0, row_tile = seg - head * sp.tiles;
    bool fresh = true;    // the next tile is the first of its piece
    bool piece0 = false;  // whether the piece starts its segment
    int then_first, then_n, then_len;
    auto peek = [&]() {  // the sequence after b, asked for early
      if (b + 1 >= c.num_seqs) return;
      seq_rows(c, b + 1, then_first, then_n);
      then_len = seq_len(c, b + 1);
    };
    peek();
    auto next = [&](Look& k) -> bool {  // the cursor's next tile; starts its page lookup
      if (left <= 0) return false;
      if (at >= sp.units) {
        at = -cut.extra;
        fresh = true;
        if (++row_tile >= sp.tiles) {
          row_tile = 0;
          if (++head >= c.nkv) {
            head = 0;
            do {
              if (++b >= c.num_seqs) {
                left = 0;
                return false;
              }
              sp.make(P, then_first, then_n, then_len, TP, ROWS);
              peek();
            } while (sp.tiles == 0);
          }
        }
      }
      if (at < 0) {
        at = 0;
        if (--left <= 0) return false;
      }
      if (fresh) {
        qslot = qslot + 1 == NST ? 0 : qslot + 1;
        piece0 = at == 0;
      }
      TileDesc& d = k.d;
      const int row0 = row_tile * ROWS;
      d.head = head;
      d.q0 = row0 ? row0 / P.group : 0;
      d.g0 = row0 - d.q0 * P.group;
      d.nrows = min(sp.rows - row0, ROWS);
      d.pos0 = sp.lo + at * TP;
      d.npos = max(min(TP, sp.hi - d.pos0), 0);
      d.qslot = qslot;
      d.first = sp.first;
      d.count = sp.count;
      d.p0 = sp.p0;
      d.flags = (fresh ? T_FIRST : 0) | (piece0 ? T_FROM0 : 0);
      ++at;
      left -= cut.scale;
      if (at == sp.units) d.flags |= T_LAST | T_TOEND;
      if (left <= 0) d.flags |= T_LAST;
      // every row sees every position, were all pages there
      if (d.npos == TP && d.pos0 + TP - 1 <= d.p0 && (P.window < 0 || d.pos0 >= d.p0 + d.count - 1 - P.window))
        d.flags |= T_FULL;
      fresh = false;
#pragma unroll
      for (int i = 0; i < TP / 32; ++i) {
        const int j = d.pos0 + i * 32 + lane;
        k.page[i] = -1;
        k.in_page[i] = 0;
        if (i * 32 + lane < d.npos) {
          const int slot = c.page_shift >= 0 ? j >> c.page_shift : j / c.page_size;
          k.page[i] = c.table[(int64_t)b * c.table_stride + slot];
          k.in_page[i] = j - slot * c.page_size;
        }
      }
      return true;
    };

    int tile = 0;
    Look now, then;
    bool have = next(now);
    if (!have) {  // no tile's first slot is in the range: a tile of nothing ends the consumers
      if (lane == 0) {
        *(TileDesc*)desc = TileDesc{0, 0, 0, 0, 0, 0, T_FIRST | T_END, 0, 0, 0, 0, {0u, 0u}};
        plan[0] = NOTHING;
      }
      bar_arrive<AHEAD_THREADS>(AHEAD);
      return;
    }
    while (have) {
      have = next(then);
      const int slot = tile % NST;
      TileDesc& nd = now.d;
      if (!have) nd.flags |= T_END;
      bool all = true;
      const char *const kh = c.k + nd.head * c.k_head, *const vh = c.v + nd.head * c.v_head;
#pragma unroll
      for (int i = 0; i < TP / 32; ++i) {
        const bool ok = (unsigned)now.page[i] < (unsigned)c.num_pages;
        const char** const to = rows + (tile & 1) * 2 * TP + i * 32 + lane;
        to[0] = ok ? kh + now.page[i] * c.k_page + now.in_page[i] * c.k_row : nullptr;
        to[TP] = ok ? vh + now.page[i] * c.v_page + now.in_page[i] * c.v_row : nullptr;
        nd.mask[i] = __ballot_sync(0xffffffffu, ok);
        all = all && nd.mask[i] == 0xffffffffu;
      }
      if (tile >= NST) bar_sync<EMPTY_THREADS>(EMPTY + slot);
      if (lane == 0) {
        *(TileDesc*)((char*)desc + slot * 64) = nd;
        // whole halves of 32 rows: what the consumers look at
        plan[tile & 1] = all ? TP | ALL_THERE : min((nd.npos + 31) & ~31, TP);
      }
      bar_sync<AHEAD_THREADS>(AHEAD);
      now = then;
      ++tile;
    }
    if (lane == 0) plan[tile & 1] = DONE;
    bar_arrive<AHEAD_THREADS>(AHEAD);
    // no arrival is left over
    for (int k = max(tile - NST, 0); k < tile - 1; ++k) bar_sync<EMPTY_THREADS>(EMPTY + k % NST);
    return;
  }

  if constexpr (L::SIMT) consume_simt<HD, NR>(P, ring, p_own, wmax, wsum, desc, warp, lane);
  else consume_mma<T, HD, NR>(P, ring, p_own, wmax, wsum, desc, warp, lane);
}

// Adds up the partials of the segment that starts in CTA blockIdx.x and is cut
// by its end: one row of it per blockIdx.y.  Which that is follows from the
// lengths, as in the kernel before, and is found while that one runs; then one
// round trip to memory brings statistics and values together (the first PRE
// partials of a group of lanes are fetched before their weights are known).
template <typename T, int HD, int ROWS, int TP>
__global__ void __launch_bounds__(AT_JOIN_THREADS) paged_attn_join_kernel(const __grid_constant__ PagedAttnParams P) {
  constexpr int LANES = HD / 4, GROUPS = AT_JOIN_THREADS / LANES, PRE = 4;
  __shared__ float4 sums[GROUPS][LANES];
  __shared__ int64_t sh[20];
  const int tid = threadIdx.x, r = blockIdx.y, lane = tid % LANES, grp = tid / LANES;
  // the kernel before waited for everything that these lengths come from
  const Cut cut = locate<AT_JOIN_THREADS, TP, ROWS>(P, sh, [](const Cut& k) { return k.begin(blockIdx.x + 1) - 1; });
  __syncthreads();
  SeqPlan sp;
  int n = 0, head = 0, row = 0;
  if ((int64_t)blockIdx.x < cut.ctas && sh[9] >= 0) {
    const int64_t end = cut.begin(blockIdx.x + 1), off = sh[9];  // the range's last slot
    sp.load(P, (int)sh[8], TP, ROWS);
    const int64_t slots = cut.slots(sp.units), seg = div_small(off, slots), base = end - 1 - (off - seg * slots);
    const int64_t from = base + cut.extra, to = base + slots - cut.scale;  // its first and last tile's first slots
    if (from >= cut.begin(blockIdx.x) && from < end && to >= end)
      n = (int)(min(cut.owner(to), cut.ctas - 1) - blockIdx.x + 1);
    head = (int)div_small(seg, max(sp.tiles, 1));
    row = (int)(seg - (int64_t)head * sp.tiles) * ROWS + r;
  }
  pdl_enter();
  if (n < 1 || row >= sp.rows || head >= P.c.nkv) return;
  // partial i: slot 1 of this CTA, then slot 0 of the ones behind it
  auto part = [&](int i) { return P.part + ((int64_t)(blockIdx.x + i) * 2 + (i == 0)) * slot_floats(ROWS, HD); };
  auto stat = [&](int i) { return *(const float2*)(part(i) + ROWS * HD + r * 2); };
  float4 pre[PRE];
  float pre_m[PRE];
#pragma unroll
  for (int k = 0; k < PRE; ++k)
    if (grp + k * GROUPS < n) {
      pre[k] = *(const float4*)(part(grp + k * GROUPS) + r * HD + lane * 4);
      pre_m[k] = stat(grp + k * GROUPS).x;
    }
  // every warp finds the same maximum and sum
  float m = -INFINITY, l = 0.f;
  auto join = [&](float m2, float l2) {
    const float M = fmaxf(m, m2), base = M == -INFINITY ? 0.f : M;
    l = l * ex2(m - base) + l2 * ex2(m2 - base);
    m = M;
  };
#pragma unroll 4
  for (int i = tid & 31; i < n; i += 32) {
    const float2 s = stat(i);
    join(s.x, s.y);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) join(__shfl_xor_sync(0xffffffffu, m, o), __shfl_xor_sync(0xffffffffu, l, o));
  const float base = m == -INFINITY ? 0.f : m;
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
  auto add = [&](float m2, const float4& v) {
    const float w = ex2(m2 - base);
    a.x += w * v.x;
    a.y += w * v.y;
    a.z += w * v.z;
    a.w += w * v.w;
  };
#pragma unroll
  for (int k = 0; k < PRE; ++k)
    if (grp + k * GROUPS < n) add(pre_m[k], pre[k]);
#pragma unroll 4
  for (int i = grp + PRE * GROUPS; i < n; i += GROUPS) add(stat(i).x, *(const float4*)(part(i) + r * HD + lane * 4));
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
  const float inv = l == 0.f ? 0.f : __fdividef(1.f, l);
  const int qi = row / P.group;
  char* o = P.out + (int64_t)(sp.first + qi) * P.o_tok + (int64_t)(head * P.group + row - qi * P.group) * P.o_head;
  if (sizeof(T) == 4 || P.out_f32) {
    ((float4*)o)[lane] = make_float4(a.x * inv, a.y * inv, a.z * inv, a.w * inv);
  } else if constexpr (sizeof(T) == 2) {
    ((uint2*)o)[lane] = make_uint2(pack2<T>(a.x * inv, a.y * inv), pack2<T>(a.z * inv, a.w * inv));
  }
}

// ------------------------------------------------------------------- host
// Row tiles of 8, 16 or 32 rows: the smallest that holds a sequence's rows for one
// KV head.  More rows than 32 take several tiles, each reading K and V again, from
// L2: 64 at a time, with their spills and fewer CTAs, measured 264 against 157 us
// (64 rows, head_dim 256), 124 against 108 (128) and 90 against 76 (32).
// f32 with at most four rows: 1, 2 or 4 of them on the FMA units (a negative
// count).
template <typename T>
int pick_nr(const PagedAttnParams& p) {
  const int64_t rows = (int64_t)p.max_rows * p.group;
  if (sizeof(T) == 4 && rows <= 4) return rows <= 1 ? -1 : rows <= 2 ? -2 : -4;
  return rows <= 8 ? 1 : rows <= 16 ? 2 : 4;
}

// One tile at most in any segment: none is cut, and nothing needs joining.
template <typename T, int HD, int NR>
bool uncut(const PagedAttnParams& p) {
  int64_t span = (int64_t)p.c.pages_per_seq * p.c.page_size;
  if (p.window >= 0) span = std::min(span, p.window + p.max_rows);
  return span <= Tile<T, HD, NR>::TP;
}

template <typename T, int HD, int NR>
int64_t workspace_nr(const PagedAttnParams& p) {
  if (uncut<T, HD, NR>(p)) return 0;
  const int64_t ctas = (int64_t)device_sm_count() * Tile<T, HD, NR>::CTAS;
  return ctas * 2 * slot_floats(Tile<T, HD, NR>::ROWS, HD) * 4;
}

template <typename T, int HD, int NR>
void launch_nr(PagedAttnParams p, cudaStream_t s) {
  using L = Tile<T, HD, NR>;
  const int ctas = device_sm_count() * L::CTAS;
  const bool cut = !uncut<T, HD, NR>(p);
  p.mul = p.softcap > 0.f ? p.scale / p.softcap : p.scale * 1.4426950408889634f;
  p.cap2 = p.softcap * 1.4426950408889634f;
  p.group_mul = p.group > 1 ? (uint32_t)((((uint64_t)1 << 32) + p.group - 1) / p.group) : 0;
  ensure_smem_optin((const void*)paged_attn_kernel<T, HD, NR>, L::SMEM);
  launch_k(paged_attn_kernel<T, HD, NR>, dim3(ctas), L::THREADS, L::SMEM, s, 1, p);
  if (cut) {
    const int rows = (int)std::min<int64_t>((int64_t)p.max_rows * p.group, L::ROWS);
    launch_k(paged_attn_join_kernel<T, HD, L::ROWS, L::TP>, dim3(ctas, rows), AT_JOIN_THREADS, 0, s, 1, p);
  }
}

template <typename T, int HD, class F>
auto with_nr(const PagedAttnParams& p, F f) {
  const int nr = pick_nr<T>(p);
  if constexpr (sizeof(T) == 4) {
    if (nr == -1) return f(std::integral_constant<int, -1>());
    if (nr == -2) return f(std::integral_constant<int, -2>());
    if (nr == -4) return f(std::integral_constant<int, -4>());
  }
  switch (nr) {
    case 1: return f(std::integral_constant<int, 1>());
    case 2: return f(std::integral_constant<int, 2>());
    default: return f(std::integral_constant<int, 4>());
  }
}
template <typename T, class F>
auto with_hd(const PagedAttnParams& p, F f) {
  switch (p.hd) {
    case 32: return with_nr<T, 32>(p, [&](auto nr) { return f(std::integral_constant<int, 32>(), nr); });
    case 64: return with_nr<T, 64>(p, [&](auto nr) { return f(std::integral_constant<int, 64>(), nr); });
    case 128: return with_nr<T, 128>(p, [&](auto nr) { return f(std::integral_constant<int, 128>(), nr); });
    default: return with_nr<T, 256>(p, [&](auto nr) { return f(std::integral_constant<int, 256>(), nr); });
  }
}

template <typename T>
int64_t attention_workspace_of(const PagedAttnParams& p) {
  return with_hd<T>(p, [&](auto hd, auto nr) { return workspace_nr<T, decltype(hd)::value, decltype(nr)::value>(p); });
}
template <typename T>
void launch_attention_of(const PagedAttnParams& p, cudaStream_t s) {
  with_hd<T>(p, [&](auto hd, auto nr) { launch_nr<T, decltype(hd)::value, decltype(nr)::value>(p, s); });
}

}  // namespace
}  // namespace cljxla
