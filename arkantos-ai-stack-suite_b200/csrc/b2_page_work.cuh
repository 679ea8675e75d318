// How the page attention kernels divide their work.
//
// The rows of one kv head and sequence are its new tokens times the G query
// heads that share the kv head (row r: token r / G, head r % G), cut into
// tiles of R rows.  A tile attends to positions [lo, hi) of its sequence, in
// units of BK positions.  All units of a call, in the order (kv head,
// sequence, tile, unit), are dealt out in equal consecutive runs to the CTAs
// of one wave: a ragged batch, a single long sequence and a triangular prompt
// all fill the machine, with no plan made on the host, so lengths may live on
// the device and a call can be captured.  A tile whose units fall to several
// CTAs is finished by a second kernel from their partial results (fp32
// weighted sums, maximum and sum of each row), always in unit order, so the
// result does not depend on timing.
#pragma once

#include "b2_common.cuh"
#include "b2_pages.hpp"

namespace b2 {

// Division by a number fixed for a call, for 0 <= n < 2^31: the product with
// floor(2^(31 + l) / d) + 1, l = ceil(log2 d), shifted (exact for 31-bit n).
// The kernels divide row numbers by G at every change of tiles, and the code
// of a general division is fetched cold there.
struct FastDiv {
  uint32_t d = 1, magic = 0, shift = 0;
  __host__ static FastDiv of(uint32_t d) {
    FastDiv f;
    f.d = d;
    if (d > 1) {
      uint32_t l = 0;
      while ((1u << l) < d) ++l;
      f.magic = (uint32_t)(((uint64_t)1 << (31 + l)) / d + 1);
      f.shift = l - 1;
    }
    return f;
  }
  __device__ __forceinline__ int div(int n) const { return magic ? (int)(__umulhi((uint32_t)n, magic) >> shift) : n; }
};

struct PageWork {
  PageSeqs b;
  FastDiv G;                                     // query heads of a kv head
  int ps_log2, n_kv, window, rows_log2, bk_log2;   // rows of a tile, positions of a unit
  __host__ __device__ int rows() const { return 1 << rows_log2; }
  __host__ __device__ int bk() const { return 1 << bk_log2; }
};

struct TileAt {
  int h, s, t;        // kv head, sequence, tile
  int rows_total;     // rows of the sequence
  int first, q0;      // position and token row of the sequence's first new token
  int lo_unit;        // first unit (of bk positions) the tile attends to
  int units;          // at least 1: a tile with nothing to see still writes zeros
  int lo, hi;         // its positions
};

__device__ __forceinline__ int tiles_of(const PageWork& w, const SeqSpan& sp) {
  return (sp.len * (int)w.G.d + w.rows() - 1) >> w.rows_log2;
}

__device__ __forceinline__ void tile_range(const PageWork& w, const SeqSpan& sp, int t, TileAt& a) {
  const int total = sp.len * (int)w.G.d;
  const int last = min((t + 1) << w.rows_log2, total) - 1;
  const int p_lo = sp.first + w.G.div(t << w.rows_log2), p_hi = sp.first + w.G.div(last);
  const int lo = w.window > 0 ? max(0, p_lo - w.window + 1) : 0;
  const int hi = max(0, min(p_hi + 1, sp.kv));
  a.lo_unit = lo >> w.bk_log2;
  a.units = max(1, ((hi + w.bk() - 1) >> w.bk_log2) - a.lo_unit);
  a.lo = lo;
  a.hi = hi;
}

__device__ __forceinline__ void tile_load(const PageWork& w, TileAt& a) {
  const SeqSpan sp = seq_span(w.b, w.ps_log2, a.s);
  a.rows_total = sp.len * (int)w.G.d;
  a.first = sp.first;
  a.q0 = sp.q0;
  tile_range(w, sp, a.t, a);
}

// How the units of a call fall to its CTAs: n CTAs get work, the first `rem`
// of them base + 1 units, the others base.  Fewer than 2^31 units.
struct Deal {
  int n, base, rem;
  __device__ __forceinline__ int start(int cta) const { return cta * base + min(cta, rem); }
  // the CTA that holds unit u
  __device__ __forceinline__ int cta_of(int u) const {
    const int cut = rem * (base + 1);
    return u < cut ? (int)((unsigned)u / (unsigned)(base + 1)) : rem + (int)((unsigned)(u - cut) / (unsigned)base);
  }
};

// The share of the calling CTA: units [u, u_end), the first of them `off`
// units into tile `at`.
struct Share {
  Deal deal;
  int u, u_end;
  int off;
  TileAt at;
};

// Block-wide: the units of every sequence (for one kv head) into sums, shared
// memory of n_seq ints.  A barrier must follow.
__device__ __forceinline__ void sum_units(const PageWork& w, int* sums) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, warps = blockDim.x >> 5;
  if (w.b.max_q * (int64_t)w.G.d <= w.rows()) {   // one tile at most: a thread per sequence
    for (int s = tid; s < w.b.n_seq; s += blockDim.x) {
      const SeqSpan sp = seq_span(w.b, w.ps_log2, s);
      const int tiles = tiles_of(w, sp);
      int sum = 0;
      for (int t = 0; t < tiles; ++t) {
        TileAt a;
        tile_range(w, sp, t, a);
        sum += a.units;
      }
      sums[s] = sum;
    }
  } else {                           // a warp per sequence, lanes over its tiles
    for (int s = warp; s < w.b.n_seq; s += warps) {
      const SeqSpan sp = seq_span(w.b, w.ps_log2, s);
      const int tiles = tiles_of(w, sp);
      int sum = 0;
      for (int t = lane; t < tiles; t += 32) {
        TileAt a;
        tile_range(w, sp, t, a);
        sum += a.units;
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if (lane == 0) sums[s] = sum;
    }
  }
}

// Warp-wide, from the sums: the share of CTA `cta` of `ctas`.  Returns false
// for a CTA without work.
__device__ __forceinline__ bool find_share(const PageWork& w, int cta, int ctas, const int* sums, Share& sh) {
  const int lane = threadIdx.x & 31;
  int per_head = 0;
  for (int s0 = 0; s0 < w.b.n_seq; s0 += 32) {
    int v = s0 + lane < w.b.n_seq ? sums[s0 + lane] : 0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    per_head += v;
  }
  const int total = per_head * w.n_kv;
  sh.deal.n = min(total, ctas);
  if (cta >= sh.deal.n) return false;
  sh.deal.base = (int)((unsigned)total / (unsigned)sh.deal.n);
  sh.deal.rem = total - sh.deal.base * sh.deal.n;
  sh.u = sh.deal.start(cta);
  sh.u_end = sh.deal.start(cta + 1);
  sh.at.h = (int)((unsigned)sh.u / (unsigned)per_head);
  int rem = sh.u - sh.at.h * per_head;
  sh.at.s = -1;
  for (int s0 = 0; s0 < w.b.n_seq; s0 += 32) {
    const int v = s0 + lane < w.b.n_seq ? sums[s0 + lane] : 0;
    int run = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, run, o);
      if (lane >= o) run += u;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, rem < run);
    if (hit) {
      const int at = __ffs(hit) - 1;
      sh.at.s = s0 + at;
      rem -= __shfl_sync(0xffffffffu, run - v, at);
      break;
    }
    rem -= __shfl_sync(0xffffffffu, run, 31);
  }
  const SeqSpan sp = seq_span(w.b, w.ps_log2, sh.at.s);
  const int tiles = tiles_of(w, sp);
  for (int t0 = 0; t0 < tiles; t0 += 32) {
    TileAt a;
    a.units = 0;
    if (t0 + lane < tiles) tile_range(w, sp, t0 + lane, a);
    int run = a.units;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, run, o);
      if (lane >= o) run += u;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, rem < run);
    if (hit) {
      const int at = __ffs(hit) - 1;
      sh.at.t = t0 + at;
      rem -= __shfl_sync(0xffffffffu, run - a.units, at);
      break;
    }
    rem -= __shfl_sync(0xffffffffu, run, 31);
  }
  sh.off = rem;
  tile_load(w, sh.at);
  return true;
}

// The tile after `a` (which has a successor: the caller has units left).
__device__ __forceinline__ void next_tile(const PageWork& w, TileAt& a) {
  if ((a.t + 1) << w.rows_log2 < a.rows_total) {
    ++a.t;
  } else {
    a.t = 0;
    do {
      if (++a.s == w.b.n_seq) {
        a.s = 0;
        ++a.h;
      }
      const SeqSpan sp = seq_span(w.b, w.ps_log2, a.s);
      if (sp.len > 0) break;
    } while (true);
  }
  tile_load(w, a);
}

// What the finishing kernel needs about the tile that starts in a CTA's share
// and runs past its end (at most one per CTA): its rows, the CTA that ends it
// and the slot of its first partial result.  A CTA's other partial result,
// the rest of a tile that began before it, is in slot 2·cta.
struct SplitTile {
  int32_t h, s, t, last, slot, rows, q0, pad;
};

// Workspace: [ctas] SplitTile, then 2·ctas slots of rows · (hd + 2) floats
// (the weighted sums of all rows, then (maximum, sum) of each).
__host__ __device__ inline size_t split_bytes(int ctas) { return (size_t)ctas * sizeof(SplitTile); }
__host__ __device__ inline size_t slot_floats(int rows, int hd) { return (size_t)rows * (hd + 2); }

// Most CTAs an attention kernel is launched with (the workspace has room for them).
constexpr int kPageMaxCtasPerSm = 4;

// Finishes the tiles that were split over CTAs (b2_page_attn.cu).
int launch_page_join(const PageWork& w, const SplitTile* split, const float* slots, int ctas, int hd, int n_head,
                     void* out, bool out_f32, cudaStream_t s);

}  // namespace b2
