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

struct PageWork {
  PageSeqs b;
  int ps_log2, n_kv, G, window, rows, bk;   // rows of a tile, positions of a unit
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
  return (sp.len * w.G + w.rows - 1) / w.rows;
}

__device__ __forceinline__ void tile_range(const PageWork& w, const SeqSpan& sp, int t, TileAt& a) {
  const int total = sp.len * w.G;
  const int last = min((t + 1) * w.rows, total) - 1;
  const int p_lo = sp.first + (t * w.rows) / w.G, p_hi = sp.first + last / w.G;
  const int lo = w.window > 0 ? max(0, p_lo - w.window + 1) : 0;
  const int hi = max(0, min(p_hi + 1, sp.kv));
  a.lo_unit = lo / w.bk;
  a.units = max(1, (hi + w.bk - 1) / w.bk - a.lo_unit);
  a.lo = lo;
  a.hi = hi;
}

__device__ __forceinline__ void tile_load(const PageWork& w, TileAt& a) {
  const SeqSpan sp = seq_span(w.b, w.ps_log2, a.s);
  a.rows_total = sp.len * w.G;
  a.first = sp.first;
  a.q0 = sp.q0;
  tile_range(w, sp, a.t, a);
}

// The share of the calling CTA: units [u, u_end), the first of them `off`
// units into tile `at`.  n is the number of CTAs that got work; total the
// units of the call.
struct Share {
  int64_t u, u_end, total;
  int n;
  int off;
  TileAt at;
};

// Block-wide: the units of every sequence (for one kv head) into sums, shared
// memory of n_seq ints.  A barrier must follow.
__device__ __forceinline__ void sum_units(const PageWork& w, int* sums) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, warps = blockDim.x >> 5;
  if (w.b.max_q * w.G <= w.rows) {   // one tile at most: a thread per sequence
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
  int64_t per_head = 0;
  for (int s0 = 0; s0 < w.b.n_seq; s0 += 32) {
    int v = s0 + lane < w.b.n_seq ? sums[s0 + lane] : 0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    per_head += v;
  }
  sh.total = per_head * w.n_kv;
  sh.n = (int)(sh.total < ctas ? sh.total : ctas);
  if (cta >= sh.n) return false;
  sh.u = sh.total * cta / sh.n;
  sh.u_end = sh.total * (cta + 1) / sh.n;
  sh.at.h = (int)(sh.u / per_head);
  int64_t rem = sh.u - sh.at.h * per_head;
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
  sh.off = (int)rem;
  tile_load(w, sh.at);
  return true;
}

// The tile after `a` (which has a successor: the caller has units left).
__device__ __forceinline__ void next_tile(const PageWork& w, TileAt& a) {
  if ((a.t + 1) * w.rows < a.rows_total) {
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

// The CTA that holds unit u: the largest c with floor(total·c / n) <= u.
__device__ __forceinline__ int cta_of_unit(int64_t u, int64_t total, int n) {
  return (int)(((u + 1) * n - 1) / total);
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
