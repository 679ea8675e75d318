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
// CTAs is finished by the last of them from all their partial results (fp32
// weighted sums, maximum and sum of each row), always in unit order, so the
// result does not depend on timing.  (A second kernel for that took 3 us of a
// single token's 13, and 9 us behind a 512-token chunk.)
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
  float join_per_tile;                             // see find_share
  int fair;                                        // units of a sequence that n_seq · n_kv of them keep below 2^31
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

// Whether a call's units are too many to count: the launcher bounds them for
// sequences that divide the tokens, but q_start is the device's, and sequences
// that overlap could pass 2^31.
__device__ __forceinline__ bool too_many_units(const PageWork& w, const int* sums) {
  int64_t total = 0;
  for (int s = 0; s < w.b.n_seq; ++s) total += sums[s];
  return total * w.n_kv >= ((int64_t)1 << 31);
}

// Warp-wide, from the sums: the share of CTA `cta` of `ctas`.  Returns false
// for a CTA without work, and for a batch with more units than can be counted.
// A tile of U units in shares of k takes k units' time and that of joining U/k
// parts; with j the units' time that a part takes to join, k = sqrt(j U) is
// best, U the mean over the tiles (join_per_tile is j over the number of
// tiles), and no CTA gets fewer.
__device__ __forceinline__ bool find_share(const PageWork& w, int cta, int ctas, const int* sums, Share& sh) {
  const int lane = threadIdx.x & 31;
  int per_head = 0;
  bool more = false;
  for (int s0 = 0; s0 < w.b.n_seq; s0 += 32) {
    int v = s0 + lane < w.b.n_seq ? sums[s0 + lane] : 0;
    more = more || v > w.fair;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    per_head += v;
  }
  if (__any_sync(0xffffffffu, more) && too_many_units(w, sums)) return false;
  const int total = per_head * w.n_kv;
  const int least = max(1, (int)ceilf(sqrtf(w.join_per_tile * (float)total)));
  sh.deal.n = min((int)((unsigned)(total + least - 1) / (unsigned)least), ctas);
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

// How a tile that is split over CTAs is put together: its parts come from n
// CTAs beginning with cta0, the first one's partial result in slot0, the
// others' in slot 2·cta.  A CTA has two slots, one for the rest of a tile that
// began before its share or with it, one for a tile that runs past its end.
struct Split {
  int cta0, n, slot0, slot;   // n = 0: the tile is not split
};
__device__ __forceinline__ Split split_of(const Share& sh, int cta, int u_hi) {
  Split p = {0, 0, 0, 0};
  if (sh.off == 0 && u_hi == sh.at.units) return p;
  const int start = sh.u - sh.off;   // the tile's first unit among all
  p.cta0 = sh.deal.cta_of(start);
  p.n = sh.deal.cta_of(start + sh.at.units - 1) - p.cta0 + 1;
  p.slot0 = 2 * p.cta0 + (sh.deal.start(p.cta0) == start ? 0 : 1);
  p.slot = cta == p.cta0 ? p.slot0 : 2 * cta;
  return p;
}

// Workspace: counters of the parts that have arrived, 8 a CTA (by the CTA that
// begins a tile; a warp of the tile each), zero between calls; then two slots
// a CTA of rows · (hd + 2) floats (the weighted sums of all rows, then
// (maximum, sum) of each).
constexpr int kPageMaxCtasPerSm = 4;   // most CTAs an attention kernel is launched with
__host__ __device__ inline size_t counter_bytes(int ctas) { return (size_t)ctas * 32; }
__host__ __device__ inline size_t slot_floats(int rows, int hd) { return (size_t)rows * (hd + 2); }

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Whether the calling warp's part is the last of its n: the parts' rows are
// then visible to it.  All lanes have written theirs; the counter is left at
// zero.
__device__ __forceinline__ bool part_arrives(unsigned* counter, int n) {
  __threadfence();
  __syncwarp();
  unsigned last = 0;
  if ((threadIdx.x & 31) == 0) {
    last = atomicAdd(counter, 1u) == (unsigned)(n - 1);
    if (last) *counter = 0;
    __threadfence();
  }
  return __shfl_sync(0xffffffffu, last, 0) != 0;
}

// HD/32 values of a row and lane, from a partial result and to the output.
template <int V>
__device__ __forceinline__ void load_part(const float* src, float (&x)[V]) {
  if constexpr (V == 4) {
    const float4 f = __ldcg(reinterpret_cast<const float4*>(src));
    x[0] = f.x, x[1] = f.y, x[2] = f.z, x[3] = f.w;
  } else if constexpr (V == 2) {
    const float2 f = __ldcg(reinterpret_cast<const float2*>(src));
    x[0] = f.x, x[1] = f.y;
  } else {
#pragma unroll
    for (int v = 0; v < V; ++v) x[v] = __ldcg(src + v);
  }
}
template <int V>
__device__ __forceinline__ void store_joined(void* out, bool f32, int64_t at, const float (&x)[V], float inv) {
  if (f32) {
    float* d = static_cast<float*>(out) + at;
    if constexpr (V == 4) {
      *reinterpret_cast<float4*>(d) = make_float4(x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv);
    } else {
#pragma unroll
      for (int v = 0; v < V; ++v) d[v] = x[v] * inv;
    }
  } else {
    __half* d = static_cast<__half*>(out) + at;
    if constexpr (V % 2 == 0) {
#pragma unroll
      for (int v = 0; v < V; v += 2) *reinterpret_cast<__half2*>(d + v) = __floats2half2_rn(x[v] * inv, x[v + 1] * inv);
    } else {
#pragma unroll
      for (int v = 0; v < V; ++v) d[v] = __float2half_rn(x[v] * inv);
    }
  }
}
// A part's weight for a row with maximum m and sum l in it: a part that saw
// nothing of the row adds nothing; a sum without a maximum comes from scores
// that are all NaN.  Any other weight stays positive, too small for finite
// values to count, so that an infinite or NaN value of a low score is not lost.
constexpr float kLeastWeight = 1.17549435e-38f;
__device__ __forceinline__ float part_weight(float m, float l, float top) {
  return l == 0.f ? 0.f : m == -INFINITY ? 1.f : fmaxf(ex2(m - top), kLeastWeight);
}

// Rows row .. row + min(R, n_rows) - 1 of a split tile from its parts, by one
// warp: w_i = 2^(m_i − M), the weighted sums added in the CTAs' order and
// divided by the joined sum.  e: where row `row` + lane starts in the output.
//
// Few rows of many parts (a single token's): the weights are formed a lane per
// part, 32 parts at a time, and U parts' rows are loaded at once.
template <int HD, int R, int U>
__device__ __forceinline__ void join_parts(const float* slots, int tile_rows, const Split& p, int row, int n_rows,
                                           int64_t e, void* out, bool f32) {
  constexpr int V = HD / 32;
  const int lane = threadIdx.x & 31;
  const int64_t size = (int64_t)slot_floats(tile_rows, HD);
  auto part = [&](int i) { return slots + (i == 0 ? p.slot0 : 2 * (p.cta0 + i)) * size; };
  auto stat = [&](int i, int r) {   // (maximum, sum) of a row in a part
    const int at = row + min(r, n_rows - 1);
    return i < p.n ? __ldcg(reinterpret_cast<const float2*>(part(i) + tile_rows * HD + 2 * at)) : make_float2(-INFINITY, 0.f);
  };
  float top[R], sum[R], acc[R][V];
  float2 kept[R];   // the first 32 parts'
#pragma unroll
  for (int r = 0; r < R; ++r) {
    kept[r] = stat(lane, r);
    top[r] = kept[r].x;
    sum[r] = 0.f;
#pragma unroll
    for (int v = 0; v < V; ++v) acc[r][v] = 0.f;
  }
  float x[U][R][V];
  auto fetch = [&](int i0) {
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int r = 0; r < R; ++r)
        load_part<V>(part(min(i0 + u, p.n - 1)) + (row + min(r, n_rows - 1)) * HD + lane * V, x[u][r]);
  };
  fetch(0);   // on their way with the statistics
#pragma unroll 1
  for (int i0 = 32; i0 < p.n; i0 += 32) {
#pragma unroll
    for (int r = 0; r < R; ++r) top[r] = fmaxf(top[r], stat(i0 + lane, r).x);
  }
#pragma unroll
  for (int r = 0; r < R; ++r) top[r] = warp_max(top[r]);
#pragma unroll 1
  for (int i0 = 0; i0 < p.n; i0 += 32) {
    float wt[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const float2 ml = i0 == 0 ? kept[r] : stat(i0 + lane, r);
      wt[r] = part_weight(ml.x, ml.y, top[r]);
      sum[r] += wt[r] * ml.y;
    }
    const int m = min(32, p.n - i0);
#pragma unroll 1
    for (int i1 = 0; i1 < m; i1 += U) {
      if (i0 + i1 > 0) fetch(i0 + i1);
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const float wr = i1 + u < m ? __shfl_sync(0xffffffffu, wt[r], i1 + u) : 0.f;
          if (wr != 0.f) {
#pragma unroll
            for (int v = 0; v < V; ++v) acc[r][v] += wr * x[u][r][v];
          }
        }
    }
  }
#pragma unroll
  for (int r = 0; r < R; ++r) {
    sum[r] = warp_sum(sum[r]);
    const int64_t at = __shfl_sync(0xffffffffu, e, r) + lane * V;
    if (r < n_rows) store_joined<V>(out, f32, at, acc[r], sum[r] != 0.f ? 1.f / sum[r] : 0.f);
  }
}

// Many rows of few parts: a lane holds one row's maximum, weight and sum, and
// a part's R rows are loaded at once.
template <int HD, int R>
__device__ __forceinline__ void join_rows(const float* slots, int tile_rows, const Split& p, int row, int n_rows,
                                          int64_t e, void* out, bool f32) {
  constexpr int V = HD / 32;
  const int lane = threadIdx.x & 31, own = row + min(lane, min(R, n_rows) - 1);
  const int64_t size = (int64_t)slot_floats(tile_rows, HD);
  auto part = [&](int i) { return slots + (i == 0 ? p.slot0 : 2 * (p.cta0 + i)) * size; };
  float top = -INFINITY;
#pragma unroll 4
  for (int i = 0; i < p.n; ++i) top = fmaxf(top, __ldcg(part(i) + tile_rows * HD + 2 * own));
  float sum = 0.f, acc[R][V];
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int v = 0; v < V; ++v) acc[r][v] = 0.f;
#pragma unroll 1
  for (int i = 0; i < p.n; ++i) {
    const float* q = part(i);
    const float2 ml = __ldcg(reinterpret_cast<const float2*>(q + tile_rows * HD + 2 * own));
    float x[R][V];
#pragma unroll
    for (int r = 0; r < R; ++r) load_part<V>(q + (row + min(r, n_rows - 1)) * HD + lane * V, x[r]);
    const float wt = part_weight(ml.x, ml.y, top);
    sum += wt * ml.y;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const float wr = __shfl_sync(0xffffffffu, wt, r);
      if (wr != 0.f) {
#pragma unroll
        for (int v = 0; v < V; ++v) acc[r][v] += wr * x[r][v];
      }
    }
  }
  const float inv = sum != 0.f ? 1.f / sum : 0.f;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const float ir = __shfl_sync(0xffffffffu, inv, r);
    const int64_t at = __shfl_sync(0xffffffffu, e, r) + lane * V;
    if (r < n_rows) store_joined<V>(out, f32, at, acc[r], ir);
  }
}

}  // namespace b2
