// Attention of few rows over the paged cache: single tokens, short chunks,
// and every cache type and head size (b2_page_rows_*.cu instantiate it).
//
//   o_r = Σ_t e^{s_rt − m_r} v_t / Σ_t e^{s_rt − m_r},   s_rt = scale · q_r·k_t
//
// in one pass over the positions with the running maximum m and sum of each
// row.  What bounds a decode step is the read of K and V; the rows of one kv
// head (its G query heads) share that read, and their products go to the
// tensor pipe through mma.sync m16n8k16: with at most 16 rows per kv head a
// tcgen05 tile of 128 rows would be 90 % padding and its operands would still
// pass through shared memory.
//
// Exactness.  Cache values enter the products exactly: fp16 as they are,
// Q8_0 / Q4_0 as their integer codes in fp16, the block scale applied in fp32
// to K's block sums and to p for V (a row of K or V is never rounded to
// fp16).  In the SPLIT form a tile has 8 rows: rows 0-7 of q's operand hold the
// high fp16 part of q, rows 8-15 the remainder (each row times the scale's
// mantissa and a power of two that brings its largest value near 2^14, so the
// parts are good for any size of q; another power of two makes the scores
// exponents), and the weights, also as two parts, are the 8-column operand of
// O^T = V^T·P^T, which is where the scores' lanes already hold them; so fp32
// queries keep 22 bits and the output is good to fp32 accuracy, with half the
// accumulators that P·V would take.  The FULL form (fp16 queries and outputs)
// rounds p once to fp16, over a quantized V its product with the block scale,
// an error of the size of the fp16 output's.  Accumulators, maxima and sums
// are fp32.
//
// Measured: 32 sequences of 4048 over fp16 pages 91 us, 5.8 TB/s; 16 of 4096
// over Q8_0 54 us, 2.8 TB/s, where the instructions that turn codes into
// operands bound it (issue slots half used, warps waiting on their latency).
//
// Layout.  A unit is 64 positions.  One warp brings K and V through a ring of
// stages that runs on over the tiles of a CTA's share, looking pages up a unit
// ahead: fp16 rows by tensor copies of a page and 64 dims, 128-byte swizzled
// for ldmatrix; quantized rows, whose 16 bytes of scales already put them on
// different banks, by plain bulk copies of a page's run.  (Copies of 16 bytes
// a thread took 150 cycles each to issue, more than the products.)  Table
// entries outside the pool read as zeros; rows past the tile's positions are
// left as they come: K's scores there are masked, V is zeroed before use.
// The other 4 warps compute.  WM = 1: they take 16 positions each of the one
// 16-row operand and their results are joined at the end of a tile; quantized
// rows go from their stored bytes straight into the operands' registers: the
// order of the dims within a block is free in q·k (q is loaded in the same
// order), and for V a byte permute pairs two positions' codes, which fixes the
// dims a lane holds of the result.  WM = 4: each warp has its own
// 16-row operand and runs over all 64 positions; quantized rows are unpacked
// to fp16 codes once for all of them.
#pragma once

#include <atomic>

#include <cuda.h>
#include <cudaTypedefs.h>

#include "b2_page_work.cuh"

namespace b2 {

struct PageRowsArgs {
  PageView c;
  PageWork w;
  const void* q;
  void* out;
  int n_head, q_f32;
  float scale_log2;          // scale · log2(e)
  float q_mul;               // the same as q_mul · 2^c_exp, 1 <= |q_mul| < 2 or 0
  int c_exp;
  FastDiv cpr_k, cpr_v;      // 16-byte chunks of a row
  int64_t pool_rows;
  int* status;
  unsigned* counters;
  float* slots;
};

constexpr int kRowsThreads = 128, kRowsBk = 64, kMaxDevices = 64;   // computing threads, positions of a unit

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool on) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(on ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }
__device__ __forceinline__ void ldsm4(uint32_t a, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(a)
               : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t a, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(a)
               : "memory");
}
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t h2(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
// (lo, hi) as fp16 pairs: the rounded values and what the rounding left.
__device__ __forceinline__ void h2_split(float lo, float hi, uint32_t& head, uint32_t& rest) {
  const __half2 v = __floats2half2_rn(lo, hi);
  const float2 f = __half22float2(v);
  head = *reinterpret_cast<const uint32_t*>(&v);
  rest = h2(lo - f.x, hi - f.y);
}

// The exponent that brings a largest magnitude (as bits; zeros, infinities and
// NaNs too) to [2^13, 2^14), as far as 2^e stays normal.
__device__ __forceinline__ int q_fit(uint32_t bits) { return min(140 - (int)(bits >> 23), 100); }
__device__ __forceinline__ float pow2(int e) { return __int_as_float((e + 127) << 23); }

// Bytes 0-3 of w (signed codes) as four exact fp16 values: a byte b + 128 in
// the low bits of 0x6400 is 1024 + b + 128.
__device__ __forceinline__ void s8x4_to_h2(uint32_t w, uint32_t& a, uint32_t& b) {
  w ^= 0x80808080u;
  const uint32_t x = __byte_perm(w, 0x64646464u, 0x4140), y = __byte_perm(w, 0x64646464u, 0x4342);
  const __half2 off = __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));   // 1152
  const __half2 p = __hsub2(*reinterpret_cast<const __half2*>(&x), off);
  const __half2 q = __hsub2(*reinterpret_cast<const __half2*>(&y), off);
  a = *reinterpret_cast<const uint32_t*>(&p);
  b = *reinterpret_cast<const uint32_t*>(&q);
}

// p is carried times 2^offset so that its fp16 parts stay normal; the sum of
// the weights carries the same factor.  With a quantized V the operand is p·d,
// d the block scale, and the offset is 15 + e, 2^e the power of two that brings
// the largest |d| so far into [1/2, 1): the operand uses fp16's whole range
// whatever the size of V (error of the result for V of size 1e-3 over Q8_0:
// 4.3e-7, with one offset for all sizes 4.5e-5).  When a larger d comes, e falls
// and the sums with it, exactly.
constexpr float kOffset = 10.f, kOffsetQ = 15.f;
constexpr int kFitMost = 23;   // e for the smallest fp16 scale, 2^-24

// An fp16 (or unpacked) operand: [dims / 64][64 rows][128 bytes], 16-byte
// chunk c of row r at c ^ (r % 8).
template <int HD>
struct RowsSmem {
  static constexpr int blocks = (HD + 63) / 64;
  static constexpr int tile = blocks * kRowsBk * 128;
  static constexpr int scales = (HD / 32) * kRowsBk * 4;
  __host__ __device__ static int raw(int rb) { return kRowsBk * rb; }
  // chunk of 8 values of a row
  __device__ static __forceinline__ uint32_t at(int row, int chunk) {
    return (uint32_t)((chunk >> 3) * (kRowsBk * 128) + row * 128 + (((chunk & 7) ^ (row & 7)) << 4));
  }
};
template <int HD, bool KQ, bool VQ>
__host__ __device__ inline int rows_stage_bytes(int rb_k, int rb_v) {
  return (KQ ? RowsSmem<HD>::raw(rb_k) : RowsSmem<HD>::tile) + (VQ ? RowsSmem<HD>::raw(rb_v) : RowsSmem<HD>::tile);
}
template <int HD, bool KQ, bool VQ, int WM>
__host__ __device__ inline int rows_conv_bytes() {
  return WM == 1 ? 0
                 : (KQ ? RowsSmem<HD>::tile + RowsSmem<HD>::scales : 0) + (VQ ? RowsSmem<HD>::tile + RowsSmem<HD>::scales : 0);
}
// CTAs meant for an SM: registers and the ring are cut to fit.  Reading
// quantized rows is bound by the latency of the code's own steps, not by HBM,
// and gains from a third (64 sequences of 4096 over Q8_0: 167 -> 156 us when
// that was measured, 164 now); fp16 rows of head_dim 128 do not (97 us against
// 98 for 32 of them).
template <int HD, bool KQ, bool VQ, bool SPLIT>
__host__ __device__ constexpr int rows_ctas() {
  return HD == 256 ? 1 : HD == 64 || (KQ && VQ && SPLIT) ? 3 : 2;
}
// Room for a tile's queries (WM = 1).
template <int HD, bool SPLIT, int WM>
__host__ __device__ constexpr int rows_q_bytes() {
  return WM == 1 ? (SPLIT ? 8 * HD * 4 : 16 * HD * 2) : 0;
}
constexpr int kRowsStagesMax = 8, kRowsCtrl = 1024;
// SPLIT, warps along the positions: units between two additions, with
// rounding, of the result so far to an fp32 sum.  The tensor pipe cuts a sum at
// each of the unit's two steps; over a share of 512 units that was 3.4e-5 of
// the result, now 1.1e-6.
constexpr int kRowsFlush = 16;
constexpr int kWaitPolls = 1 << 22;   // polls of a wait, each suspended by the hardware for a while

__device__ __forceinline__ void tma_2d(uint32_t dst, const CUtensorMap* map, int x, int y, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(
          dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(x), "r"(y)
      : "memory");
}
__device__ __forceinline__ void fence_async_proxy() {
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}
// The computing warps' barrier, and one that tells whether any thread said so.
__device__ __forceinline__ void bar_compute() { asm volatile("barrier.cta.sync 1, 128;" ::: "memory"); }
__device__ __forceinline__ bool bar_compute_or(int x) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.s32 p, %1, 0;\n\tbarrier.cta.red.or.pred q, 1, 128, p;\n\tselp.u32 %0, 1, 0, q;\n\t}\n"
      : "=r"(r)
      : "r"(x)
      : "memory");
  return r != 0;
}

// Bytes 0-3 of w, 4-bit codes 0..15 (offset 8), as exact fp16 values - 8..7.
__device__ __forceinline__ void n4x4_to_h2(uint32_t w, uint32_t& a, uint32_t& b) {
  const uint32_t x = __byte_perm(w, 0x64646464u, 0x4140), y = __byte_perm(w, 0x64646464u, 0x4342);
  const __half2 off = __halves2half2(__ushort_as_half(0x6408), __ushort_as_half(0x6408));   // 1032
  const __half2 p = __hsub2(*reinterpret_cast<const __half2*>(&x), off);
  const __half2 q = __hsub2(*reinterpret_cast<const __half2*>(&y), off);
  a = *reinterpret_cast<const uint32_t*>(&p);
  b = *reinterpret_cast<const uint32_t*>(&q);
}
// Bytes of two positions' words as (position, next position) pairs of fp16:
// out[t] from byte t of each.  `off`: 1152 for signed codes (their top bits
// flipped before), 1032 for 4-bit ones.
__device__ __forceinline__ void pair_to_h2(uint32_t w0, uint32_t w1, uint32_t off, uint32_t (&out)[4]) {
  const uint32_t lo = __byte_perm(w0, w1, 0x5140), hi = __byte_perm(w0, w1, 0x7362);
  const uint32_t x[4] = {__byte_perm(lo, 0x64646464u, 0x4140), __byte_perm(lo, 0x64646464u, 0x4342),
                         __byte_perm(hi, 0x64646464u, 0x4140), __byte_perm(hi, 0x64646464u, 0x4342)};
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    const __half2 v = __hsub2(*reinterpret_cast<const __half2*>(&x[t]), *reinterpret_cast<const __half2*>(&off));
    out[t] = *reinterpret_cast<const uint32_t*>(&v);
  }
}
// The NB block scales behind a row's codes.
template <int NB>
__device__ __forceinline__ void row_scales(const uint8_t* p, float (&d)[NB]) {
  uint32_t w[(NB + 1) / 2];
  if constexpr (NB == 8) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
  } else if constexpr (NB > 2) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    w[0] = v.x, w[1] = v.y;
  } else {
    w[0] = *reinterpret_cast<const uint32_t*>(p);
  }
#pragma unroll
  for (int b = 0; b < NB; ++b) d[b] = h2f((uint16_t)(w[b / 2] >> (16 * (b & 1))));
}

template <int HD, bool KQ, bool VQ, bool SPLIT, int WM>
__global__ void __launch_bounds__(kRowsThreads + 32, rows_ctas<HD, KQ, VQ, SPLIT>())
    page_rows_kernel(const PageRowsArgs a, int stages, const __grid_constant__ CUtensorMap k_map,
                     const __grid_constant__ CUtensorMap v_map) {
  using L = RowsSmem<HD>;
  constexpr int WK = 4 / WM;                   // warps along the positions
  constexpr int KEYS = kRowsBk / WK;           // positions of a warp in a unit
  constexpr int NC = WM == 1 ? 16 : 32;        // positions per softmax step
  constexpr int NT = NC / 8, KS = HD / 16, NB = HD / 32, OT = SPLIT ? HD / 16 : HD / 8;   // OT: tiles of the result
  constexpr int WROWS = SPLIT ? 8 : 16;        // rows of a warp's operand
  constexpr bool KD = KQ && WM == 1, VD = VQ && WM == 1;   // stored bytes straight into registers
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem);      // [stages]
  uint64_t* empty = full + kRowsStagesMax;                 // [stages]
  uint64_t* t_full = empty + kRowsStagesMax;               // a tile and its queries have come,
  uint64_t* t_empty = t_full + 1;                          // and been taken
  int* abort_flag = reinterpret_cast<int*>(smem + 256);
  int* last_part = abort_flag + 1;
  // [2] by unit (WM = 4): the largest scale of V, as bits, where the offset must fall
  uint32_t* v_top = reinterpret_cast<uint32_t*>(smem + 264);
  TileAt* tile = reinterpret_cast<TileAt*>(smem + 320);
  constexpr int kQRows = rows_q_bytes<HD, SPLIT, WM>();
  uint8_t* q_rows = smem + kRowsCtrl;                      // WM = 1: the tile's queries as they are in q
  uint8_t* ring = q_rows + kQRows;

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid == 0) {
    for (int i = 0; i < stages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 4);
    }
    mbar_init(t_full, 1);
    mbar_init(t_empty, 4);
    *abort_flag = 0;
    v_top[0] = v_top[1] = 0;
    *tile = TileAt{};   // what the warps would read if the first one never came
    tile->units = 1;
    fence_mbar_init();
  }
  if (warp == 4 && lane < 2 && !(lane ? VQ : KQ))
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(lane ? &v_map : &k_map)) : "memory");
  pdl_wait();
  pdl_launch_dependents();

  const int wm = WM == 1 ? 0 : warp, wk = WM == 1 ? warp : 0;
  const int g = lane >> 2, j = lane & 3;
  const PageView& c = a.c;
  const PageWork& w = a.w;
  const int G = (int)w.G.d;

  const int stage_bytes = rows_stage_bytes<HD, KQ, VQ>(c.rb_k, c.rb_v);
  const int k_bytes = KQ ? L::raw(c.rb_k) : L::tile;
  Share sh;
  int* sums = reinterpret_cast<int*>(ring);
  sum_units(w, sums);
  __syncthreads();
  const bool have = find_share(w, blockIdx.x, gridDim.x, sums, sh);   // every warp finds the same place
  if (!have) return;
  __syncthreads();   // the sums are read, the stages take their place

  // A wait; after one in the CTA has expired all others return.
  auto wait = [&](uint64_t* bar, uint32_t parity, int code) -> bool {
    for (int i = 0; !mbar_try_wait(bar, parity); ++i)
      if (i == kWaitPolls || *reinterpret_cast<volatile int*>(abort_flag)) {
        *reinterpret_cast<volatile int*>(abort_flag) = 1;
        if (a.status) atomicExch(a.status, code);
        return false;
      }
    return true;
  };

  if (warp == 4) {
    // ---------------- K and V ----------------
    fence_async_proxy();
    const int n_units = sh.u_end - sh.u;
    const int run_log2 = min(c.ps_log2, 6), run = 1 << run_log2, runs = kRowsBk >> run_log2;   // rows of a copy
    const int nk = KQ ? 1 : L::blocks, nv = VQ ? 1 : L::blocks;   // copies of a run
    const int total = runs * (nk + nv);
    constexpr int PER = (8 * 2 * L::blocks + 31) / 32;            // copies of a lane, pages of 8 positions
    int y[PER], next_y[PER];                                      // row of each copy's run, -1: zeros
    auto look_up = [&](int (&row)[PER]) {
#pragma unroll
      for (int e = 0; e < PER; ++e) {
        const int i = lane + 32 * e, p = (sh.at.lo_unit + sh.off) * kRowsBk + (i & (runs - 1)) * run;
        row[e] = -1;
        if (i < total && p < sh.at.hi && p + run > sh.at.lo) row[e] = (int)page_row(w.b, c, sh.at.s, sh.at.h, p);
      }
    };
    look_up(next_y);
    bool ok = true, wrote = false;
    int n = 0, n_tiles = 0;
    // hands the tile at sh.at to the computing warps
    auto send_tile = [&]() {
      if (n_tiles > 0) ok = __all_sync(0xffffffffu, wait(t_empty, (n_tiles - 1) & 1, 53));
      ++n_tiles;
      if (!ok) return;
      const TileAt& at = sh.at;
      const int row0 = at.t << w.rows_log2, rows = min(w.rows(), at.rows_total - row0);
      const int es = a.q_f32 ? 4 : 2;
      if (lane == 0) {
        *tile = at;
        mbar_arrive_expect_tx(t_full, WM == 1 ? rows * HD * es : 0);
      }
      __syncwarp();
      if (WM == 1 && lane < rows) {
        const int rr = row0 + lane, tok = w.G.div(rr);
        const int64_t e = ((int64_t)(at.q0 + tok) * a.n_head + at.h * G + rr - tok * G) * HD;
        bulk_g2s(q_rows + lane * HD * es, static_cast<const uint8_t*>(a.q) + e * es, HD * es, t_full);
      }
    };
    send_tile();
    for (; n < n_units && ok; ++n) {
      uint8_t* st = ring + (n % stages) * stage_bytes;
      uint64_t* bar = &full[n % stages];
      const int key0 = (sh.at.lo_unit + sh.off) * kRowsBk, lo = sh.at.lo, hi = sh.at.hi;
      uint32_t bytes = 0;
#pragma unroll
      for (int e = 0; e < PER; ++e) {
        y[e] = next_y[e];
        const int i = lane + 32 * e, r = i >> (6 - run_log2);   // which copy of its run
        // runs without a page that the tile needs are zeroed by hand when quantized
        if (i < total) bytes += r < nk ? (KQ ? (y[e] >= 0 ? run * c.rb_k : 0) : run * 128)
                                       : (VQ ? (y[e] >= 0 ? run * c.rb_v : 0) : run * 128);
      }
      bytes = __reduce_add_sync(0xffffffffu, bytes);
      if (n + 1 < n_units) {
        if (++sh.off == sh.at.units) {
          next_tile(w, sh.at);
          sh.off = 0;
        }
        look_up(next_y);
      }
      const bool new_tile = n + 1 < n_units && sh.off == 0;
      if (n >= stages) ok = __all_sync(0xffffffffu, wait(&empty[n % stages], (n / stages - 1) & 1, 50));
      if (!ok) break;
      if (wrote) fence_async_proxy();   // a stage may hold rows zeroed by hand
#pragma unroll
      for (int e = 0; e < PER; ++e) {
        const int i = lane + 32 * e, r = i >> (6 - run_log2), first = (i & (runs - 1)) * run;
        const bool is_v = r >= nk, quant = is_v ? VQ : KQ;
        bool zero = false;
        if (i < total && quant && y[e] < 0) {
          const int p = key0 + first;
          if (p < hi && p + run > lo) {   // a missing page, not a run past the positions
            uint4* d = reinterpret_cast<uint4*>(st + (is_v ? k_bytes : 0) + first * (is_v ? c.rb_v : c.rb_k));
            for (int x = 0; x < run * (is_v ? c.rb_v : c.rb_k) / 16; ++x) d[x] = make_uint4(0, 0, 0, 0);
            zero = true;
          }
        }
        wrote |= __any_sync(0xffffffffu, zero);
      }
      __syncwarp();
      if (lane == 0) mbar_arrive_expect_tx(bar, bytes);
      __syncwarp();
#pragma unroll
      for (int e = 0; e < PER; ++e) {
        const int i = lane + 32 * e, r = i >> (6 - run_log2), first = (i & (runs - 1)) * run;
        if (i >= total) continue;
        if (r < nk) {
          if (!KQ)
            tma_2d(smem_u32(st) + r * (kRowsBk * 128) + first * 128, &k_map, r * 64, (int)(y[e] < 0 ? a.pool_rows : y[e]), bar);
          else if (y[e] >= 0)
            bulk_g2s(st + first * c.rb_k, c.k + (int64_t)y[e] * c.rb_k, run * c.rb_k, bar);
        } else {
          if (!VQ)
            tma_2d(smem_u32(st + k_bytes) + (r - nk) * (kRowsBk * 128) + first * 128, &v_map, (r - nk) * 64,
                   (int)(y[e] < 0 ? a.pool_rows : y[e]), bar);
          else if (y[e] >= 0)
            bulk_g2s(st + k_bytes + first * c.rb_v, c.v + (int64_t)y[e] * c.rb_v, run * c.rb_v, bar);
        }
      }
      if (new_tile) send_tile();
    }
    if (n_tiles > 0) mbar_wait_bounded(t_full, (n_tiles - 1) & 1, a.status, 54);
    // every copy issued has landed before the CTA may end
    for (int i = max(0, n - stages); i < n; ++i) mbar_wait_bounded(&full[i % stages], (i / stages) & 1, a.status, 51);
    return;
  }

  uint8_t* conv_k = ring + stages * stage_bytes;
  float* scale_k = reinterpret_cast<float*>(conv_k + L::tile);
  uint8_t* conv_v = conv_k + (KQ ? L::tile + L::scales : 0);
  float* scale_v = reinterpret_cast<float*>(conv_v + L::tile);

  // Quantized rows of a stage -> fp16 codes and fp32 scales [block][position] (WM = 4).
  auto unpack = [&](const uint8_t* raw, int type, int rb, uint8_t* dst, float* sc, const FastDiv& cpr, int lo, int hi,
                    bool guard, float& top) {
    int found = 0;   // infinite or NaN scales, taken out when guarded; rows outside [lo, hi) count as zeros
    top = 0.f;       // the largest scale
    const int cb = type == B2_Q8_0 ? HD : HD / 2;
    const int cpk = (int)cpr.d - 1, total = kRowsBk * (int)cpr.d;   // a row: code chunks, then the scales'
#pragma unroll 2
    for (int i = tid; i < total; i += kRowsThreads) {
      const int key = cpr.div(i), ch = i - key * (int)cpr.d;
      const uint8_t* row = raw + key * rb;
      if (ch == cpk) {
        float d[NB];
        row_scales<NB>(row + cb, d);
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          if (key < lo || key >= hi) d[b] = 0.f;
          if (guard && !(fabsf(d[b]) <= 65504.f)) d[b] = 0.f, found = 1;
          top = fmaxf(top, fabsf(d[b]));
          sc[b * kRowsBk + key] = d[b];
        }
        continue;
      }
      const uint4 x = *reinterpret_cast<const uint4*>(row + ch * 16);
      uint32_t h[8];
      if (type == B2_Q8_0) {
        s8x4_to_h2(x.x, h[0], h[1]);
        s8x4_to_h2(x.y, h[2], h[3]);
        s8x4_to_h2(x.z, h[4], h[5]);
        s8x4_to_h2(x.w, h[6], h[7]);
        *reinterpret_cast<uint4*>(dst + L::at(key, 2 * ch)) = make_uint4(h[0], h[1], h[2], h[3]);
        *reinterpret_cast<uint4*>(dst + L::at(key, 2 * ch + 1)) = make_uint4(h[4], h[5], h[6], h[7]);
      } else {
        n4x4_to_h2(x.x & 0x0F0F0F0Fu, h[0], h[1]);
        n4x4_to_h2(x.y & 0x0F0F0F0Fu, h[2], h[3]);
        n4x4_to_h2(x.z & 0x0F0F0F0Fu, h[4], h[5]);
        n4x4_to_h2(x.w & 0x0F0F0F0Fu, h[6], h[7]);
        *reinterpret_cast<uint4*>(dst + L::at(key, 4 * ch)) = make_uint4(h[0], h[1], h[2], h[3]);
        *reinterpret_cast<uint4*>(dst + L::at(key, 4 * ch + 1)) = make_uint4(h[4], h[5], h[6], h[7]);
        n4x4_to_h2((x.x >> 4) & 0x0F0F0F0Fu, h[0], h[1]);
        n4x4_to_h2((x.y >> 4) & 0x0F0F0F0Fu, h[2], h[3]);
        n4x4_to_h2((x.z >> 4) & 0x0F0F0F0Fu, h[4], h[5]);
        n4x4_to_h2((x.w >> 4) & 0x0F0F0F0Fu, h[6], h[7]);
        *reinterpret_cast<uint4*>(dst + L::at(key, 4 * ch + 2)) = make_uint4(h[0], h[1], h[2], h[3]);
        *reinterpret_cast<uint4*>(dst + L::at(key, 4 * ch + 3)) = make_uint4(h[4], h[5], h[6], h[7]);
      }
    }
    return found;
  };

  int done = 0;   // units of the share so far
  for (int n_tile = 0; sh.u < sh.u_end; ++n_tile) {
    wait(t_full, n_tile & 1, 55);
    const TileAt at = *tile;
    sh.at.units = at.units;
    const int u_lo = sh.off, u_hi = min(at.units, u_lo + (sh.u_end - sh.u));
    const int row0 = at.t << w.rows_log2;
    const int rows = min(w.rows(), at.rows_total - row0);
    // where row r of the tile stands in q and out
    auto place = [&](int r) -> int64_t {
      const int rr = row0 + r, tok = w.G.div(rr);
      return ((int64_t)(at.q0 + tok) * a.n_head + at.h * G + rr - tok * G) * HD;
    };

    // ---- queries: registers, split in two parts, or as they are; in
    // the dims' order within a block of 32 that the K operand is loaded in ----
    uint32_t qf[KS][4];
    int p0 = -1, p1 = -1;   // positions of rows g and g + 8 (-1: sees nothing)
    float cs = 1.f;   // SPLIT: from scores to exponents, a power of two of the row
    {
      const int r = wm * WROWS + g, r1 = r + 8;
      const bool on0 = r < rows, on1 = !SPLIT && r1 < rows;
      if (on0) p0 = at.first + w.G.div(row0 + r);
      if (on1) p1 = at.first + w.G.div(row0 + r1);
      // WM = 1: from shared memory, else from q itself
      const uint8_t* x0;
      const uint8_t* x1;
      if constexpr (WM == 1) {
        x0 = q_rows + (on0 ? r : 0) * HD * (a.q_f32 ? 4 : 2);
        x1 = q_rows + (on1 ? r1 : 0) * HD * (a.q_f32 ? 4 : 2);
      } else {
        x0 = static_cast<const uint8_t*>(a.q) + place(on0 ? r : 0) * (a.q_f32 ? 4 : 2);
        x1 = static_cast<const uint8_t*>(a.q) + place(on1 ? r1 : 0) * (a.q_f32 ? 4 : 2);
      }
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        // dims of operand columns 2j, 2j + 1 and 2j + 8, 2j + 9
        const int d0 = KD ? (ks / 2) * 32 + (ks & 1) * 16 + 4 * j : ks * 16 + 2 * j, d1 = KD ? d0 + 2 : d0 + 8;
        if constexpr (SPLIT) {
          float2 x = make_float2(0.f, 0.f), y = x;
          if (on0) {
            if (a.q_f32) {
              x = *reinterpret_cast<const float2*>(x0 + 4 * d0);
              y = *reinterpret_cast<const float2*>(x0 + 4 * d1);
            } else {
              x = __half22float2(*reinterpret_cast<const __half2*>(x0 + 2 * d0));
              y = __half22float2(*reinterpret_cast<const __half2*>(x0 + 2 * d1));
            }
          }
          qf[ks][0] = __float_as_uint(x.x), qf[ks][1] = __float_as_uint(x.y);
          qf[ks][2] = __float_as_uint(y.x), qf[ks][3] = __float_as_uint(y.y);
        } else {
          qf[ks][0] = on0 ? *reinterpret_cast<const uint32_t*>(x0 + 2 * d0) : 0u;
          qf[ks][1] = on1 ? *reinterpret_cast<const uint32_t*>(x1 + 2 * d0) : 0u;
          qf[ks][2] = on0 ? *reinterpret_cast<const uint32_t*>(x0 + 2 * d1) : 0u;
          qf[ks][3] = on1 ? *reinterpret_cast<const uint32_t*>(x1 + 2 * d1) : 0u;
        }
      }
      if constexpr (SPLIT) {
        uint32_t top = 0;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
          for (int e = 0; e < 4; ++e) top = max(top, qf[ks][e] & 0x7FFFFFFFu);
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const int fit = q_fit(top);
        const float f = a.q_mul * pow2(fit);
        cs = pow2(min(max(a.c_exp - fit, -120), 120));
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          const uint32_t x = qf[ks][2], y = qf[ks][3];
          h2_split(__uint_as_float(qf[ks][0]) * f, __uint_as_float(qf[ks][1]) * f, qf[ks][0], qf[ks][1]);
          h2_split(__uint_as_float(x) * f, __uint_as_float(y) * f, qf[ks][2], qf[ks][3]);
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(t_empty);
    }

    float o[OT][4];
#pragma unroll
    for (int d = 0; d < OT; ++d)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[d][e] = 0.f;
    // the row (of the warp's) and the dim that o[d][e] belongs to
    auto o_row = [&](int e) { return SPLIT ? 2 * j + (e & 1) : g + 8 * (e >> 1); };
    auto o_dim = [&](int d, int e) {
      if constexpr (SPLIT) return VD ? (d >> 1) * 32 + 4 * g + 2 * (d & 1) + (e >> 1) : d * 16 + g + 8 * (e >> 1);
      return VD ? (d >> 2) * 32 + 8 * j + 4 * (e & 1) + (d & 3) : d * 8 + 2 * j + (e & 1);
    };
    // a value of rows g and g + 8 (x0, x1), for the row of o[.][e]
    auto by_row = [&](float x0, float x1, float (&f)[4]) {
      if constexpr (SPLIT) {
        f[0] = f[2] = __shfl_sync(0xffffffffu, x0, 8 * j);
        f[1] = f[3] = __shfl_sync(0xffffffffu, x0, 8 * j + 4);
      } else {
        f[0] = f[1] = x0;
        f[2] = f[3] = x1;
      }
    };
    float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;   // rows g and g + 8 (SPLIT: row g)
    float off = VQ ? kOffsetQ + kFitMost : kOffset, fit = VQ ? pow2(kFitMost) : 1.f;   // fit: 2^e of the offset
    auto fit_scales = [&](float top) {   // top: the same in every lane
      top = fminf(top, 65504.f);         // what an infinite scale does to its rows needs no room
      if (top * fit < 1.f) return;
      const int e_old = (__float_as_int(fit) >> 23) - 127, e = 126 - (__float_as_int(top) >> 23);
      const float r = pow2(e - e_old);
#pragma unroll
      for (int d = 0; d < OT; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[d][i] *= r;
      l0 *= r;
      l1 *= r;
      fit = pow2(e);
      off = kOffsetQ + e;
    };
    // Where the exponents of a row with maximum m are counted from: a row that
    // has seen nothing keeps m = -inf and counts from 0.  Rounded up, so that no
    // weight passes 2^off where the offset is below the spacing of scores.
    auto origin = [&](float m) { return __fsub_ru(m == -INFINITY ? 0.f : SPLIT ? m * cs : m, off); };
    // positions every live row sees need no mask
    const int p_min = at.first + w.G.div(row0), p_max = at.first + w.G.div(row0 + rows - 1);

    // WM = 1: [4 warps][16] (maximum, sum), then [4 warps][WROWS][HD] sums, after
    // the ring.  Until the tile's end SPLIT keeps its fp32 sums there, a lane's
    // own (see kRowsFlush), with the maximum and the offset they are relative to.
    float2* ml = reinterpret_cast<float2*>(ring + stages * stage_bytes);
    float* so = reinterpret_cast<float*>(ml + 64);
    float4* own_sum = reinterpret_cast<float4*>(so + warp * WROWS * HD) + lane;
    auto add_sums = [&]() {   // to o
      const float2 rel = ml[warp * 16 + g];
      float x = rel.x == -INFINITY ? 0.f : ex2(origin(rel.x) - origin(m0)), f[4];
      if constexpr (VQ) x *= pow2((__float_as_int(fit) >> 23) - (__float_as_int(rel.y) >> 23));
      by_row(x, x, f);
#pragma unroll
      for (int d = 0; d < OT; ++d) {
        const float4 y = own_sum[d * 32];
        o[d][0] = fmaf(y.x, f[0], o[d][0]);
        o[d][1] = fmaf(y.y, f[1], o[d][1]);
        o[d][2] = fmaf(y.z, f[2], o[d][2]);
        o[d][3] = fmaf(y.w, f[3], o[d][3]);
      }
      __syncwarp();
    };

    for (int u = u_lo; u < u_hi; ++u, ++done) {
      if (SPLIT && WM == 1 && u > u_lo && (u - u_lo) % kRowsFlush == 0) {
        if (u - u_lo > kRowsFlush) add_sums();
#pragma unroll
        for (int d = 0; d < OT; ++d) {
          own_sum[d * 32] = make_float4(o[d][0], o[d][1], o[d][2], o[d][3]);
          o[d][0] = o[d][1] = o[d][2] = o[d][3] = 0.f;
        }
        if (j == 0) ml[warp * 16 + g] = make_float2(m0, fit);
        __syncwarp();
      }
      uint8_t* st = ring + (done % stages) * stage_bytes;
      const int key0 = (at.lo_unit + u) * kRowsBk;
      const bool edge = key0 + kRowsBk > at.hi || key0 + kRowsBk - 1 > p_min ||
                        (w.window > 0 && key0 <= p_max - w.window);
      // A value that some row must not see can still reach it as 0·v when v is
      // infinite or NaN.  Such values are taken out of the operand and added
      // at the end to the rows that do see them.
      const bool guard = edge && p_max > p_min;
      int found = 0;
      bool bad = false;
      wait(&full[done % stages], (done / stages) & 1, 52);
      uint8_t* Kt = KQ && !KD ? conv_k : st;
      uint8_t* Vt = VQ && !VD ? conv_v : st + k_bytes;
      const int v_lo = edge ? at.lo - key0 : 0, v_hi = edge ? at.hi - key0 : kRowsBk;   // rows of V the tile sees
      if constexpr (WM == 4) {
        if constexpr (KQ || VQ) bar_compute();   // the last unit's operands are done with
        float top;
        if constexpr (KQ) unpack(st, c.type_k, c.rb_k, conv_k, scale_k, a.cpr_k, 0, kRowsBk, false, top);
        if constexpr (VQ) {
          found = unpack(st + k_bytes, c.type_v, c.rb_v, conv_v, scale_v, a.cpr_v, v_lo, v_hi, guard, top);
          if (top * fit >= 1.f) atomicMax(&v_top[done & 1], __float_as_uint(top));   // the offset must fall
        }
      }
      if (!VQ && edge) {
        // WM = 1: a warp looks over its own positions
        constexpr int CH = L::blocks * 8;
        const int n = (WM == 1 ? KEYS : kRowsBk) * CH;
        for (int i = WM == 1 ? lane : tid; i < n; i += WM == 1 ? 32 : kRowsThreads) {
          const int key = (WM == 1 ? wk * KEYS : 0) + i / CH;
          uint4* q = reinterpret_cast<uint4*>(Vt + L::at(key, i % CH));
          if (key < v_lo || key >= v_hi) {
            *q = make_uint4(0, 0, 0, 0);
          } else if (guard) {
            uint4 x = *q;
            uint32_t* v = reinterpret_cast<uint32_t*>(&x);
            bool changed = false;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              if ((v[e] & 0x7C00u) == 0x7C00u) v[e] &= 0xFFFF0000u, changed = true;
              if ((v[e] & 0x7C000000u) == 0x7C000000u) v[e] &= 0xFFFFu, changed = true;
            }
            if (changed) *q = x, found = 1;
          }
        }
        // a later copy into this stage must not be overtaken by these stores
        fence_async_proxy();
      }
      if constexpr (WM == 4) {
        if (edge)
          bad = bar_compute_or(found);
        else if (KQ || VQ)
          bar_compute();
        if constexpr (VQ) {
          fit_scales(__uint_as_float(*reinterpret_cast<volatile uint32_t*>(&v_top[done & 1])));
          if (tid == 0) v_top[(done + 1) & 1] = 0;   // read before the barrier above, used after the next unit's first
        }
      } else if (!VQ && edge) {
        __syncwarp();
        bad = __any_sync(0xffffffffu, found);
      }
      const uint32_t ks_base = smem_u32(Kt), vs_base = smem_u32(Vt);

      for (int c0 = 0; c0 < KEYS; c0 += NC) {
        const int kw = wk * KEYS + c0;   // first position of this step within the unit
        // ---- S = Q·K^T ----
        float s[NT][4];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          float acc[4] = {0.f, 0.f, 0.f, 0.f};
          if constexpr (KD) {
            // the row of operand column g; scales of positions 2j, 2j + 1
            const uint8_t* kr = Kt + (kw + n * 8 + g) * c.rb_k;
            const uint8_t* sr = Kt + (kw + n * 8 + 2 * j) * c.rb_k + (c.type_k == B2_Q8_0 ? HD : HD / 2);
            uint32_t x[NB][2];
            if (c.type_k == B2_Q8_0) {
#pragma unroll
              for (int b = 0; b < NB; ++b) {
                x[b][0] = *reinterpret_cast<const uint32_t*>(kr + b * 32 + 4 * j);
                x[b][1] = *reinterpret_cast<const uint32_t*>(kr + b * 32 + 16 + 4 * j);
              }
            } else {
#pragma unroll
              for (int b = 0; b < NB; ++b) {
                const uint32_t v = *reinterpret_cast<const uint32_t*>(kr + b * 16 + 4 * j);
                x[b][0] = (uint32_t)nib_lo_s8(v);
                x[b][1] = (uint32_t)nib_hi_s8(v);
              }
            }
            float da[NB], db[NB];
            row_scales<NB>(sr, da);
            row_scales<NB>(sr + c.rb_k, db);
            float t[NB][4];
#pragma unroll
            for (int b = 0; b < NB; ++b) {
              uint32_t kf[4];
              s8x4_to_h2(x[b][0], kf[0], kf[1]);
              s8x4_to_h2(x[b][1], kf[2], kf[3]);
              t[b][0] = t[b][1] = t[b][2] = t[b][3] = 0.f;
              mma16816(t[b], qf[2 * b], kf[0], kf[1]);
              mma16816(t[b], qf[2 * b + 1], kf[2], kf[3]);
            }
#pragma unroll
            for (int b = 0; b < NB; ++b) {
              acc[0] = fmaf(t[b][0], da[b], acc[0]);
              acc[1] = fmaf(t[b][1], db[b], acc[1]);
              acc[2] = fmaf(t[b][2], da[b], acc[2]);
              acc[3] = fmaf(t[b][3], db[b], acc[3]);
            }
          } else {
#pragma unroll
            for (int b = 0; b < NB; ++b) {
              uint32_t kf[4];   // 8 positions x 32 dims
              ldsm4(ks_base + L::at(kw + n * 8 + (lane & 7), b * 4 + (lane >> 3)), kf);
              if constexpr (KQ) {
                float t[4] = {0.f, 0.f, 0.f, 0.f};
                mma16816(t, qf[2 * b], kf[0], kf[1]);
                mma16816(t, qf[2 * b + 1], kf[2], kf[3]);
                const float2 d = *reinterpret_cast<const float2*>(scale_k + b * kRowsBk + kw + n * 8 + 2 * j);
                acc[0] = fmaf(t[0], d.x, acc[0]);
                acc[1] = fmaf(t[1], d.y, acc[1]);
                acc[2] = fmaf(t[2], d.x, acc[2]);
                acc[3] = fmaf(t[3], d.y, acc[3]);
              } else {
                mma16816(acc, qf[2 * b], kf[0], kf[1]);
                mma16816(acc, qf[2 * b + 1], kf[2], kf[3]);
              }
            }
          }
          if constexpr (SPLIT) {
            s[n][0] = acc[0] + acc[2];
            s[n][1] = acc[1] + acc[3];
            s[n][2] = s[n][3] = 0.f;
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) s[n][e] = acc[e] * a.scale_log2;
          }
          if (edge) {
            const int t0 = key0 + kw + n * 8 + 2 * j;
#pragma unroll
            for (int e = 0; e < (SPLIT ? 2 : 4); ++e) {
              const int t = t0 + (e & 1), p = e < 2 ? p0 : p1;
              if (t > p || t >= at.hi || (w.window > 0 && t <= p - w.window)) s[n][e] = -INFINITY;
            }
          }
        }
        // VD: this step's words of V, on their way while the weights are formed
        uint32_t vw[VD ? NB : 1][4];
        float sc[VD ? 4 : 1][NB];   // scales of positions 2j, 2j+1, 2j+8, 2j+9
        if constexpr (VD) {
          const uint8_t* vr = Vt + (kw + 2 * j) * c.rb_v;
          const bool q8 = c.type_v == B2_Q8_0;
#pragma unroll
          for (int b = 0; b < NB; ++b) {
            const uint8_t* q = vr + (q8 ? b * 32 + 4 * g : b * 16 + 4 * (g & 3));
            vw[b][0] = *reinterpret_cast<const uint32_t*>(q);
            vw[b][1] = *reinterpret_cast<const uint32_t*>(q + c.rb_v);
            vw[b][2] = *reinterpret_cast<const uint32_t*>(q + 8 * c.rb_v);
            vw[b][3] = *reinterpret_cast<const uint32_t*>(q + 9 * c.rb_v);
          }
          const uint8_t* sr = vr + (q8 ? HD : HD / 2);
          row_scales<NB>(sr, sc[0]);
          row_scales<NB>(sr + c.rb_v, sc[1]);
          row_scales<NB>(sr + 8 * c.rb_v, sc[2]);
          row_scales<NB>(sr + 9 * c.rb_v, sc[3]);
          if (edge) {
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const int key = kw + 2 * j + (r & 1) + (r >> 1) * 8;
#pragma unroll
              for (int b = 0; b < NB; ++b) {
                if (key < v_lo || key >= v_hi) sc[r][b] = 0.f;
                if (guard && !(fabsf(sc[r][b]) <= 65504.f)) sc[r][b] = 0.f, found = 1;
              }
            }
          }
          float top = 0.f;
#pragma unroll
          for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int b = 0; b < NB; ++b) top = fmaxf(top, fabsf(sc[r][b]));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
          fit_scales(fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2)));   // lanes of the same j hold the same
        }
        // ---- running maximum and sum ----
        float n0 = m0, n1 = m1;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          n0 = fmaxf(n0, fmaxf(s[n][0], s[n][1]));
          if constexpr (!SPLIT) n1 = fmaxf(n1, fmaxf(s[n][2], s[n][3]));
        }
#pragma unroll
        for (int x = 1; x < 4; x <<= 1) {
          n0 = fmaxf(n0, __shfl_xor_sync(0xffffffffu, n0, x));
          if constexpr (!SPLIT) n1 = fmaxf(n1, __shfl_xor_sync(0xffffffffu, n1, x));
        }
        const float r0 = origin(n0), r1 = origin(n1);
        if (__any_sync(0xffffffffu, n0 != m0 || (!SPLIT && n1 != m1))) {
          const float f0 = m0 == -INFINITY ? 0.f : ex2(origin(m0) - r0), f1 = m1 == -INFINITY ? 0.f : ex2(origin(m1) - r1);
          l0 *= f0;
          l1 *= f1;
          float f[4];
          by_row(f0, f1, f);
#pragma unroll
          for (int d = 0; d < OT; ++d)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[d][e] *= f[e];
          m0 = n0;
          m1 = n1;
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          s[n][0] = ex2(SPLIT ? fmaf(s[n][0], cs, -r0) : s[n][0] - r0);
          s[n][1] = ex2(SPLIT ? fmaf(s[n][1], cs, -r0) : s[n][1] - r0);
          l0 += s[n][0] + s[n][1];
          if constexpr (!SPLIT) {
            s[n][2] = ex2(s[n][2] - r1);
            s[n][3] = ex2(s[n][3] - r1);
            l1 += s[n][2] + s[n][3];
          }
        }
        // ---- O += P·V ----
#pragma unroll
        for (int k = 0; k < NC / 16; ++k) {
          uint32_t pf[4];
          const float* x = s[2 * k];
          const float* y = s[2 * k + 1];
          // FULL: rows g and g + 8; SPLIT: high parts pf[0], pf[2], the others' pf[1], pf[3]
          auto operand = [&](float a0, float a1, float b0, float b1) {   // scales of positions 2j, 2j+1, 2j+8, 2j+9
            if constexpr (SPLIT) {
              h2_split(x[0] * a0, x[1] * a1, pf[0], pf[1]);
              h2_split(y[0] * b0, y[1] * b1, pf[2], pf[3]);
            } else {
              pf[0] = h2(x[0] * a0, x[1] * a1);
              pf[1] = h2(x[2] * a0, x[3] * a1);
              pf[2] = h2(y[0] * b0, y[1] * b1);
              pf[3] = h2(y[2] * b0, y[3] * b1);
            }
          };
          if constexpr (!VQ) operand(1.f, 1.f, 1.f, 1.f);
#pragma unroll
          for (int b = 0; b < NB; ++b) {
            if constexpr (VD) {
              operand(sc[0][b], sc[1][b], sc[2][b], sc[3][b]);
              uint32_t v0[4], v1[4];   // positions 2j, 2j+1 and 2j+8, 2j+9 of dims 4g + t of the block
              if (c.type_v == B2_Q8_0) {
                pair_to_h2(vw[b][0] ^ 0x80808080u, vw[b][1] ^ 0x80808080u, 0x64806480u, v0);
                pair_to_h2(vw[b][2] ^ 0x80808080u, vw[b][3] ^ 0x80808080u, 0x64806480u, v1);
              } else {
                const int sf = g & 4;   // values 16..31 are the high nibbles
                pair_to_h2((vw[b][0] >> sf) & 0x0F0F0F0Fu, (vw[b][1] >> sf) & 0x0F0F0F0Fu, 0x64086408u, v0);
                pair_to_h2((vw[b][2] >> sf) & 0x0F0F0F0Fu, (vw[b][3] >> sf) & 0x0F0F0F0Fu, 0x64086408u, v1);
              }
              if constexpr (SPLIT) {
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                  const uint32_t av[4] = {v0[2 * t], v0[2 * t + 1], v1[2 * t], v1[2 * t + 1]};
                  mma16816(o[b * 2 + t], av, pf[0], pf[2]);
                  mma16816(o[b * 2 + t], av, pf[1], pf[3]);
                }
              } else {
#pragma unroll
                for (int t = 0; t < 4; ++t) mma16816(o[b * 4 + t], pf, v0[t], v1[t]);
              }
            } else {
              if constexpr (VQ) {
                const float* q = scale_v + b * kRowsBk + kw + k * 16 + 2 * j;
                const float2 da = *reinterpret_cast<const float2*>(q), db = *reinterpret_cast<const float2*>(q + 8);
                operand(da.x, da.y, db.x, db.y);
              }
#pragma unroll
              for (int d = 0; d < 2; ++d) {
                uint32_t vf[4];   // 16 positions x 16 dims
                if constexpr (SPLIT) {
                  ldsm4_t(vs_base + L::at(kw + k * 16 + (lane & 7) + (lane >> 4) * 8, b * 4 + 2 * d + ((lane >> 3) & 1)), vf);
                  if constexpr (WM == 4) {
                    // the tensor pipe cuts its sums to fp32; over a chunk's many
                    // positions in one warp that would show, so 16 positions at
                    // a time are added with rounding
                    float t[4] = {0.f, 0.f, 0.f, 0.f};
                    mma16816(t, vf, pf[1], pf[3]);
                    mma16816(t, vf, pf[0], pf[2]);
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[b * 2 + d][e] += t[e];
                  } else {
                    mma16816(o[b * 2 + d], vf, pf[0], pf[2]);
                    mma16816(o[b * 2 + d], vf, pf[1], pf[3]);
                  }
                } else {
                  ldsm4_t(vs_base + L::at(kw + k * 16 + (lane & 15), b * 4 + 2 * d + (lane >> 4)), vf);
                  mma16816(o[b * 4 + 2 * d], pf, vf[0], vf[1]);
                  mma16816(o[b * 4 + 2 * d + 1], pf, vf[2], vf[3]);
                }
              }
            }
          }
        }
      }
      if (VD && guard) bad = __any_sync(0xffffffffu, found);
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[done % stages]);
      if (bad) {
        // infinite and NaN values of V, to the rows that see them (their
        // weight is positive, so the value itself decides the sum)
        float pos[4];
        by_row(__int_as_float(p0), __int_as_float(p1), pos);
        for (int key = wk * KEYS; key < (wk + 1) * KEYS; ++key) {
          const int t = key0 + key;
          if (t < at.lo || t >= at.hi) continue;
          const int64_t row = page_row(w.b, c, at.s, at.h, t);
          if (row < 0) continue;
          const uint8_t* vr = c.v + row * c.rb_v;
#pragma unroll
          for (int d = 0; d < OT; ++d)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int i = o_dim(d, e), p = __float_as_int(pos[e]);
              float v;
              if constexpr (VQ) {
                const float sc = h2f(*reinterpret_cast<const uint16_t*>(
                    vr + (c.type_v == B2_Q8_0 ? HD : HD / 2) + 2 * (i >> 5)));
                const int code = c.type_v == B2_Q8_0
                                     ? (int)(int8_t)vr[i]
                                     : ((vr[(i >> 5) * 16 + (i & 15)] >> ((i & 16) ? 4 : 0)) & 15) - 8;
                v = (float)code * sc;
              } else {
                v = h2f(reinterpret_cast<const uint16_t*>(vr)[i]);
              }
              if (!(fabsf(v) <= 3.4e38f) && t <= p && !(w.window > 0 && t <= p - w.window)) o[d][e] += v;
            }
        }
      }
    }

    if (SPLIT && WM == 1 && u_hi - u_lo > kRowsFlush) add_sums();
    if constexpr (VQ) {   // warps and parts meet with the same offset
      const float r = pow2(127 - (__float_as_int(fit) >> 23));
#pragma unroll
      for (int d = 0; d < OT; ++d)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[d][e] *= r;
      l0 *= r;
      l1 *= r;
    }
    if (m0 != -INFINITY) m0 = origin(m0) + off;
    if (m1 != -INFINITY) m1 = origin(m1) + off;
    // ---- join the lanes' sums, and for WM = 1 the warps ----
#pragma unroll
    for (int x = 1; x < 4; x <<= 1) {
      l0 += __shfl_xor_sync(0xffffffffu, l0, x);
      if constexpr (!SPLIT) l1 += __shfl_xor_sync(0xffffffffu, l1, x);
    }
    const Split split = split_of(sh, blockIdx.x, u_hi);
    const bool whole = split.n == 0;
    float* part = a.slots + (int64_t)split.slot * slot_floats(w.rows(), HD);
    float* part_ml = part + w.rows() * HD;
    auto put = [&](int r, int d, float x) {   // value d of row r, normalized, or a partial result
      if (!whole)
        part[r * HD + d] = x;
      else if (a.q_f32)
        static_cast<float*>(a.out)[place(r) + d] = x;
      else
        static_cast<__half*>(a.out)[place(r) + d] = __float2half_rn(x);
    };

    if constexpr (WM == 1) {
      if (j == 0) {
        ml[warp * 16 + g] = make_float2(m0, l0);
        if constexpr (!SPLIT) ml[warp * 16 + g + 8] = make_float2(m1, l1);
      }
      bar_compute();
      auto top = [&](int r) {
        return fmaxf(fmaxf(ml[r].x, ml[16 + r].x), fmaxf(ml[32 + r].x, ml[48 + r].x));
      };
      // a warp that saw nothing of a row contributes nothing, not 0·NaN
      float f[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 x = ml[warp * 16 + o_row(e)];
        f[e] = part_weight(x.x, x.y, top(o_row(e)));
      }
#pragma unroll
      for (int d = 0; d < OT; ++d)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          so[(warp * WROWS + o_row(e)) * HD + o_dim(d, e)] = f[e] != 0.f ? o[d][e] * f[e] : 0.f;
      bar_compute();
      for (int i = tid; i < rows * HD; i += kRowsThreads) {
        const int r = i / HD, d = i - r * HD;
        const float t = top(r);
        float x = 0.f, l = 0.f;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const float2 e = ml[q * 16 + r];
          x += so[(q * WROWS + r) * HD + d];
          l += e.x == -INFINITY ? e.y : e.y * ex2(e.x - t);
        }
        if (whole)
          x *= l != 0.f ? 1.f / l : 0.f;
        else if (d == 0)
          *reinterpret_cast<float2*>(part_ml + 2 * r) = make_float2(t, l);
        put(r, d, x);
      }
      if (!whole) {
        // all warps' shares of the rows are written before one counts the part
        __threadfence();
        bar_compute();
        if (warp == 0) {
          const bool last = part_arrives(a.counters + split.cta0 * 8, split.n);
          if (lane == 0) *last_part = last;
        }
        bar_compute();
        if (*reinterpret_cast<volatile int*>(last_part)) {
          constexpr int R = WROWS / 4;
          const int r = warp * R;
          if (r < rows)
            join_parts<HD, R, 16 / R>(a.slots, w.rows(), split, r, rows - r, place(min(r + lane, rows - 1)), a.out,
                                      a.q_f32 != 0);
        }
      }
      bar_compute();   // the join's space is free for the next tile
    } else {
      const int r = wm * WROWS + g;
      float f[4];
      by_row(!whole ? 1.f : l0 != 0.f ? 1.f / l0 : 0.f, !whole ? 1.f : l1 != 0.f ? 1.f / l1 : 0.f, f);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (wm * WROWS + o_row(e) < rows) {
#pragma unroll
          for (int d = 0; d < OT; ++d) put(wm * WROWS + o_row(e), o_dim(d, e), o[d][e] * f[e]);
        }
      if (!whole && wm * WROWS < rows) {
        if (j == 0) {
          if (r < rows) *reinterpret_cast<float2*>(part_ml + 2 * r) = make_float2(m0, l0);
          if constexpr (!SPLIT)
            if (r + 8 < rows) *reinterpret_cast<float2*>(part_ml + 2 * (r + 8)) = make_float2(m1, l1);
        }
        if (part_arrives(a.counters + split.cta0 * 8 + warp, split.n)) {
          constexpr int R = HD == 256 ? 4 : 8;
          for (int r0 = wm * WROWS; r0 < min((wm + 1) * WROWS, rows); r0 += R)
            join_rows<HD, R>(a.slots, w.rows(), split, r0, rows - r0, place(min(r0 + lane, rows - 1)), a.out,
                             a.q_f32 != 0);
        }
      }
    }

    sh.u += u_hi - u_lo;
    sh.off = 0;
  }
}

int launch_page_rows_64(const PageRowsArgs& a, bool split, int wm, cudaStream_t s);
int launch_page_rows_96(const PageRowsArgs& a, bool split, int wm, cudaStream_t s);
int launch_page_rows_128(const PageRowsArgs& a, bool split, int wm, cudaStream_t s);
int launch_page_rows_256(const PageRowsArgs& a, bool split, int wm, cudaStream_t s);

// Tensor map of one layer's pool as [rows][hd] fp16, copied in boxes of
// box_rows x 64 dims, 128-byte swizzled (b2_page_tc.cu).
int page_pool_map(const void* base, int hd, int64_t rows, int box_rows, CUtensorMap* map);

// The ring, then what the tile's end needs beside it (WM = 1: the next tile's
// units are already on their way).
template <int HD, bool KQ, bool VQ, bool SPLIT, int WM>
inline int rows_smem_bytes(const PageRowsArgs& a, int stages) {
  const int ring = stages * rows_stage_bytes<HD, KQ, VQ>(a.c.rb_k, a.c.rb_v) + rows_conv_bytes<HD, KQ, VQ, WM>();
  const int join = WM == 1 ? 64 * 8 + 4 * (SPLIT ? 8 : 16) * HD * 4 : 0, sums = kPageMaxSeq * 4;
  return 1024 + kRowsCtrl + rows_q_bytes<HD, SPLIT, WM>() + std::max(ring + join, sums);   // the first for alignment
}

template <int HD, bool KQ, bool VQ, bool SPLIT, int WM>
int launch_page_rows_one(PageRowsArgs a, cudaStream_t s) {
  int stages = kRowsStagesMax;
  while (stages > 2 && rows_smem_bytes<HD, KQ, VQ, SPLIT, WM>(a, stages) > (227 / rows_ctas<HD, KQ, VQ, SPLIT>() - 1) * 1024) --stages;
  const int smem = rows_smem_bytes<HD, KQ, VQ, SPLIT, WM>(a, stages);
  auto kern = page_rows_kernel<HD, KQ, VQ, SPLIT, WM>;
  // looked up once per device and cache type pair
  static std::atomic<int> resident[kMaxDevices][2][2];
  int dev = 0;
  B2_CUDA_TRY(cudaGetDevice(&dev));
  B2_CHECK_ARG(dev < kMaxDevices, "device index");
  std::atomic<int>& known = resident[dev][a.c.type_k == B2_Q4_0][a.c.type_v == B2_Q4_0];
  int per_sm = known.load(std::memory_order_relaxed);
  if (per_sm == 0) {
    B2_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024));
    B2_CUDA_TRY(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kern, kRowsThreads + 32, smem));
    per_sm = std::max(1, std::min(per_sm, kPageMaxCtasPerSm));
    known.store(per_sm, std::memory_order_relaxed);
  }
  a.cpr_k = FastDiv::of(a.c.rb_k / 16);
  a.cpr_v = FastDiv::of(a.c.rb_v / 16);
  CUtensorMap km = {}, vm = {};
  const int box = std::min(1 << a.c.ps_log2, kRowsBk);
  int rc = B2_OK;
  if (!KQ) rc = page_pool_map(a.c.k, HD, a.pool_rows, box, &km);
  if (rc == B2_OK && !VQ) rc = page_pool_map(a.c.v, HD, a.pool_rows, box, &vm);
  if (rc != B2_OK) return rc;
  const int ctas = per_sm * sm_count();
  return launch_pdl(kern, dim3(ctas), dim3(kRowsThreads + 32), (size_t)smem, s, a, stages, km, vm);
}

template <int HD>
int launch_page_rows_hd(const PageRowsArgs& a, bool split, int wm, cudaStream_t s) {
  const bool kq = a.c.type_k != B2_F16, vq = a.c.type_v != B2_F16;
  // many rows over fp16 pages of these head sizes go to the tensor-core kernel
  constexpr bool kTc = HD == 64 || HD == 128;
#define B2_ROWS(KQ, VQ)                                                                             \
  if (kq == KQ && vq == VQ) {                                                                       \
    if (wm == 1)                                                                                    \
      return split ? launch_page_rows_one<HD, KQ, VQ, true, 1>(a, s)                                \
                   : launch_page_rows_one<HD, KQ, VQ, false, 1>(a, s);                              \
    if constexpr (KQ || VQ || !kTc)                                                                 \
      return split ? launch_page_rows_one<HD, KQ, VQ, true, 4>(a, s)                                \
                   : launch_page_rows_one<HD, KQ, VQ, false, 4>(a, s);                              \
  }
  B2_ROWS(false, false)
  B2_ROWS(true, false)
  B2_ROWS(false, true)
  B2_ROWS(true, true)
#undef B2_ROWS
  return B2_ERR_UNSUPPORTED;
}

}  // namespace b2
