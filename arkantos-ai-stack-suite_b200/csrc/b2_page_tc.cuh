// Attention of many rows over the paged cache on the 5th-generation tensor
// cores: chunks of a prompt, whole prompts, and steps that mix them with
// single tokens, over fp16 pages with head_dim 64 or 128.
//
//   o_r = Σ_t e^{s_rt − m_r} v_t / Σ_t e^{s_rt − m_r},   s_rt = scale · q_r·k_t
//
// A CTA works on a tile of 256 rows (token, query head) of one kv head as two
// halves of 128, and on units of 128 positions.  Per unit and half one 128 x
// 128 product S = Q·K^T and one 128 x hd product O += P·V run on tcgen05, S, P
// and O in TMEM; while the softmax of one half runs on its 128 threads (a
// thread owns a row: no exchange between lanes), the other half's products
// run.  Both products of a unit cost 128·128·hd multiply-adds a half, 2048
// tensor cycles for hd 128 and both halves; its 32768 exponentials take as
// many cycles of the special-function pipe, so the two bound the kernel
// together.
//
//   warps 0-3, 4-7  softmax of halves 0, 1; they also bring their rows of Q
//                   into shared memory and write the result
//   warp 8          issues the products from one thread
//   warp 9          brings K and V: one tensor copy per page and 64 dims, the
//                   lanes issuing side by side; pages past the tile's
//                   positions and table entries outside the pool are sent out
//                   of the map's range, which fills zeros
//
// The running maximum of a row is raised only when it grew by more than 2^8
// (the weights are relative to the old one until then: at most 2^15 with
// their offset of 2^7, inside fp16's range), so O is rarely rescaled.
//
// SPLIT (fp32 queries): q and p as two fp16 parts each, high and remainder,
// two products instead of one; both parts of p take exactly S's columns.
// FULL rounds p once to fp16, the error of the fp16 output itself.
//
// V rows that a tile must not see are zeroed in shared memory by half 0's
// threads before the unit's product, and infinite or NaN values of units that
// only some rows see wholly are taken out and added to the rows that see
// them at the end, so nothing masked reaches a row as 0·NaN.
//
// Every wait is bounded: an expired one records a code in *status and ends
// the other waits.
#pragma once

#include <cuda.h>
#include <cudaTypedefs.h>

#include "b2_page_rows.cuh"

namespace b2 {

struct PageTcArgs {
  PageView c;
  PageWork w;
  const void* q;
  void* out;
  int n_head;
  float scale_log2;
  int box_rows_log2;      // rows of a tensor copy: min(page_size, 128)
  int64_t pool_rows;      // rows of the layer's pool
  SplitTile* split;
  float* slots;
  int* status;
};

constexpr int kTcRows = 256, kTcBk = 128, kTcThreads = 384;
constexpr float kTcOffset = 7.f, kTcRaise = 8.f;

template <int HD, bool SPLIT>
struct TcSmem {
  static constexpr int half_q = 128 * HD * 2;                        // one fp16 part of a half's queries
  static constexpr int q = 2 * half_q * (SPLIT ? 2 : 1);
  static constexpr int tile = kTcBk * HD * 2;
  static constexpr int stages = HD == 128 ? (SPLIT ? 3 : 5) : 8;
  static constexpr int ctrl = 1024;
  static constexpr int bytes = ctrl + q + stages * tile + 1024;      // the last for alignment
};

// ---- tcgen05 -------------------------------------------------------------------------------
// K-major, 128-byte swizzle: rows of 64 fp16, 8-row groups 1024 bytes apart.
__device__ __forceinline__ uint64_t tc_desc_k(uint32_t saddr) {
  return (uint64_t)((saddr >> 4) & 0x3FFF) | ((uint64_t)1 << 16) | ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) |
         ((uint64_t)2 << 61);
}
// N-major (V: rows are positions, the k of P·V; 64 dims of a row contiguous):
// 64-dim blocks 128 rows apart, 8-row groups 1024 bytes apart.
__device__ __forceinline__ uint64_t tc_desc_n(uint32_t saddr) {
  return (uint64_t)((saddr >> 4) & 0x3FFF) | ((uint64_t)((kTcBk * 128) >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
         ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
// fp16 operands, fp32 accumulators, M = 128.
constexpr uint32_t tc_idesc(int n, bool b_n_major) {
  return (1u << 4) | ((b_n_major ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}
__device__ __forceinline__ void tc_mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)acc)
      : "memory");
}
__device__ __forceinline__ void tc_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"((uint32_t)acc)
      : "memory");
}
__device__ __forceinline__ void tc_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_async_proxy() {
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}

// Columns of the warp's 32 lanes; the wait is in the same asm block, so no
// register can be used before it.
__device__ __forceinline__ void tmem_ld32(uint32_t t, float* r) {
  uint32_t* u = reinterpret_cast<uint32_t*>(r);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
      "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n\ttcgen05.wait::ld.sync.aligned;"
      : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7]), "=r"(u[8]),
        "=r"(u[9]), "=r"(u[10]), "=r"(u[11]), "=r"(u[12]), "=r"(u[13]), "=r"(u[14]), "=r"(u[15]), "=r"(u[16]),
        "=r"(u[17]), "=r"(u[18]), "=r"(u[19]), "=r"(u[20]), "=r"(u[21]), "=r"(u[22]), "=r"(u[23]), "=r"(u[24]),
        "=r"(u[25]), "=r"(u[26]), "=r"(u[27]), "=r"(u[28]), "=r"(u[29]), "=r"(u[30]), "=r"(u[31])
      : "r"(t)
      : "memory");
}
__device__ __forceinline__ void tmem_ld64(uint32_t t, float* r) {
  uint32_t* u = reinterpret_cast<uint32_t*>(r);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x64.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,"
      "%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,%47,%48,%49,%50,%51,%52,%53,%54,%55,%56,%57,%58,%59,%60,%61,%62,%63}, [%64];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7]), "=r"(u[8]),
        "=r"(u[9]), "=r"(u[10]), "=r"(u[11]), "=r"(u[12]), "=r"(u[13]), "=r"(u[14]), "=r"(u[15]), "=r"(u[16]),
        "=r"(u[17]), "=r"(u[18]), "=r"(u[19]), "=r"(u[20]), "=r"(u[21]), "=r"(u[22]), "=r"(u[23]), "=r"(u[24]),
        "=r"(u[25]), "=r"(u[26]), "=r"(u[27]), "=r"(u[28]), "=r"(u[29]), "=r"(u[30]), "=r"(u[31]), "=r"(u[32]),
        "=r"(u[33]), "=r"(u[34]), "=r"(u[35]), "=r"(u[36]), "=r"(u[37]), "=r"(u[38]), "=r"(u[39]), "=r"(u[40]),
        "=r"(u[41]), "=r"(u[42]), "=r"(u[43]), "=r"(u[44]), "=r"(u[45]), "=r"(u[46]), "=r"(u[47]), "=r"(u[48]),
        "=r"(u[49]), "=r"(u[50]), "=r"(u[51]), "=r"(u[52]), "=r"(u[53]), "=r"(u[54]), "=r"(u[55]), "=r"(u[56]),
        "=r"(u[57]), "=r"(u[58]), "=r"(u[59]), "=r"(u[60]), "=r"(u[61]), "=r"(u[62]), "=r"(u[63])
      : "r"(t)
      : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t t, float* r) {
  uint32_t* u = reinterpret_cast<uint32_t*>(r);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7]), "=r"(u[8]),
        "=r"(u[9]), "=r"(u[10]), "=r"(u[11]), "=r"(u[12]), "=r"(u[13]), "=r"(u[14]), "=r"(u[15])
      : "r"(t)
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t t, const uint32_t* u) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(t),
      "r"(u[0]), "r"(u[1]), "r"(u[2]), "r"(u[3]), "r"(u[4]), "r"(u[5]), "r"(u[6]), "r"(u[7]), "r"(u[8]), "r"(u[9]),
      "r"(u[10]), "r"(u[11]), "r"(u[12]), "r"(u[13]), "r"(u[14]), "r"(u[15])
      : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ void tma_2d(uint32_t dst, const CUtensorMap* map, int x, int y, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(
          dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(x), "r"(y)
      : "memory");
}

template <int HD, bool SPLIT>
__global__ void __launch_bounds__(kTcThreads, 1)
    page_tc_kernel(const PageTcArgs a, const __grid_constant__ CUtensorMap k_map,
                   const __grid_constant__ CUtensorMap v_map) {
  using L = TcSmem<HD, SPLIT>;
  constexpr int NS = L::stages;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  uint64_t* kv_full = reinterpret_cast<uint64_t*>(smem);   // [NS]
  uint64_t* kv_empty = kv_full + NS;                       // [NS]
  uint64_t* q_full = kv_empty + NS;                        // [2]
  uint64_t* s_full = q_full + 2;                           // [2]
  uint64_t* p_full = s_full + 2;                           // [2]
  uint64_t* o_full = p_full + 2;                           // [2]
  uint64_t* done = o_full + 2;                             // [1]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + 512);
  int* abort_flag = reinterpret_cast<int*>(smem + 516);
  int* bad_seen = reinterpret_cast<int*>(smem + 520);      // 1 + the last segment with values taken out of V
  uint8_t* Qs = smem + L::ctrl;                            // [half][part][hd/64][128 rows][128 B]
  uint8_t* Ts = Qs + L::q;                                 // ring of K and V tiles [hd/64][128 rows][128 B]

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (int i = 0; i < NS; ++i) {
      mbar_init(&kv_full[i], 1);
      mbar_init(&kv_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_full[i], 128);
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 128);
      mbar_init(&o_full[i], 1);
    }
    mbar_init(done, 1);
    *abort_flag = 0;
    *bad_seen = 0;
    fence_mbar_init();
  }
  if (warp == 8) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                 "r"(512)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  pdl_wait();
  Share sh;
  const PageWork& w = a.w;
  const bool have = find_share(w, blockIdx.x, gridDim.x, reinterpret_cast<int*>(Qs), sh);
  tc_before();
  __syncthreads();   // barriers, the TMEM address; the sums in the queries' place are read
  tc_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(tmem_slot);
  pdl_launch_dependents();   // only now: a later kernel must not take the TMEM before this CTA has it

  auto wait = [&](uint64_t* bar, uint32_t parity, int code) -> bool {
    if (*reinterpret_cast<volatile int*>(abort_flag)) return false;
    if (mbar_wait_bounded(bar, parity, a.status, code)) return true;
    *reinterpret_cast<volatile int*>(abort_flag) = 1;
    return false;
  };
  // the units [lo, hi) of the current tile that fall into the share
  auto seg_end = [&]() {
    return sh.u_end - sh.u < sh.at.units - sh.off ? sh.off + (int)(sh.u_end - sh.u) : sh.at.units;
  };
  auto advance = [&](int u_hi) {
    sh.u += u_hi - sh.off;
    sh.off = 0;
    if (sh.u < sh.u_end) next_tile(w, sh.at);
  };
  auto unit_edge = [&](const TileAt& at, int key0) {
    const int row0 = at.t * kTcRows, last = min(row0 + kTcRows, at.rows_total) - 1;
    return key0 + kTcBk > at.hi || key0 + kTcBk - 1 > at.first + row0 / w.G ||
           (w.window > 0 && key0 <= at.first + last / w.G - w.window);
  };

  // Registers move from the last four warps to the softmax warps: 2 x 184 + 136
  // a lane of each scheduler, the 3 x 168 of the launch.
  if (!have && tid == 0) {
    SplitTile rec = {};
    rec.last = -1;
    a.split[blockIdx.x] = rec;
  }
  if (!have) sh.u = sh.u_end = 0;
  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 136;");
  if (warp == 9) {
    // ---------------- K and V ----------------
    const int per = 128 >> a.box_rows_log2;              // copies of 64 dims per tile
    const int rows_box = 1 << a.box_rows_log2;
    const int bx = lane % per, bh = lane / per;          // this lane's copy: rows bx·rows_box, dims 64·bh
    int n = 0;
    bool ok = true;
    while (ok && sh.u < sh.u_end) {
      const TileAt& at = sh.at;
      const int u_hi = seg_end();
      for (int u = sh.off; ok && u < u_hi; ++u) {
        const int p = (at.lo_unit + u) * kTcBk + bx * rows_box;
        int64_t row = -1;
        if (bh < HD / 64 && p < at.hi && p + rows_box > at.lo) row = page_row(w.b, a.c, at.s, at.h, p);
        const int y = (int)(row < 0 ? a.pool_rows : row);
#pragma unroll
        for (int kv = 0; kv < 2 && ok; ++kv, ++n) {
          const int st = n % NS;
          if (n >= NS) ok = wait(&kv_empty[st], ((n / NS) - 1) & 1, 50);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          if (lane == 0) mbar_arrive_expect_tx(&kv_full[st], L::tile);
          __syncwarp();
          if (bh < HD / 64)
            tma_2d(smem_u32(Ts + st * L::tile + bh * (kTcBk * 128) + bx * rows_box * 128), kv ? &v_map : &k_map, bh * 64,
                   y, &kv_full[st]);
        }
      }
      advance(u_hi);
    }
    // every copy issued has landed before the CTA may end
    for (int i = max(0, n - NS); i < n; ++i) mbar_wait_bounded(&kv_full[i % NS], (i / NS) & 1, a.status, 51);
  } else if (warp == 8) {
    // ---------------- products ----------------
    if (lane == 0) {
      constexpr uint32_t id_s = tc_idesc(128, false), id_o = tc_idesc(HD, true);
      int n = 0, seg[2] = {0, 0}, pn[2] = {0, 0};   // ring position, segments and P tiles of each half so far
      bool ok = true;
      auto qk = [&](int i, int st) {
#pragma unroll
        for (int part = 0; part < (SPLIT ? 2 : 1); ++part)
#pragma unroll
          for (int ks = 0; ks < HD / 16; ++ks) {
            const uint32_t off = (ks / 4) * (128 * 128) + (ks % 4) * 32;
            const uint32_t q = smem_u32(Qs) + (i * (SPLIT ? 2 : 1) + part) * L::half_q + off;
            tc_mma_ss(tmem + i * 128, tc_desc_k(q), tc_desc_k(smem_u32(Ts) + st * L::tile + off), id_s, (part | ks) != 0);
          }
        tc_commit(&s_full[i]);
      };
      auto pv = [&](int i, int st, bool acc) {
#pragma unroll
        for (int part = 0; part < (SPLIT ? 2 : 1); ++part)
#pragma unroll
          for (int ks = 0; ks < kTcBk / 16; ++ks)
            tc_mma_ts(tmem + 256 + i * 128, tmem + i * 128 + (SPLIT ? (ks / 2) * 32 + part * 16 + (ks & 1) * 8 : ks * 8),
                      tc_desc_n(smem_u32(Ts) + st * L::tile + ks * 2048), id_o, acc || (part | ks) != 0);
      };
      while (ok && sh.u < sh.u_end) {
        const int u_lo = sh.off, u_hi = seg_end();
        const int halves = min(kTcRows, sh.at.rows_total - sh.at.t * kTcRows) > 128 ? 2 : 1;
        ok = wait(&kv_full[n % NS], (n / NS) & 1, 60);
        for (int i = 0; i < halves && ok; ++i) {
          ok = wait(&q_full[i], seg[i] & 1, 61);
          tc_after();
          if (ok) qk(i, n % NS);
          ++seg[i];
        }
        if (ok) tc_commit(&kv_empty[n % NS]);
        ++n;
        for (int u = u_lo; ok && u < u_hi; ++u) {
          const int sv = n % NS, sk = (n + 1) % NS;
          const bool more = u + 1 < u_hi;
          ok = wait(&kv_full[sv], (n / NS) & 1, 62);
          for (int i = 0; i < halves && ok; ++i) {
            ok = wait(&p_full[i], pn[i] & 1, 63);
            ++pn[i];
            tc_after();
            if (!ok) break;
            pv(i, sv, u > u_lo);
            if (i == halves - 1) tc_commit(&kv_empty[sv]);
            if (more) {
              if (i == 0) ok = wait(&kv_full[sk], ((n + 1) / NS) & 1, 64);
              if (!ok) break;
              qk(i, sk);
              if (i == halves - 1) tc_commit(&kv_empty[sk]);
            } else {
              tc_commit(&o_full[i]);
            }
          }
          n += more ? 2 : 1;
        }
        advance(u_hi);
      }
      tc_commit(done);   // every product has completed before TMEM is given back
      mbar_wait_bounded(done, 0, a.status, 65);
    }
  }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 184;");
    // ---------------- softmax: a thread owns row 128·half + its lane of TMEM ----------------
    const int half = warp >> 2, r_in = tid & 127;
    const uint32_t tm = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const uint32_t ts = tm + half * 128, to = tm + 256 + half * 128;
    const float c = SPLIT ? 1.f : fmaxf(fabsf(a.scale_log2), 1e-30f);   // the sign went into the queries
    int n_seg = 0, n_s = 0, n_kv = 0, seg_id = 0;   // segments and S tiles of this half; units and segments of all
    bool ok = true, first_tile = true;
    SplitTile rec = {};
    rec.last = -1;
    while (ok && sh.u < sh.u_end) {
      const TileAt& at = sh.at;
      const int u_lo = sh.off, u_hi = seg_end();
      const int row0 = at.t * kTcRows, rows = min(kTcRows, at.rows_total - row0);
      const bool whole = u_lo == 0 && u_hi == at.units;
      const int slot = u_lo == 0 && !first_tile ? 2 * blockIdx.x + 1 : 2 * blockIdx.x;
      if (half * 128 < rows) {
        const int r = half * 128 + r_in;
        const bool on = r < rows;
        const int rr = row0 + (on ? r : 0), tok = rr / w.G;
        const int p = on ? at.first + tok : -1;
        const int64_t e0 = ((int64_t)(at.q0 + tok) * a.n_head + at.h * w.G + (rr - tok * w.G)) * HD;
        // ---- this row of Q, swizzled for the products ----
        {
          uint8_t* qd = Qs + half * (SPLIT ? 2 : 1) * L::half_q;
          const uint32_t sign = !SPLIT && a.scale_log2 < 0.f ? 0x80008000u : 0u;
#pragma unroll 4
          for (int ch = 0; ch < HD / 8; ++ch) {
            const uint32_t at_q = (ch / 8) * (128 * 128) + r_in * 128 + (((ch & 7) ^ (r_in & 7)) << 4);
            if constexpr (SPLIT) {
              float4 x = make_float4(0.f, 0.f, 0.f, 0.f), y = x;
              if (on) {
                const float4* q = reinterpret_cast<const float4*>(static_cast<const float*>(a.q) + e0 + ch * 8);
                x = __ldg(q);
                y = __ldg(q + 1);
              }
              uint4 hi, lo;
              const float f = a.scale_log2;
              h2_split(x.x * f, x.y * f, hi.x, lo.x);
              h2_split(x.z * f, x.w * f, hi.y, lo.y);
              h2_split(y.x * f, y.y * f, hi.z, lo.z);
              h2_split(y.z * f, y.w * f, hi.w, lo.w);
              *reinterpret_cast<uint4*>(qd + at_q) = hi;
              *reinterpret_cast<uint4*>(qd + L::half_q + at_q) = lo;
            } else {
              uint4 x = make_uint4(0, 0, 0, 0);
              if (on) x = __ldg(reinterpret_cast<const uint4*>(static_cast<const __half*>(a.q) + e0 + ch * 8));
              x.x ^= sign;
              x.y ^= sign;
              x.z ^= sign;
              x.w ^= sign;
              *reinterpret_cast<uint4*>(qd + at_q) = x;
            }
          }
          fence_async_proxy();
          mbar_arrive(&q_full[half]);
        }
        float m = -INFINITY, l = 0.f;
        for (int u = u_lo; u < u_hi && ok; ++u) {
          const int key0 = (at.lo_unit + u) * kTcBk;
          const bool edge = unit_edge(at, key0);
          ok = wait(&s_full[half], n_s & 1, 70);
          ++n_s;
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          tc_after();
          // The columns past 63 give their maximum, then the first 64 stay in
          // registers: their weights go where they came from before the others
          // are read again.
          float s[64];
          // this row sees columns [lo, hi)
          const int hi = min(p + 1, at.hi) - key0, lo = w.window > 0 ? p - w.window + 1 - key0 : 0;
          auto load = [&](int h) {
            tmem_ld64(ts + h * 64, s);
            if (edge) {
#pragma unroll
              for (int i = 0; i < 64; ++i)
                if (i + h * 64 >= hi || i + h * 64 < lo) s[i] = -INFINITY;
            }
          };
          float top = -INFINITY, top1 = -INFINITY;
          load(1);
#pragma unroll
          for (int i = 0; i < 64; i += 2) {
            top = fmaxf(top, s[i]);
            top1 = fmaxf(top1, s[i + 1]);
          }
          load(0);
#pragma unroll
          for (int i = 0; i < 64; i += 2) {
            top = fmaxf(top, s[i]);
            top1 = fmaxf(top1, s[i + 1]);
          }
          top = fmaxf(top, top1) * c;
          const bool raise = top > m + kTcRaise || (m == -INFINITY && top > m);
          if (__any_sync(0xffffffffu, raise)) {
            const float nm = raise ? top : m;
            const float f = m == -INFINITY ? 0.f : ex2(m - nm);
            const float g = raise ? f : 1.f;                      // the other rows keep their maximum
            if (u > u_lo) {
              float o[16];
#pragma unroll 1
              for (int i = 0; i < HD / 16; ++i) {
                tmem_ld16(to + i * 16, o);
#pragma unroll
                for (int e = 0; e < 16; ++e) o[e] *= g;
                tmem_st16(to + i * 16, reinterpret_cast<const uint32_t*>(o));
              }
            }
            l *= g;
            m = nm;
          }
          const float rs = (m == -INFINITY ? 0.f : m) - kTcOffset;
          float l0 = 0.f, l1 = 0.f;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            if (h) load(1);
#pragma unroll
            for (int i = 0; i < 64; i += 2) {
              s[i] = ex2(fmaf(s[i], c, -rs));
              s[i + 1] = ex2(fmaf(s[i + 1], c, -rs));
              l0 += s[i];
              l1 += s[i + 1];
            }
            // FULL: 64 columns of weights over S's first 64.  SPLIT: the two
            // parts of 32 positions over their own 32 columns.
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              uint32_t ph[16], pl[16];
#pragma unroll
              for (int e = 0; e < 16; ++e) {
                if constexpr (SPLIT)
                  h2_split(s[i * 32 + 2 * e], s[i * 32 + 2 * e + 1], ph[e], pl[e]);
                else
                  ph[e] = h2(s[i * 32 + 2 * e], s[i * 32 + 2 * e + 1]);
              }
              if constexpr (SPLIT) {
                tmem_st16(ts + h * 64 + i * 32, ph);
                tmem_st16(ts + h * 64 + i * 32 + 16, pl);
              } else {
                tmem_st16(ts + h * 32 + i * 16, ph);
              }
            }
          }
          l += l0 + l1;
          tmem_wait_st();
          if (half == 0 && edge) {
            // V of a unit that some rows do not see wholly
            const int nv = 2 * (n_kv + u - u_lo) + 1, st = nv % NS;
            ok = wait(&kv_full[st], (nv / NS) & 1, 71);
            uint8_t* V = Ts + st * L::tile;
            int found = 0;
            const int key = key0 + r_in;
            const bool none = key >= at.hi || key < at.lo;
#pragma unroll 4
            for (int ch = 0; ch < HD / 8; ++ch) {
              uint4* q = reinterpret_cast<uint4*>(V + (ch / 8) * (kTcBk * 128) + r_in * 128 + ((ch & 7) << 4));
              uint4 x = *q;
              const uint4 was = x;
              uint32_t* v = reinterpret_cast<uint32_t*>(&x);
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                if (none) v[e] = 0u;
                if ((v[e] & 0x7C00u) == 0x7C00u) v[e] &= 0xFFFF0000u, found = 1;
                if ((v[e] & 0x7C000000u) == 0x7C000000u) v[e] &= 0xFFFFu, found = 1;
              }
              if (x.x != was.x || x.y != was.y || x.z != was.z || x.w != was.w) *q = x;
            }
            if (found) *reinterpret_cast<volatile int*>(bad_seen) = seg_id + 1;
            fence_async_proxy();
          }
          tc_before();
          mbar_arrive(&p_full[half]);
        }
        // ---- the result ----
        if (ok) ok = wait(&o_full[half], n_seg & 1, 72);
        ++n_seg;
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        tc_after();
        const float inv = !whole ? 1.f : l != 0.f ? 1.f / l : 0.f;
        float* part = a.slots + (int64_t)slot * slot_floats(kTcRows, HD);
        const bool bad = *reinterpret_cast<volatile int*>(bad_seen) > seg_id;
#pragma unroll 1
        for (int i = 0; i < HD / 32; ++i) {
          float o[32];
          tmem_ld32(to + i * 32, o);
          if (bad && on) {
            for (int u = u_lo; u < u_hi; ++u) {
              const int key0 = (at.lo_unit + u) * kTcBk;
              if (!unit_edge(at, key0)) continue;
              const int t1 = min(min(p + 1, at.hi), key0 + kTcBk);
              for (int t = max(max(at.lo, key0), w.window > 0 ? p - w.window + 1 : 0); t < t1; ++t) {
                const int64_t row = page_row(w.b, a.c, at.s, at.h, t);
                if (row < 0) continue;
                const __half* v = reinterpret_cast<const __half*>(a.c.v + row * a.c.rb_v) + i * 32;
#pragma unroll
                for (int e = 0; e < 32; ++e) {
                  const float f = __half2float(v[e]);
                  if (!(fabsf(f) <= 65504.f)) o[e] += f;
                }
              }
            }
          }
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] *= inv;
          if (!on) continue;
          if (!whole) {
#pragma unroll
            for (int e = 0; e < 32; e += 4)
              *reinterpret_cast<float4*>(part + r * HD + i * 32 + e) = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
          } else if constexpr (SPLIT) {
#pragma unroll
            for (int e = 0; e < 32; e += 4)
              *reinterpret_cast<float4*>(static_cast<float*>(a.out) + e0 + i * 32 + e) =
                  make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
          } else {
#pragma unroll
            for (int e = 0; e < 32; e += 8)
              *reinterpret_cast<uint4*>(static_cast<__half*>(a.out) + e0 + i * 32 + e) =
                  make_uint4(h2(o[e], o[e + 1]), h2(o[e + 2], o[e + 3]), h2(o[e + 4], o[e + 5]), h2(o[e + 6], o[e + 7]));
          }
        }
        if (!whole && on) *reinterpret_cast<float2*>(part + kTcRows * HD + 2 * r) = make_float2(m, l);
        tc_before();
      }
      if (u_lo == 0 && u_hi < at.units) {
        rec.h = at.h;
        rec.s = at.s;
        rec.t = at.t;
        rec.rows = rows;
        rec.q0 = at.q0;
        rec.slot = slot;
        rec.last = cta_of_unit(sh.u + at.units - 1, sh.total, sh.n);
      }
      n_kv += u_hi - u_lo;
      ++seg_id;
      first_tile = false;
      advance(u_hi);
    }
    if (have && tid == 0) a.split[blockIdx.x] = rec;
  }
  tc_before();
  __syncthreads();
  if (warp == 8) {
    tc_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
  }
}

int launch_page_tc(PageTcArgs a, int hd, bool split, int page_size, cudaStream_t s);
// Pools a tensor map can describe, in pages that hold whole 8-row groups.
inline bool page_tc_ok(const PageView& c, int hd) {
  return (hd == 64 || hd == 128) && c.type_k == B2_F16 && c.type_v == B2_F16 && c.ps_log2 >= 3 &&
         (((int64_t)c.n_pages * c.n_kv) << c.ps_log2) < (int64_t)1 << 31;
}

}  // namespace b2
