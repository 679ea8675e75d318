// Page attention: the choice of kernel, and the kernel that finishes tiles
// split over several CTAs.
#include <math.h>

#include "b2_page_tc.cuh"

namespace b2 {
namespace {

constexpr int kJoinThreads = 128;

// One warp per row of a split tile: its partial results (w_i = 2^(m_i − M))
// added in unit order, divided by the joined sum.  Lanes first share the
// CTAs' (m, l) pairs, then each lane adds its dims over the CTAs.
template <int HD>
__global__ void __launch_bounds__(kJoinThreads)
    page_join_kernel(const PageWork w, const SplitTile* __restrict__ split, const float* __restrict__ slots,
                     int n_head, void* __restrict__ out, int out_f32) {
  pdl_wait();
  pdl_launch_dependents();
  const SplitTile t = split[blockIdx.x];
  if (t.last < 0) return;
  constexpr int V = HD / 32;   // values of a lane
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int n = t.last - (int)blockIdx.x + 1;
  const int64_t slot = (int64_t)slot_floats(w.rows(), HD);
  auto part = [&](int i) { return slots + (i == 0 ? t.slot : 2 * ((int)blockIdx.x + i)) * slot; };
  for (int r = blockIdx.y * (kJoinThreads / 32) + warp; r < t.rows; r += gridDim.y * (kJoinThreads / 32)) {
    float top = -INFINITY;
    for (int i = lane; i < n; i += 32) top = fmaxf(top, part(i)[w.rows() * HD + 2 * r]);
    top = warp_max(top);
    float o[V], sum = 0.f;
#pragma unroll
    for (int e = 0; e < V; ++e) o[e] = 0.f;
    for (int i0 = 0; i0 < n; i0 += 32) {
      float wt = 0.f, l = 0.f;
      if (i0 + lane < n) {
        const float2 ml = *reinterpret_cast<const float2*>(part(i0 + lane) + w.rows() * HD + 2 * r);
        l = ml.y;
        wt = ml.x == -INFINITY ? (l != 0.f ? 1.f : 0.f) : ex2(ml.x - top);   // l != 0 there: only NaN scores
      }
      const int m = min(32, n - i0);
#pragma unroll 4
      for (int i = 0; i < m; ++i) {
        const float wi = __shfl_sync(0xffffffffu, wt, i), li = __shfl_sync(0xffffffffu, l, i);
        const float* p = part(i0 + i) + r * HD + lane;
        if (li != 0.f) {   // a CTA that saw nothing of the row adds nothing
          sum += wi * li;
#pragma unroll
          for (int e = 0; e < V; ++e) o[e] += wi * p[e * 32];
        }
      }
    }
    const float inv = sum != 0.f ? 1.f / sum : 0.f;
    const int rr = (t.t << w.rows_log2) + r, tok = w.G.div(rr), G = (int)w.G.d;
    const int64_t at = ((int64_t)(t.q0 + tok) * n_head + t.h * G + rr - tok * G) * HD + lane;
#pragma unroll
    for (int e = 0; e < V; ++e) {
      if (out_f32)
        static_cast<float*>(out)[at + e * 32] = o[e] * inv;
      else
        static_cast<__half*>(out)[at + e * 32] = __float2half_rn(o[e] * inv);
    }
  }
}

// Which kernel takes a call, by the most rows a sequence has per kv head.
struct Plan {
  bool tc, split;
  int wm, rows, bk, max_ctas;
};
Plan plan_of(const PageAttnArgs& a) {
  const int64_t rows = (int64_t)a.b.max_q * (a.n_head / a.c.n_kv);
  const bool f32 = a.type_q == B2_F32;
  Plan p;
  p.tc = rows > 32 && page_tc_ok(a.c, a.hd);
  p.split = f32 || (!p.tc && rows <= 8);
  if (p.tc) {
    p.wm = 0;
    p.rows = kTcRows;
    p.bk = kTcBk;
    p.max_ctas = sm_count();
  } else {
    p.wm = rows <= (p.split ? 8 : 16) ? 1 : 4;
    p.rows = (p.split ? 8 : 16) * p.wm;
    p.bk = kRowsBk;
    p.max_ctas = kPageMaxCtasPerSm * sm_count();
  }
  return p;
}
PageWork work_of(const PageAttnArgs& a, const Plan& p) {
  PageWork w = {};
  w.b = a.b;
  w.ps_log2 = a.c.ps_log2;
  w.n_kv = a.c.n_kv;
  w.G = FastDiv::of(a.n_head / a.c.n_kv);
  w.window = a.window;
  while (w.rows() < p.rows) ++w.rows_log2;
  while (w.bk() < p.bk) ++w.bk_log2;
  return w;
}

}  // namespace

int launch_page_join(const PageWork& w, const SplitTile* split, const float* slots, int ctas, int hd, int n_head,
                     void* out, bool out_f32, cudaStream_t s) {
  // a CTA of 4 rows per slice: large tiles are finished by many CTAs
  const dim3 grid(ctas, std::min(16, (w.rows() + 3) / 4)), block(kJoinThreads);
#define B2_JOIN(HD) \
  if (hd == HD) return launch_pdl(page_join_kernel<HD>, grid, block, 0, s, w, split, slots, n_head, out, (int)out_f32);
  B2_JOIN(64)
  B2_JOIN(96)
  B2_JOIN(128)
  B2_JOIN(256)
#undef B2_JOIN
  return B2_ERR_UNSUPPORTED;
}

size_t page_attn_workspace(const PageAttnArgs& a) {
  const Plan p = plan_of(a);
  return split_bytes(p.max_ctas) + 2 * (size_t)p.max_ctas * slot_floats(p.rows, a.hd) * 4;
}

int launch_page_attn(const PageAttnArgs& a, cudaStream_t s) {
  const Plan p = plan_of(a);
  // the units of a call are counted in 31 bits
  const int64_t tiles = ((int64_t)a.b.n_tok * (a.n_head / a.c.n_kv)) / p.rows + a.b.n_seq;
  B2_CHECK_ARG(a.c.n_kv * tiles * ((((int64_t)a.b.max_pages << a.c.ps_log2) / p.bk) + 2) < ((int64_t)1 << 31),
               "page_attn: too many tokens for such a long table");
  const float scale_log2 = (float)((double)a.scale * 1.4426950408889634);
  SplitTile* split = reinterpret_cast<SplitTile*>(a.ws);
  float* slots = reinterpret_cast<float*>(a.ws + split_bytes(p.max_ctas));
  if (p.tc) {
    PageTcArgs t;
    t.c = a.c;
    t.w = work_of(a, p);
    t.q = a.q;
    t.out = a.out;
    t.n_head = a.n_head;
    t.scale_log2 = scale_log2;
    t.split = split;
    t.slots = slots;
    t.status = a.status;
    return launch_page_tc(t, a.hd, p.split, 1 << a.c.ps_log2, s);
  }
  PageRowsArgs r;
  r.c = a.c;
  r.w = work_of(a, p);
  r.q = a.q;
  r.out = a.out;
  r.n_head = a.n_head;
  r.q_f32 = a.type_q == B2_F32;
  r.scale_log2 = scale_log2;
  r.split = split;
  r.slots = slots;
  switch (a.hd) {
    case 64: return launch_page_rows_64(r, p.split, p.wm, s);
    case 96: return launch_page_rows_96(r, p.split, p.wm, s);
    case 128: return launch_page_rows_128(r, p.split, p.wm, s);
    case 256: return launch_page_rows_256(r, p.split, p.wm, s);
    default: break;
  }
  set_error("page_attn: head_dim %d (64, 96, 128 and 256 are supported)", a.hd);
  return B2_ERR_UNSUPPORTED;
}

}  // namespace b2
