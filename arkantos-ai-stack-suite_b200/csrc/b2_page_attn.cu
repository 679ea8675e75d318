// Page attention: the choice of kernel and its launch.
#include <math.h>

#include "b2_page_tc.cuh"

namespace b2 {
namespace {

// Which kernel takes a call, by the most rows a sequence has per kv head (new
// tokens times the query heads that share it).  Up to kFewRows: the few-row
// kernel with its warps along the positions.  More: the tensor-core kernel
// where it reads the cache, else the few-row kernel with its warps along the
// rows.  One kernel takes all sequences of a call: running both, each on the
// sequences of its kind, was slower (a step of 12 single tokens and 4 chunks
// of 129 over 300-2049 positions: 81 us against 47 with fp16 queries in one
// run; 49 now), since the second begins when the first has ended.
constexpr int kFewRows = 16;
struct Plan {
  bool tc, split;
  int wm, rows, bk, max_ctas;
};
Plan plan_of(const PageAttnArgs& a) {
  const int64_t rows = (int64_t)a.b.max_q * (a.n_head / a.c.n_kv);
  const bool f32 = a.type_q == B2_F32;
  Plan p;
  p.tc = rows > kFewRows && page_tc_ok(a.c, a.hd);
  p.split = f32 || (!p.tc && rows <= 8);
  if (p.tc) {
    p.wm = 0;
    p.rows = kTcRows;
    p.bk = kTcBk;
    p.max_ctas = sm_count();
  } else {
    p.wm = rows <= kFewRows ? 1 : 4;
    p.rows = (p.split ? 8 : 16) * p.wm;
    p.bk = kRowsBk;
    p.max_ctas = kPageMaxCtasPerSm * sm_count();
  }
  return p;
}
// Units' time that a warp takes to join a part of a split tile (see find_share).
// One sequence's 8 tokens over 512, 4096 and 16384 fp16 positions, all measured
// in one run: 22, 74 and 65 us when every CTA gets some of them, 19, 33 and 56
// with 0.4 (now 18, 31, 53); 0.25 gives 22, 43, 64, 0.6 19, 37, 59 and 1.5 24,
// 36, 56.  The few-row kernel's units and tiles are smaller: fp32 queries over
// Q8_0 20, 54, 76 against 20, 41, 76 with 0.1 (now 21, 42, 80); 0.4 gives 24,
// 45, 80.
constexpr float kJoinTc = 0.4f, kJoinRows = 0.1f;
PageWork work_of(const PageAttnArgs& a, const Plan& p) {
  PageWork w = {};
  w.b = a.b;
  w.ps_log2 = a.c.ps_log2;
  w.n_kv = a.c.n_kv;
  w.G = FastDiv::of(a.n_head / a.c.n_kv);
  w.window = a.window;
  w.fair = (int)((((int64_t)1 << 31) - 1) / ((int64_t)a.c.n_kv * a.b.n_seq));
  while (w.rows() < p.rows) ++w.rows_log2;
  while (w.bk() < p.bk) ++w.bk_log2;
  if (p.wm != 1) {   // one warp joins 32 rows; with few rows the join is spread over lanes and parts, and cheap
    const int64_t tiles = (int64_t)a.c.n_kv * (a.b.n_seq + (((int64_t)a.b.n_tok * (a.n_head / a.c.n_kv)) >> w.rows_log2));
    w.join_per_tile = (p.tc ? kJoinTc : kJoinRows) / (float)tiles;
  }
  return w;
}

}  // namespace

size_t page_attn_counters(const PageAttnArgs&) { return counter_bytes(kPageMaxCtasPerSm * sm_count()); }

size_t page_attn_workspace(const PageAttnArgs& a) {
  const Plan p = plan_of(a);
  size_t floats = 2 * (size_t)p.max_ctas * slot_floats(p.rows, a.hd);
  if (p.tc && p.split) floats += (size_t)p.max_ctas * p.rows * a.hd;   // the running sums
  return page_attn_counters(a) + floats * 4;
}

int launch_page_attn(const PageAttnArgs& a, cudaStream_t s) {
  const Plan p = plan_of(a);
  // the units of a call are counted in 31 bits
  const int64_t tiles = ((int64_t)a.b.n_tok * (a.n_head / a.c.n_kv)) / p.rows + a.b.n_seq;
  B2_CHECK_ARG(a.c.n_kv * tiles * ((((int64_t)a.b.max_pages << a.c.ps_log2) / p.bk) + 2) < ((int64_t)1 << 31),
               "page_attn: too many tokens for such a long table");
  const int64_t pool_rows = ((int64_t)a.c.n_pages * a.c.n_kv) << a.c.ps_log2;
  B2_CHECK_ARG(pool_rows < ((int64_t)1 << 31), "page_attn: rows of a layer's pool below 2^31");
  const float scale_log2 = (float)((double)a.scale * 1.4426950408889634);
  int c_exp;
  const float q_mul = 2.f * frexpf(scale_log2, &c_exp);
  --c_exp;
  unsigned* counters = reinterpret_cast<unsigned*>(a.ws);
  float* slots = reinterpret_cast<float*>(a.ws + page_attn_counters(a));
  if (p.tc) {
    PageTcArgs t;
    t.c = a.c;
    t.w = work_of(a, p);
    t.q = a.q;
    t.out = a.out;
    t.n_head = a.n_head;
    t.scale_log2 = scale_log2;
    t.q_mul = q_mul;
    t.c_exp = c_exp;
    t.counters = counters;
    t.slots = slots;
    t.sums = slots + 2 * (size_t)p.max_ctas * slot_floats(p.rows, a.hd);
    t.status = a.status;
    t.pool_rows = pool_rows;
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
  r.q_mul = q_mul;
  r.c_exp = c_exp;
  r.counters = counters;
  r.pool_rows = pool_rows;
  r.status = a.status;
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
