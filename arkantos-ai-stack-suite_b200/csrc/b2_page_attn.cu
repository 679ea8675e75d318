// Page attention: the choice of kernel and its launch.
#include "b2_page_tc.cuh"

namespace b2 {
namespace {

// Which kernel takes a call, by the most rows a sequence has per kv head (new
// tokens times the query heads that share it).  Up to kFewRows: the few-row
// kernel with its warps along the positions.  More: the tensor-core kernel
// where it reads the cache, else the few-row kernel with its warps along the
// rows.  One kernel takes all sequences of a call: running both, each on the
// sequences of its kind, was slower (a step of 12 single tokens and 4 chunks
// of 129 over 300-2049 positions: 81 us against 47 with fp16 queries), since
// the second begins when the first has ended.
constexpr int kFewRows = 16;
// Quantized pages under fp16 queries and more than kFewRows rows: the positions
// that the call attends to are first written to the workspace as fp16 rows,
// rounded once, and the tensor-core kernel reads those (the few-row kernel
// would unpack K and V anew for every 64 rows).  Over Q8_0, with it and
// without: eight prompts 290 us and 2356, a 512-token chunk over 4096
// positions 62 and 317, 8 x 16 tokens over 4096 89 and 107, 5 tokens over 512
// 25 and 27.  The workspace is sized by the table's capacity, hence its bound:
// past it the pages are read as they are.
constexpr int kExpandTile = 64;
constexpr int64_t kExpandBytes = (int64_t)1 << 30;
int64_t expand_bytes(const PageAttnArgs& a) {   // of K or V
  return (((int64_t)a.b.n_seq * a.b.max_pages * a.c.n_kv) << a.c.ps_log2) * a.hd * 2;
}
// Room for the pages' table in front of them.
size_t expand_table_bytes(const PageAttnArgs& a) { return ((size_t)a.b.n_seq * a.b.max_pages * 4 + 255) & ~(size_t)255; }
struct Plan {
  bool tc, split, expand;
  int wm, rows, bk, max_ctas;
};
Plan plan_of(const PageAttnArgs& a) {
  const int64_t rows = (int64_t)a.b.max_q * (a.n_head / a.c.n_kv);
  const bool f32 = a.type_q == B2_F32;
  Plan p;
  p.expand = !f32 && rows > kFewRows && page_tc_hd(a.hd) && !page_tc_ok(a.c, a.hd) && a.c.n_kv < 32768 &&
             2 * expand_bytes(a) <= kExpandBytes;
  p.tc = p.expand || (rows > kFewRows && page_tc_ok(a.c, a.hd));
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
// One sequence's 8 tokens over 512, 4096 and 16384 fp16 positions: 22, 74 and
// 65 us when every CTA gets some of them, 19, 33 and 56 with 0.4; 0.25 gives
// 22, 43, 64, 0.6 19, 37, 59 and 1.5 24, 36, 56.  The few-row kernel's units and
// tiles are smaller: fp32 queries over Q8_0 20, 54, 76 against 20, 41, 76 with
// 0.1; 0.4 gives 24, 45, 80.
constexpr float kJoinTc = 0.4f, kJoinRows = 0.1f;
PageWork work_of(const PageAttnArgs& a, const Plan& p) {
  PageWork w = {};
  w.b = a.b;
  w.ps_log2 = a.c.ps_log2;
  w.n_kv = a.c.n_kv;
  w.G = FastDiv::of(a.n_head / a.c.n_kv);
  w.window = a.window;
  while (w.rows() < p.rows) ++w.rows_log2;
  while (w.bk() < p.bk) ++w.bk_log2;
  if (p.wm != 1) {   // one warp joins 32 rows; with few rows the join is spread over lanes and parts, and cheap
    const int64_t tiles = (int64_t)a.c.n_kv * (a.b.n_seq + (((int64_t)a.b.n_tok * (a.n_head / a.c.n_kv)) >> w.rows_log2));
    w.join_per_tile = (p.tc ? kJoinTc : kJoinRows) / (float)tiles;
  }
  return w;
}

// 16 values of a cache row, as stored.
struct Piece {
  uint4 x0, x1;   // fp16: all; codes: x0
  __half d;       // their block's scale
};
template <int HD>
__device__ __forceinline__ Piece load_piece(const uint8_t* row, int type, int piece) {
  Piece r = {};
  const uint4* x = reinterpret_cast<const uint4*>(row);
  if (type == B2_F16) {
    r.x0 = __ldg(x + 2 * piece);
    r.x1 = __ldg(x + 2 * piece + 1);
    return r;
  }
  const bool q8 = type == B2_Q8_0;
  r.x0 = __ldg(x + (q8 ? piece : piece >> 1));
  r.d = __ldg(reinterpret_cast<const __half*>(row + (q8 ? HD : HD / 2)) + (piece >> 1));
  return r;
}
// -> fp16, each value rounded once (codes are exact in fp16).
__device__ __forceinline__ void piece_values(const Piece& r, int type, int piece, uint32_t (&h)[8]) {
  const uint4& x = r.x0;
  if (type == B2_F16) {
    h[0] = x.x, h[1] = x.y, h[2] = x.z, h[3] = x.w;
    h[4] = r.x1.x, h[5] = r.x1.y, h[6] = r.x1.z, h[7] = r.x1.w;
    return;
  }
  if (type == B2_Q8_0) {
    s8x4_to_h2(x.x, h[0], h[1]);
    s8x4_to_h2(x.y, h[2], h[3]);
    s8x4_to_h2(x.z, h[4], h[5]);
    s8x4_to_h2(x.w, h[6], h[7]);
  } else {   // a block's low nibbles are its first half
    const int sh = (piece & 1) * 4;
    n4x4_to_h2((x.x >> sh) & 0x0F0F0F0Fu, h[0], h[1]);
    n4x4_to_h2((x.y >> sh) & 0x0F0F0F0Fu, h[2], h[3]);
    n4x4_to_h2((x.z >> sh) & 0x0F0F0F0Fu, h[4], h[5]);
    n4x4_to_h2((x.w >> sh) & 0x0F0F0F0Fu, h[6], h[7]);
  }
  const __half2 d = __half2half2(r.d);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const __half2 v = __hmul2(*reinterpret_cast<const __half2*>(&h[i]), d);
    h[i] = *reinterpret_cast<const uint32_t*>(&v);
  }
}

// The attended positions of each sequence as fp16 rows: page s·max_pages + i of
// a pool of the same page size, entered so in the new table.  Entries outside
// the cache's pool become zeros.  A CTA takes 64 positions of one kv head's K
// or V, a thread 16 values of each of PER rows, whose loads are all under way
// before the first is used.
template <int HD>
__global__ void __launch_bounds__(256)
page_expand_kernel(PageView c, PageSeqs b, int window, uint8_t* k, uint8_t* v, int32_t* table) {
  constexpr int PIECES = HD / 16, ROWS = 256 / PIECES, PER = kExpandTile / ROWS;
  pdl_wait();
  pdl_launch_dependents();
  const int s = blockIdx.z, h = blockIdx.y >> 1, p0 = blockIdx.x * kExpandTile;
  const bool is_v = blockIdx.y & 1;
  const SeqSpan q = seq_span(b, c.ps_log2, s);
  const int lo = window > 0 ? max(q.first - window + 1, 0) : 0;
  if (q.len == 0 || p0 >= q.kv || p0 + kExpandTile <= lo) return;
  if (blockIdx.y == 0) {
    const int page = (p0 >> c.ps_log2) + threadIdx.x;
    if (page <= (p0 + kExpandTile - 1) >> c.ps_log2 && page < b.max_pages)
      table[s * b.max_pages + page] = s * b.max_pages + page;
  }
  const int type = is_v ? c.type_v : c.type_k, rb = is_v ? c.rb_v : c.rb_k;
  const uint8_t* pool = is_v ? c.v : c.k;
  const int piece = threadIdx.x % PIECES, p = p0 + threadIdx.x / PIECES;
  int64_t row[PER];
  Piece x[PER] = {};
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int pi = p + i * ROWS;
    row[i] = pi >= lo && pi < q.kv ? page_row(b, c, s, h, pi) : -1;
  }
#pragma unroll
  for (int i = 0; i < PER; ++i)
    if (row[i] >= 0) x[i] = load_piece<HD>(pool + row[i] * rb, type, piece);
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int pi = p + i * ROWS;
    if (pi < lo || pi >= q.kv) continue;
    uint32_t y[8] = {};
    if (row[i] >= 0) piece_values(x[i], type, piece, y);
    const int64_t to = ((((int64_t)s * b.max_pages + (pi >> c.ps_log2)) * c.n_kv + h) << c.ps_log2) +
                       (pi & ((1 << c.ps_log2) - 1));
    uint4* dst = reinterpret_cast<uint4*>((is_v ? v : k) + to * (HD * 2)) + 2 * piece;
    dst[0] = make_uint4(y[0], y[1], y[2], y[3]);
    dst[1] = make_uint4(y[4], y[5], y[6], y[7]);
  }
}

// Expands the call's pages at `at` and has it read those instead.
int expand_pages(PageAttnArgs& a, uint8_t* at, cudaStream_t s) {
  int32_t* table = reinterpret_cast<int32_t*>(at);
  uint8_t* k = at + expand_table_bytes(a);
  uint8_t* v = k + expand_bytes(a);
  const int positions = a.b.max_pages << a.c.ps_log2;
  const dim3 grid((positions + kExpandTile - 1) / kExpandTile, a.c.n_kv * 2, a.b.n_seq);
  const int rc = a.hd == 128
                     ? launch_pdl(page_expand_kernel<128>, grid, dim3(256), 0, s, a.c, a.b, a.window, k, v, table)
                     : launch_pdl(page_expand_kernel<64>, grid, dim3(256), 0, s, a.c, a.b, a.window, k, v, table);
  a.b.table = table;
  a.c.k = k;
  a.c.v = v;
  a.c.n_pages = a.b.n_seq * a.b.max_pages;
  a.c.type_k = a.c.type_v = B2_F16;
  a.c.rb_k = a.c.rb_v = a.hd * 2;
  return rc;
}

size_t own_bytes(const PageAttnArgs& a, const Plan& p) {   // counters and partial results, whole 256 bytes
  size_t floats = 2 * (size_t)p.max_ctas * slot_floats(p.rows, a.hd);
  if (p.tc && p.split) floats += (size_t)p.max_ctas * p.rows * a.hd;   // the running sums
  return (page_attn_counters(a) + floats * 4 + 255) & ~(size_t)255;
}

}  // namespace

size_t page_attn_counters(const PageAttnArgs&) { return counter_bytes(kPageMaxCtasPerSm * sm_count()); }

size_t page_attn_workspace(const PageAttnArgs& a) {
  const Plan p = plan_of(a);
  return own_bytes(a, p) + (p.expand ? expand_table_bytes(a) + 2 * (size_t)expand_bytes(a) : 0);
}

int launch_page_attn(const PageAttnArgs& args, cudaStream_t s) {
  PageAttnArgs a = args;
  const Plan p = plan_of(a);
  // the units of a call are counted in 31 bits
  const int64_t tiles = ((int64_t)a.b.n_tok * (a.n_head / a.c.n_kv)) / p.rows + a.b.n_seq;
  B2_CHECK_ARG(a.c.n_kv * tiles * ((((int64_t)a.b.max_pages << a.c.ps_log2) / p.bk) + 2) < ((int64_t)1 << 31),
               "page_attn: too many tokens for such a long table");
  if (p.expand) {
    const int rc = expand_pages(a, a.ws + own_bytes(a, p), s);
    if (rc != B2_OK) return rc;
  }
  const int64_t pool_rows = ((int64_t)a.c.n_pages * a.c.n_kv) << a.c.ps_log2;
  B2_CHECK_ARG(pool_rows < ((int64_t)1 << 31), "page_attn: rows of a layer's pool below 2^31");
  const float scale_log2 = (float)((double)a.scale * 1.4426950408889634);
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
