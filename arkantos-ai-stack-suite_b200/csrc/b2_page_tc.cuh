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
// many cycles of the special-function pipe.  Neither is reached: a unit takes
// some 3500 cycles, the length of a half's own chain of score product,
// maximum, exponentials and second product, of which two run side by side
// (TMEM holds no third half).  2048 tokens over 16384 positions, 32 heads of
// 128: 449 us or 1150 TFLOP/s, the tensor pipe 57 % busy; SPLIT 920 us.  Eight
// prompts of 1500-2048 tokens: 276 us in a short run, 300-310 once a long one
// has lowered the clocks.  Two threads a row (16 softmax warps) shortened the
// chain less than their exchange of maxima cost (274 us against 267, when both
// were measured in one short run).
//
//   warps 0-3, 4-7  softmax of halves 0, 1, and their results
//   warp 8          issues the products from one thread
//   warp 9          brings K and V: one tensor copy per page and 64 dims, the
//                   lanes issuing side by side; pages past the tile's
//                   positions and table entries outside the pool are sent out
//                   of the map's range, which fills zeros
//   warp 10         walks the tiles of the CTA's share and hands them to the
//                   other warps through a short ring in shared memory; brings
//                   the next tile's Q as soon as the last product of this
//                   one's has read it (SPLIT: the softmax warps do, after
//                   their results: both parts need the whole of that space)
//   warp 11         looks over V of units that not every row sees whole
//
// The next tile's first product is issued before this tile's results are out,
// and results leave through shared memory so that a warp writes whole
// segments of rows: with a few units per tile (a prompt of 2000 tokens has 7
// on average) the change of tiles costs as much as the units otherwise.
//
// The running maximum of a row is raised only when it grew by more than 2^8
// (the weights are relative to the old one until then: at most 2^15 with
// their offset of 2^7, inside fp16's range), so O is rarely rescaled.
//
// SPLIT (fp32 queries): q and p as two fp16 parts each, high and remainder,
// two products instead of one; both parts of p take exactly S's columns.  A
// row of q is brought near 2^14 by a power of two first, taken back in its
// scores, so the parts are good for any size of q.
// The tensor pipe cuts its sums to fp32 at every step of 16, so an O that runs
// over all positions loses accuracy with their number (7.8e-6 of the result
// at 8192); after every 3 units SPLIT therefore adds it, rounded, to a sum in
// the workspace and begins anew.
// FULL rounds p once to fp16, an error of the size of the fp16 output's, and
// leaves its sums to the pipe (2.6e-4 of the result with 32768 positions in one
// CTA, 1.0e-3 with 262144).
//
// V rows that a tile must not see are zeroed in shared memory before the
// unit's product, and infinite or NaN values of units that only some rows see
// whole are taken out and added to the rows that see them at the end, so
// nothing masked reaches a row as 0·NaN.
//
// The product warp stays converged and elects a lane at each issue, which
// keeps descriptors in uniform registers: with a branch of one lane around all
// of it a unit took 4800 cycles instead of 4250.  It looks for K and V ahead
// of need and waits for little else than the weights.  The walk over the
// tiles exists once and the code is kept short: with everything inlined in
// every role it was 160 KB, and its fetches showed at every change of tiles.
//
// Every wait is bounded: an expired one records a code in *status and ends
// the other waits; warps leave whole, copies in flight are waited for and TMEM
// is given back.  Parts of split tiles may then never be counted: the
// workspace's counters have to be cleared again.
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
  float scale_log2;       // FULL: scores to exponents; SPLIT: q_mul · 2^c_exp, 1 <= |q_mul| < 2 or 0
  float q_mul;
  int c_exp;
  int box_rows_log2;      // rows of a tensor copy: min(page_size, 128)
  int q_map;              // FULL: Q comes by tensor copies (G divides 128)
  int o_map;              // FULL: results leave by tensor copies (G divides 32)
  int64_t pool_rows;      // rows of the layer's pool
  unsigned* counters;
  float* slots;
  float* sums;            // SPLIT: [ctas][2 halves][hd / 4][128 rows] float4
  int* status;
};

constexpr int kTcRows = 256, kTcBk = 128, kTcThreads = 384;
constexpr float kTcOffset = 7.f, kTcRaise = 8.f;
// SPLIT: units between two additions of O to its fp32 sum.  2, 3, 4, 8 and
// never give 1.0, 1.2, 1.5, 2.0 and 2.2e-6 on a mixed step over 300-2049
// positions, where fp32 arithmetic gives 0.9e-6, in 84, 81, 80, 78 and 72 us;
// over 16384 positions in one CTA, values of one sign, never gives 8.5e-5.
constexpr int kTcFlush = 3;

template <int HD, bool SPLIT>
struct TcSmem {
  static constexpr int half_q = 128 * HD * 2;                        // one fp16 part of a half's queries
  static constexpr int q = 2 * half_q * (SPLIT ? 2 : 1);
  static constexpr int tile = kTcBk * HD * 2;
  static constexpr int stages = HD == 128 ? (SPLIT ? 3 : 4) : 7;
  static constexpr int ctrl = 1024;
  // Results on their way out, 32 rows x 32 columns of fp32 a warp; SPLIT uses
  // the space of the warp's own queries, which are done by then.
  static constexpr int out = SPLIT ? 0 : 8 * 32 * 128;
  static constexpr int bytes = ctrl + q + stages * tile + out + 1024;   // the last for alignment
};

// ---- tcgen05 -------------------------------------------------------------------------------
// Shared-memory descriptors, 128-byte swizzle, 8-row groups 1024 bytes apart.
// The high word is the same for all; the low one is the address in 16-byte
// steps and the distance of 64-value blocks along M or N, which only N-major
// operands use (V: rows are positions, the k of P·V, 64 dims of a row
// contiguous; blocks of 64 dims are 128 rows apart).
constexpr uint32_t kDescHi = (1024 >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t desc_k(uint32_t saddr) { return (saddr >> 4) | (1u << 16); }
__device__ __forceinline__ uint32_t desc_n(uint32_t saddr) { return (saddr >> 4) | ((uint32_t)((kTcBk * 128) >> 4) << 16); }
// fp16 operands, fp32 accumulators, M = 128.
constexpr uint32_t tc_idesc(int n, bool b_n_major) {
  return (1u << 4) | ((b_n_major ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}
__device__ __forceinline__ void tc_mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 x, y;\n\tmov.b64 x, {%1, %3};\n\tmov.b64 y, {%2, %3};\n\tsetp.ne.b32 p, %5, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %4, p;\n\t}\n" ::"r"(d),
      "r"(a), "r"(b), "r"(kDescHi), "r"(idesc), "r"(acc)
      : "memory");
}
__device__ __forceinline__ void tc_mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 y;\n\tmov.b64 y, {%2, %3};\n\tsetp.ne.b32 p, %5, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], y, %4, p;\n\t}\n" ::"r"(d),
      "r"(a), "r"(b), "r"(kDescHi), "r"(idesc), "r"(acc)
      : "memory");
}
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}\n" : "=r"(p));
  return p != 0;
}
__device__ __forceinline__ uint32_t uniform(uint32_t x) { return __shfl_sync(0xffffffffu, x, 0); }
__device__ __forceinline__ void tc_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
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
__device__ __forceinline__ void tmem_ld128(uint32_t t, float* r) {
  uint32_t* u = reinterpret_cast<uint32_t*>(r);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x128.b32 {"
      "%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,"
      "%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,%47,%48,%49,%50,%51,%52,%53,%54,%55,%56,%57,%58,%59,%60,%61,%62,%63,"
      "%64,%65,%66,%67,%68,%69,%70,%71,%72,%73,%74,%75,%76,%77,%78,%79,%80,%81,%82,%83,%84,%85,%86,%87,%88,%89,%90,%91,%92,%93,%94,%95,"
      "%96,%97,%98,%99,%100,%101,%102,%103,%104,%105,%106,%107,%108,%109,%110,%111,%112,%113,%114,%115,%116,%117,%118,%119,%120,%121,%122,%123,%124,%125,%126,%127}, [%128];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7]), "=r"(u[8]),
        "=r"(u[9]), "=r"(u[10]), "=r"(u[11]), "=r"(u[12]), "=r"(u[13]), "=r"(u[14]), "=r"(u[15]), "=r"(u[16]),
        "=r"(u[17]), "=r"(u[18]), "=r"(u[19]), "=r"(u[20]), "=r"(u[21]), "=r"(u[22]), "=r"(u[23]), "=r"(u[24]),
        "=r"(u[25]), "=r"(u[26]), "=r"(u[27]), "=r"(u[28]), "=r"(u[29]), "=r"(u[30]), "=r"(u[31]), "=r"(u[32]),
        "=r"(u[33]), "=r"(u[34]), "=r"(u[35]), "=r"(u[36]), "=r"(u[37]), "=r"(u[38]), "=r"(u[39]), "=r"(u[40]),
        "=r"(u[41]), "=r"(u[42]), "=r"(u[43]), "=r"(u[44]), "=r"(u[45]), "=r"(u[46]), "=r"(u[47]), "=r"(u[48]),
        "=r"(u[49]), "=r"(u[50]), "=r"(u[51]), "=r"(u[52]), "=r"(u[53]), "=r"(u[54]), "=r"(u[55]), "=r"(u[56]),
        "=r"(u[57]), "=r"(u[58]), "=r"(u[59]), "=r"(u[60]), "=r"(u[61]), "=r"(u[62]), "=r"(u[63]), "=r"(u[64]),
        "=r"(u[65]), "=r"(u[66]), "=r"(u[67]), "=r"(u[68]), "=r"(u[69]), "=r"(u[70]), "=r"(u[71]), "=r"(u[72]),
        "=r"(u[73]), "=r"(u[74]), "=r"(u[75]), "=r"(u[76]), "=r"(u[77]), "=r"(u[78]), "=r"(u[79]), "=r"(u[80]),
        "=r"(u[81]), "=r"(u[82]), "=r"(u[83]), "=r"(u[84]), "=r"(u[85]), "=r"(u[86]), "=r"(u[87]), "=r"(u[88]),
        "=r"(u[89]), "=r"(u[90]), "=r"(u[91]), "=r"(u[92]), "=r"(u[93]), "=r"(u[94]), "=r"(u[95]), "=r"(u[96]),
        "=r"(u[97]), "=r"(u[98]), "=r"(u[99]), "=r"(u[100]), "=r"(u[101]), "=r"(u[102]), "=r"(u[103]), "=r"(u[104]),
        "=r"(u[105]), "=r"(u[106]), "=r"(u[107]), "=r"(u[108]), "=r"(u[109]), "=r"(u[110]), "=r"(u[111]), "=r"(u[112]),
        "=r"(u[113]), "=r"(u[114]), "=r"(u[115]), "=r"(u[116]), "=r"(u[117]), "=r"(u[118]), "=r"(u[119]), "=r"(u[120]),
        "=r"(u[121]), "=r"(u[122]), "=r"(u[123]), "=r"(u[124]), "=r"(u[125]), "=r"(u[126]), "=r"(u[127])
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

// Two fp32 operations in one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n\t.reg .b64 x, y, z, r;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\t"
      "fma.rn.f32x2 r, x, y, z;\n\tmov.b64 {%0, %1}, r;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 x, y, r;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\t"
      "add.rn.f32x2 r, x, y;\n\tmov.b64 {%0, %1}, r;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
// Maxima that keep a NaN, so that a row with a NaN score becomes NaN whole.
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ void tma_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(
          dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z)
      : "memory");
}
// Shared memory to a tensor, and the waits for a thread's stores: until their
// shared memory has been read, until they are done.
__device__ __forceinline__ void tma_store_3d(const CUtensorMap* map, int x, int y, int z, uint32_t src) {
  asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%2, %3, %4}], [%1];\n\t"
               "cp.async.bulk.commit_group;" ::"l"(reinterpret_cast<uint64_t>(map)),
               "r"(src), "r"(x), "r"(y), "r"(z)
               : "memory");
}
__device__ __forceinline__ void tma_store_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
__device__ __forceinline__ void tma_store_done() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }

// A tile of the CTA's share as the warps see it.
struct TcTile {
  int h, s, q0, first;            // kv head, sequence; its first new token's row and position
  int row0, rows;                 // first row (of the sequence's) and rows of the tile
  int key0, units;                // first position and units of this CTA's part; units = 0: no more tiles
  int lo, hi, p_min, p_max;       // positions attended to; those of the first and last row
  Split split;                    // of a tile that other CTAs share
};
static_assert(sizeof(TcTile) == 64, "four 16-byte words");
constexpr int kTcTiles = 4;       // ring of tiles

// Whether some row of the tile does not see the unit at key0 whole.
__device__ __forceinline__ bool tc_edge(const TcTile& t, int key0, int window) {
  return key0 + kTcBk > t.hi || key0 + kTcBk - 1 > t.p_min || (window > 0 && key0 <= t.p_max - window);
}

template <int HD, bool SPLIT>
__global__ void __launch_bounds__(kTcThreads, 1)
    page_tc_kernel(const PageTcArgs a, const __grid_constant__ CUtensorMap k_map,
                   const __grid_constant__ CUtensorMap v_map, const __grid_constant__ CUtensorMap q_map,
                   const __grid_constant__ CUtensorMap o_map) {
  using L = TcSmem<HD, SPLIT>;
  constexpr int NS = L::stages, PARTS = SPLIT ? 2 : 1;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  // The ring's stages hold K and V of the units in turn; a stage's release is
  // counted by stage, an arrival by unit and operand, so that warp 11, which
  // waits for V alone, meets every phase of the barriers it waits on.
  uint64_t* k_full = reinterpret_cast<uint64_t*>(smem);    // [NS]
  uint64_t* v_full = k_full + NS;                          // [NS]
  uint64_t* kv_empty = v_full + NS;                        // [NS]
  uint64_t* v_ok = kv_empty + NS;                          // [NS], by unit: V has been looked over
  uint64_t* q_full = v_ok + NS;                            // [2]
  uint64_t* s_full = q_full + 2;                           // [2]
  uint64_t* p_full = s_full + 2;                           // [2] first 64 positions, [2] the others
  uint64_t* o_full = p_full + 4;                           // [2]
  uint64_t* q_empty = o_full + 2;                          // [2]
  uint64_t* t_full = q_empty + 2;                          // [kTcTiles]
  uint64_t* t_empty = t_full + kTcTiles;                   // [kTcTiles]
  uint64_t* done = t_empty + kTcTiles;                     // [1]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + 512);
  int* abort_flag = reinterpret_cast<int*>(smem + 516);
  int* bad_seen = reinterpret_cast<int*>(smem + 520);      // 1 + the last tile with values taken out of V
  TcTile* tiles = reinterpret_cast<TcTile*>(smem + 640);   // [kTcTiles]
  uint8_t* Qs = smem + L::ctrl;                            // [half][part][hd/64][128 rows][128 B]
  uint8_t* Ts = Qs + L::q;                                 // ring of K and V tiles [hd/64][128 rows][128 B]
  static_assert(8 * (4 * NS + 15 + 2 * kTcTiles) <= 512 && 640 + kTcTiles * 64 <= L::ctrl, "control block");

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (int i = 0; i < NS; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&v_full[i], 1);
      mbar_init(&v_ok[i], 32);
      mbar_init(&kv_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_full[i], SPLIT ? 128 : a.q_map ? 1 : 32);
      mbar_init(&q_empty[i], 1);
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 128);
      mbar_init(&p_full[2 + i], 128);
      mbar_init(&o_full[i], 1);
    }
    for (int i = 0; i < kTcTiles; ++i) {
      mbar_init(&t_full[i], 1);
      mbar_init(&t_empty[i], 11);   // warps 0-9 and 11
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
  if (warp == 9 && lane < 4)
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(lane == 0   ? &k_map
                                                                              : lane == 1 ? &v_map
                                                                              : lane == 2 ? &q_map
                                                                                          : &o_map))
                 : "memory");
  pdl_wait();
  const PageWork& w = a.w;
  sum_units(w, reinterpret_cast<int*>(Ts));
  tc_before();
  __syncthreads();   // barriers, the TMEM address, the sums
  tc_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(tmem_slot);
  pdl_launch_dependents();   // only now: a later kernel must not take the TMEM before this CTA has it

  // A wait of one thread; after one in the CTA has expired all others return.
  // Lanes may learn of that at different polls, so a warp votes before any of
  // them leaves a loop: what follows asks for all 32.
  auto wait = [&](uint64_t* bar, uint32_t parity, int code) -> bool {
    for (int i = 0; !mbar_try_wait(bar, parity); ++i)
      if (i == kWaitPolls || *reinterpret_cast<volatile int*>(abort_flag)) {
        *reinterpret_cast<volatile int*>(abort_flag) = 1;
        if (a.status) atomicExch(a.status, code);
        return false;
      }
    return true;
  };
  auto warp_wait = [&](uint64_t* bar, uint32_t parity, int code) -> bool {
    return __all_sync(0xffffffffu, wait(bar, parity, code));
  };
  // The n-th tile of the share, copied out of the ring (whole warps).
  auto take_tile = [&](int n, TcTile& t) -> bool {
    if (!warp_wait(&t_full[n % kTcTiles], (n / kTcTiles) & 1, 90)) return false;
    const int4* src = reinterpret_cast<const int4*>(&tiles[n % kTcTiles]);
    int4* dst = reinterpret_cast<int4*>(&t);
#pragma unroll
    for (int i = 0; i < 4; ++i) dst[i] = src[i];
    __syncwarp();
    if (lane == 0) mbar_arrive(&t_empty[n % kTcTiles]);
    return t.units > 0;
  };

  // Registers move from the last four warps to the softmax warps: 2 x 200 + 104
  // a lane of each scheduler, the 3 x 168 of the launch.
  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 104;");
    if (warp == 9) {
      // ---------------- K and V ----------------
      // the sums gave way to the ring once warp 10 has its share, which the
      // first tile tells
      const int per = 128 >> a.box_rows_log2;              // copies of 64 dims per operand
      const int rows_box = 1 << a.box_rows_log2;
      const int bx = lane % per, bh = lane / per;          // this lane's copy: rows bx·rows_box, dims 64·bh
      int n = 0;
      bool ok = true;
      TcTile t;
      for (int nt = 0; ok && take_tile(nt, t); ++nt) {
        if (nt == 0) fence_async_proxy();
        // the unit's row in the pool; looked up a unit ahead
        auto look_up = [&](int u) {
          const int p = t.key0 + u * kTcBk + bx * rows_box;
          int64_t row = -1;
          if (bh < HD / 64 && p < t.hi && p + rows_box > t.lo) row = page_row(w.b, a.c, t.s, t.h, p);
          return (int)(row < 0 ? a.pool_rows : row);
        };
        int next_y = look_up(0);
        for (int u = 0; ok && u < t.units; ++u) {
          const int y = next_y;
          if (u + 1 < t.units) next_y = look_up(u + 1);
#pragma unroll
          for (int kv = 0; kv < 2; ++kv, ++n) {
            const int st = n % NS;
            uint64_t* full = (kv ? v_full : k_full) + (n / 2) % NS;
            if (n >= NS) ok = warp_wait(&kv_empty[st], ((n / NS) - 1) & 1, 50);
            if (!ok) break;
            if (lane == 0) mbar_arrive_expect_tx(full, L::tile);
            __syncwarp();
            if (bh < HD / 64)
              tma_2d(smem_u32(Ts + st * L::tile + bh * (kTcBk * 128) + bx * rows_box * 128), kv ? &v_map : &k_map,
                     bh * 64, y, full);
          }
        }
        __syncwarp();
      }
      // every copy issued has landed before the CTA may end
      for (int i = max(0, n - NS); i < n; ++i)
        mbar_wait_bounded(((i & 1) ? v_full : k_full) + (i / 2) % NS, (i / 2 / NS) & 1, a.status, 51);
    } else if (warp == 10) {
      // ---------------- tiles, Q (FULL) ----------------
      Share sh;
      const bool have = find_share(w, blockIdx.x, gridDim.x, reinterpret_cast<const int*>(Ts), sh);
      if (!have) sh.u = sh.u_end = 0;
      __syncwarp();   // the sums are read: the ring may take their place
      constexpr int LR = HD / 8, RI = 32 / LR;   // lanes per row of Q, rows per step
      const int ch = lane % LR, rl = lane / LR;
      const int G = (int)w.G.d, step_tok = w.G.div(RI), step_g = RI - step_tok * G;
      int fills[2] = {0, 0};
      bool ok = true;
      for (int nt = 0; ok; ++nt) {
        if (nt >= kTcTiles) ok = warp_wait(&t_empty[nt % kTcTiles], (nt / kTcTiles - 1) & 1, 91);
        if (!ok) break;
        TcTile t = {};
        const bool more = sh.u < sh.u_end;
        if (more) {
          const TileAt& at = sh.at;
          const int u_hi = min(at.units, sh.off + (sh.u_end - sh.u));
          t.h = at.h;
          t.s = at.s;
          t.q0 = at.q0;
          t.first = at.first;
          t.row0 = at.t * kTcRows;
          t.rows = min(kTcRows, at.rows_total - t.row0);
          t.key0 = (at.lo_unit + sh.off) * kTcBk;
          t.units = u_hi - sh.off;
          t.lo = at.lo;
          t.hi = at.hi;
          t.p_min = at.first + w.G.div(t.row0);
          t.p_max = at.first + w.G.div(t.row0 + t.rows - 1);
          t.split = split_of(sh, blockIdx.x, u_hi);
          sh.u += t.units;
          sh.off = 0;
        }
        if (lane == 0) {
          tiles[nt % kTcTiles] = t;
          mbar_arrive(&t_full[nt % kTcTiles]);
        }
        if (!more) break;
        if constexpr (!SPLIT) {
          const int halves = t.rows > 128 ? 2 : 1;
          if (a.q_map) {
            // 128/G tokens x G heads x 64 dims a copy: the rows' own order.
            // Rows past the sequence are other tokens' and are not written.
            const int z = t.q0 + w.G.div(t.row0), dz = w.G.div(128);
            for (int i = 0; i < halves && ok; ++i) {
              if (fills[i] > 0) ok = warp_wait(&q_empty[i], (fills[i] - 1) & 1, 80);
              if (!ok) break;
              ++fills[i];
              if (lane == 0) mbar_arrive_expect_tx(&q_full[i], L::half_q);
              __syncwarp();
              if (lane < HD / 64)
                tma_3d(smem_u32(Qs) + i * L::half_q + lane * (128 * 128), &q_map, lane * 64, t.h * G, z + i * dz, &q_full[i]);
            }
          } else {
            const __half* src = static_cast<const __half*>(a.q) + ((int64_t)t.q0 * a.n_head + t.h * G) * HD + ch * 8;
            int tok = w.G.div(t.row0 + rl), g = (t.row0 + rl) - tok * G;
            for (int i = 0; i < halves && ok; ++i) {
              if (fills[i] > 0) ok = warp_wait(&q_empty[i], (fills[i] - 1) & 1, 80);
              if (!ok) break;
              ++fills[i];
              const uint32_t qd = smem_u32(Qs) + i * L::half_q + (ch / 8) * (128 * 128);
#pragma unroll 2
              for (int r = rl; r < 128; r += RI) {
                const bool live = i * 128 + r < t.rows;
                cp_async16(qd + r * 128 + (((ch & 7) ^ (r & 7)) << 4),
                           live ? src + ((int64_t)tok * a.n_head + g) * HD : src, live);
                tok += step_tok;
                g += step_g;
                if (g >= G) {
                  g -= G;
                  ++tok;
                }
              }
              cp_async_wait_all();
              fence_async_proxy();
              mbar_arrive(&q_full[i]);
            }
          }
        }
        if (sh.u < sh.u_end) next_tile(w, sh.at);
      }
      // the queries' copies have landed before the CTA may end
      if (!SPLIT && a.q_map)
        for (int i = 0; i < 2; ++i)
          if (fills[i] > 0) mbar_wait_bounded(&q_full[i], (fills[i] - 1) & 1, a.status, 81);
    } else if (warp == 11) {
      // ---------------- V of units that some rows do not see whole ----------------
      int n = 0;
      bool ok = true;
      TcTile t;
      for (int nt = 0; ok && take_tile(nt, t); ++nt) {
        for (int u = 0; ok && u < t.units; ++u, ++n) {
          const int key0 = t.key0 + u * kTcBk;
          ok = warp_wait(&v_full[n % NS], (n / NS) & 1, 71);
          if (!ok) break;
          if (tc_edge(t, key0, w.window)) {
            // zeros where the tile sees nothing; of the others only positions
            // that some row does not see are looked over
            uint8_t* V = Ts + ((2 * n + 1) % NS) * L::tile;
            const int r_hi = max(min(t.hi - key0, kTcBk), 0), r_lo = min(max(t.lo - key0, 0), r_hi);
            const int below = w.window > 0 ? min(max(t.p_max - w.window + 1 - key0, r_lo), r_hi) : r_lo;
            const int above = max(min(t.p_min + 1 - key0, r_hi), below);
#pragma unroll 1
            for (int blk = 0; blk < HD / 64; ++blk) {
              uint4* q = reinterpret_cast<uint4*>(V + blk * (kTcBk * 128));
#pragma unroll 1
              for (int i = lane; i < kTcBk * 8; i += 32)
                if (i < r_lo * 8 || i >= r_hi * 8) q[i] = make_uint4(0, 0, 0, 0);
              uint32_t any = 0;   // bit 15 or 31: an exponent of all ones
#pragma unroll 1
              for (int part = 0; part < 2; ++part) {
                const int i1 = (part ? r_hi : below) * 8;
#pragma unroll 8
                for (int i = (part ? above : r_lo) * 8 + lane; i < i1; i += 32) {
                  const uint4 x = q[i];
                  any |= ((x.x & 0x7FFF7FFFu) + 0x04000400u) | ((x.y & 0x7FFF7FFFu) + 0x04000400u) |
                         ((x.z & 0x7FFF7FFFu) + 0x04000400u) | ((x.w & 0x7FFF7FFFu) + 0x04000400u);
                }
              }
              if (__any_sync(0xffffffffu, (any & 0x80008000u) != 0)) {
                uint32_t* v = reinterpret_cast<uint32_t*>(q);
#pragma unroll 1
                for (int i = r_lo * 32 + lane; i < r_hi * 32; i += 32) {
                  uint32_t x = v[i];
                  if ((x & 0x7C00u) == 0x7C00u) x &= 0xFFFF0000u;
                  if ((x & 0x7C000000u) == 0x7C000000u) x &= 0xFFFFu;
                  v[i] = x;
                }
                *reinterpret_cast<volatile int*>(bad_seen) = nt + 1;
              }
            }
            fence_async_proxy();
          }
          mbar_arrive(&v_ok[n % NS]);
        }
      }
    } else {
      // ---------------- products (a converged warp; one lane issues) ----------------
      // a negative scale negates Q (SPLIT has that in Q already)
      const uint32_t id_s = tc_idesc(128, false) | (!SPLIT && a.scale_log2 < 0.f ? 1u << 13 : 0u);
      constexpr uint32_t id_o = tc_idesc(HD, true);
      const uint32_t q_desc = uniform(desc_k(smem_u32(Qs))), k_desc = uniform(desc_k(smem_u32(Ts))),
                     v_desc = uniform(desc_n(smem_u32(Ts))), tm = uniform(tmem);
      int n = 0, nq[2] = {0, 0}, np[2] = {0, 0};   // ring position; Q and P tiles of each half so far
      bool ok = true;
      auto qk = [&](int i, uint32_t kd) {          // in the elected lane
        const uint32_t qd = q_desc + i * PARTS * (L::half_q >> 4);
        // the remainders first: the sum is cut to fp32 at every step, and these
        // steps' sums are small
#pragma unroll
        for (int part = PARTS - 1; part >= 0; --part)
#pragma unroll
          for (int ks = 0; ks < HD / 16; ++ks) {
            const uint32_t off = ((ks / 4) * (128 * 128) + (ks % 4) * 32) >> 4;
            tc_mma_ss(tm + i * 128, qd + part * (L::half_q >> 4) + off, kd + off, id_s, part != PARTS - 1 || ks != 0);
          }
        tc_commit(&s_full[i]);
      };
      auto pv = [&](int i, uint32_t vd, int h, uint32_t acc) {   // 64 positions; in the elected lane
#pragma unroll
        for (int part = 0; part < PARTS; ++part)
#pragma unroll
          for (int k4 = 0; k4 < 4; ++k4) {
            const int ks = h * 4 + k4;
            const uint32_t p = SPLIT ? (ks / 2) * 32 + part * 16 + (ks & 1) * 8 : ks * 8;
            tc_mma_ts(tm + 256 + i * 128, tm + i * 128 + p, vd + ks * (2048 >> 4), id_o, (part | k4) ? 1u : acc);
          }
      };
      // S of a tile's first unit
      auto open_tile = [&](const TcTile& t) {
        ok = wait(&k_full[(n / 2) % NS], (n / 2 / NS) & 1, 60);
        const uint32_t kd = uniform(k_desc + (n % NS) * (L::tile >> 4));
#pragma unroll
        for (int i = 0; i < 2; ++i)
          if (i == 0 || t.rows > 128) {
            ok = ok && wait(&q_full[i], nq[i]++ & 1, 61);
            tc_after();
            if (elect_one()) {
              qk(i, kd);
              if (!SPLIT && t.units == 1) tc_commit(&q_empty[i]);
            }
            __syncwarp();
          }
        if (elect_one()) tc_commit(&kv_empty[n % NS]);
        __syncwarp();
        ++n;
        ok = __all_sync(0xffffffffu, ok);
      };
      TcTile t;
      int nt = 0;
      bool have = take_tile(nt++, t);
      if (have) open_tile(t);
      while (ok && have) {
        const bool two = t.rows > 128;
        for (int u = 0; u < t.units; ++u) {
          const int sv = n % NS, sk = (n + 1) % NS;
          const bool more = u + 1 < t.units;
          const uint32_t vd = uniform(v_desc + sv * (L::tile >> 4)), kd = uniform(k_desc + sk * (L::tile >> 4)),
                         add = uniform(SPLIT ? u % kTcFlush != 0 : u > 0);
          // K of the next unit and V of this one came while the softmax ran:
          // these waits are not on its path
          ok = wait(&v_ok[(n / 2) % NS], (n / 2 / NS) & 1, 62) &&
               (!more || wait(&k_full[((n + 1) / 2) % NS], ((n + 1) / 2 / NS) & 1, 65));
#pragma unroll
          for (int i = 0; i < 2; ++i)
            if (i == 0 || two) {
              ok = ok && wait(&p_full[i], np[i] & 1, 63);
              tc_after();
              if (elect_one()) pv(i, vd, 0, add);
              __syncwarp();
              ok = ok && wait(&p_full[2 + i], np[i]++ & 1, 64);
              tc_after();
              if (elect_one()) {
                pv(i, vd, 1, 1u);
                if (i == 1 || !two) tc_commit(&kv_empty[sv]);
                if (more) {
                  qk(i, kd);
                  if (!SPLIT && u + 2 == t.units) tc_commit(&q_empty[i]);
                  if (i == 1 || !two) tc_commit(&kv_empty[sk]);
                } else {
                  tc_commit(&o_full[i]);
                }
              }
              __syncwarp();
            }
          n += more ? 2 : 1;
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
        }
        if (!ok) break;
        have = take_tile(nt++, t);
        if (have) open_tile(t);
      }
      if (elect_one()) tc_commit(done);   // every product has completed before TMEM is given back
      __syncwarp();
      mbar_wait_bounded(done, 0, a.status, 67);
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 200;");
    // ---------------- softmax: a thread owns row 128·half + its lane of TMEM ----------------
    const int half = warp >> 2, r = tid, r_in = tid & 127;   // row of the tile, of the half
    const uint32_t tm = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const uint32_t ts = tm + half * 128, to = tm + 256 + half * 128;
    int n_o = 0, n_s = 0;   // tiles and units of this half so far
    bool ok = true;
    for (int nt = 0; ok; ++nt) {
      // The tile stays in the ring until its results are out: what the units
      // need is in registers, the rest is read where it is used.
      ok = warp_wait(&t_full[nt % kTcTiles], (nt / kTcTiles) & 1, 90);
      if (!ok) break;
      const TcTile& t = tiles[nt % kTcTiles];
      auto leave_tile = [&]() {
        __syncwarp();
        if (lane == 0) mbar_arrive(&t_empty[nt % kTcTiles]);
      };
      const int units = t.units, tile_key0 = t.key0, tile_hi = t.hi;
      if (units == 0) break;
      if (half * 128 >= t.rows) {
        leave_tile();
        continue;
      }
      const bool on = r < t.rows;
      // position, and place in q and out, of a row of the tile
      auto token_of = [&](int row) { return w.G.div(t.row0 + row); };
      auto place_of = [&](int row) {
        const int tok = token_of(row), G = (int)w.G.d;
        return ((int64_t)(t.q0 + tok) * a.n_head + t.h * G + (t.row0 + row - tok * G)) * HD;
      };
      const int p = on ? t.first + token_of(r) : -1;
      // from products to exponents: the product takes the sign, and a masked
      // score of minus infinity must not meet a zero.  SPLIT: a power of two of
      // each row.
      float c = fmaxf(fabsf(a.scale_log2), 1e-30f);
      if constexpr (SPLIT) {
        // ---- the warp's 32 rows of Q, a row (hd 64: two) per step, as two
        // parts, each row times the scale's mantissa and a power of two that
        // brings its largest value near 2^14 ----
        constexpr int LR = HD / 4, RI = 32 / LR, B = 8;
        uint8_t* qd = Qs + half * 2 * L::half_q;
        const int ch = lane % LR;   // 4 values
        uint32_t own_top = 0;       // of the row this thread will own
        const int64_t e0 = place_of(on ? r : 0);
#pragma unroll 1
        for (int it = 0; it < 32 / RI; it += B) {
          float4 x[B];
#pragma unroll
          for (int e = 0; e < B; ++e) {
            const int rl = (it + e) * RI + lane / LR;
            const int64_t at_r = __shfl_sync(0xffffffffu, e0, rl);
            const bool live = __shfl_sync(0xffffffffu, (int)on, rl);
            x[e] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (live) x[e] = __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(a.q) + at_r) + ch);
          }
          // largest magnitudes of the rows, a bound by their upper 16 bits: of two steps at once
          uint32_t pair[B / 2];
#pragma unroll
          for (int e = 0; e < B; e += 2) {
            uint32_t top[2];
#pragma unroll
            for (int i = 0; i < 2; ++i)
              top[i] = max(max(__float_as_uint(fabsf(x[e + i].x)), __float_as_uint(fabsf(x[e + i].y))),
                           max(__float_as_uint(fabsf(x[e + i].z)), __float_as_uint(fabsf(x[e + i].w))));
            if constexpr (LR == 32) {
              pair[e / 2] = __byte_perm(__reduce_max_sync(0xffffffffu, top[0]), __reduce_max_sync(0xffffffffu, top[1]), 0x7632);
            } else {
              pair[e / 2] = __byte_perm(top[0], top[1], 0x7632);
#pragma unroll
              for (int i = 1; i < LR; i <<= 1) pair[e / 2] = __vmaxu2(pair[e / 2], __shfl_xor_sync(0xffffffffu, pair[e / 2], i));
            }
            const uint32_t to_own = RI == 1 ? pair[e / 2] : __shfl_sync(0xffffffffu, pair[e / 2], (lane % RI) * LR);
            if (lane / RI == it + e) own_top = to_own << 16;
            if (lane / RI == it + e + 1) own_top = to_own;
          }
#pragma unroll
          for (int e = 0; e < B; ++e) {
            const int rl = (warp & 3) * 32 + (it + e) * RI + lane / LR;
            const float f = a.q_mul * pow2(q_fit(e & 1 ? pair[e / 2] : pair[e / 2] << 16));
            uint2 hi, lo;
            h2_split(x[e].x * f, x[e].y * f, hi.x, lo.x);
            h2_split(x[e].z * f, x[e].w * f, hi.y, lo.y);
            uint8_t* d = qd + (ch / 16) * (128 * 128) + rl * 128 + ((((ch >> 1) & 7) ^ (rl & 7)) << 4) + (ch & 1) * 8;
            *reinterpret_cast<uint2*>(d) = hi;
            *reinterpret_cast<uint2*>(d + L::half_q) = lo;
          }
        }
        fence_async_proxy();
        mbar_arrive(&q_full[half]);
        c = pow2(min(max(a.c_exp - q_fit(own_top), -120), 120));
      }
      float m = -INFINITY, l = 0.f, m_sum = -INFINITY;   // m_sum: the maximum that the sum is relative to
      // FULL: c is no power of two, so far from zero the rounding of m would be
      // more than an exponent may be off by; there the scores in TMEM are made
      // relative to the maximum first, as the product left both.
      float m_raw = -INFINITY;
      bool far = false;
      float4* sum_row = SPLIT ? reinterpret_cast<float4*>(a.sums) + ((int64_t)blockIdx.x * 2 + half) * (HD / 4) * 128 + r_in : nullptr;
      for (int u = 0; u < units; ++u) {
        const int key0 = tile_key0 + u * kTcBk;
        const bool edge = tc_edge(t, key0, w.window);
        ok = warp_wait(&s_full[half], n_s++ & 1, 70);
        if (!ok) break;
        tc_after();
        if (SPLIT && u > 0 && u % kTcFlush == 0) {   // O of the last units is complete
          const float f = m_sum == -INFINITY ? 0.f : ex2(m_sum - m);
#pragma unroll 1
          for (int i = 0; i < HD / 32; ++i) {
            float o[32];
            tmem_ld32(to + i * 32, o);
            float4 x[8];
            if (u > kTcFlush) {
#pragma unroll
              for (int e = 0; e < 8; ++e) x[e] = __ldcg(sum_row + (i * 8 + e) * 128);
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              float4 y = make_float4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
              if (u > kTcFlush)
                y = make_float4(fmaf(x[e].x, f, y.x), fmaf(x[e].y, f, y.y), fmaf(x[e].z, f, y.z), fmaf(x[e].w, f, y.w));
              __stcg(sum_row + (i * 8 + e) * 128, y);
            }
          }
          m_sum = m;
        }
        bool shifted = false;   // the scores in TMEM are relative to m_raw already
        float s[128];
      [[maybe_unused]] load_scores:
        tmem_ld128(ts, s);
        // this row sees columns [lo, hi)
        const int hi = min(p + 1, tile_hi) - key0, lo = w.window > 0 ? p - w.window + 1 - key0 : 0;
        if (edge) {
#pragma unroll
          for (int i = 0; i < 128; ++i)
            if (i >= hi) s[i] = -INFINITY;
          if (w.window > 0) {
#pragma unroll
            for (int i = 0; i < 128; ++i)
              if (i < lo) s[i] = -INFINITY;
          }
        }
        float top[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
        for (int i = 4; i < 124; i += 8)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            top[e] = max3_nan(top[e], s[i + e], s[i + 4 + e]);

#pragma unroll
        for (int e = 0; e < 4; ++e) top[e] = max_nan(top[e], s[124 + e]);
        const float raw = max_nan(max_nan(top[0], top[1]), max_nan(top[2], top[3])), high = raw * c;
        // both roundings towards less, so that no weight passes 2^15 where the
        // offsets are below the spacing of scores
        bool raise = !(high <= __fadd_rd(m, kTcRaise));   // from -inf, and to NaN, always
        if (!shifted && __any_sync(0xffffffffu, raise || far)) {
          if (!SPLIT && far) raise = raise || raw > m_raw;
          const float nm = raise ? high : m;
          const float f = m == -INFINITY ? 0.f : ex2(SPLIT ? m - nm : (m_raw - (raise ? raw : m_raw)) * c);
          const float g = raise ? f : 1.f;            // the other rows keep their maximum
          if (u > 0) {
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
          if constexpr (!SPLIT) {
            m_raw = raise ? raw : m_raw;
            far = __any_sync(0xffffffffu, fabsf(m) > 4194304.f && m != -INFINITY);
            if (far) {
              float x[16];
#pragma unroll 1
              for (int i = 0; i < 8; ++i) {
                tmem_ld16(ts + i * 16, x);
#pragma unroll
                for (int e = 0; e < 16; ++e) x[e] -= m_raw == -INFINITY ? 0.f : m_raw;
                tmem_st16(ts + i * 16, reinterpret_cast<const uint32_t*>(x));
              }
              tmem_wait_st();
              shifted = true;
              goto load_scores;
            }
          }
        }
        const float rs = __fsub_rd(kTcOffset, m == -INFINITY || shifted ? 0.f : m);
        float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
        for (int h = 0; h < 4; ++h) {
#pragma unroll
          for (int i = h * 32; i < h * 32 + 32; i += 2) {
            const float2 x = fma2(make_float2(s[i], s[i + 1]), make_float2(c, c), make_float2(rs, rs));
            s[i] = ex2(x.x);
            s[i + 1] = ex2(x.y);
            sum[(i >> 1) & 1] = add2(sum[(i >> 1) & 1], make_float2(s[i], s[i + 1]));
          }
          // FULL: 64 columns of weights over S's first 64.  SPLIT: the two
          // parts of 32 positions over their own 32 columns.
          uint32_t ph[16], pl[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            if constexpr (SPLIT)
              h2_split(s[h * 32 + 2 * e], s[h * 32 + 2 * e + 1], ph[e], pl[e]);
            else
              ph[e] = h2(s[h * 32 + 2 * e], s[h * 32 + 2 * e + 1]);
          }
          if constexpr (SPLIT) {
            tmem_st16(ts + h * 32, ph);
            tmem_st16(ts + h * 32 + 16, pl);
          } else {
            tmem_st16(ts + h * 16, ph);
          }
          if (h & 1) {   // 64 positions: their product can begin
            tmem_wait_st();
            tc_before();
            mbar_arrive(&p_full[h - 1 + half]);
          }
        }
        l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
      }
      // ---- the result ----
      if (ok) ok = warp_wait(&o_full[half], n_o++ & 1, 72);
      if (!ok) break;
      tc_after();
      const bool whole = t.split.n == 0;
      const int64_t e0 = place_of(on ? r : 0);
      const float inv = !whole ? 1.f : l != 0.f ? 1.f / l : 0.f;
      float* part = a.slots + (int64_t)t.split.slot * slot_floats(kTcRows, HD);
      // Through shared memory, 32 columns at a time: 16-byte chunks of a row,
      // moved so that neither side meets a bank conflict, then segments of rows.
      uint8_t* stage = SPLIT ? Qs + half * 2 * L::half_q + (warp & 3) * 4096 : Ts + NS * L::tile + warp * 4096;
      const bool wide = SPLIT || !whole;   // fp32 out
      // Whole warps of rows of a whole tile leave as a tensor copy of 32/G
      // tokens x G heads x 64 dims.
      const int warp_row = (half * 4 + (warp & 3)) * 32;
      const bool by_copy = !SPLIT && whole && a.o_map && warp_row + 32 <= t.rows;
      if (by_copy) {
#pragma unroll 1
        for (int blk = 0; blk < HD / 64; ++blk) {
          if (lane == 0) tma_store_read();   // the space is free again
          __syncwarp();
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            float o[32];
            tmem_ld32(to + blk * 64 + i * 32, o);
#pragma unroll
            for (int ch = 0; ch < 4; ++ch)
              *reinterpret_cast<uint4*>(stage + lane * 128 + (((i * 4 + ch) ^ (lane & 7)) << 4)) =
                  make_uint4(h2(o[8 * ch] * inv, o[8 * ch + 1] * inv), h2(o[8 * ch + 2] * inv, o[8 * ch + 3] * inv),
                             h2(o[8 * ch + 4] * inv, o[8 * ch + 5] * inv), h2(o[8 * ch + 6] * inv, o[8 * ch + 7] * inv));
          }
          fence_async_proxy();
          __syncwarp();
          if (lane == 0)
            tma_store_3d(&o_map, blk * 64, t.h * (int)w.G.d, t.q0 + token_of(warp_row), smem_u32(stage));
        }
      }
#pragma unroll 1
      for (int i = by_copy ? HD / 32 : 0; i < HD / 32; ++i) {
        float o[32];
        tmem_ld32(to + i * 32, o);
        if (SPLIT && units > kTcFlush) {
          const float f = m_sum == -INFINITY ? 0.f : ex2(m_sum - m);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float4 x = __ldcg(sum_row + (i * 8 + e) * 128);
            o[4 * e] = fmaf(x.x, f, o[4 * e]);
            o[4 * e + 1] = fmaf(x.y, f, o[4 * e + 1]);
            o[4 * e + 2] = fmaf(x.z, f, o[4 * e + 2]);
            o[4 * e + 3] = fmaf(x.w, f, o[4 * e + 3]);
          }
        }
#pragma unroll
        for (int e = 0; e < 32; ++e) o[e] *= inv;
        if (!SPLIT && lane == 0) tma_store_read();   // an earlier tile's copy may still read the space
        __syncwarp();
        if (wide) {
#pragma unroll
          for (int ch = 0; ch < 8; ++ch)
            *reinterpret_cast<float4*>(stage + lane * 128 + ((ch ^ (lane & 7)) << 4)) =
                make_float4(o[4 * ch], o[4 * ch + 1], o[4 * ch + 2], o[4 * ch + 3]);
        } else {
#pragma unroll
          for (int ch = 0; ch < 4; ++ch)
            *reinterpret_cast<uint4*>(stage + lane * 64 + ((ch ^ ((lane >> 1) & 3)) << 4)) =
                make_uint4(h2(o[8 * ch], o[8 * ch + 1]), h2(o[8 * ch + 2], o[8 * ch + 3]),
                           h2(o[8 * ch + 4], o[8 * ch + 5]), h2(o[8 * ch + 6], o[8 * ch + 7]));
        }
        __syncwarp();
        if (wide) {
          const int ch = lane & 7;
#pragma unroll 2
          for (int it = 0; it < 8; ++it) {
            const int rl = it * 4 + (lane >> 3), rt = half * 128 + (warp & 3) * 32 + rl;
            const float4 x = *reinterpret_cast<const float4*>(stage + rl * 128 + ((ch ^ (rl & 7)) << 4));
            const int64_t at_r = __shfl_sync(0xffffffffu, e0, rl);
            float* dst = whole ? static_cast<float*>(a.out) + at_r : part + rt * HD;
            if (rt < t.rows) *reinterpret_cast<float4*>(dst + i * 32 + ch * 4) = x;
          }
        } else {
          const int ch = lane & 3;
#pragma unroll 2
          for (int it = 0; it < 4; ++it) {
            const int rl = it * 8 + (lane >> 2), rt = half * 128 + (warp & 3) * 32 + rl;
            const uint4 x = *reinterpret_cast<const uint4*>(stage + rl * 64 + ((ch ^ ((rl >> 1) & 3)) << 4));
            const int64_t at_r = __shfl_sync(0xffffffffu, e0, rl);
            if (rt < t.rows) *reinterpret_cast<uint4*>(static_cast<__half*>(a.out) + at_r + i * 32 + ch * 8) = x;
          }
        }
      }
      if (!whole && on) *reinterpret_cast<float2*>(part + kTcRows * HD + 2 * r) = make_float2(m, l);
      if (*reinterpret_cast<volatile int*>(bad_seen) > nt) {
        // infinite and NaN values that were taken out of V, to the rows that
        // see them: their weight is positive, so the value decides the sum
        if (lane == 0) tma_store_done();
        __syncwarp();
        for (int u = 0; u < t.units && on; ++u) {
          const int key0 = t.key0 + u * kTcBk;
          if (!tc_edge(t, key0, w.window)) continue;
          const int t1 = min(min(p + 1, t.hi), key0 + kTcBk);
#pragma unroll 1
          for (int pos = max(max(t.lo, key0), w.window > 0 ? p - w.window + 1 : 0); pos < t1; ++pos) {
            const int64_t row = page_row(w.b, a.c, t.s, t.h, pos);
            if (row < 0) continue;
            const __half* v = reinterpret_cast<const __half*>(a.c.v + row * a.c.rb_v);
#pragma unroll 1
            for (int d = 0; d < HD; ++d) {
              const float f = __half2float(v[d]);
              if (fabsf(f) <= 65504.f) continue;
              if (!whole)
                part[r * HD + d] += f;
              else if (SPLIT)
                static_cast<float*>(a.out)[e0 + d] += f;
              else
                static_cast<__half*>(a.out)[e0 + d] =
                    __float2half_rn(__half2float(static_cast<__half*>(a.out)[e0 + d]) + f);
            }
          }
        }
      }
      if (!whole && warp_row < t.rows) {
        if (part_arrives(a.counters + t.split.cta0 * 8 + half * 4 + (warp & 3), t.split.n)) {
          constexpr int R = 16;
#pragma unroll 1
          for (int r0 = 0; r0 < 32 && warp_row + r0 < t.rows; r0 += R)
            join_rows<HD, R>(a.slots, kTcRows, t.split, warp_row + r0, t.rows - warp_row - r0,
                             __shfl_sync(0xffffffffu, e0, (lane + r0) & 31), a.out, SPLIT);
        }
      }
      tc_before();
      leave_tile();
    }
    if (!SPLIT && lane == 0) tma_store_done();   // results are out before the CTA ends
  }
  tc_before();
  __syncthreads();
  if (warp == 8) {
    tc_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
  }
}

int launch_page_tc(PageTcArgs a, int hd, bool split, int page_size, cudaStream_t s);
// The caches this kernel reads.
inline bool page_tc_ok(const PageView& c, int hd) {
  return (hd == 64 || hd == 128) && c.type_k == B2_F16 && c.type_v == B2_F16;
}

}  // namespace b2
