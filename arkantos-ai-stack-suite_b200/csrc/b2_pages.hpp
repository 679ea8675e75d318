// Paged K/V cache: the structures the page kernels share, and their launchers
// (b2_pages.cu, b2_page_attn*.cu).
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "b2_internal.hpp"
#include "b2_layers.hpp"

namespace b2 {

// A pool and a step's batch, as kernels take them (see b2_page_cache and
// b2_page_batch).  k and v point at the layer the call works on.
struct PageView {
  uint8_t* k = nullptr;
  uint8_t* v = nullptr;
  int32_t n_pages = 0, ps_log2 = 0, n_kv = 0, type_k = 0, type_v = 0, rb_k = 0, rb_v = 0;
};
struct PageSeqs {
  const int32_t* q_start = nullptr;
  const int32_t* kv_len = nullptr;
  const int32_t* table = nullptr;
  int32_t n_seq = 0, max_pages = 0, n_tok = 0, max_q = 0;
};
constexpr int kPageMaxSeq = 1024;   // sequences a call takes (their work is summed in shared memory)

// The new tokens of one sequence: token rows [q0, q0 + len), positions
// [first, kv), every value clamped into the arrays the call was given, so a
// malformed batch cannot send a kernel outside them.
struct SeqSpan {
  int q0, len, kv, first;
};
#if defined(__CUDACC__)
__device__ __forceinline__ SeqSpan seq_span(const PageSeqs& b, int ps_log2, int s) {
  SeqSpan r;
  r.q0 = min(max(b.q_start[s], 0), b.n_tok);
  r.len = max(min(b.q_start[s + 1], b.n_tok) - r.q0, 0);
  r.kv = min(max(b.kv_len[s], 0), b.max_pages << ps_log2);
  r.first = r.kv - r.len;
  return r;
}
// Row (of n_pages · n_kv · page_size rows) of position p of sequence s and kv
// head h, or -1 when the table names no page of the pool.
__device__ __forceinline__ int64_t page_row(const PageSeqs& b, const PageView& c, int s, int h, int p) {
  const int page = __ldg(b.table + (int64_t)s * b.max_pages + (p >> c.ps_log2));
  if ((unsigned)page >= (unsigned)c.n_pages) return -1;
  return (((int64_t)page * c.n_kv + h) << c.ps_log2) + (p & ((1 << c.ps_log2) - 1));
}
#endif

struct RopeStoreArgs {
  PageView c;
  PageSeqs b;
  const void* x = nullptr;         // [n_tok][n_head + 2 n_kv][hd]
  void* q = nullptr;               // [n_tok][n_head][hd]
  const int32_t* pos = nullptr;    // [n_axes][n_tok]
  const uint8_t* axis = nullptr;   // [rot / 2] or null
  const float* rope = nullptr;     // [n_pos][rot]
  int n_head = 0, hd = 0, n_axes = 0, n_pos = 0, rot = 0, style = 0, type_x = 0, type_q = 0;
};
int launch_page_rope_store(const RopeStoreArgs& a, cudaStream_t s);

struct PageAttnArgs {
  PageView c;
  PageSeqs b;
  const void* q = nullptr;
  void* out = nullptr;
  int n_head = 0, hd = 0, type_q = 0, window = 0;
  float scale = 1.0f;
  uint8_t* ws = nullptr;
  int* status = nullptr;
};
// Bytes of the workspace, and of its counters, which come first and are zero
// between calls.
size_t page_attn_workspace(const PageAttnArgs& a);
size_t page_attn_counters(const PageAttnArgs& a);
int launch_page_attn(const PageAttnArgs& a, cudaStream_t s);

// Whole pages src[i] -> dst[i] in every layer; bytes per page and layer of K and V.
int launch_page_copy(uint8_t* k, uint8_t* v, int n_layer, int64_t n_pages, int64_t page_k, int64_t page_v,
                     const int32_t* src, const int32_t* dst, int n, cudaStream_t s);
int launch_page_gather(const PageView& c, int n_layer, const PageSeqs& dst, const int32_t* keep,
                       const int32_t* src_table, cudaStream_t s);

}  // namespace b2
