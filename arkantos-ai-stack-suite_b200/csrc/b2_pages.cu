// Paged K/V cache: rotary positions with several axes and the page store, page
// copies and the gather of kept positions.  The pool of a layer is
// [n_pages][n_kv][page_size] rows (kv_row_bytes each), so the positions of one
// page and head are contiguous.
//
// All three move bytes and do next to no arithmetic: what bounds them is HBM at
// large sizes and the latency of one launch at small ones.
#include "b2_common.cuh"
#include "b2_page_work.cuh"

namespace b2 {
namespace {

// ---- rotary + store ---------------------------------------------------------------------------
// Token i of sequence s sits at cache position p = kv_len[s] − len + i and
// carries one rotary position per axis.  Pair j of a head takes its angle's
// (cos, sin) from row pos[axis[j]][token] of the table:
//   (a, b) -> (a·c − b·n, a·n + b·c), the products and the sum each rounded
// to fp32 as rope_kv_kernel rounds them; (a, b) are values (2j, 2j + 1), or
// (j, j + rot/2) of a head whose halves are paired.  Values past `rot` and
// the v heads pass unchanged.
//
// A CTA takes a few tokens (of a decode step: a share of one token's heads).
// Where they go is looked up once, and their rot/2 (cos, sin) pairs, the same
// for every head, are gathered through the axis map into shared memory.  A
// thread makes 8 values, two runs of 4 half a head apart (or one run, see the
// launch): 16-byte loads, 8- or 16-byte stores, and the 8 threads of a
// 32-value block share its scale by shuffles when the cache is quantized.
// With 4 values a thread and one token a CTA the instructions bound it: 118 us
// for 14192 tokens of 48 heads of 128 whether they came as fp32 or fp16.
// 4 tokens by 128 threads: 86 us (94 % of a plain copy's rate); 1 by 256: 99, 8 by 128: 95.
constexpr int kStoreThreads = 128, kStoreTokens = 4;

template <typename T>
__device__ __forceinline__ float4 load4(const T* p) {
  if constexpr (sizeof(T) == 4) {
    return __ldg(reinterpret_cast<const float4*>(p));
  } else {
    const uint2 w = __ldg(reinterpret_cast<const uint2*>(p));
    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&w.x));
    const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&w.y));
    return make_float4(a.x, a.y, b.x, b.y);
  }
}
__device__ __forceinline__ uint2 half4(float4 v) {
  const __half2 a = __floats2half2_rn(v.x, v.y), b = __floats2half2_rn(v.z, v.w);
  return make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
}

// 4 values y of a cache row at i = 4·(thread's place in the row); for the
// quantized types the 8 lanes of a 32-value block call this together and
// form the codes and the scale that kv_store (b2_layers.cu) forms.
__device__ __forceinline__ void store_row4(uint8_t* row, int type, int hd, int i, float4 y) {
  if (type == B2_F16) {
    if (row) *reinterpret_cast<uint2*>(row + 2 * i) = half4(y);
    return;
  }
  const float v[4] = {y.x, y.y, y.z, y.w};
  const int sub = (i >> 2) & 7;                       // place in the block
  const uint32_t lanes = 0xFFu << (threadIdx.x & 24); // the block's 8 lanes
  if (type == B2_Q8_0) {
    float amax = fmaxf(fmaxf(fabsf(y.x), fabsf(y.y)), fmaxf(fabsf(y.z), fabsf(y.w)));
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) amax = fmaxf(amax, __shfl_xor_sync(lanes, amax, o));
    const float id = amax != 0.0f ? __fdiv_rn(127.0f, amax) : 0.0f;
    uint32_t w = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float t = __fmul_rn(v[e], id);
      int q = __float2int_rz(t >= 0.0f ? __fadd_rn(t, 0.5f) : __fsub_rn(t, 0.5f));
      q = q < -127 ? -127 : (q > 127 ? 127 : q);
      w |= (uint32_t)(uint8_t)(int8_t)q << (8 * e);
    }
    if (!row) return;
    *reinterpret_cast<uint32_t*>(row + i) = w;
    if (sub == 0)
      *reinterpret_cast<uint16_t*>(row + hd + 2 * (i >> 5)) = f2h_rn(__fmul_rn(amax, 1.0f / 127.0f));
    return;
  }
  // Q4_0: the value of largest magnitude, the first such
  float av = 0.0f, mx = 0.0f;
  int idx = 32;
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (fabsf(v[e]) > av) {
      av = fabsf(v[e]);
      mx = v[e];
      idx = 4 * sub + e;
    }
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) {
    const float a2 = __shfl_xor_sync(lanes, av, o), m2 = __shfl_xor_sync(lanes, mx, o);
    const int i2 = __shfl_xor_sync(lanes, idx, o);
    if (a2 > av || (a2 == av && i2 < idx)) {
      av = a2;
      mx = m2;
      idx = i2;
    }
  }
  const float d = __fdiv_rn(mx, -8.0f);
  const float id = d != 0.0f ? __fdiv_rn(1.0f, d) : 0.0f;
  uint32_t w = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int c = __float2int_rz(__fadd_rn(__fmul_rn(v[e], id), 8.5f));
    w |= (uint32_t)(c < 15 ? c : 15) << (8 * e);
  }
  const uint32_t hi = __shfl_down_sync(lanes, w, 4, 8);   // values 16..31 are the high nibbles
  if (!row) return;
  if (sub < 4) *reinterpret_cast<uint32_t*>(row + (i >> 5) * 16 + 4 * sub) = w | (hi << 4);
  if (sub == 0) *reinterpret_cast<uint16_t*>(row + hd / 2 + 2 * (i >> 5)) = f2h_rn(d);
}

template <typename TX, typename TQ, bool PAIR>
__global__ void __launch_bounds__(kStoreThreads)
    page_rope_store_kernel(const RopeStoreArgs a, const int n_here, const FastDiv row_div, const FastDiv head_div) {
  __shared__ __align__(16) float2 cs[kStoreTokens][128];   // rot <= 256
  __shared__ int s_seq[kStoreTokens], s_bad[kStoreTokens];
  __shared__ int64_t s_row[kStoreTokens];    // the position's row of kv head 0; -1: nothing stored, -2: not a token
  pdl_wait();
  pdl_launch_dependents();
  const int tok0 = blockIdx.x * n_here, n = min(n_here, a.b.n_tok - tok0), tid = threadIdx.x;
  const int hd = a.hd, g4 = hd / 4, heads = a.n_head + 2 * a.c.n_kv, half = a.rot / 2, total = heads * g4;
  if (tid < kStoreTokens) {
    s_seq[tid] = -1;
    s_bad[tid] = 0;
  }
  __syncthreads();
  // the tokens' sequences: one parallel look at the boundaries
  for (int s = tid; s < a.b.n_seq; s += kStoreThreads) {
    const int lo = a.b.q_start[s] - tok0, hi = a.b.q_start[s + 1] - tok0;
    for (int t = max(lo, 0); t < min(hi, n); ++t) s_seq[t] = s;
  }
  for (int i = tid; i < n * half; i += kStoreThreads) {
    const int t = i / half, j = i - t * half;
    const int ax = a.axis ? a.axis[j] : 0;
    const int p = ax < a.n_axes ? a.pos[(int64_t)ax * a.b.n_tok + tok0 + t] : -1;
    if (p >= 0 && p < a.n_pos)
      cs[t][j] = reinterpret_cast<const float2*>(a.rope)[(int64_t)p * half + j];
    else
      s_bad[t] = 1;
  }
  __syncthreads();
  if (tid < n) {
    int64_t row = -2;
    if (s_seq[tid] >= 0) {
      const SeqSpan sp = seq_span(a.b, a.c.ps_log2, s_seq[tid]);
      const int p = sp.first + (tok0 + tid - sp.q0);
      row = p >= 0 && !s_bad[tid] ? page_row(a.b, a.c, s_seq[tid], 0, p) : -1;
    }
    s_row[tid] = row;
  }
  __syncthreads();
  // 4 values at i: both of a pair's sides here (style 0), rotated
  auto turn_adjacent = [&](const float2* c, int i, float4 y) {
    const float4 r = *reinterpret_cast<const float4*>(c + i / 2);
    return make_float4(__fsub_rn(__fmul_rn(y.x, r.x), __fmul_rn(y.y, r.y)),
                       __fadd_rn(__fmul_rn(y.x, r.y), __fmul_rn(y.y, r.x)),
                       __fsub_rn(__fmul_rn(y.z, r.z), __fmul_rn(y.w, r.w)),
                       __fadd_rn(__fmul_rn(y.z, r.w), __fmul_rn(y.w, r.z)));
  };
  auto low = [](float a, float b, float c, float n) { return __fsub_rn(__fmul_rn(a, c), __fmul_rn(b, n)); };
  auto high = [](float a, float b, float c, float n) { return __fadd_rn(__fmul_rn(a, n), __fmul_rn(b, c)); };
  const int per_row = PAIR ? total / 2 : total, gw = PAIR ? g4 / 2 : g4;
  for (int i0 = blockIdx.y * kStoreThreads + tid; i0 < n * per_row; i0 += gridDim.y * kStoreThreads) {
    // hd is a multiple of 32 (PAIR: 64), so the 8 threads of a block always run together
    const int t = row_div.div(i0), g = i0 - t * per_row, head = head_div.div(g), i = 4 * (g - head * gw);
    const int64_t row0 = s_row[t];
    if (row0 == -2) continue;   // a row past the last sequence
    const bool live = row0 >= 0;
    const TX* xr = static_cast<const TX*>(a.x) + ((int64_t)(tok0 + t) * heads + head) * hd;
    const int i2 = i + hd / 2;   // PAIR: this thread's other 4 values
    float4 y = load4(xr + i), z = make_float4(0.f, 0.f, 0.f, 0.f);
    if constexpr (PAIR) z = load4(xr + i2);
    if (head < a.n_head + a.c.n_kv) {
      if (a.style == 0) {
        if (i < a.rot) y = turn_adjacent(cs[t], i, y);
        if (PAIR && i2 < a.rot) z = turn_adjacent(cs[t], i2, z);
      } else if (PAIR) {   // rot = hd: (y, z) are the pairs
        const float4 r0 = *reinterpret_cast<const float4*>(&cs[t][i]), r1 = *reinterpret_cast<const float4*>(&cs[t][i + 2]);
        const float4 u = y;
        y = make_float4(low(u.x, z.x, r0.x, r0.y), low(u.y, z.y, r0.z, r0.w), low(u.z, z.z, r1.x, r1.y),
                        low(u.w, z.w, r1.z, r1.w));
        z = make_float4(high(u.x, z.x, r0.x, r0.y), high(u.y, z.y, r0.z, r0.w), high(u.z, z.z, r1.x, r1.y),
                        high(u.w, z.w, r1.z, r1.w));
      } else if (i < a.rot) {
        const bool lo = i < half;
        const int j = lo ? i : i - half;
        const float4 o = load4(xr + (lo ? i + half : j));
        const float4 r0 = *reinterpret_cast<const float4*>(&cs[t][j]), r1 = *reinterpret_cast<const float4*>(&cs[t][j + 2]);
        y = lo ? make_float4(low(y.x, o.x, r0.x, r0.y), low(y.y, o.y, r0.z, r0.w), low(y.z, o.z, r1.x, r1.y),
                             low(y.w, o.w, r1.z, r1.w))
               : make_float4(high(o.x, y.x, r0.x, r0.y), high(o.y, y.y, r0.z, r0.w), high(o.z, y.z, r1.x, r1.y),
                             high(o.w, y.w, r1.z, r1.w));
      }
    }
    if (head < a.n_head) {
      TQ* q = static_cast<TQ*>(a.q) + ((int64_t)(tok0 + t) * a.n_head + head) * hd + i;
      if (!live) y = z = make_float4(0.f, 0.f, 0.f, 0.f);   // no place in the cache, or no angle: a zero q row
      if constexpr (sizeof(TQ) == 4) {
        *reinterpret_cast<float4*>(q) = y;
        if constexpr (PAIR) *reinterpret_cast<float4*>(q + hd / 2) = z;
      } else {
        *reinterpret_cast<uint2*>(q) = half4(y);
        if constexpr (PAIR) *reinterpret_cast<uint2*>(q + hd / 2) = half4(z);
      }
    } else {
      const bool is_v = head >= a.n_head + a.c.n_kv;
      const int kh = head - a.n_head - (is_v ? a.c.n_kv : 0);
      const int rb = is_v ? a.c.rb_v : a.c.rb_k, type = is_v ? a.c.type_v : a.c.type_k;
      uint8_t* row = live ? (is_v ? a.c.v : a.c.k) + (row0 + ((int64_t)kh << a.c.ps_log2)) * rb : nullptr;
      store_row4(row, type, hd, i, y);
      if constexpr (PAIR) store_row4(row, type, hd, i2, z);
    }
  }
}

// ---- page copies ------------------------------------------------------------------------------
// The pairs travel as kernel parameters: no upload, nothing for the stream to
// wait for, and the call can be captured.
constexpr int kCopyPairs = 256, kCopyThreads = 256, kCopyVec = 4;
struct CopyPairs {
  int32_t src[kCopyPairs], dst[kCopyPairs];
};
__global__ void __launch_bounds__(kCopyThreads)
    page_copy_kernel(uint8_t* k, uint8_t* v, int64_t n_pages, int64_t page_k, int64_t page_v,
                     const __grid_constant__ CopyPairs pairs) {
  pdl_wait();
  pdl_launch_dependents();
  const bool is_v = blockIdx.z & 1;
  const int64_t layer = blockIdx.z >> 1, bytes = is_v ? page_v : page_k;
  uint8_t* base = (is_v ? v : k) + layer * n_pages * bytes;
  const uint4* src = reinterpret_cast<const uint4*>(base + pairs.src[blockIdx.y] * bytes);
  uint4* dst = reinterpret_cast<uint4*>(base + pairs.dst[blockIdx.y] * bytes);
  const int64_t n = bytes / 16;
  for (int64_t i0 = (int64_t)blockIdx.x * kCopyThreads * kCopyVec + threadIdx.x; i0 < n;
       i0 += (int64_t)gridDim.x * kCopyThreads * kCopyVec) {
    uint4 w[kCopyVec];
#pragma unroll
    for (int e = 0; e < kCopyVec; ++e)
      if (i0 + e * kCopyThreads < n) w[e] = __ldcs(src + i0 + e * kCopyThreads);
#pragma unroll
    for (int e = 0; e < kCopyVec; ++e)
      if (i0 + e * kCopyThreads < n) dst[i0 + e * kCopyThreads] = w[e];
  }
}

// ---- gather of kept positions -------------------------------------------------------------------
// Row j of sequence s's kept list (position keep[j] of the old table) becomes
// position j − keep_start[s] of the new table, in every layer, for K and V.
// One CTA moves 32 kept positions of one layer's K or V: their old and new
// rows are looked up once for all heads, then each head's rows go as 16-byte
// vectors, consecutive threads along a row and on to the next position, whose
// row follows in memory within a page.
constexpr int kGatherRows = 32, kGatherThreads = 256;
__global__ void __launch_bounds__(kGatherThreads)
    page_gather_kernel(const PageView c, int64_t layer_rows, const PageSeqs b, const int32_t* __restrict__ keep,
                       const int32_t* __restrict__ src_table) {
  __shared__ int64_t from[kGatherRows], to[kGatherRows];
  pdl_wait();
  pdl_launch_dependents();
  const bool is_v = blockIdx.y & 1;
  const int64_t layer = blockIdx.y >> 1;
  const int j0 = blockIdx.x * kGatherRows, tid = threadIdx.x;
  if (tid < kGatherRows) {
    const int j = j0 + tid;
    int64_t f = -1, t = -1;
    if (j < b.n_tok) {
      int lo = 0, hi = b.n_seq;   // the last s with keep_start[s] <= j
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (b.q_start[mid] <= j) lo = mid + 1; else hi = mid;
      }
      const int s = lo - 1;
      if (s >= 0 && j < b.q_start[s + 1]) {
        const int p = keep[j], np = j - b.q_start[s], cap = b.max_pages << c.ps_log2;
        if (p >= 0 && p < cap && np < cap) {
          PageSeqs old = b;
          old.table = src_table;
          f = page_row(old, c, s, 0, p);
          t = page_row(b, c, s, 0, np);
        }
      }
    }
    from[tid] = t >= 0 && t != f ? f : -1;   // a row that stays where it is needs no copy
    to[tid] = t;
  }
  __syncthreads();
  const int rb = is_v ? c.rb_v : c.rb_k, cpr = rb / 16;
  uint8_t* base = (is_v ? c.v : c.k) + layer * layer_rows * rb;
  const int per_head = kGatherRows * cpr, total = c.n_kv * per_head;
  constexpr int U = 4;
  for (int i0 = tid; i0 < total; i0 += U * kGatherThreads) {
    uint4 w[U];
    int64_t dst[U];
#pragma unroll
    for (int e = 0; e < U; ++e) {
      const int i = i0 + e * kGatherThreads;
      dst[e] = -1;
      if (i < total) {
        const int h = i / per_head, r = (i - h * per_head) / cpr, ch = i - h * per_head - r * cpr;
        if (from[r] >= 0) {
          w[e] = *reinterpret_cast<const uint4*>(base + (from[r] + ((int64_t)h << c.ps_log2)) * rb + ch * 16);
          dst[e] = (to[r] + ((int64_t)h << c.ps_log2)) * rb + ch * 16;
        }
      }
    }
#pragma unroll
    for (int e = 0; e < U; ++e)
      if (dst[e] >= 0) *reinterpret_cast<uint4*>(base + dst[e]) = w[e];
  }
}

}  // namespace

int launch_page_rope_store(const RopeStoreArgs& a, cudaStream_t s) {
  // Few tokens: a token's heads are split over up to one CTA per 256 vectors,
  // so that a decode step still covers the SMs.  Many: a CTA takes several
  // tokens and looks their places up at once.
  const int row = (a.n_head + 2 * a.c.n_kv) * a.hd / 4;   // vectors of a token
  const int n_here = a.b.n_tok >= 4 * kStoreTokens * kSMs ? kStoreTokens : 1;
  const int most = (row + kStoreThreads - 1) / kStoreThreads, want = (2 * kSMs + a.b.n_tok - 1) / a.b.n_tok;
  const dim3 grid((a.b.n_tok + n_here - 1) / n_here, std::max(1, std::min(most, want))), block(kStoreThreads);
  // 8 values a thread, a half head apart, where those are whole blocks and hold
  // both sides of a half-split pair; else 4
  const bool pair = a.hd % 64 == 0 && (a.style == 0 || a.rot == a.hd);
  const FastDiv rd = FastDiv::of(pair ? row / 2 : row), hdv = FastDiv::of(pair ? a.hd / 8 : a.hd / 4);
#define B2_STORE(TX, TQ)                                                                                       \
  return pair ? launch_pdl(page_rope_store_kernel<TX, TQ, true>, grid, block, 0, s, a, n_here, rd, hdv)        \
              : launch_pdl(page_rope_store_kernel<TX, TQ, false>, grid, block, 0, s, a, n_here, rd, hdv);
  if (a.type_x == B2_F32) {
    if (a.type_q == B2_F32) B2_STORE(float, float)
    B2_STORE(float, __half)
  }
  if (a.type_q == B2_F32) B2_STORE(__half, float)
  B2_STORE(__half, __half)
#undef B2_STORE
}

int launch_page_copy(uint8_t* k, uint8_t* v, int n_layer, int64_t n_pages, int64_t page_k, int64_t page_v,
                     const int32_t* src, const int32_t* dst, int n, cudaStream_t s) {
  const int64_t vecs = std::max(page_k, page_v) / 16, per = kCopyThreads * kCopyVec;
  const unsigned x = (unsigned)std::min<int64_t>((vecs + per - 1) / per, 64);
  for (int i0 = 0; i0 < n; i0 += kCopyPairs) {
    CopyPairs p;
    const int m = std::min(n - i0, kCopyPairs);
    for (int i = 0; i < m; ++i) {
      p.src[i] = src[i0 + i];
      p.dst[i] = dst[i0 + i];
    }
    for (int i = m; i < kCopyPairs; ++i) p.src[i] = p.dst[i] = 0;
    const int rc = launch_pdl(page_copy_kernel, dim3(x, m, 2 * n_layer), dim3(kCopyThreads), 0, s, k, v, n_pages,
                              page_k, page_v, p);
    if (rc != B2_OK) return rc;
  }
  return B2_OK;
}

int launch_page_gather(const PageView& c, int n_layer, const PageSeqs& dst, const int32_t* keep,
                       const int32_t* src_table, cudaStream_t s) {
  const int64_t layer_rows = ((int64_t)c.n_pages * c.n_kv) << c.ps_log2;
  return launch_pdl(page_gather_kernel, dim3((dst.n_tok + kGatherRows - 1) / kGatherRows, 2 * n_layer),
                    dim3(kGatherThreads), 0, s, c, layer_rows, dst, keep, src_table);
}

}  // namespace b2
