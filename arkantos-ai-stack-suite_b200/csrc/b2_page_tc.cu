// Launch of the tensor-core page attention (see b2_page_tc.cuh).
#include "b2_page_tc.cuh"

namespace b2 {
namespace {

int encode_map(CUtensorMap* map, const void* base, int rank, const cuuint64_t* dims, const cuuint64_t* strides,
           const cuuint32_t* box) {
  static std::atomic<PFN_cuTensorMapEncodeTiled> found{nullptr};
  PFN_cuTensorMapEncodeTiled fn = found.load(std::memory_order_relaxed);
  if (!fn) {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult qr;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &qr) != cudaSuccess || !p) {
      set_error("page_attn: cuTensorMapEncodeTiled unavailable");
      return B2_ERR_CUDA;
    }
    fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled>(p);
    found.store(fn, std::memory_order_relaxed);
  }
  const cuuint32_t step[3] = {1, 1, 1};
  const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, (cuuint32_t)rank, const_cast<void*>(base), dims, strides,
                        box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                        CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    set_error("page_attn: tensor map rejected (CUresult %d)", (int)r);
    return B2_ERR_CUDA;
  }
  return B2_OK;
}

// Queries or results [n_tok][n_head][hd], copied as `rows` rows (token, head of
// the group) x 64 dims.
int rows_map(const void* q, int hd, int n_head, int n_tok, int G, int rows, CUtensorMap* map) {
  const cuuint64_t dims[3] = {(cuuint64_t)hd, (cuuint64_t)n_head, (cuuint64_t)n_tok};
  const cuuint64_t strides[2] = {(cuuint64_t)hd * 2, (cuuint64_t)n_head * hd * 2};
  const cuuint32_t box[3] = {64, (cuuint32_t)G, (cuuint32_t)(rows / G)};
  return encode_map(map, q, 3, dims, strides, box);
}

template <int HD, bool SPLIT>
int launch(const PageTcArgs& a, const CUtensorMap& km, const CUtensorMap& vm, const CUtensorMap& qm,
           const CUtensorMap& om, cudaStream_t s) {
  auto kern = page_tc_kernel<HD, SPLIT>;
  static std::atomic<int> ready[kMaxDevices];
  int dev = 0;
  B2_CUDA_TRY(cudaGetDevice(&dev));
  B2_CHECK_ARG(dev < kMaxDevices, "device index");
  if (!ready[dev].load(std::memory_order_relaxed)) {
    B2_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, TcSmem<HD, SPLIT>::bytes));
    ready[dev].store(1, std::memory_order_relaxed);
  }
  const int ctas = sm_count();   // one per SM: the kernel takes all of TMEM
  return launch_pdl(kern, dim3(ctas), dim3(kTcThreads), (size_t)TcSmem<HD, SPLIT>::bytes, s, a, km, vm, qm, om);
}

}  // namespace

int page_pool_map(const void* base, int hd, int64_t rows, int box_rows, CUtensorMap* map) {
  const cuuint64_t dims[2] = {(cuuint64_t)hd, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)hd * 2};
  const cuuint32_t box[2] = {64, (cuuint32_t)box_rows};
  return encode_map(map, base, 2, dims, strides, box);
}

int launch_page_tc(PageTcArgs a, int hd, bool split, int page_size, cudaStream_t s) {
  const int box = std::min(page_size, kTcBk);
  a.box_rows_log2 = 0;
  while ((1 << a.box_rows_log2) < box) ++a.box_rows_log2;
  CUtensorMap km, vm, qm = {}, om = {};
  int rc = page_pool_map(a.c.k, hd, a.pool_rows, box, &km);
  if (rc == B2_OK) rc = page_pool_map(a.c.v, hd, a.pool_rows, box, &vm);
  const int G = (int)a.w.G.d;
  a.q_map = !split && 128 % G == 0;
  a.o_map = !split && 32 % G == 0;
  if (rc == B2_OK && a.q_map) rc = rows_map(a.q, hd, a.n_head, a.w.b.n_tok, G, 128, &qm);
  if (rc == B2_OK && a.o_map) rc = rows_map(a.out, hd, a.n_head, a.w.b.n_tok, G, 32, &om);
  if (rc != B2_OK) return rc;
  if (hd == 128) return split ? launch<128, true>(a, km, vm, qm, om, s) : launch<128, false>(a, km, vm, qm, om, s);
  return split ? launch<64, true>(a, km, vm, qm, om, s) : launch<64, false>(a, km, vm, qm, om, s);
}

}  // namespace b2
