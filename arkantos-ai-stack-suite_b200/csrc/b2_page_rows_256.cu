// Page attention of few rows, head_dim 256 (see b2_page_rows.cuh).
#include "b2_page_rows.cuh"

namespace b2 {

int launch_page_rows_256(const PageRowsArgs& a, bool split, int wm, cudaStream_t s) {
  return launch_page_rows_hd<256>(a, split, wm, s);
}

}  // namespace b2
