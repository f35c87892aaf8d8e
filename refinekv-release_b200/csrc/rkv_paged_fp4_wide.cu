// paged_kernel over pools of 4 bits for nine to sixteen queries a KV head.
#include "rkv_paged_fp4.cuh"

namespace rkv {

cudaError_t launch_paged_fp4_wide(const Fp4Pages& pages, const PagedParams& p, int ctas,
                                  cudaStream_t stream) {
  return launch_fp4<2>(pages, p, ctas, stream);
}

}  // namespace rkv
