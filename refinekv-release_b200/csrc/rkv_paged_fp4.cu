// paged_kernel over pools of 4 bits: up to eight queries a KV head (rkv_paged_fp4_wide.cu
// has the instances for more; they are compiled apart because they take long).
#include "rkv_paged_fp4.cuh"

namespace rkv {

cudaError_t launch_paged_fp4(const Fp4Pages& pages, const PagedParams& p, int ctas,
                             cudaStream_t stream) {
  return p.group <= 8 ? launch_fp4<1>(pages, p, ctas, stream)
                      : launch_paged_fp4_wide(pages, p, ctas, stream);
}

PagedLayout fp4_layout(int64_t group, int64_t dim, int sms) {
  const auto layout = [&](auto pool) { return pool_layout<decltype(pool)>(sms); };
  return group <= 8 ? by_dim<1>(dim, layout) : by_dim<2>(dim, layout);
}

}  // namespace rkv
