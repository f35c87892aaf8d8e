// paged_kernel over bf16 pools with a cap, a bias, a prefix or the logits kept, and
// the sums of the weights that tokens get.
//
// Weights: with the logits x_gj of the attention (kept in the call's scratch, fp32)
// and each query's sum lse_g,  W_j += sum_g e^(x_gj - lse_g)  over the queries g of
// the KV head, in this order.  Bound: HBM or L2, 4 (G + 2) bytes a token and KV
// head; the attention writes 4 G of them (128K tokens, 8 KV heads, G 4: 6 us, 25 MB).
#include "rkv_paged_bf16.cuh"

namespace rkv {

cudaError_t launch_paged_more(const PagedMaps& maps, const PagedParams& p, int D, int ctas,
                              cudaStream_t stream) {
  return launch_bf16<true>(maps, p, D, ctas, stream);
}

namespace {

constexpr int kWeightThreads = 256, kWeightTokens = 4;  // of a thread
constexpr int kChunk = kWeightThreads * kWeightTokens;

__global__ void __launch_bounds__(kWeightThreads)
    weights_kernel(const __grid_constant__ WeightParams w, const __grid_constant__ PagedParams p,
                   unsigned each) {
  pdl_wait();
  pdl_launch_dependents();
  const int row = static_cast<int>(blockIdx.x / each), seq = row / p.heads;
  const int part = static_cast<int>(blockIdx.x - static_cast<unsigned>(row) * each);
  const int head = row - seq * p.heads;
  const int length = clamp_length(p, seq);
  const int low = first_visible(p, length), prefix = min(p.prefix, low);
  const float* scores =
      p.scores + static_cast<int64_t>(row) * p.group * p.capacity;
  const float* lse = p.lse + static_cast<int64_t>(row) * p.group;
  float* weights = w.weights + seq * w.seq_stride + head * w.head_stride;
  for (int64_t base = static_cast<int64_t>(part) * kChunk; base < length;
       base += static_cast<int64_t>(each) * kChunk) {
    const int j = static_cast<int>(base) + threadIdx.x * kWeightTokens;
    if (j >= length || (j >= prefix && j + kWeightTokens <= low)) continue;
    float sum[kWeightTokens] = {0.f, 0.f, 0.f, 0.f};
    for (int g = 0; g < p.group; ++g) {
      const float total = lse[g];
      // A query without a finite sum (nothing visible, a NaN, a bad page) adds nothing.
      if (!(fabsf(total) < INFINITY)) continue;
      // The capacity is a multiple of 16 tokens, so the four are the row's own.
      const float4 x = *reinterpret_cast<const float4*>(
          scores + static_cast<int64_t>(g) * p.capacity + j);
      sum[0] += __expf(x.x - total);
      sum[1] += __expf(x.y - total);
      sum[2] += __expf(x.z - total);
      sum[3] += __expf(x.w - total);
    }
#pragma unroll
    for (int i = 0; i < kWeightTokens; ++i) {
      const int at = j + i;
      if (at < length && (at >= low || at < prefix)) weights[at] += sum[i];
    }
  }
}

}  // namespace

cudaError_t launch_weights(const WeightParams& w, const PagedParams& p, cudaStream_t stream) {
  int sms = 0;
  if (device_sms(&sms) != RKV_OK) return cudaErrorInvalidDevice;
  const int64_t rows = static_cast<int64_t>(p.sequences) * p.heads;
  // Enough CTAs to fill the device whatever the number of rows; a row's CTAs
  // take its chunks in turn.
  const int64_t chunks = (p.capacity + kChunk - 1) / kChunk;
  const int64_t each = std::max<int64_t>(1, std::min<int64_t>(chunks, (8 * sms + rows - 1) / rows));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(rows * each));  // at most 2^24 + 8 SMs' worth
  cfg.blockDim = dim3(kWeightThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, weights_kernel, w, p, static_cast<unsigned>(each));
}

}  // namespace rkv
