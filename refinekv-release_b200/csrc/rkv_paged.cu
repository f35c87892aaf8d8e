// Dense attention of one new token per sequence over a page pool.
//
// One CTA per (query head, sequence), four warps: warp w takes the visible
// rows w, w + 4, ... with an online softmax (a lane holds dim / 32 channels),
// and the warps' partials are merged in shared memory.
#include <string>

#include "refinekv_b200.h"
#include "rkv_device.cuh"
#include "rkv_kernels.h"

namespace rkv {
void set_last_error(const std::string& message);

namespace {

constexpr int kWarps = 4;

template <int C>
__global__ void __launch_bounds__(kWarps * 32) paged_kernel(const __grid_constant__ PagedParams p) {
  __shared__ float sm_m[kWarps], sm_l[kWarps], sm_o[kWarps][C * 32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int row = blockIdx.x, seq = blockIdx.y, head = row / p.group;
  int64_t length = p.lengths[seq];
  const int64_t most = p.table_blocks << p.block_shift;
  if (length < 0 || length > most) {
    if (threadIdx.x == 0) atomicOr(p.status, kStatusBadInput);
    length = length < 0 ? 0 : most;
  }
  const int64_t low = p.window > 0 && length > p.window ? length - p.window : 0;
  float q[C], o[C];
#pragma unroll
  for (int i = 0; i < C; ++i) {
    const int64_t at = seq * p.q_seq + row * p.q_head + lane * C + i;
    q[i] = p.query_f32 ? bf16_round(static_cast<const float*>(p.query)[at])
                       : __bfloat162float(static_cast<const __nv_bfloat16*>(p.query)[at]);
    o[i] = 0.f;
  }
  float m = -INFINITY, l = 0.f;
  for (int64_t j = low + warp; j < length; j += kWarps) {
    int64_t page = p.page_table[seq * p.page_table_stride + (j >> p.block_shift)];
    if (page < 0 || page >= p.pool_pages) {
      if (lane == 0) atomicOr(p.status, kStatusBadInput);
      page = 0;
    }
    const int64_t in = j & ((1 << p.block_shift) - 1);
    const __nv_bfloat16* k = p.keys + page * p.k_page + head * p.k_head + in * p.k_row + lane * C;
    const __nv_bfloat16* v = p.values + page * p.v_page + head * p.v_head + in * p.v_row + lane * C;
    float x = 0.f;
#pragma unroll
    for (int i = 0; i < C; ++i) x += q[i] * __bfloat162float(k[i]);
    for (int s = 16; s > 0; s >>= 1) x += __shfl_xor_sync(0xffffffffu, x, s);
    x *= p.scale;
    const float top = fmaxf(m, x), ref = top == -INFINITY ? 0.f : top;
    const float keep = __expf(m - ref), w = __expf(x - ref);
    m = top;
    l = l * keep + w;
#pragma unroll
    for (int i = 0; i < C; ++i) o[i] = o[i] * keep + w * __bfloat162float(v[i]);
  }
  if (lane == 0) {
    sm_m[warp] = m;
    sm_l[warp] = l;
  }
#pragma unroll
  for (int i = 0; i < C; ++i) sm_o[warp][lane * C + i] = o[i];
  __syncthreads();
  float top = -INFINITY, sum = 0.f;
  for (int w = 0; w < kWarps; ++w) top = fmaxf(top, sm_m[w]);
  const float ref = top == -INFINITY ? 0.f : top;
  for (int w = 0; w < kWarps; ++w) sum += sm_l[w] * __expf(sm_m[w] - ref);
  const int64_t out_row = static_cast<int64_t>(seq) * p.heads * p.group + row;
  for (int d = threadIdx.x; d < p.dim; d += blockDim.x) {
    float acc = 0.f;
    for (int w = 0; w < kWarps; ++w) acc += sm_o[w][d] * __expf(sm_m[w] - ref);
    // An empty row is zero; a row whose every logit is -inf is 0 / 0 as the formula has it.
    const float y = length > low ? acc / sum : 0.f;
    if (p.query_f32) static_cast<float*>(p.out)[out_row * p.dim + d] = y;
    else static_cast<__nv_bfloat16*>(p.out)[out_row * p.dim + d] = __float2bfloat16_rn(y);
  }
  if (p.lse != nullptr && threadIdx.x == 0) p.lse[out_row] = ref + logf(sum);
}

template <int C>
cudaError_t launch_c(const PagedParams& p, cudaStream_t stream) {
  paged_kernel<C><<<dim3(p.heads * p.group, p.sequences), kWarps * 32, 0, stream>>>(p);
  return cudaGetLastError();
}

int reject(int code, const char* message) {
  set_last_error(message);
  return code;
}

}  // namespace

cudaError_t launch_paged(const PagedParams& p, cudaStream_t stream) {
  switch (p.dim / 32) {
    case 1: return launch_c<1>(p, stream);
    case 2: return launch_c<2>(p, stream);
    case 3: return launch_c<3>(p, stream);
    case 4: return launch_c<4>(p, stream);
    case 5: return launch_c<5>(p, stream);
    case 6: return launch_c<6>(p, stream);
    case 7: return launch_c<7>(p, stream);
    default: return launch_c<8>(p, stream);
  }
}

}  // namespace rkv

extern "C" {

size_t rkv_paged_workspace_size(int64_t group, int64_t head_dim) {
  if (group < 1 || group > rkv::kMaxGroup || head_dim < 32 || head_dim > 256 || head_dim % 32) {
    return 0;
  }
  return 256;
}

int rkv_paged_attention(const rkv_paged_args* a, void* stream) {
  using namespace rkv;
  set_last_error("");
  if (a == nullptr) return reject(RKV_ERR_INVALID_ARGUMENT, "args is null");
  if (a->head_dim < 32 || a->head_dim > 256 || a->head_dim % 32 != 0) {
    return reject(RKV_ERR_UNSUPPORTED, "head_dim must be a multiple of 32 in [32, 256]");
  }
  if (a->block_size != 16 && a->block_size != 32 && a->block_size != 64) {
    return reject(RKV_ERR_UNSUPPORTED, "block_size must be 16, 32 or 64");
  }
  if (a->group < 1 || a->group > kMaxGroup) {
    return reject(RKV_ERR_UNSUPPORTED, "group must be 1..16");
  }
  if (a->sequences < 0 || a->sequences > 8192 || a->kv_heads < 1 || a->kv_heads > 4096) {
    return reject(RKV_ERR_UNSUPPORTED, "at most 8192 sequences and 4096 KV heads");
  }
  if (a->query_dtype != RKV_DTYPE_BF16 && a->query_dtype != RKV_DTYPE_F32) {
    return reject(RKV_ERR_INVALID_ARGUMENT, "query dtype must be bf16 or fp32");
  }
  if (a->window < 0 || a->table_blocks < 0 || a->table_blocks > (1LL << 31) / a->block_size - 1 ||
      a->page_table_stride < 0 || a->pool_pages < 0 || a->pool_pages > (1LL << 31) - 1) {
    return reject(RKV_ERR_INVALID_ARGUMENT, "window, page table or pool sizes are out of range");
  }
  if (a->sequences == 0) return RKV_OK;
  if (!a->query || !a->output || !a->lengths ||
      (a->table_blocks > 0 && (!a->page_table || !a->key_pool || !a->value_pool))) {
    return reject(RKV_ERR_INVALID_ARGUMENT,
                  "query, output, pools, page_table and lengths must be non-null");
  }
  if (a->table_blocks > 0 && a->pool_pages < 1) {
    return reject(RKV_ERR_INVALID_ARGUMENT, "the pool has no pages");
  }
  const size_t need = rkv_paged_workspace_size(a->group, a->head_dim);
  if (a->workspace == nullptr || a->workspace_size < static_cast<int64_t>(need)) {
    return reject(RKV_ERR_WORKSPACE, "workspace is missing or too small");
  }
  const int width = a->query_dtype == RKV_DTYPE_F32 ? 4 : 2;
  uintptr_t bits = reinterpret_cast<uintptr_t>(a->query) | reinterpret_cast<uintptr_t>(a->output) |
                   reinterpret_cast<uintptr_t>(a->key_pool) |
                   reinterpret_cast<uintptr_t>(a->value_pool);
  for (int64_t s : a->query_strides) bits |= static_cast<uintptr_t>(s * width);
  for (int64_t s : a->key_pool_strides) bits |= static_cast<uintptr_t>(s * 2);
  for (int64_t s : a->value_pool_strides) bits |= static_cast<uintptr_t>(s * 2);
  if (bits & 15u) {
    return reject(RKV_ERR_ALIGNMENT, "pointers and strides must be 16-byte aligned");
  }
  PagedParams p = {};
  p.query = a->query;
  p.q_seq = a->query_strides[0];
  p.q_head = a->query_strides[1];
  p.query_f32 = a->query_dtype == RKV_DTYPE_F32;
  p.out = a->output;
  p.lse = a->lse;
  p.keys = static_cast<const __nv_bfloat16*>(a->key_pool);
  p.values = static_cast<const __nv_bfloat16*>(a->value_pool);
  p.k_page = a->key_pool_strides[0];
  p.k_head = a->key_pool_strides[1];
  p.k_row = a->key_pool_strides[2];
  p.v_page = a->value_pool_strides[0];
  p.v_head = a->value_pool_strides[1];
  p.v_row = a->value_pool_strides[2];
  p.page_table = a->page_table;
  p.page_table_stride = a->page_table_stride;
  p.lengths = a->lengths;
  p.sequences = static_cast<int>(a->sequences);
  p.heads = static_cast<int>(a->kv_heads);
  p.group = static_cast<int>(a->group);
  p.dim = static_cast<int>(a->head_dim);
  p.block_shift = a->block_size == 16 ? 4 : a->block_size == 32 ? 5 : 6;
  p.table_blocks = a->table_blocks;
  p.pool_pages = a->pool_pages;
  p.window = a->window;
  p.scale = static_cast<float>(a->scale);
  p.status = static_cast<int*>(a->workspace);
  const cudaError_t err = launch_paged(p, static_cast<cudaStream_t>(stream));
  if (err != cudaSuccess) {
    set_last_error(std::string("paged attention launch: ") + cudaGetErrorString(err));
    return RKV_ERR_CUDA;
  }
  return RKV_OK;
}

}  // extern "C"
