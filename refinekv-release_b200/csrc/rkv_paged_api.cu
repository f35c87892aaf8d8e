// The C entries of the attention over a page pool, and its instances for bf16 pools
// without a cap, a bias, a prefix or weights' sums.
#include <algorithm>
#include <cmath>
#include <string>

#include "rkv_paged_bf16.cuh"

namespace rkv {
void set_last_error(const std::string& message);

namespace {

int reject(int code, const char* message) {
  set_last_error(message);
  return code;
}

int padded(int64_t dim) { return static_cast<int>((dim + 63) / 64 * 64); }

PagedLayout bf16_layout(int64_t group, int64_t dim, int sms) {
  const auto by_group = [&](auto one, auto two) {
    return group <= 8 ? pool_layout<decltype(one)>(sms) : pool_layout<decltype(two)>(sms);
  };
  switch (padded(dim)) {
    case 64: return by_group(Bf16Pool<64, 1>{}, Bf16Pool<64, 2>{});
    case 128: return by_group(Bf16Pool<128, 1>{}, Bf16Pool<128, 2>{});
    case 192: return by_group(Bf16Pool<192, 1>{}, Bf16Pool<192, 2>{});
    default: return by_group(Bf16Pool<256, 1>{}, Bf16Pool<256, 2>{});
  }
}

size_t workspace_size(int64_t group, int64_t head_dim, bool fp4) {
  int sms = 0;
  if (group < 1 || group > kMaxGroup || head_dim < 32 || head_dim > 256 || head_dim % 32 ||
      device_sms(&sms) != RKV_OK || sms > kMostCtas) {
    return 0;
  }
  return (fp4 ? fp4_layout(group, head_dim, sms) : bf16_layout(group, head_dim, sms)).bytes;
}

// A call checked, and what its launch takes.
struct Prepared {
  PagedParams p;
  PagedMaps maps;  // of bf16 pools
  int D, ctas;
  bool nothing;  // no sequences
};

int prepare(const rkv_paged_args* a, bool fp4, Prepared* out) {
  if (a->head_dim < 32 || a->head_dim > 256 || a->head_dim % 32 != 0) {
    return reject(RKV_ERR_UNSUPPORTED, "head_dim must be a multiple of 32 in [32, 256]");
  }
  if (a->block_size != 16 && a->block_size != 32 && a->block_size != 64) {
    return reject(RKV_ERR_UNSUPPORTED, "block_size must be 16, 32 or 64");
  }
  if (a->group < 1 || a->group > kMaxGroup) {
    return reject(RKV_ERR_UNSUPPORTED, "group must be 1..16");
  }
  if (a->sequences < 0 || a->sequences > kMostSequences || a->kv_heads < 1 ||
      a->kv_heads > kMostPagedHeads) {
    return reject(RKV_ERR_UNSUPPORTED, "at most 4096 sequences and 4096 KV heads");
  }
  if (a->query_dtype != RKV_DTYPE_BF16 && a->query_dtype != RKV_DTYPE_F32) {
    return reject(RKV_ERR_INVALID_ARGUMENT, "query dtype must be bf16 or fp32");
  }
  if (a->window < 0 || a->table_blocks < 0 ||
      a->table_blocks > kMostPagedTokens / a->block_size || a->page_table_stride < 0 ||
      a->pool_pages < 0 || a->pool_pages > (1LL << 31) - 1) {
    return reject(RKV_ERR_INVALID_ARGUMENT, "window, page table or pool sizes are out of range");
  }
  const int D = padded(a->head_dim), R = fp4 ? kFp4Rows : tile_rows(D);
  const int64_t tiles = a->sequences * a->kv_heads * ((a->table_blocks * a->block_size + R - 1) / R);
  if (tiles > (1LL << 31) - 1) {  // a product below 2^13 * 2^12 * 2^25
    return reject(RKV_ERR_UNSUPPORTED, "the page table covers more rows than are counted");
  }
  out->nothing = a->sequences == 0;
  if (out->nothing) return RKV_OK;
  if (!a->query || !a->output || !a->lengths || !a->key_pool || !a->value_pool ||
      !a->page_table) {
    return reject(RKV_ERR_INVALID_ARGUMENT,
                  "query, output, pools, page_table and lengths must be non-null");
  }
  if (a->pool_pages < 1) return reject(RKV_ERR_INVALID_ARGUMENT, "the pool has no pages");
  if (a->workspace == nullptr || a->workspace_size < static_cast<int64_t>(kHeader)) {
    return reject(RKV_ERR_WORKSPACE, "workspace is missing or too small");
  }
  const int width = a->query_dtype == RKV_DTYPE_F32 ? 4 : 2, pool_width = fp4 ? 1 : 2;
  uintptr_t bits = reinterpret_cast<uintptr_t>(a->query) | reinterpret_cast<uintptr_t>(a->output);
  bits |= reinterpret_cast<uintptr_t>(a->key_pool) | reinterpret_cast<uintptr_t>(a->value_pool);
  for (int64_t s : a->query_strides) bits |= static_cast<uintptr_t>(s * width);
  for (int i = 0; i < (fp4 ? 2 : 3); ++i) {
    bits |= static_cast<uintptr_t>(a->key_pool_strides[i] * pool_width);
    bits |= static_cast<uintptr_t>(a->value_pool_strides[i] * pool_width);
  }
  if (bits & 15u) {
    return reject(RKV_ERR_ALIGNMENT, "pointers and strides must be 16-byte aligned");
  }
  if (!aligned_to(4, {a->page_table, a->lengths, a->lse})) {
    return reject(RKV_ERR_ALIGNMENT,
                  "page_table, lengths and lse must be aligned to their elements");
  }
  int rc = RKV_OK, sms = 0;
  const int box_rows = static_cast<int>(std::min<int64_t>(R, a->block_size));
  const int64_t *ks = a->key_pool_strides, *vs = a->value_pool_strides;
  if (!fp4 &&
      ((rc = pool_map(&out->maps.keys, a->key_pool, a->head_dim, a->block_size, box_rows,
                      a->kv_heads, a->pool_pages, ks[2], ks[1], ks[0], "key_pool")) != RKV_OK ||
       (rc = pool_map(&out->maps.values, a->value_pool, a->head_dim, a->block_size, box_rows,
                      a->kv_heads, a->pool_pages, vs[2], vs[1], vs[0], "value_pool")) != RKV_OK)) {
    return rc;
  }
  if ((rc = device_sms(&sms)) != RKV_OK) return rc;
  if (sms > kMostCtas) return reject(RKV_ERR_UNSUPPORTED, "more SMs than the workspace counts");
  const PagedLayout layout = fp4 ? fp4_layout(a->group, a->head_dim, sms)
                                 : bf16_layout(a->group, a->head_dim, sms);
  if (a->workspace_size < static_cast<int64_t>(layout.bytes) ||
      (reinterpret_cast<uintptr_t>(a->workspace) & 255u) != 0) {
    return reject(RKV_ERR_WORKSPACE, "workspace is too small or not 256-byte aligned");
  }
  char* ws = static_cast<char*>(a->workspace);
  PagedParams& p = out->p;
  p = {};
  p.query = a->query;
  p.q_seq = a->query_strides[0];
  p.q_head = a->query_strides[1];
  p.query_f32 = a->query_dtype == RKV_DTYPE_F32;
  p.out = a->output;
  p.lse = a->lse;
  p.page_table = a->page_table;
  p.page_table_stride = a->page_table_stride;
  p.lengths = a->lengths;
  p.sequences = static_cast<int>(a->sequences);
  p.heads = static_cast<int>(a->kv_heads);
  p.group = static_cast<int>(a->group);
  p.dim = static_cast<int>(a->head_dim);
  p.block_shift = a->block_size == 16 ? 4 : a->block_size == 32 ? 5 : 6;
  p.capacity = static_cast<int>(a->table_blocks * a->block_size);
  p.pool_pages = static_cast<int>(a->pool_pages);
  p.window = static_cast<int>(std::min<int64_t>(a->window, kMostPagedTokens));
  p.scale = static_cast<float>(a->scale);
  p.status = reinterpret_cast<int*>(ws);
  p.counters = reinterpret_cast<int*>(ws + kCounterBytes);
  p.warp_partials = reinterpret_cast<float*>(ws + layout.warp_partials);
  p.cta_partials = reinterpret_cast<float*>(ws + layout.cta_partials);
  p.group_partials = reinterpret_cast<float*>(ws + layout.group_partials);
  out->D = D;
  out->ctas = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(sms, tiles)));
  return RKV_OK;
}

int launched(cudaError_t err) {
  if (err == cudaSuccess) return RKV_OK;
  set_last_error(std::string("paged attention launch: ") + cudaGetErrorString(err));
  return RKV_ERR_CUDA;
}

}  // namespace

}  // namespace rkv

extern "C" {

size_t rkv_paged_workspace_size(int64_t group, int64_t head_dim) {
  return rkv::workspace_size(group, head_dim, false);
}

size_t rkv_paged_more_workspace_size(int64_t group, int64_t head_dim, int64_t pool_dtype) {
  if (pool_dtype != RKV_DTYPE_BF16 && pool_dtype != RKV_DTYPE_FP4) return 0;
  return rkv::workspace_size(group, head_dim, pool_dtype == RKV_DTYPE_FP4);
}

int rkv_paged_attention(const rkv_paged_args* a, void* stream) {
  using namespace rkv;
  set_last_error("");
  if (a == nullptr) return reject(RKV_ERR_INVALID_ARGUMENT, "args is null");
  Prepared call;
  const int rc = prepare(a, false, &call);
  if (rc != RKV_OK || call.nothing) return rc;
  return launched(
      launch_bf16<false>(call.maps, call.p, call.D, call.ctas, static_cast<cudaStream_t>(stream)));
}

int rkv_paged_attention_more(const rkv_paged_more_args* args, void* stream) {
  using namespace rkv;
  set_last_error("");
  if (args == nullptr) return reject(RKV_ERR_INVALID_ARGUMENT, "args is null");
  const rkv_paged_args* a = &args->base;
  const bool fp4 = args->pool_dtype == RKV_DTYPE_FP4;
  if (!fp4 && args->pool_dtype != RKV_DTYPE_BF16) {
    return reject(RKV_ERR_INVALID_ARGUMENT, "pools are bf16 or fp4");
  }
  if (!fp4 && (args->key_scale != nullptr || args->value_scale != nullptr)) {
    return reject(RKV_ERR_INVALID_ARGUMENT, "scales belong to an fp4 pool");
  }
  const float softcap = static_cast<float>(args->softcap);
  // Below the normal numbers its reciprocal could be infinite.
  if (!(args->softcap == 0 || std::isnormal(softcap)) || softcap < 0.f) {
    return reject(RKV_ERR_INVALID_ARGUMENT, "softcap must be finite and positive, or 0 for none");
  }
  if (args->prefix < 0) return reject(RKV_ERR_INVALID_ARGUMENT, "prefix must not be negative");
  if (!aligned_to(4, {args->slopes, args->key_scale, args->value_scale, args->weights})) {
    return reject(RKV_ERR_ALIGNMENT, "slopes, scales and weights must be aligned to their elements");
  }
  Prepared call;
  int rc = prepare(a, fp4, &call);
  if (rc != RKV_OK || call.nothing) return rc;
  PagedParams& p = call.p;
  p.prefix = static_cast<int>(std::min<int64_t>(args->prefix, kMostPagedTokens));
  p.softcap = softcap;
  p.slopes = args->slopes;
  p.key_scale = args->key_scale;
  p.value_scale = args->value_scale;
  WeightParams w = {};
  if (args->weights != nullptr) {
    if (a->lse == nullptr || args->scores == nullptr) {
      return reject(RKV_ERR_INVALID_ARGUMENT, "weights need lse and scores");
    }
    if (args->weight_width < p.capacity || args->weight_strides[0] < 0 ||
        args->weight_strides[1] < 0) {
      return reject(RKV_ERR_INVALID_ARGUMENT,
                    "a row of weights must hold as many tokens as the page table");
    }
    // At most 2^12 * 2^12 * 2^4 rows of 2^30 tokens.
    const int64_t rows = a->sequences * a->kv_heads * a->group;
    if (p.capacity > 0 && rows > (1LL << 58) / p.capacity) {
      return reject(RKV_ERR_UNSUPPORTED, "more scores than are counted");
    }
    if (args->scores_size < rows * p.capacity * 4) {
      return reject(RKV_ERR_WORKSPACE, "scores are too small");
    }
    if (!aligned_to(16, {args->scores})) {
      return reject(RKV_ERR_ALIGNMENT, "scores must be 16-byte aligned");
    }
    p.scores = args->scores;
    w.weights = args->weights;
    w.seq_stride = args->weight_strides[0];
    w.head_stride = args->weight_strides[1];
  }
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t err;
  if (fp4) {
    Fp4Pages pages = {};
    pages.pool[0] = static_cast<const uint8_t*>(a->key_pool);
    pages.pool[1] = static_cast<const uint8_t*>(a->value_pool);
    for (int i = 0; i < 2; ++i) {
      const int64_t* strides = i ? a->value_pool_strides : a->key_pool_strides;
      if (strides[0] < 0 || strides[1] < 0 || strides[0] >> 36 != 0 || strides[1] >> 36 != 0) {
        return reject(RKV_ERR_UNSUPPORTED, "pool strides must lie below 2^36 bytes");
      }
      pages.page[i] = static_cast<uint32_t>(strides[0] / 16);
      pages.head[i] = static_cast<uint32_t>(strides[1] / 16);
    }
    err = launch_paged_fp4(pages, p, call.ctas, st);
  } else {
    err = launch_paged_more(call.maps, p, call.D, call.ctas, st);
  }
  if (err == cudaSuccess && w.weights != nullptr) err = launch_weights(w, p, st);
  return launched(err);
}

}  // extern "C"
