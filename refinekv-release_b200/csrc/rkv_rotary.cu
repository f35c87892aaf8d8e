// Rotary positions and the append of new tokens to a page pool.
//
// Both are one pass over rows of head_dim channels: read a row, rotate its
// rotary channels by the position's row of the cos/sin table, write it to a
// tensor or to the pool's page.  Bound: HBM on long inputs (every element
// read once and written once, a few flops per pair), latency on single
// tokens.
//
// A unit of work is 2V channels of one head: for a rotated half-layout unit
// the V channels at c and the V at c + rotary/2 (the two halves of V pairs),
// for an interleaved or copied one 2V consecutive channels.  V is 16 bytes of
// elements, or 1 where strides, alignment or a rotary width that is no
// multiple of 2V forbid 16-byte accesses.
#include <algorithm>
#include <string>

#include "refinekv_b200.h"
#include "rkv_device.cuh"
#include "rkv_kernels.h"

namespace rkv {
void set_last_error(const std::string& message);

namespace {

template <typename T, int V>
struct alignas(V * sizeof(T)) Pack {
  T at[V];
};

__device__ __forceinline__ float widen(float x) { return x; }
__device__ __forceinline__ float widen(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T>
__device__ __forceinline__ T narrow(float x);
template <>
__device__ __forceinline__ float narrow<float>(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 narrow<__nv_bfloat16>(float x) {
  return __float2bfloat16_rn(x);
}

template <typename T, int V>
__device__ __forceinline__ void load_pack(const T* from, float (&x)[V]) {
  const Pack<T, V> p = *reinterpret_cast<const Pack<T, V>*>(from);
#pragma unroll
  for (int i = 0; i < V; ++i) x[i] = widen(p.at[i]);
}

template <typename T, int V>
__device__ __forceinline__ void store_pack(T* to, const float (&x)[V]) {
  Pack<T, V> p;
#pragma unroll
  for (int i = 0; i < V; ++i) p.at[i] = narrow<T>(x[i]);
  *reinterpret_cast<Pack<T, V>*>(to) = p;
}

// V cosines or sines: at most 16 bytes a load.
template <int V>
__device__ __forceinline__ void load_table(const float* from, float (&x)[V]) {
  constexpr int W = V < 4 ? V : 4;
#pragma unroll
  for (int i = 0; i < V; i += W) {
    const Pack<float, W> p = *reinterpret_cast<const Pack<float, W>*>(from + i);
#pragma unroll
    for (int j = 0; j < W; ++j) x[i + j] = p.at[j];
  }
}

// One product pair of the rotation.  Products and sums are rounded one by one
// (no fused multiply-add): the result then depends on nothing but its
// operands, so rotating alone, rotating while appending and the formula in
// fp32 agree bit for bit.
__device__ __forceinline__ void turn(float& a, float& b, float c, float s) {
  const float y = __fsub_rn(__fmul_rn(a, c), __fmul_rn(b, s));
  const float z = __fadd_rn(__fmul_rn(b, c), __fmul_rn(a, s));
  a = y;
  b = z;
}

template <typename T, int V, bool Interleaved, bool Append>
__global__ void __launch_bounds__(512) rows_kernel(const __grid_constant__ RowsParams p) {
  const int per_head = p.dim / (2 * V), turned = p.rotary / (2 * V);
  const int q_units = p.query.heads * per_head, k_units = p.key.heads * per_head;
  const int units = q_units + k_units + (Append ? p.value.heads * per_head : 0);
  pdl_wait();
  pdl_launch_dependents();
  for (int64_t n = blockIdx.x; n < p.batch * p.tokens; n += gridDim.x) {
    const int64_t b = p.batch > 1 ? n / p.tokens : 0, t = n - b * p.tokens;
    const int64_t at = b * p.pos_b + t * p.pos_t;
    const int64_t pos = p.pos_i64 ? static_cast<const int64_t*>(p.positions)[at]
                                  : static_cast<const int32_t*>(p.positions)[at];
    const bool known = p.rotary == 0 || (pos >= 0 && pos < p.table_rows);
    const float* table = p.cos_sin + (known ? pos : 0) * p.table_stride;
    bool keep = true;  // the token's rows go to the pool
    int64_t page = 0, row = 0;
    if (Append) {
      keep = pos >= 0;
      if (keep) {
        const int64_t seq = p.sequence_ids != nullptr ? p.sequence_ids[n] : n;
        const int64_t block = pos >> p.block_shift;
        row = pos - (block << p.block_shift);
        bool ok = known && seq >= 0 && seq < p.sequences && block < p.table_blocks;
        if (ok) {
          page = p.page_table[seq * p.page_table_stride + block];
          ok = page >= 0 && page < p.pool_pages;
        }
        if (!ok) {
          keep = false;
          if (threadIdx.x == 0 && p.status != nullptr) atomicOr(p.status, kStatusBadInput);
        }
      }
    }
    for (int u = threadIdx.x; u < units; u += blockDim.x) {
      const int kind = u < q_units ? 0 : u < q_units + k_units ? 1 : 2;
      const RowStream& s = kind == 0 ? p.query : kind == 1 ? p.key : p.value;
      const int v = u - (kind == 0 ? 0 : kind == 1 ? q_units : q_units + k_units);
      const int h = v / per_head, c = v - h * per_head;
      const bool rotate = c < turned && kind < 2;
      const int first = rotate && !Interleaved ? c * V : c * 2 * V;
      const int second = rotate && !Interleaved ? p.rotary / 2 + c * V : c * 2 * V + V;
      if (Append && kind > 0 && !keep) continue;
      const T* in = static_cast<const T*>(s.in) + b * s.in_b + t * s.in_t + h * s.in_h;
      float x[V], y[V];
      load_pack<T, V>(in + first, x);
      load_pack<T, V>(in + second, y);
      if (rotate) {
        float cs[V], sn[V];
        load_table<V>(table + c * V, cs);
        load_table<V>(table + p.rotary / 2 + c * V, sn);
        if (Interleaved) {
          if constexpr (V == 1) {
            turn(x[0], y[0], cs[0], p.sign * sn[0]);
          } else {
#pragma unroll
            for (int i = 0; i < V / 2; ++i) {
              turn(x[2 * i], x[2 * i + 1], cs[i], p.sign * sn[i]);
              turn(y[2 * i], y[2 * i + 1], cs[V / 2 + i], p.sign * sn[V / 2 + i]);
            }
          }
        } else {
#pragma unroll
          for (int i = 0; i < V; ++i) turn(x[i], y[i], cs[i], p.sign * sn[i]);
        }
        if (!known) {
#pragma unroll
          for (int i = 0; i < V; ++i) x[i] = y[i] = __int_as_float(0x7fc00000);
        }
      }
      if (Append && kind > 0) {
        __nv_bfloat16* out = static_cast<__nv_bfloat16*>(s.out) + page * s.out_b + row * s.out_t +
                             h * s.out_h;
        store_pack<__nv_bfloat16, V>(out + first, x);
        store_pack<__nv_bfloat16, V>(out + second, y);
      } else {
        if (Append && pos < 0) {
#pragma unroll
          for (int i = 0; i < V; ++i) x[i] = y[i] = 0.f;
        }
        T* out = static_cast<T*>(s.out) + b * s.out_b + t * s.out_t + h * s.out_h;
        store_pack<T, V>(out + first, x);
        store_pack<T, V>(out + second, y);
      }
    }
  }
}

template <typename T, int V, bool Interleaved, bool Append>
cudaError_t launch_rows_t(const RowsParams& p, cudaStream_t stream) {
  const int heads = p.query.heads + p.key.heads + (Append ? p.value.heads : 0);
  const int units = heads * (p.dim / (2 * V));
  const int threads = std::min(512, (units + 31) / 32 * 32);
  const int64_t rows = p.batch * p.tokens;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(rows));
  cfg.blockDim = dim3(threads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, rows_kernel<T, V, Interleaved, Append>, p);
}

template <typename T, int V>
cudaError_t launch_rows_v(const RowsParams& p, bool interleaved, bool append, cudaStream_t stream) {
  if (append) {
    return interleaved ? launch_rows_t<T, V, true, true>(p, stream)
                       : launch_rows_t<T, V, false, true>(p, stream);
  }
  return interleaved ? launch_rows_t<T, V, true, false>(p, stream)
                     : launch_rows_t<T, V, false, false>(p, stream);
}

int reject(int code, const char* message) {
  set_last_error(message);
  return code;
}

// Whether rows that start at `base` with these element strides can be read in
// pieces of `bytes`.
bool aligned_rows(const void* base, std::initializer_list<int64_t> strides, int width, int bytes) {
  uintptr_t bits = reinterpret_cast<uintptr_t>(base);
  for (int64_t s : strides) bits |= static_cast<uintptr_t>(s * width);
  return (bits & (bytes - 1)) == 0;
}

bool aligned_stream(const RowStream& s, int in_width, int out_width, int in_bytes, int out_bytes) {
  return s.heads == 0 ||
         (aligned_rows(s.in, {s.in_b, s.in_t, s.in_h}, in_width, in_bytes) &&
          aligned_rows(s.out, {s.out_b, s.out_t, s.out_h}, out_width, out_bytes));
}

constexpr int64_t kMostTokens = (1LL << 31) - 1;  // the grid's x extent
constexpr int64_t kMostHeads = 1 << 16;

// The rotation's arguments, shared by the two entry points.
int check_rotation(const float* cos_sin, int64_t rotary, int64_t dim, int64_t rows,
                   int64_t stride) {
  if (cos_sin == nullptr) return reject(RKV_ERR_INVALID_ARGUMENT, "cos_sin is null");
  if (rotary < 2 || rotary % 2 != 0 || rotary > dim) {
    return reject(RKV_ERR_INVALID_ARGUMENT, "rotary_dim must be even in [2, head_dim]");
  }
  if (rows < 1 || stride < rotary) {
    return reject(RKV_ERR_INVALID_ARGUMENT, "cos_sin rows must hold rotary_dim entries");
  }
  if ((reinterpret_cast<uintptr_t>(cos_sin) & 3u) != 0) {
    return reject(RKV_ERR_ALIGNMENT, "cos_sin is not aligned to its elements");
  }
  return RKV_OK;
}

int finish(RowsParams& p, int64_t dtype, bool interleaved, bool append, int64_t heads,
           void* stream) {
  const bool f32 = dtype == RKV_DTYPE_F32;
  const int width = f32 ? 4 : 2, out_width = append ? 2 : width;
  if (!aligned_stream(p.query, width, width, width, width) ||
      !aligned_stream(p.key, width, out_width, width, out_width) ||
      !aligned_stream(p.value, width, out_width, width, out_width)) {
    return reject(RKV_ERR_ALIGNMENT, "rows are not aligned to their elements");
  }
  if (p.batch * p.tokens == 0 || heads == 0) return RKV_OK;
  const int v = 16 / width, out_bytes = append ? v * 2 : 16;
  const bool vector = p.dim % (2 * v) == 0 && p.rotary % (2 * v) == 0 &&
                      aligned_stream(p.query, width, width, 16, 16) &&
                      aligned_stream(p.key, width, out_width, 16, out_bytes) &&
                      aligned_stream(p.value, width, out_width, 16, out_bytes) &&
                      (p.rotary == 0 || aligned_rows(p.cos_sin, {p.table_stride}, 4, 16));
  const cudaError_t err =
      launch_rows(p, f32, vector, interleaved, append, static_cast<cudaStream_t>(stream));
  if (err != cudaSuccess) {
    set_last_error(std::string("rotary launch: ") + cudaGetErrorString(err));
    return RKV_ERR_CUDA;
  }
  return RKV_OK;
}

}  // namespace

cudaError_t launch_rows(const RowsParams& p, bool f32, bool vector, bool interleaved, bool append,
                        cudaStream_t stream) {
  if (f32) {
    return vector ? launch_rows_v<float, 4>(p, interleaved, append, stream)
                  : launch_rows_v<float, 1>(p, interleaved, append, stream);
  }
  return vector ? launch_rows_v<__nv_bfloat16, 8>(p, interleaved, append, stream)
                : launch_rows_v<__nv_bfloat16, 1>(p, interleaved, append, stream);
}

}  // namespace rkv

extern "C" {

int rkv_rotary(const rkv_rotary_args* a, void* stream) {
  using namespace rkv;
  set_last_error("");
  if (a == nullptr) return reject(RKV_ERR_INVALID_ARGUMENT, "args is null");
  if (a->batch < 0 || a->tokens < 0 || a->query_heads < 0 || a->key_heads < 0 ||
      a->query_heads > kMostHeads || a->key_heads > kMostHeads || a->batch > kMostTokens ||
      a->tokens > kMostTokens || a->batch * a->tokens > kMostTokens) {
    return reject(RKV_ERR_INVALID_ARGUMENT, "batch, tokens and heads are out of range");
  }
  if (a->head_dim < 2 || a->head_dim > 1024 || a->head_dim % 2 != 0) {
    return reject(RKV_ERR_UNSUPPORTED, "head_dim must be even in [2, 1024]");
  }
  if (a->dtype != RKV_DTYPE_BF16 && a->dtype != RKV_DTYPE_F32) {
    return reject(RKV_ERR_INVALID_ARGUMENT, "dtype must be bf16 or fp32");
  }
  const int rc = check_rotation(a->cos_sin, a->rotary_dim, a->head_dim, a->table_rows,
                                a->table_stride);
  if (rc != RKV_OK) return rc;
  if (a->batch * a->tokens > 0 &&
      (a->positions == nullptr || (a->query_heads > 0 && (!a->query || !a->query_out)) ||
       (a->key_heads > 0 && (!a->key || !a->key_out)))) {
    return reject(RKV_ERR_INVALID_ARGUMENT, "positions, rows and outputs must be non-null");
  }
  RowsParams p = {};
  const auto row_stream = [](const void* in, void* out, const int64_t* is, const int64_t* os,
                             int64_t heads) {
    return RowStream{in, out, is[0], is[1], is[2], os[0], os[1], os[2], static_cast<int>(heads)};
  };
  p.query = row_stream(a->query, a->query_out, a->query_strides, a->query_out_strides,
                       a->query_heads);
  p.key = row_stream(a->key, a->key_out, a->key_strides, a->key_out_strides, a->key_heads);
  p.dim = static_cast<int>(a->head_dim);
  p.rotary = static_cast<int>(a->rotary_dim);
  p.sign = a->inverse ? -1.f : 1.f;
  p.cos_sin = a->cos_sin;
  p.table_rows = a->table_rows;
  p.table_stride = a->table_stride;
  p.positions = a->positions;
  p.pos_b = a->position_strides[0];
  p.pos_t = a->position_strides[1];
  p.pos_i64 = a->positions_i64 != 0;
  p.batch = a->batch;
  p.tokens = a->tokens;
  return finish(p, a->dtype, a->interleaved != 0, false, a->query_heads + a->key_heads, stream);
}

int rkv_paged_append(const rkv_append_args* a, void* stream) {
  using namespace rkv;
  set_last_error("");
  if (a == nullptr) return reject(RKV_ERR_INVALID_ARGUMENT, "args is null");
  if (a->tokens < 0 || a->tokens > kMostTokens || a->kv_heads < 1 || a->kv_heads > kMostHeads ||
      a->query_heads < 0 || a->query_heads > kMostHeads || a->sequences < 0 ||
      a->table_blocks < 0 || a->pool_pages < 0 || a->page_table_stride < 0) {
    return reject(RKV_ERR_INVALID_ARGUMENT, "tokens, heads, sequences or pages are out of range");
  }
  if (a->head_dim < 32 || a->head_dim > 256 || a->head_dim % 32 != 0) {
    return reject(RKV_ERR_UNSUPPORTED, "head_dim must be a multiple of 32 in [32, 256]");
  }
  if (a->block_size != 16 && a->block_size != 32 && a->block_size != 64) {
    return reject(RKV_ERR_UNSUPPORTED, "block_size must be 16, 32 or 64");
  }
  if (a->dtype != RKV_DTYPE_BF16 && a->dtype != RKV_DTYPE_F32) {
    return reject(RKV_ERR_INVALID_ARGUMENT, "dtype must be bf16 or fp32");
  }
  if (a->cos_sin != nullptr) {
    const int rc = check_rotation(a->cos_sin, a->rotary_dim, a->head_dim, a->table_rows,
                                  a->table_stride);
    if (rc != RKV_OK) return rc;
  }
  if (a->tokens > 0 && (!a->key || !a->value || !a->key_pool || !a->value_pool ||
                        !a->page_table || !a->positions)) {
    return reject(RKV_ERR_INVALID_ARGUMENT,
                  "rows, pools, page_table and positions must be non-null");
  }
  if (a->tokens > 0 && a->query_heads > 0 && (!a->query || !a->query_out)) {
    return reject(RKV_ERR_INVALID_ARGUMENT, "query and query_out must be non-null");
  }
  RowsParams p = {};
  p.query = RowStream{a->query, a->query_out, 0, a->query_strides[0], a->query_strides[1],
                      0, a->query_out_strides[0], a->query_out_strides[1],
                      static_cast<int>(a->query_heads)};
  const auto pool_stream = [&](const void* in, void* out, const int64_t* is, const int64_t* os) {
    return RowStream{in, out, 0, is[0], is[1], os[0], os[2], os[1],
                     static_cast<int>(a->kv_heads)};
  };
  p.key = pool_stream(a->key, a->key_pool, a->key_strides, a->key_pool_strides);
  p.value = pool_stream(a->value, a->value_pool, a->value_strides, a->value_pool_strides);
  p.dim = static_cast<int>(a->head_dim);
  p.rotary = a->cos_sin != nullptr ? static_cast<int>(a->rotary_dim) : 0;
  p.sign = 1.f;
  p.cos_sin = a->cos_sin;
  p.table_rows = a->table_rows;
  p.table_stride = a->table_stride;
  p.positions = a->positions;
  p.pos_t = 1;
  p.pos_i64 = a->positions_i64 != 0;
  p.batch = 1;
  p.tokens = a->tokens;
  p.page_table = a->page_table;
  p.page_table_stride = a->page_table_stride;
  p.sequence_ids = a->sequence_ids;
  p.sequences = a->sequences;
  p.table_blocks = a->table_blocks;
  p.pool_pages = a->pool_pages;
  p.block_shift = a->block_size == 16 ? 4 : a->block_size == 32 ? 5 : 6;
  p.status = a->status;
  return finish(p, a->dtype, a->interleaved != 0, true, a->query_heads + a->kv_heads, stream);
}

}  // extern "C"
