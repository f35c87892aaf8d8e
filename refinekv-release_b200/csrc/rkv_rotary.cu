// Rotary positions and the append of new tokens to a page pool.
//
// Both are one pass over rows of head_dim channels: read a row, rotate its
// rotary channels by the position's row of the cos/sin table, write it to a
// tensor or to the pool's page.  Bound: HBM on long inputs (every element
// read once and written once, a few flops per pair), latency on single
// tokens.  Measured on B200 (graph replay): 8192 tokens of 40 bf16 heads, D
// 128: 29 us, 172 MB, 0.90 of the measured copy rate; 24.5K prompt tokens into
// the pool, 48 heads each: 116 us, 653 MB, 0.86; one token: 2.1 to 2.4 us (eight
// appended: 2.5 to 2.8).
//
// What it took: CTAs that stay and take token after token (one CTA a token
// launched too slowly: 45 us for the 8192), the pieces of a row kept as they
// lie in memory and turned in place (as arrays of floats they went to local
// memory: 44 us), two heads in flight per thread (one: 35 us, three: 33), 1024
// resident threads an SM (768: 34 us).
//
// A unit of work is 2V channels of one head: for a rotated half-layout unit
// the V channels at c and the V at c + rotary/2 (the two halves of V pairs),
// for an interleaved or copied one 2V consecutive channels.  V is 16 bytes of
// elements, or 1 where strides, alignment or a rotary width that is no
// multiple of 2V forbid 16-byte accesses (the 8192 tokens then take 111 us).
#include <algorithm>
#include <string>

#include "refinekv_b200.h"
#include "rkv_device.cuh"
#include "rkv_kernels.h"

namespace rkv {
void set_last_error(const std::string& message);

namespace {

// V consecutive elements as they lie in memory.
template <typename T, int V>
struct Piece {
  uint32_t word[4];  // 16 bytes
  __device__ void load(const T* from) {
    const uint4 x = *reinterpret_cast<const uint4*>(from);
    word[0] = x.x, word[1] = x.y, word[2] = x.z, word[3] = x.w;
  }
  __device__ void store(T* to) const {
    *reinterpret_cast<uint4*>(to) = make_uint4(word[0], word[1], word[2], word[3]);
  }
};

template <typename T>
struct Piece<T, 1> {
  T one;
  __device__ void load(const T* from) { one = *from; }
  __device__ void store(T* to) const { *to = one; }
};

__device__ __forceinline__ float low(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float high(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }
__device__ __forceinline__ float widen(float x) { return x; }
__device__ __forceinline__ float widen(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void narrow(float& to, float x) { to = x; }
__device__ __forceinline__ void narrow(__nv_bfloat16& to, float x) { to = __float2bfloat16_rn(x); }

// The piece rounded to bf16 (as it is when it holds bf16).
__device__ __forceinline__ void store_bf16(const Piece<__nv_bfloat16, 8>& x, __nv_bfloat16* to) {
  x.store(to);
}
__device__ __forceinline__ void store_bf16(const Piece<float, 4>& x, __nv_bfloat16* to) {
  *reinterpret_cast<uint2*>(to) =
      make_uint2(pack_bf16(__uint_as_float(x.word[0]), __uint_as_float(x.word[1])),
                 pack_bf16(__uint_as_float(x.word[2]), __uint_as_float(x.word[3])));
}
template <typename T>
__device__ __forceinline__ void store_bf16(const Piece<T, 1>& x, __nv_bfloat16* to) {
  narrow(*to, widen(x.one));
}

template <typename T, int V>
__device__ __forceinline__ void clear(Piece<T, V>& x) {
  x.word[0] = x.word[1] = x.word[2] = x.word[3] = 0;
}
template <typename T>
__device__ __forceinline__ void clear(Piece<T, 1>& x) { narrow(x.one, 0.f); }

// V cosines or sines: at most 16 bytes a load.
template <int V>
__device__ __forceinline__ void load_table(const float* from, float (&x)[V]) {
  constexpr int W = V < 4 ? V : 4;
#pragma unroll
  for (int i = 0; i < V; i += W) {
    if constexpr (W == 4) {
      const float4 four = *reinterpret_cast<const float4*>(from + i);
      x[i] = four.x, x[i + 1] = four.y, x[i + 2] = four.z, x[i + 3] = four.w;
    } else {
      x[i] = from[i];
    }
  }
}

// One pair (a, b) turned.  Products and sums are rounded one by one (no fused
// multiply-add): the result then depends on nothing but its operands, so
// rotating alone, rotating while appending and the formula in fp32 agree bit
// for bit.  (The two-wide fp32 instructions would halve the arithmetic, but
// their products and sums are fused by the assembler.)
__device__ __forceinline__ void turn1(float& a, float& b, float c, float s) {
  const float y = __fsub_rn(__fmul_rn(a, c), __fmul_rn(b, s));
  b = __fadd_rn(__fmul_rn(b, c), __fmul_rn(a, s));
  a = y;
}

// Two pairs.
__device__ __forceinline__ void turn2(float2& a, float2& b, float2 c, float2 s) {
  turn1(a.x, b.x, c.x, s.x);
  turn1(a.y, b.y, c.y, s.y);
}

// The V pairs of a unit's two pieces turned: (p_i, q_i), or interleaved the
// neighbours of p and then those of q.
template <bool Interleaved>
__device__ __forceinline__ void turn(Piece<__nv_bfloat16, 8>& p, Piece<__nv_bfloat16, 8>& q,
                                     const float (&c)[8], const float (&s)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {  // pairs 2 i and 2 i + 1
    const float2 c2 = make_float2(c[2 * i], c[2 * i + 1]);
    const float2 s2 = make_float2(s[2 * i], s[2 * i + 1]);
    if constexpr (Interleaved) {
      uint32_t& w0 = i < 2 ? p.word[2 * i] : q.word[2 * i - 4];
      uint32_t& w1 = i < 2 ? p.word[2 * i + 1] : q.word[2 * i - 3];
      float2 a = make_float2(low(w0), low(w1)), b = make_float2(high(w0), high(w1));
      turn2(a, b, c2, s2);
      w0 = pack_bf16(a.x, b.x);
      w1 = pack_bf16(a.y, b.y);
    } else {
      float2 a = make_float2(low(p.word[i]), high(p.word[i]));
      float2 b = make_float2(low(q.word[i]), high(q.word[i]));
      turn2(a, b, c2, s2);
      p.word[i] = pack_bf16(a.x, a.y);
      q.word[i] = pack_bf16(b.x, b.y);
    }
  }
}

template <bool Interleaved>
__device__ __forceinline__ void turn(Piece<float, 4>& p, Piece<float, 4>& q, const float (&c)[4],
                                     const float (&s)[4]) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    uint32_t& a0 = Interleaved ? (i ? q : p).word[0] : p.word[2 * i];
    uint32_t& b0 = Interleaved ? (i ? q : p).word[1] : q.word[2 * i];
    uint32_t& a1 = Interleaved ? (i ? q : p).word[2] : p.word[2 * i + 1];
    uint32_t& b1 = Interleaved ? (i ? q : p).word[3] : q.word[2 * i + 1];
    float2 a = make_float2(__uint_as_float(a0), __uint_as_float(a1));
    float2 b = make_float2(__uint_as_float(b0), __uint_as_float(b1));
    turn2(a, b, make_float2(c[2 * i], c[2 * i + 1]), make_float2(s[2 * i], s[2 * i + 1]));
    a0 = __float_as_uint(a.x), a1 = __float_as_uint(a.y);
    b0 = __float_as_uint(b.x), b1 = __float_as_uint(b.y);
  }
}

template <bool Interleaved, typename T>
__device__ __forceinline__ void turn(Piece<T, 1>& p, Piece<T, 1>& q, const float (&c)[1],
                                     const float (&s)[1]) {
  float a = widen(p.one), b = widen(q.one);
  turn1(a, b, c[0], s[0]);
  narrow(p.one, a);
  narrow(q.one, b);
}

// A CTA takes the heads of one blockIdx.y and every gridDim.x-th token; the
// next token's position is requested ahead.  A thread keeps its channels (unit
// c) of kHeads heads, so their cosines and sines are loaded once a token and
// the heads' addresses worked out once.
constexpr int kHeads = 2;
// Vector units: CTAs of up to 256 threads, four to an SM or more (64 registers).
constexpr int row_threads(int V) { return V == 1 ? 512 : 256; }
constexpr int row_ctas(int V) { return V == 1 ? 2 : 4; }

template <typename T, int V, bool Interleaved, bool Append>
__global__ void __launch_bounds__(row_threads(V), row_ctas(V))
    rows_kernel(const __grid_constant__ RowsParams p) {
  const int per_head = p.dim / (2 * V);
  const int stride = blockDim.x / per_head, c = threadIdx.x % per_head;
  const int k_from = p.query.heads, v_from = k_from + p.key.heads;
  const int heads = v_from + (Append ? p.value.heads : 0);
  const bool rotary = c < p.rotary / (2 * V);
  // The unit's two pieces; unrotated rows are copied in the same pieces.
  const bool halves = !Interleaved && rotary;
  const int first = halves ? c * V : c * 2 * V;
  const int gap = halves ? p.rotary / 2 : V;
  int kind[kHeads];  // 0 query, 1 key, 2 value, -1 nothing
  int64_t in_at[kHeads], out_at[kHeads];
#pragma unroll
  for (int u = 0; u < kHeads; ++u) {
    const int lane_head = threadIdx.x / per_head;
    const int head = (blockIdx.y * kHeads + u) * stride + lane_head;
    kind[u] = lane_head >= stride || head >= heads ? -1 : head < k_from ? 0 : head < v_from ? 1 : 2;
    const RowStream& s = kind[u] <= 0 ? p.query : kind[u] == 1 ? p.key : p.value;
    const int own = head - (kind[u] <= 0 ? 0 : kind[u] == 1 ? k_from : v_from);
    in_at[u] = own * s.in_h + first;
    out_at[u] = own * s.out_h + first;
  }
  pdl_wait();
  pdl_launch_dependents();
  // Tokens are counted in 32 bits (below 2^31): their divisions are cheap.
  const unsigned tokens = static_cast<unsigned>(p.tokens);
  const unsigned count = static_cast<unsigned>(p.batch) * tokens;
  const auto position = [&](unsigned n) -> int64_t {
    const unsigned b = p.batch > 1 ? n / tokens : 0;
    const int64_t at = b * p.pos_b + (n - b * tokens) * p.pos_t;
    return p.pos_i64 ? static_cast<const int64_t*>(p.positions)[at]
                     : static_cast<const int32_t*>(p.positions)[at];
  };
  int64_t upcoming = position(blockIdx.x);
  for (unsigned n = blockIdx.x; n < count; n += gridDim.x) {
    const unsigned at_b = p.batch > 1 ? n / tokens : 0;
    const int64_t b = at_b, t = n - at_b * tokens;
    const int64_t pos = upcoming;
    Piece<T, V> in[kHeads][2];
#pragma unroll
    for (int u = 0; u < kHeads; ++u) {
      if (kind[u] < 0) continue;
      const RowStream& s = kind[u] == 0 ? p.query : !Append || kind[u] == 1 ? p.key : p.value;
      const T* from = static_cast<const T*>(s.in) + (b * s.in_b + t * s.in_t) + in_at[u];
      in[u][0].load(from);
      in[u][1].load(from + gap);
    }
    if (n + gridDim.x < count) upcoming = position(n + gridDim.x);
    const bool known = p.rotary == 0 || (pos >= 0 && pos < p.table_rows);
    float cs[V], sn[V];
    if (rotary && known) {
      const float* table = p.cos_sin + pos * p.table_stride + c * V;
      load_table<V>(table, cs);
      load_table<V>(table + p.rotary / 2, sn);
#pragma unroll
      for (int i = 0; i < V; ++i) sn[i] *= p.sign;
    } else {  // a position outside the table: NaN
#pragma unroll
      for (int i = 0; i < V; ++i) cs[i] = sn[i] = __int_as_float(0x7fc00000);
    }
    bool keep = true;  // the token's rows go to the pool
    int64_t page = 0, page_row = 0;
    if (Append) {
      keep = pos >= 0;
      if (keep) {
        const int64_t seq = p.sequence_ids != nullptr ? p.sequence_ids[n] : static_cast<int64_t>(n);
        const int64_t block = pos >> p.block_shift;
        page_row = pos - (block << p.block_shift);
        bool ok = known && seq >= 0 && seq < p.sequences && block < p.table_blocks;
        if (ok) {
          page = p.page_table[seq * p.page_table_stride + block];
          ok = page >= 0 && page < p.pool_pages;
        }
        if (!ok) {
          keep = false;
          if (threadIdx.x == 0 && blockIdx.y == 0 && p.status != nullptr) {
            atomicOr(p.status, kStatusBadInput);
          }
        }
      }
    }
#pragma unroll
    for (int u = 0; u < kHeads; ++u) {
      if (kind[u] < 0) continue;
      if (rotary && (!Append || kind[u] < 2)) turn<Interleaved>(in[u][0], in[u][1], cs, sn);
      if (Append && kind[u] > 0) {
        const RowStream& s = kind[u] == 1 ? p.key : p.value;
        if (!keep) continue;
        __nv_bfloat16* to = static_cast<__nv_bfloat16*>(s.out) +
                            (page * s.out_b + page_row * s.out_t) + out_at[u];
        store_bf16(in[u][0], to);
        store_bf16(in[u][1], to + gap);
      } else {
        if (Append && pos < 0) {
          clear(in[u][0]);
          clear(in[u][1]);
        }
        const RowStream& s = kind[u] == 0 ? p.query : p.key;
        T* to = static_cast<T*>(s.out) + (b * s.out_b + t * s.out_t) + out_at[u];
        in[u][0].store(to);
        in[u][1].store(to + gap);
      }
    }
  }
}

template <typename T, int V, bool Interleaved, bool Append>
cudaError_t launch_rows_t(const RowsParams& p, cudaStream_t stream) {
  const int heads = p.query.heads + p.key.heads + (Append ? p.value.heads : 0);
  const int per_head = p.dim / (2 * V);
  // kHeads heads a thread, as many as the CTA holds; the rest in blockIdx.y.
  const int wanted = std::min(row_threads(V), per_head * ((heads + kHeads - 1) / kHeads));
  const int threads = (wanted + 31) / 32 * 32;
  const int each = threads / per_head * kHeads, slices = (heads + each - 1) / each;
  int sms = 0;
  if (device_sms(&sms) != RKV_OK) return cudaErrorInvalidDevice;
  const int64_t resident =
      std::max<int64_t>(1, static_cast<int64_t>(sms) * std::min(32, 1024 / threads) / slices);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(std::min(p.batch * p.tokens, resident)), slices);
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
constexpr int64_t kMostHeads = 4096;

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
  if (!aligned_to(a->positions_i64 ? 8 : 4, {a->positions})) {
    return reject(RKV_ERR_ALIGNMENT, "positions are not aligned to their elements");
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
  if (!aligned_to(a->positions_i64 ? 8 : 4, {a->positions}) ||
      !aligned_to(4, {a->page_table, a->sequence_ids, a->status})) {
    return reject(RKV_ERR_ALIGNMENT,
                  "positions, page_table, sequence_ids and status must be aligned to their elements");
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
