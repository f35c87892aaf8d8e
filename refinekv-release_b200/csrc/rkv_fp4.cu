// New tokens into a page pool of 4 bits, rotated on the way, and rows of a pool
// (4 bits or bf16) back as numbers.
//
// Mathematics: y_a = x_a c - x_b s, y_b = x_b c + x_a s for the rotary pairs (each
// product and sum rounded by itself, as in the bf16 append), then per 16
// channels scale = e4m3(max |y| / 6) and code = e2m1(y / scale), both to the
// nearest, ties to even; the quotients are correctly rounded, so the codes are
// those of the formula.  Reading multiplies back.
//
// Bound: HBM on long inputs: a bf16 row of 128 channels is read (256 bytes) and
// 72 bytes written, or the other way round.
#include <algorithm>
#include <string>

#include "refinekv_b200.h"
#include "rkv_device.cuh"
#include "rkv_fp4.cuh"
#include "rkv_kernels.h"

namespace rkv {
void set_last_error(const std::string& message);

namespace {

template <typename T>
__device__ __forceinline__ float widen(T x) {
  return static_cast<float>(x);
}

__device__ __forceinline__ int64_t position_of(const RowsParams& p, unsigned n) {
  return p.pos_i64 ? static_cast<const int64_t*>(p.positions)[n]
                   : static_cast<const int32_t*>(p.positions)[n];
}

// Where a token's rows are in the pool.
struct Place {
  int64_t pos;
  int page, row;
  bool keep;   // false: padding, or out of range
  bool known;  // the position is within the rotation table, where there is one
};

__device__ __forceinline__ Place find_place(const RowsParams& p, unsigned n, bool report) {
  Place at;
  at.pos = position_of(p, n);
  at.known = p.rotary == 0 || (at.pos >= 0 && at.pos < p.table_rows);
  at.page = at.row = 0;
  at.keep = at.pos >= 0;
  if (!at.keep) return at;
  const int64_t seq = p.sequence_ids != nullptr ? p.sequence_ids[n] : static_cast<int64_t>(n);
  const int64_t block = at.pos >> p.block_shift;
  at.row = static_cast<int>(at.pos - (block << p.block_shift));
  at.keep = at.known && seq >= 0 && seq < p.sequences && block < p.table_blocks;
  if (at.keep) {
    at.page = p.page_table[seq * p.page_table_stride + block];
    at.keep = at.page >= 0 && at.page < p.pool_pages;
  }
  if (!at.keep && report && p.status != nullptr) atomicOr(p.status, kStatusBadInput);
  return at;
}

// A CTA takes every gridDim.x-th token.  Their places hang on three loads in a
// row, so a thread each finds those of up to kBatch tokens at once, ahead of the
// rows' own loads.  Returns how many (for the whole CTA).
constexpr int kBatch = 64;

__device__ __forceinline__ unsigned find_places(const RowsParams& p, Place (&places)[kBatch],
                                                unsigned first, bool report) {
  const unsigned left = (static_cast<unsigned>(p.tokens) - first + gridDim.x - 1) / gridDim.x;
  const unsigned there = min(left, min(static_cast<unsigned>(kBatch), blockDim.x));
  __syncthreads();  // the batch before is done with
  if (threadIdx.x < there) {
    places[threadIdx.x] = find_place(p, first + threadIdx.x * gridDim.x, report);
  }
  __syncthreads();
  return there;
}

// x / b correctly rounded, r being 1 / b correctly rounded: the first quotient's
// error x - q b is exact, and corrects it (Markstein 1990, on division by fused
// multiply-adds).  Ties between two codes must be met exactly (bf16 rows are full of
// them), which x r alone does not; three instructions instead of a division's ten or
// so.  Finite numbers whose quotient neither overflows nor is tiny; r = 0 gives 0
// with the sign of x.
__device__ __forceinline__ float quotient(float x, float b, float r) {
  const float q = __fmul_rn(x, r);
  return __fmaf_rn(-__fmaf_rn(b, q, -x), r, q);  // in these signs -0 stays -0
}

// The codes of 8 of the 16 channels that share a scale.
__device__ __forceinline__ uint32_t codes_of(float (&y)[8], uint32_t scale) {
  const float by = fp4_scale_value(scale), r = by > 0.f ? __frcp_rn(by) : 0.f;
#pragma unroll
  for (int j = 0; j < 8; ++j) y[j] = quotient(y[j], by, r);
  const uint32_t codes = fp4_encode(y);
  return scale == kFp4NanScale ? 0u : codes;
}

__device__ __forceinline__ uint32_t magnitude(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// Eight consecutive channels as they lie in memory, and as numbers.
template <typename T>
struct Eight;
template <>
struct Eight<__nv_bfloat16> {
  uint4 raw;
  __device__ void load(const __nv_bfloat16* from) { raw = *reinterpret_cast<const uint4*>(from); }
  __device__ void widen(float (&x)[8]) const {
    const uint32_t words[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      x[2 * j] = __uint_as_float(words[j] << 16);
      x[2 * j + 1] = __uint_as_float(words[j] & 0xffff0000u);
    }
  }
};
template <>
struct Eight<float> {
  float4 raw[2];
  __device__ void load(const float* from) {
    raw[0] = *reinterpret_cast<const float4*>(from);
    raw[1] = *reinterpret_cast<const float4*>(from + 4);
  }
  __device__ void widen(float (&x)[8]) const {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      x[4 * j] = raw[j].x, x[4 * j + 1] = raw[j].y;
      x[4 * j + 2] = raw[j].z, x[4 * j + 3] = raw[j].w;
    }
  }
};
template <typename T>
__device__ __forceinline__ void load8(const T* from, float (&x)[8]) {
  Eight<T> eight;
  eight.load(from);
  eight.widen(x);
}
__device__ __forceinline__ void store8(__nv_bfloat16* to, const float (&x)[8]) {
  *reinterpret_cast<uint4*>(to) = make_uint4(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]),
                                             pack_bf16(x[4], x[5]), pack_bf16(x[6], x[7]));
}
__device__ __forceinline__ void store8(float* to, const float (&x)[8]) {
  *reinterpret_cast<float4*>(to) = make_float4(x[0], x[1], x[2], x[3]);
  *reinterpret_cast<float4*>(to + 4) = make_float4(x[4], x[5], x[6], x[7]);
}

// A thread takes eight consecutive channels of kHeads heads of a token, and two
// neighbours share a scale.  A CTA takes the heads of one blockIdx.y; a token's rows
// are requested while the one before is worked on.  The half layout's partners are
// read by both threads that need them (the second read is in L1), so that every
// rotary width of whole pieces goes this way.
constexpr int kHeads = 2;
constexpr int kRowThreads = 256;

template <typename T, bool Interleaved>
__global__ void __launch_bounds__(kRowThreads, sizeof(T) == 2 ? 3 : 2)
    fp4_append_kernel(const __grid_constant__ RowsParams p, const float* __restrict__ key_scale,
                      const float* __restrict__ value_scale) {
  __shared__ Place places[kBatch];
  const int per_head = p.dim / 8;
  const int stride = blockDim.x / per_head, c = threadIdx.x % per_head;
  const int k_from = p.query.heads, v_from = k_from + p.key.heads, heads = v_from + p.value.heads;
  const int half = p.rotary / 2;
  const bool rotary = 8 * c < p.rotary, second = !Interleaved && 8 * c >= half;
  const int gap = second ? -half : half;                                // to the partners
  const int pair = Interleaved ? 4 * c : second ? 8 * c - half : 8 * c;  // the first one's
  int kind[kHeads], own[kHeads];  // 0 query, 1 key, 2 value, -1 nothing
  const T* in[kHeads];
  int64_t in_t[kHeads];
#pragma unroll
  for (int u = 0; u < kHeads; ++u) {
    const int lane_head = threadIdx.x / per_head;
    const int head = (blockIdx.y * kHeads + u) * stride + lane_head;
    kind[u] = lane_head >= stride || head >= heads ? -1 : head < k_from ? 0 : head < v_from ? 1 : 2;
    own[u] = head - (kind[u] <= 0 ? 0 : kind[u] == 1 ? k_from : v_from);
    const RowStream& s = kind[u] <= 0 ? p.query : kind[u] == 1 ? p.key : p.value;
    in[u] = static_cast<const T*>(s.in) + own[u] * s.in_h + 8 * c;
    in_t[u] = s.in_t;
  }
  struct Rows {
    Eight<T> x[kHeads], z[Interleaved ? 1 : kHeads];
  };
  const auto request = [&](unsigned n, Rows& rows) {
#pragma unroll
    for (int u = 0; u < kHeads; ++u) {
      if (kind[u] < 0) continue;
      const T* from = in[u] + n * in_t[u];
      rows.x[u].load(from);
      if constexpr (!Interleaved) {
        if (rotary && kind[u] < 2) rows.z[u].load(from + gap);
      }
    }
  };
  pdl_wait();
  pdl_launch_dependents();
  const unsigned tokens = static_cast<unsigned>(p.tokens);
  for (unsigned first = blockIdx.x; first < tokens; first += gridDim.x * min(kBatch, blockDim.x)) {
    Rows rows, next;
    request(first, rows);
    const unsigned there = find_places(p, places, first, blockIdx.y == 0);
    for (unsigned i = 0; i < there; ++i) {
      const unsigned n = first + i * gridDim.x;
      if (i + 1 < there) request(n + gridDim.x, next);
      const Place at = places[i];
      float cs[8], sn[8];
      if (rotary) {
        if (at.known) {
          const float* table = p.cos_sin + at.pos * p.table_stride + pair;
          if constexpr (Interleaved) {
            const float4 c4 = *reinterpret_cast<const float4*>(table);
            const float4 s4 = *reinterpret_cast<const float4*>(table + half);
            cs[0] = c4.x, cs[1] = c4.y, cs[2] = c4.z, cs[3] = c4.w;
            sn[0] = s4.x, sn[1] = s4.y, sn[2] = s4.z, sn[3] = s4.w;
          } else {
            load8(table, cs);
            load8(table + half, sn);
          }
        } else {  // a position outside the table: NaN
#pragma unroll
          for (int j = 0; j < 8; ++j) cs[j] = sn[j] = __int_as_float(0x7fc00000);
        }
      }
#pragma unroll
      for (int u = 0; u < kHeads; ++u) {
        float x[8];
        uint32_t most = 0;
        if (kind[u] >= 0) {
          rows.x[u].widen(x);
          if (rotary && kind[u] < 2) {
            // No fused multiply-add: the codes are those of the formula in fp32.
            if constexpr (Interleaved) {
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const float a = x[2 * j], b = x[2 * j + 1];
                x[2 * j] = __fsub_rn(__fmul_rn(a, cs[j]), __fmul_rn(b, sn[j]));
                x[2 * j + 1] = __fadd_rn(__fmul_rn(b, cs[j]), __fmul_rn(a, sn[j]));
              }
            } else {
              float z[8];
              rows.z[u].widen(z);
#pragma unroll
              for (int j = 0; j < 8; ++j) {
                // x c - z s is x c + (-z s), rounded the same
                const float turned = __fmul_rn(z[j], sn[j]);
                x[j] = __fadd_rn(__fmul_rn(x[j], cs[j]), second ? turned : -turned);
              }
            }
          }
          if (kind[u] == 0) {
            if (at.pos < 0) {
#pragma unroll
              for (int j = 0; j < 8; ++j) x[j] = 0.f;
            }
            store8(static_cast<T*>(p.query.out) + n * p.query.out_t + own[u] * p.query.out_h + 8 * c,
                   x);
          } else {
            const float* factors = kind[u] == 1 ? key_scale : value_scale;
            if (factors != nullptr) {
              const float by = factors[own[u]];
#pragma unroll
              for (int j = 0; j < 8; ++j) x[j] = __fdiv_rn(x[j], by);
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) most = max(most, magnitude(x[j]));
          }
        }
        most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));  // every lane comes here
        if (kind[u] > 0 && at.keep) {
          const uint32_t scale = fp4_scale_of(most);
          const RowStream& s = kind[u] == 1 ? p.key : p.value;
          uint8_t* slab = static_cast<uint8_t*>(s.out) + at.page * s.out_b + own[u] * s.out_h;
          *reinterpret_cast<uint32_t*>(slab + at.row * (p.dim / 2) + 4 * c) = codes_of(x, scale);
          if (!(c & 1)) {
            slab[(p.dim / 2 << p.block_shift) + at.row * (p.dim / 16) + c / 2] =
                static_cast<uint8_t>(scale);
          }
        }
      }
      if (i + 1 < there) rows = next;
    }
  }
}

template <typename T, bool Interleaved>
cudaError_t launch_append(const RowsParams& p, const float* key_scale, const float* value_scale,
                          cudaStream_t stream) {
  const int heads = p.query.heads + p.key.heads + p.value.heads, per_head = p.dim / 8;
  // A token's heads in as few CTAs as hold them, shared out evenly.
  const int wanted = per_head * ((heads + kHeads - 1) / kHeads);
  const int ctas = (wanted + kRowThreads - 1) / kRowThreads;
  const int threads = std::max((wanted / ctas + 31) / 32 * 32, 32);
  const int each = threads / per_head * kHeads, slices = (heads + each - 1) / each;
  int sms = 0;
  if (device_sms(&sms) != RKV_OK) return cudaErrorInvalidDevice;
  const int64_t resident = std::max<int64_t>(
      1, static_cast<int64_t>(sms) * ((sizeof(T) == 2 ? 3 : 2) * kRowThreads / threads) / slices);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(std::min(p.tokens, resident)), slices);
  cfg.blockDim = dim3(threads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, fp4_append_kernel<T, Interleaved>, p, key_scale, value_scale);
}

// One channel of a key, turned.
template <typename T>
__device__ __forceinline__ float turned(const RowsParams& p, const T* row, int d,
                                        const float* table, bool interleaved) {
  const float x = widen(row[d]);
  if (d >= p.rotary) return x;
  const int half = p.rotary / 2;
  const bool second = interleaved ? d & 1 : d >= half;
  const int pair = interleaved ? d >> 1 : second ? d - half : d;
  const int other = interleaved ? d ^ 1 : second ? d - half : d + half;
  const float c = table[pair], s = table[half + pair], z = widen(row[other]);
  return second ? __fadd_rn(__fmul_rn(x, c), __fmul_rn(z, s))
                : __fsub_rn(__fmul_rn(x, c), __fmul_rn(z, s));
}

// Any strides, alignment and rotary width, keys and values only: a thread takes
// 16 channels of a head of a token, element by element.
template <typename T, bool Interleaved>
__global__ void __launch_bounds__(256)
    fp4_append_any_kernel(const __grid_constant__ RowsParams p,
                          const float* __restrict__ key_scale,
                          const float* __restrict__ value_scale) {
  pdl_wait();
  pdl_launch_dependents();
  const int blocks = p.dim / 16, heads = p.key.heads + p.value.heads;
  const int64_t count = p.tokens * heads * blocks;
  for (int64_t i = blockIdx.x * static_cast<int64_t>(blockDim.x) + threadIdx.x; i < count;
       i += static_cast<int64_t>(gridDim.x) * blockDim.x) {
    const int64_t n = i / (heads * blocks);
    const int rest = static_cast<int>(i - n * heads * blocks);
    const int head = rest / blocks, block = rest - head * blocks;
    const bool is_key = head < p.key.heads;
    const RowStream& s = is_key ? p.key : p.value;
    const int own = is_key ? head : head - p.key.heads;
    const T* row = static_cast<const T*>(s.in) + n * s.in_t + own * s.in_h;
    const Place at = find_place(p, static_cast<unsigned>(n), rest == 0);
    if (!at.keep) continue;
    const float* table = p.rotary > 0 ? p.cos_sin + at.pos * p.table_stride : nullptr;
    const float* factors = is_key ? key_scale : value_scale;
    float y[2][8];
    uint32_t most = 0;
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const int d = 16 * block + j;
      float x = is_key ? turned(p, row, d, table, Interleaved) : widen(row[d]);
      if (factors != nullptr) x = __fdiv_rn(x, factors[own]);
      y[j >> 3][j & 7] = x;
      most = max(most, magnitude(x));
    }
    const uint32_t scale = fp4_scale_of(most);
    uint8_t* slab = static_cast<uint8_t*>(s.out) + at.page * s.out_b + own * s.out_h;
    *reinterpret_cast<uint2*>(slab + at.row * (p.dim / 2) + 8 * block) =
        make_uint2(codes_of(y[0], scale), codes_of(y[1], scale));
    slab[(p.dim / 2 << p.block_shift) + at.row * blocks + block] = static_cast<uint8_t>(scale);
  }
}

// Rows of a pool back as numbers.  A thread takes eight channels of a head of the CTA's
// tokens, kAhead of them in flight at once.
constexpr int kAhead = 4;

template <typename Out, bool Fp4>
__global__ void __launch_bounds__(256)
    read_kernel(const __grid_constant__ RowsParams p, const float* __restrict__ key_scale,
                const float* __restrict__ value_scale) {
  __shared__ Place places[kBatch];
  const int units = p.dim / 8, heads = 2 * p.key.heads;
  // The thread's unit; blockIdx.y has the rest of a token's.
  const int all = heads * units, mine = blockIdx.y * blockDim.x + threadIdx.x;
  const int head = mine / units, unit = mine - head * units;
  const bool there_is = mine < all, is_key = head < p.key.heads;
  const RowStream& s = is_key ? p.key : p.value;
  const int own = is_key ? head : head - p.key.heads;
  pdl_wait();
  pdl_launch_dependents();
  const float* factors = is_key ? key_scale : value_scale;
  const bool scaled = there_is && factors != nullptr;
  const float factor = scaled ? factors[own] : 1.f;
  const unsigned tokens = static_cast<unsigned>(p.tokens);
  for (unsigned first = blockIdx.x; first < tokens; first += gridDim.x * min(kBatch, blockDim.x)) {
    const unsigned there = find_places(p, places, first, blockIdx.y == 0);
    if (!there_is) continue;
    for (unsigned i = 0; i < there; i += kAhead) {
      uint32_t codes[kAhead], scale[kAhead];
      Eight<__nv_bfloat16> rows[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        if (i + u >= there || !places[i + u].keep) continue;
        const Place& at = places[i + u];
        if constexpr (Fp4) {
          const uint8_t* slab = static_cast<const uint8_t*>(s.in) + at.page * s.in_b + own * s.in_h;
          codes[u] = *reinterpret_cast<const uint32_t*>(slab + at.row * (p.dim / 2) + 4 * unit);
          scale[u] = slab[(p.dim / 2 << p.block_shift) + at.row * (p.dim / 16) + unit / 2];
        } else {
          rows[u].load(static_cast<const __nv_bfloat16*>(s.in) + at.page * s.in_b +
                       at.row * s.in_t + own * s.in_h + 8 * unit);
        }
      }
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        if (i + u >= there) continue;
        const Place& at = places[i + u];
        float x[8];
        if (!at.keep) {
#pragma unroll
          for (int j = 0; j < 8; ++j) x[j] = at.pos < 0 ? 0.f : __int_as_float(0x7fc00000);
        } else if constexpr (Fp4) {
          uint32_t pairs[4];
          fp4_decode(codes[u], pairs);
          const float by = fp4_scale_value(scale[u]);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float2 two = __half22float2(*reinterpret_cast<const __half2*>(&pairs[j]));
            x[2 * j] = two.x * by;  // exact
            x[2 * j + 1] = two.y * by;
          }
          if (scaled) {
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] *= factor;
          }
        } else {
          rows[u].widen(x);
        }
        const int64_t n = first + (i + u) * gridDim.x;
        store8(static_cast<Out*>(s.out) + n * s.out_t + own * s.out_h + 8 * unit, x);
      }
    }
  }
}

template <typename Out, bool Fp4>
cudaError_t launch_read(const RowsParams& p, const float* key_scale, const float* value_scale,
                        cudaStream_t stream) {
  const int units = 2 * p.key.heads * (p.dim / 8);
  const int threads = std::min(256, (units + 31) / 32 * 32), slices = (units + threads - 1) / threads;
  int sms = 0;
  if (device_sms(&sms) != RKV_OK) return cudaErrorInvalidDevice;
  const int64_t resident = std::max<int64_t>(1, static_cast<int64_t>(sms) * (2048 / threads) / slices);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(std::min(p.tokens, resident)), slices);
  cfg.blockDim = dim3(threads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, read_kernel<Out, Fp4>, p, key_scale, value_scale);
}

template <typename Kernel>
cudaError_t launch_units(Kernel kernel, const RowsParams& p, int64_t units, const float* key_scale,
                         const float* value_scale, cudaStream_t stream) {
  int sms = 0;
  if (device_sms(&sms) != RKV_OK) return cudaErrorInvalidDevice;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(std::min<int64_t>((units + 255) / 256, sms * 8)));
  cfg.blockDim = dim3(256);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, p, key_scale, value_scale);
}

int reject(int code, const char* message) {
  set_last_error(message);
  return code;
}

bool aligned_rows(const void* base, std::initializer_list<int64_t> strides, int width, int bytes) {
  uintptr_t bits = reinterpret_cast<uintptr_t>(base);
  for (int64_t s : strides) bits |= static_cast<uintptr_t>(s * width);
  return (bits & static_cast<uintptr_t>(bytes - 1)) == 0;
}

constexpr int64_t kMostTokens = (1LL << 31) - 1;

// What both entry points ask of a pool and its tokens.
int check_pool(int64_t tokens, int64_t heads, int64_t sequences, int64_t table_blocks,
               int64_t table_stride, int64_t pages, int64_t dim, int64_t block) {
  if (tokens < 0 || tokens > kMostTokens || heads < 1 || heads > kMostPagedHeads || sequences < 0 ||
      table_blocks < 0 || pages < 0 || table_stride < 0) {
    return reject(RKV_ERR_INVALID_ARGUMENT, "tokens, heads, sequences or pages are out of range");
  }
  if (dim < 32 || dim > 256 || dim % 32 != 0) {
    return reject(RKV_ERR_UNSUPPORTED, "head_dim must be a multiple of 32 in [32, 256]");
  }
  if (block != 16 && block != 32 && block != 64) {
    return reject(RKV_ERR_UNSUPPORTED, "block_size must be 16, 32 or 64");
  }
  return RKV_OK;
}

template <typename Args>
void set_pool(RowsParams& p, const Args& a) {
  p.dim = static_cast<int>(a.head_dim);
  p.sign = 1.f;
  p.positions = a.positions;
  p.pos_t = 1;
  p.pos_i64 = a.positions_i64 != 0;
  p.batch = 1;
  p.tokens = a.tokens;
  p.page_table = a.page_table;
  p.page_table_stride = a.page_table_stride;
  p.sequence_ids = a.sequence_ids;
  p.sequences = a.sequences;
  p.table_blocks = a.table_blocks;
  p.pool_pages = a.pool_pages;
  p.block_shift = a.block_size == 16 ? 4 : a.block_size == 32 ? 5 : 6;
  p.status = a.status;
}

int launched(cudaError_t err, const char* what) {
  if (err == cudaSuccess) return RKV_OK;
  set_last_error(std::string(what) + " launch: " + cudaGetErrorString(err));
  return RKV_ERR_CUDA;
}

}  // namespace
}  // namespace rkv

extern "C" {

int rkv_paged_append_fp4(const rkv_append_fp4_args* args, void* stream) {
  using namespace rkv;
  set_last_error("");
  if (args == nullptr) return reject(RKV_ERR_INVALID_ARGUMENT, "args is null");
  const rkv_append_args* a = &args->rows;
  int rc = check_pool(a->tokens, a->kv_heads, a->sequences, a->table_blocks, a->page_table_stride,
                      a->pool_pages, a->head_dim, a->block_size);
  if (rc != RKV_OK) return rc;
  if (a->query_heads < 0 || a->query_heads > kMostPagedHeads) {
    return reject(RKV_ERR_INVALID_ARGUMENT, "query heads are out of range");
  }
  if (a->dtype != RKV_DTYPE_BF16 && a->dtype != RKV_DTYPE_F32) {
    return reject(RKV_ERR_INVALID_ARGUMENT, "dtype must be bf16 or fp32");
  }
  if (a->cos_sin != nullptr) {
    if (a->rotary_dim < 2 || a->rotary_dim % 2 != 0 || a->rotary_dim > a->head_dim) {
      return reject(RKV_ERR_INVALID_ARGUMENT, "rotary_dim must be even in [2, head_dim]");
    }
    if (a->table_rows < 1 || a->table_stride < a->rotary_dim) {
      return reject(RKV_ERR_INVALID_ARGUMENT, "cos_sin rows must hold rotary_dim entries");
    }
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
      !aligned_to(4, {a->page_table, a->sequence_ids, a->status, a->cos_sin, args->key_scale,
                      args->value_scale})) {
    return reject(RKV_ERR_ALIGNMENT, "positions, page_table, sequence_ids, cos_sin, scales and "
                                     "status must be aligned to their elements");
  }
  const bool f32 = a->dtype == RKV_DTYPE_F32;
  const int width = f32 ? 4 : 2;
  const auto rows_aligned = [&](int bytes) {
    return aligned_rows(a->key, {a->key_strides[0], a->key_strides[1]}, width, bytes) &&
           aligned_rows(a->value, {a->value_strides[0], a->value_strides[1]}, width, bytes) &&
           (a->query_heads == 0 ||
            (aligned_rows(a->query, {a->query_strides[0], a->query_strides[1]}, width, bytes) &&
             aligned_rows(a->query_out, {a->query_out_strides[0], a->query_out_strides[1]}, width,
                          bytes)));
  };
  if (!rows_aligned(width)) return reject(RKV_ERR_ALIGNMENT, "rows are not aligned to their elements");
  const int64_t *ks = a->key_pool_strides, *vs = a->value_pool_strides;
  if (!aligned_rows(a->key_pool, {ks[0], ks[1]}, 1, 16) ||
      !aligned_rows(a->value_pool, {vs[0], vs[1]}, 1, 16)) {
    return reject(RKV_ERR_ALIGNMENT, "pools and their strides must be multiples of 16 bytes");
  }
  RowsParams p = {};
  set_pool(p, *a);
  p.query = RowStream{a->query, a->query_out, 0, a->query_strides[0], a->query_strides[1],
                      0, a->query_out_strides[0], a->query_out_strides[1],
                      static_cast<int>(a->query_heads)};
  const int heads = static_cast<int>(a->kv_heads);
  p.key = RowStream{a->key, a->key_pool, 0, a->key_strides[0], a->key_strides[1], ks[0], 0, ks[1],
                    heads};
  p.value = RowStream{a->value, a->value_pool, 0, a->value_strides[0], a->value_strides[1], vs[0],
                      0, vs[1], heads};
  p.rotary = a->cos_sin != nullptr ? static_cast<int>(a->rotary_dim) : 0;
  p.cos_sin = a->cos_sin;
  p.table_rows = a->table_rows;
  p.table_stride = a->table_stride;
  if (p.tokens == 0) return RKV_OK;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool inter = a->interleaved != 0;
  const bool pieces = rows_aligned(16) && (inter ? p.rotary : p.rotary / 2) % 8 == 0 &&
                      (p.rotary == 0 || aligned_rows(p.cos_sin, {p.table_stride}, 4, 16));
  if (pieces) {
    const auto append = [&](auto launch) { return launch(p, args->key_scale, args->value_scale, st); };
    return launched(f32 ? (inter ? append(launch_append<float, true>)
                                 : append(launch_append<float, false>))
                        : (inter ? append(launch_append<__nv_bfloat16, true>)
                                 : append(launch_append<__nv_bfloat16, false>)),
                    "append");
  }
  const int64_t units = p.tokens * 2 * heads * (p.dim / 16);
  const auto any = [&](auto kernel) {
    return launch_units(kernel, p, units, args->key_scale, args->value_scale, st);
  };
  cudaError_t err = f32 ? (inter ? any(fp4_append_any_kernel<float, true>)
                                 : any(fp4_append_any_kernel<float, false>))
                        : (inter ? any(fp4_append_any_kernel<__nv_bfloat16, true>)
                                 : any(fp4_append_any_kernel<__nv_bfloat16, false>));
  if (err == cudaSuccess && p.query.heads > 0) {  // the queries as in the bf16 append
    p.key.heads = p.value.heads = 0;
    err = launch_rows(p, f32, false, inter, true, st);
  }
  return launched(err, "append");
}

int rkv_paged_read(const rkv_read_args* a, void* stream) {
  using namespace rkv;
  set_last_error("");
  if (a == nullptr) return reject(RKV_ERR_INVALID_ARGUMENT, "args is null");
  const int rc = check_pool(a->tokens, a->kv_heads, a->sequences, a->table_blocks,
                            a->page_table_stride, a->pool_pages, a->head_dim, a->block_size);
  if (rc != RKV_OK) return rc;
  const bool fp4 = a->pool_dtype == RKV_DTYPE_FP4;
  if ((!fp4 && a->pool_dtype != RKV_DTYPE_BF16) ||
      (a->dtype != RKV_DTYPE_BF16 && a->dtype != RKV_DTYPE_F32)) {
    return reject(RKV_ERR_INVALID_ARGUMENT, "pools are bf16 or fp4, rows bf16 or fp32");
  }
  if (!fp4 && (a->key_scale != nullptr || a->value_scale != nullptr)) {
    return reject(RKV_ERR_INVALID_ARGUMENT, "scales belong to an fp4 pool");
  }
  if (a->tokens > 0 && (!a->key_out || !a->value_out || !a->key_pool || !a->value_pool ||
                        !a->page_table || !a->positions)) {
    return reject(RKV_ERR_INVALID_ARGUMENT,
                  "rows, pools, page_table and positions must be non-null");
  }
  if (!aligned_to(a->positions_i64 ? 8 : 4, {a->positions}) ||
      !aligned_to(4, {a->page_table, a->sequence_ids, a->status, a->key_scale, a->value_scale})) {
    return reject(RKV_ERR_ALIGNMENT, "positions, page_table, sequence_ids, scales and status must "
                                     "be aligned to their elements");
  }
  const int out_width = a->dtype == RKV_DTYPE_F32 ? 4 : 2, width = fp4 ? 1 : 2;
  const int64_t *ks = a->key_pool_strides, *vs = a->value_pool_strides;
  if (!aligned_rows(a->key_pool, {ks[0], ks[1], fp4 ? 0 : ks[2]}, width, 16) ||
      !aligned_rows(a->value_pool, {vs[0], vs[1], fp4 ? 0 : vs[2]}, width, 16) ||
      !aligned_rows(a->key_out, {a->key_out_strides[0], a->key_out_strides[1]}, out_width, 16) ||
      !aligned_rows(a->value_out, {a->value_out_strides[0], a->value_out_strides[1]}, out_width,
                    16)) {
    return reject(RKV_ERR_ALIGNMENT, "pools, rows and their strides must be multiples of 16 bytes");
  }
  RowsParams p = {};
  set_pool(p, *a);
  const int heads = static_cast<int>(a->kv_heads);
  p.key = RowStream{a->key_pool, a->key_out, ks[0], ks[2], ks[1], 0, a->key_out_strides[0],
                    a->key_out_strides[1], heads};
  p.value = RowStream{a->value_pool, a->value_out, vs[0], vs[2], vs[1], 0, a->value_out_strides[0],
                      a->value_out_strides[1], heads};
  if (p.tokens == 0) return RKV_OK;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const auto read = [&](auto launch) { return launch(p, a->key_scale, a->value_scale, st); };
  const cudaError_t err = out_width == 4 ? (fp4 ? read(launch_read<float, true>)
                                                : read(launch_read<float, false>))
                                         : (fp4 ? read(launch_read<__nv_bfloat16, true>)
                                                : read(launch_read<__nv_bfloat16, false>));
  return launched(err, "read");
}

}  // extern "C"
