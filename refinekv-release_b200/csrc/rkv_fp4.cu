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
// 72 bytes written, or the other way round.  24.5K tokens of 8 KV heads read back into
// bf16 (128 MB): 33 us, 3.9 TB/s, bound by latency: loads and the barriers of a batch of
// tokens (issue 61 %, of 13 cycles between a warp's instructions 3.8 wait for memory and
// 1.5 at a barrier).  From a bf16 pool (217 MB) 40 us, 5.4 TB/s.
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
constexpr int kBatch = 32;

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

// x / factor for any two numbers, as far as its code can tell: quotient(x * lift, by, inverse).
// `lift` is a power of two that brings the factor into [1/2, 1) (a subnormal one to 2^-23 or
// more), with its sign; so x * lift is exact, or infinite where x / factor is, or so small that
// the code is a zero, with the right sign.  A quotient that overflows is NaN instead of infinite,
// and both make 16 channels NaN.  One product more than `quotient` alone.
struct Divisor {
  float lift, by;
  __device__ void set(float factor) {
    const int exponent = static_cast<int>(__float_as_uint(factor) >> 23 & 0xffu);
    lift = copysignf(ldexpf(1.f, exponent > 0 ? 126 - exponent : 126), factor);
    by = factor * lift;
    if (fabsf(factor) == INFINITY) {
      lift = copysignf(0.f, factor);
      by = 1.f;
    }
  }
  __device__ void divide(float (&x)[2][8]) const {
    const float inverse = __frcp_rn(by);
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      x[j >> 3][j & 7] = quotient(x[j >> 3][j & 7] * lift, by, inverse);
    }
  }
};

// The scale of 16 channels whose greatest magnitude is `most`: most / 6 rounded to
// e4m3, at most 448.  A channel that is infinite or NaN makes it NaN, and with it all
// 16.
__device__ __forceinline__ uint32_t scale_of(float most) {
  uint16_t two;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %1;" : "=h"(two) : "f"(quotient(most, 6.f, 1.f / 6.f)));
  return most < INFINITY ? two & 0xffu : kFp4NanScale;
}

// The codes of 8 of the 16 channels that share a scale.
__device__ __forceinline__ uint32_t codes_of(float (&y)[8], uint32_t scale) {
  const float by = fp4_scale_value(scale), r = by > 0.f ? __frcp_rn(by) : 0.f;
#pragma unroll
  for (int j = 0; j < 8; ++j) y[j] = quotient(y[j], by, r);
  const uint32_t codes = fp4_encode(y);
  return scale == kFp4NanScale ? 0u : codes;
}

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

// The greatest magnitude of eight channels; NaN if one is.
__device__ __forceinline__ float greatest(const float (&x)[8]) {
  float most = fabsf(x[0]);
#pragma unroll
  for (int j = 1; j < 7; j += 2) {
    asm("max.NaN.f32 %0, %0, %1, %2;" : "+f"(most) : "f"(fabsf(x[j])), "f"(fabsf(x[j + 1])));
  }
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(most) : "f"(fabsf(x[7])));
  return most;
}

// A unit of work is two pieces of eight channels of one head: for a rotated
// half-layout unit c the channels at 8 c and at 8 c + rotary / 2 (the two halves of
// eight pairs), for an interleaved or copied one the 16 from 16 c.  Pieces 2 i and
// 2 i + 1 share a scale, wherever in the warp they are, so a warp holds whole heads.
// A thread keeps its unit of kHeads heads, so the table's row is read once a token;
// a CTA takes the heads of one blockIdx.y, and a token's rows are requested while
// the one before is worked on.  Measured (24.5K prompt tokens of 32 + 8 + 8 bf16 heads, D
// 128, half layout): 116 us, 530 MB; with single pieces, whose partners are read
// twice, 202 and twice the instructions; with the table's rows read from L2 for each
// token instead of ahead for a batch 149; one head a thread and 1.5 times the warps 138;
// two heads and 80 registers, which spill, 158.  fp32 rows, which spill 32 to 64 bytes: 192.
// With factors 117 and 195.
constexpr int kHeads = 2;
constexpr int kRowThreads = 256, kRowCtas = 2;

template <typename T, bool Interleaved, bool Scaled>
__global__ void __launch_bounds__(kRowThreads, kRowCtas)
    fp4_append_kernel(const __grid_constant__ RowsParams p, const float* __restrict__ key_scale,
                      const float* __restrict__ value_scale) {
  __shared__ Place places[kBatch];
  extern __shared__ float tables[];  // of the batch's tokens
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int per_head = p.dim / 16, in_warp = 32 / per_head;
  const int slot = lane / per_head, c = lane - slot * per_head;
  const int slots = (blockDim.x >> 5) * in_warp;
  const int k_from = p.query.heads, v_from = k_from + p.key.heads, heads = v_from + p.value.heads;
  const bool rotary = 16 * c < p.rotary, halves = !Interleaved && rotary;
  const int first = halves ? 8 * c : 16 * c, gap = halves ? p.rotary / 2 : 8;
  // The unit's pieces, and where the other one of each scale is.
  const int piece[2] = {first / 8, (first + gap) / 8};
  int source[2];
  bool from_second[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int other = piece[i] ^ 1, h = p.rotary / 16;
    from_second[i] = halves ? other >= h : i == 0;
    source[i] = halves ? slot * per_head + (other >= h ? other - h : other) : lane;
  }
  int kind[kHeads];  // 0 query, 1 key, 2 value, -1 nothing
  const T* in[kHeads];
  uint8_t* out[kHeads];  // of a query head, or of a KV head in page 0
  int64_t in_t[kHeads];
  // Each thread its own: in registers, which are short, fp32 rows took 207 us instead of 195.
  __shared__ Divisor divisors[Scaled ? kHeads * kRowThreads : 1];
#pragma unroll
  for (int u = 0; u < kHeads; ++u) {
    const int head = (blockIdx.y * kHeads + u) * slots + warp * in_warp + slot;
    kind[u] = slot >= in_warp || head >= heads ? -1 : head < k_from ? 0 : head < v_from ? 1 : 2;
    const RowStream& s = kind[u] <= 0 ? p.query : kind[u] == 1 ? p.key : p.value;
    const int own = head - (kind[u] <= 0 ? 0 : kind[u] == 1 ? k_from : v_from);
    in[u] = static_cast<const T*>(s.in) + own * s.in_h + first;
    in_t[u] = s.in_t;
    out[u] = kind[u] == 0
                 ? reinterpret_cast<uint8_t*>(static_cast<T*>(s.out) + own * s.out_h + first)
                 : static_cast<uint8_t*>(s.out) + own * s.out_h;
  }
  struct Rows {
    Eight<T> x[kHeads][2];
  };
  const auto request = [&](unsigned n, Rows& rows) {
#pragma unroll
    for (int u = 0; u < kHeads; ++u) {
      if (kind[u] < 0) continue;
      const T* from = in[u] + n * in_t[u];
      rows.x[u][0].load(from);
      rows.x[u][1].load(from + gap);
    }
  };
  pdl_wait();
  pdl_launch_dependents();
  if constexpr (Scaled) {
#pragma unroll
    for (int u = 0; u < kHeads; ++u) {
      const int head = (blockIdx.y * kHeads + u) * slots + warp * in_warp + slot;
      const float* factors = kind[u] == 1 ? key_scale : kind[u] == 2 ? value_scale : nullptr;
      const int own = head - (kind[u] == 1 ? k_from : v_from);
      divisors[u * kRowThreads + threadIdx.x].set(factors != nullptr ? factors[own] : 1.f);
    }
  }
  const unsigned tokens = static_cast<unsigned>(p.tokens);
  for (unsigned at_token = blockIdx.x; at_token < tokens;
       at_token += gridDim.x * min(kBatch, blockDim.x)) {
    Rows rows, next;
    request(at_token, rows);
    const unsigned there = find_places(p, places, at_token, blockIdx.y == 0);
    // The batch's rows of the table; a position outside it: NaN.
    if (p.rotary > 0) {
      const unsigned quads = p.rotary / 4;
      for (unsigned x = threadIdx.x; x < there * quads; x += blockDim.x) {
        const unsigned i = x / quads;
        const float nan = __int_as_float(0x7fc00000);
        float4 four = make_float4(nan, nan, nan, nan);
        if (places[i].known) {
          four = *reinterpret_cast<const float4*>(p.cos_sin + places[i].pos * p.table_stride +
                                                  4 * (x - i * quads));
        }
        reinterpret_cast<float4*>(tables)[x] = four;
      }
      __syncthreads();
    }
    for (unsigned i = 0; i < there; ++i) {
      const unsigned n = at_token + i * gridDim.x;
      if (i + 1 < there) request(n + gridDim.x, next);
      const Place at = places[i];
      float cs[8], sn[8];
      if (rotary) {
        const float* table = tables + i * p.rotary + 8 * c;
        load8(table, cs);
        load8(table + p.rotary / 2, sn);
      }
#pragma unroll
      for (int u = 0; u < kHeads; ++u) {
        float x[2][8];
        rows.x[u][0].widen(x[0]);
        rows.x[u][1].widen(x[1]);
        if (rotary && kind[u] < 2) {
          // No fused multiply-add: the codes are those of the formula in fp32.
          const auto turn = [](float& a, float& b, float cos, float sin) {
            const float y = __fsub_rn(__fmul_rn(a, cos), __fmul_rn(b, sin));
            b = __fadd_rn(__fmul_rn(b, cos), __fmul_rn(a, sin));
            a = y;
          };
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            if constexpr (Interleaved) {
              turn(x[j >> 2][2 * j & 7], x[j >> 2][(2 * j & 7) + 1], cs[j], sn[j]);
            } else {
              turn(x[0][j], x[1][j], cs[j], sn[j]);
            }
          }
        }
        if (kind[u] == 0) {
          T* to = reinterpret_cast<T*>(out[u]) + n * p.query.out_t;
          if (at.pos < 0) {
#pragma unroll
            for (int j = 0; j < 8; ++j) x[0][j] = x[1][j] = 0.f;
          }
          store8(to, x[0]);
          store8(to + gap, x[1]);
        }
        // Warps of queries alone have no scales to find.
        if (__all_sync(0xffffffffu, kind[u] <= 0)) continue;
        if constexpr (Scaled) divisors[u * kRowThreads + threadIdx.x].divide(x);
        const float most[2] = {greatest(x[0]), greatest(x[1])};
        uint32_t scale[2];
#pragma unroll
        for (int i2 = 0; i2 < 2; ++i2) {
          const float p0 = __shfl_sync(0xffffffffu, most[0], source[i2]);
          const float p1 = __shfl_sync(0xffffffffu, most[1], source[i2]);
          float both;
          asm("max.NaN.f32 %0, %1, %2;" : "=f"(both) : "f"(most[i2]), "f"(from_second[i2] ? p1 : p0));
          scale[i2] = scale_of(both);
        }
        if (kind[u] > 0 && at.keep) {
          const RowStream& s = kind[u] == 1 ? p.key : p.value;
          uint8_t* slab = out[u] + at.page * s.out_b;
          uint8_t* codes = slab + at.row * (p.dim / 2);
          uint8_t* scales = slab + (p.dim / 2 << p.block_shift) + at.row * (p.dim / 16);
#pragma unroll
          for (int i2 = 0; i2 < 2; ++i2) {
            *reinterpret_cast<uint32_t*>(codes + 4 * piece[i2]) = codes_of(x[i2], scale[i2]);
            if (!(piece[i2] & 1)) scales[piece[i2] / 2] = static_cast<uint8_t>(scale[i2]);
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
  const int heads = p.query.heads + p.key.heads + p.value.heads, in_warp = 32 / (p.dim / 16);
  // A token's heads in as few CTAs as hold them, shared out evenly.
  const int warps = (heads + kHeads * in_warp - 1) / (kHeads * in_warp), most = kRowThreads / 32;
  const int ctas = (warps + most - 1) / most, threads = (warps + ctas - 1) / ctas * 32;
  int sms = 0;
  if (device_sms(&sms) != RKV_OK) return cudaErrorInvalidDevice;
  const int64_t resident = std::max<int64_t>(
      1, static_cast<int64_t>(sms) * (kRowCtas * kRowThreads / threads) / ctas);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(std::min(p.tokens, resident)), ctas);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = static_cast<size_t>(kBatch) * p.rotary * 4;  // 32 KB at most
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  // Factors apart: fp32 rows without them 192 us against 203, bf16 rows 115 either way.
  if (key_scale != nullptr || value_scale != nullptr) {
    return cudaLaunchKernelEx(&cfg, fp4_append_kernel<T, Interleaved, true>, p, key_scale,
                              value_scale);
  }
  return cudaLaunchKernelEx(&cfg, fp4_append_kernel<T, Interleaved, false>, p, key_scale,
                            value_scale);
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
// The same tokens with a rotary width of 24: 413 us (fp32 rows 423).
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
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const int d = 16 * block + j;
      float x = is_key ? turned(p, row, d, table, Interleaved) : widen(row[d]);
      if (factors != nullptr) x = __fdiv_rn(x, factors[own]);
      y[j >> 3][j & 7] = x;
    }
    float most;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(most) : "f"(greatest(y[0])), "f"(greatest(y[1])));
    const uint32_t scale = scale_of(most);
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
  const bool pieces = rows_aligned(16) && p.rotary % 16 == 0 &&
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
