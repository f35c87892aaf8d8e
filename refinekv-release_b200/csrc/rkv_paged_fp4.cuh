// paged_kernel over pools of 4 bits.
//
// Mathematics.  A channel is code * scale (rkv_fp4.cuh), six significant bits,
// exact in fp16; so a tile's codes become fp16 operands (one conversion and one
// product a pair) and the matrix instructions see the very numbers that the pool
// stands for.  Queries (bf16, 8 bits) are moved by a power of two into fp16's
// range, and the weights are held in fp16 terms: one for bf16 queries (2^-11,
// against the output's own 2^-8: the error against 64 bits is that of a result rounded once,
// and two would take 170 us instead of 143), two for fp32 queries (2^-22), however small a
// weight is against the greatest of its row.  A query's channels of less than 2^-29 of its
// greatest one lose digits.
//
// Tiles hold 64 tokens, so that a page is at most one tile and a page's slab of a KV
// head is fetched by one bulk copy.  Which channels and tokens a lane holds is
// chosen so that its codes lie together: the k index of a product and the rows
// of its result may be taken in any order as long as both operands agree.
//   scores: lane 4 r + j has a quarter j of the channels of tokens r and r + 8
//     of 16 (dim 128: 16 bytes of codes and two scales each);
//   values: lane 4 g + j has an eighth g of the channels of four tokens (dim 128: 8
//     bytes of codes and one scale each), whose codes are paired by token before the
//     conversion.  Tokens 2j and 2j + 1 change places for odd j, and with them the
//     rows of the scores, or the four j of a load would hit the same banks.
//
// Bound: latency, with three warps a scheduler that each go alone through loads, conversions,
// products, votes and exponentials.  An instruction issues in 61 % of the cycles and 1.06 warps
// could have; of a warp's 4.75 cycles between two of its instructions 1.3 wait for a result
// of fixed latency, 0.7 for the other warps, 0.55 for a busy pipe (ALU 50 %, tensor 21 %), 0.2
// for memory.  16 sequences of 32K tokens (32 + 8 heads, D 128, 604 MB): 141 to 144 us, 4.2
// TB/s, 1400 warp instructions a tile of 64 tokens; 128K tokens 48.0; 333 tokens 9.6, more than
// from a bf16 pool (8.2): half of the warps have no tile, and a tile alone takes 4 us.
#pragma once

#include "rkv_fp4.cuh"
#include "rkv_paged.cu"

namespace rkv {
namespace {

__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                        uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7},"
      " {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// The same from zero.
__device__ __forceinline__ void mma_f16_first(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                              uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7},"
      " {%8, %9}, {%10, %10, %10, %10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}

// Kept behind the waits for the copies by being volatile, like them.
template <int Bytes>
__device__ __forceinline__ uint32_t lds(uint32_t at) {
  uint32_t x;
  if constexpr (Bytes == 1) asm volatile("ld.shared.u8 %0, [%1];" : "=r"(x) : "r"(at));
  if constexpr (Bytes == 2) asm volatile("ld.shared.u16 %0, [%1];" : "=r"(x) : "r"(at));
  if constexpr (Bytes == 4) asm volatile("ld.shared.u32 %0, [%1];" : "=r"(x) : "r"(at));
  return x;
}

// N words from an address that is aligned to the widest load that N allows.
template <int N>
__device__ __forceinline__ void lds_words(uint32_t at, uint32_t (&x)[N]) {
  if constexpr (N % 4 == 0) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                   : "=r"(x[i]), "=r"(x[i + 1]), "=r"(x[i + 2]), "=r"(x[i + 3])
                   : "r"(at + 4 * i));
    }
  } else if constexpr (N % 2 == 0) {
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];"
                   : "=r"(x[i]), "=r"(x[i + 1])
                   : "r"(at + 4 * i));
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = lds<4>(at + 4 * i);
  }
}

__device__ __forceinline__ uint32_t times(uint32_t a, uint32_t b) {
  const __half2 y = __hmul2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&y);
}

__device__ __forceinline__ uint32_t low_twice(uint32_t pair) {
  return __byte_perm(pair, pair, 0x1010);
}
__device__ __forceinline__ uint32_t high_twice(uint32_t pair) {
  return __byte_perm(pair, pair, 0x3232);
}
__device__ __forceinline__ float exp2_of(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Weights and their sums are held 2^13 times as large within a tile and a row's part,
// and up to 2^2 times the reference's: fp16 terms of weights down to 2^-27 of the
// greatest are then normal.  Smaller ones (below kLeast, fp16's smallest normal number) are
// held kStep times as large.
constexpr float kBoost = 13.f, kLag = 2.f;
constexpr float kUnboost = 1.f / 8192.f;
constexpr float kLeast = 1.f / 16384.f;
constexpr float kStep = 16777216.f;
// The second term of a weight is held 2^11 times as large: the first one's error is at
// most 2^-11 of the weight, so that both have the same range, and 22 bits down to kLeast.
constexpr float kFine = 2048.f;
constexpr float kLog2E = 1.44269504088896341f;

template <int Dim, int NT_>
struct Fp4Pool {
  static constexpr int D = Dim, NT = NT_, R = kFp4Rows;
  // Eight where twelve would spill.  Spilled all the same, bytes of stores a thread: 16 (D 256); with
  // 9 to 16 queries a KV head 12 (D 160), 154 (192), 560 (224), 748 (256).  8 sequences of 32K
  // tokens, 2 KV heads of 16 queries: 43 us (D 128), 55, 59 and 80 (D 256; bf16 pool: 102).
  static constexpr int W = NT == 1 && Dim <= 192 ? 12 : 8;
  static constexpr int kTile = fp4_slab_bytes(R, Dim);
  static constexpr bool kFirstInSmem = Dim <= 128;
  // Short batches: the longer ones' registers would spill with 12 warps (128K tokens 53.3
  // against 49.9 us).
  static constexpr int kJoinBatch = 4, kLongBatch = 6;
  // Kept scores apart from shape_logits: 128K tokens 57 us against 64.
  static constexpr bool kBareScores = true;
  static constexpr int kRow = Dim / 2;      // bytes of a row's codes
  static constexpr int kScales = Dim / 16;  // and of its scales
  static constexpr int kWords = Dim / 32;   // words of a lane's part of a key's codes
  static constexpr int kBytes = Dim / 16;   // bytes of a lane's part of a value's codes
  // A lane's logits, and then its weights' terms, of 16 rows each while those are not worked
  // on: 16 bytes a column tile.
  static constexpr int kLane = 16 * NT, kScratch = R / 16 * 32 * kLane;
  static_assert(warp_partial_floats(D, NT) * 4 <= 2 * kTile, "a partial waits in its warp's stage");
  using Source = Fp4Pages;
  struct Query {
    uint32_t frags[D / 16][NT][2];  // fp16, times 2^k
    float scale[NT][2];             // what the lane's columns are multiplied by
  };
  using Logits = float (&)[R / 16][NT][4];
  using Columns = float (&)[NT][2];
  using Outputs = float (&)[D / 16][NT][4];

  // Neighbouring ranges on different schedulers (warp w's is w % 4): where there are fewer
  // tiles than warps, every second range has one, and in order those would share two of
  // the four (333 tokens: 9.5 us against 10.4).
  static_assert(W % 4 == 0, "as many warps on every scheduler");
  static __device__ __forceinline__ int range_of(int warp) {
    return warp % 4 * (W / 4) + warp / 4;
  }
  // A tile takes some 4 us alone on its scheduler, so a row is worth a CTA for every
  // fourth of its tiles (1000 tokens of 8 heads: 10.7 us against 13.3 with every warp a
  // tile), but one CTA where each tile has a warp (333 tokens: 9.5 against 10.3).
  static __device__ __forceinline__ unsigned ctas_of(unsigned tiles, unsigned rows) {
    return tiles <= W * rows ? 1 : (tiles / rows + 3) / 4;
  }
  static __device__ __forceinline__ void prefetch(const Source&) {}
  static __device__ __forceinline__ int box_bytes(int rows) { return rows * (kRow + kScales); }
  // A box is a page: its slab in two pieces, so that a tile's codes lie together and its
  // scales behind them, whatever the pages' size.
  static constexpr int kPieces = 2;
  struct Lane {  // the piece that a lane fetches: from where in a slab, to where in a tile
    uint32_t from, to, bytes;
    __device__ Lane(int lane, int boxes, int box_rows) {
      const int box = lane & (boxes - 1), codes = box_rows * kRow, scales = box_rows * kScales;
      const bool second = lane >= boxes;
      from = second ? codes : 0;
      to = second ? R * kRow + box * scales : box * codes;
      bytes = second ? scales : codes;
    }
  };
  static __device__ __forceinline__ void fetch(const Source& pages, const Lane& own, int which,
                                               uint8_t* tile, uint64_t* bar, int, int head, int page,
                                               uint64_t policy) {
    const uint64_t units =
        static_cast<uint64_t>(static_cast<uint32_t>(page)) * pages.page[which] +
        static_cast<uint64_t>(static_cast<uint32_t>(head)) * pages.head[which];
    asm volatile(
        "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint"
        " [%0], [%1], %2, [%3], %4;" ::"r"(smem_addr(tile) + own.to),
        "l"(pages.pool[which] + own.from + units * 16), "r"(own.bytes), "r"(smem_addr(bar)),
        "l"(policy)
        : "memory");
  }

  // Word w of the quarter j of a query row: channels j Dim / 4 + 8 w and on.
  static __device__ __forceinline__ void load_queries(Query& q, const PagedParams& p, int seq,
                                                      int head, int lane) {
    const int64_t base = seq * p.q_seq + static_cast<int64_t>(head) * p.group * p.q_head;
    const float factor = p.scale * (p.key_scale != nullptr ? p.key_scale[head] : 1.f);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int g = nt * 8 + (lane >> 2);
      const int64_t row = base + min(g, p.group - 1) * p.q_head + (lane & 3) * (Dim / 4);
      float x[kWords][8];
      uint32_t most = 0;  // of the finite ones
#pragma unroll
      for (int w = 0; w < kWords; ++w) {
        if (p.query_f32) {
          const float4* from =
              reinterpret_cast<const float4*>(static_cast<const float*>(p.query) + row + 8 * w);
          const float4 a = from[0], b = from[1];
          const float raw[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
          for (int i = 0; i < 8; ++i) x[w][i] = bf16_round(raw[i]);
        } else {
          const uint4 four = *reinterpret_cast<const uint4*>(
              static_cast<const __nv_bfloat16*>(p.query) + row + 8 * w);
          const uint32_t raw[4] = {four.x, four.y, four.z, four.w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            x[w][2 * i] = __uint_as_float(raw[i] << 16);
            x[w][2 * i + 1] = __uint_as_float(raw[i] & 0xffff0000u);
          }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const uint32_t size = __float_as_uint(x[w][i]) & 0x7fffffffu;
          if (size < 0x7f800000u) most = max(most, size);
        }
      }
      most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
      most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
      // 2^k brings the row's greatest into [2^14, 2^15): whatever lies within 2^29
      // of it keeps all its bits.
      const int k = min(126, 141 - static_cast<int>(most >> 23));
      const float up = __int_as_float((127 + k) << 23), down = __int_as_float((127 - k) << 23);
#pragma unroll
      for (int w = 0; w < kWords; ++w)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const __half2 pair = __floats2half2_rn(x[w][2 * i] * up, x[w][2 * i + 1] * up);
          q.frags[2 * w + (i >> 1)][nt][i & 1] =
              g < p.group ? *reinterpret_cast<const uint32_t*>(&pair) : 0u;
        }
#pragma unroll
      for (int col = 0; col < 2; ++col) {
        q.scale[nt][col] = factor * __shfl_sync(0xffffffffu, down, 4 * (2 * (lane & 3) + col));
      }
    }
  }
  static __device__ __forceinline__ float column_scale(const Query& q, const PagedParams&, int nt,
                                                       int col, int lane) {
    return q.scale[nt][col];
  }
  static __device__ __forceinline__ int swapped(int r) { return r ^ (r >> 1 & 1); }
  static __device__ __forceinline__ int token_of(int mt, int half, int lane) {
    return mt * 16 + swapped(lane >> 2) + half * 8;
  }
  static __device__ __forceinline__ int channel(int dt, int half, int lane) {
    return (lane >> 2) * (Dim / 8) + 2 * dt + half;
  }

  // The scales of a lane's words of one key row, each twice in a pair.
  static __device__ __forceinline__ void key_scales(uint32_t at, int j, uint32_t (&s)[kWords]) {
    if constexpr (kWords % 4 == 0) {
#pragma unroll
      for (int i = 0; i < kWords / 4; ++i) {
        const uint32_t pair = fp4_scales(lds<2>(at + j * (kWords / 2) + 2 * i));
        s[4 * i] = s[4 * i + 1] = low_twice(pair);
        s[4 * i + 2] = s[4 * i + 3] = high_twice(pair);
      }
    } else {
#pragma unroll
      for (int w = 0; w < kWords; ++w) {
        if (kWords % 2 == 0 && w % 2 == 1) {
          s[w] = s[w - 1];
        } else {
          s[w] = low_twice(fp4_scales(lds<1>(at + ((j * kWords + w) >> 1))));
        }
      }
    }
  }

  // The rows are taken 16 at a time by loops that are not unrolled: unrolled, a tile is some
  // 1500 instructions that miss the instruction caches and spill (then 153 us against 146 for
  // 16 sequences of 32K tokens).  What outlives an iteration waits in shared memory.
  static __device__ __forceinline__ void score(uint32_t tile, const Query& q, Logits logit,
                                               uint32_t scratch, int lane, const PagedParams& p) {
    const int j = lane & 3, row = swapped(lane >> 2);
    uint32_t codes = tile + row * kRow + j * 4 * kWords;
    uint32_t scales = tile + R * kRow + row * kScales;
    uint32_t keep = scratch + lane * kLane;
#pragma unroll 1
    for (int mt = 0; mt < R / 16; ++mt) {
      float acc[NT][2][4];  // two sums of products: half as long a chain
      uint32_t a[kWords], b[kWords], sa[kWords], sb[kWords];
      lds_words(codes, a);
      lds_words(codes + 8 * kRow, b);
      key_scales(scales, j, sa);
      key_scales(scales + 8 * kScales, j, sb);
#pragma unroll
      for (int w = 0; w < kWords; ++w) {
        uint32_t x[4], y[4];
        fp4_decode(a[w], x);
        fp4_decode(b[w], y);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          x[i] = times(x[i], sa[w]);
          y[i] = times(y[i], sb[w]);
        }
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const uint32_t frag[4] = {x[2 * half], y[2 * half], x[2 * half + 1], y[2 * half + 1]};
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            const uint32_t(&b)[2] = q.frags[2 * w + half][nt];
            if (w == 0) {
              mma_f16_first(acc[nt][half], frag, b[0], b[1]);
            } else {
              mma_f16(acc[nt][half], frag, b[0], b[1]);
            }
          }
        }
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(keep + 16 * nt),
                     "f"(acc[nt][0][0] + acc[nt][1][0]), "f"(acc[nt][0][1] + acc[nt][1][1]),
                     "f"(acc[nt][0][2] + acc[nt][1][2]), "f"(acc[nt][0][3] + acc[nt][1][3]));
      }
      codes += 16 * kRow;
      scales += 16 * kScales;
      keep += 32 * kLane;
    }
#pragma unroll
    for (int mt = 0; mt < R / 16; ++mt)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
                     : "=f"(logit[mt][nt][0]), "=f"(logit[mt][nt][1]), "=f"(logit[mt][nt][2]),
                       "=f"(logit[mt][nt][3])
                     : "r"(scratch + mt * 32 * kLane + lane * kLane + 16 * nt));
      }
  }

  // Online softmax whose reference follows the maximum only when a logit exceeds it by
  // kLag (in powers of two): a vote a tile instead of six shuffles in a row, and sums
  // that are seldom rescaled.  Weights are then at most 2^(kLag + kBoost), fp16's
  // range, and a row's parts join as before: any reference serves.
  static __device__ __forceinline__ void softmax(Logits logit, Columns m, Columns l, Outputs o) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float mx[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        mx[j] = fmaxf(logit[0][nt][j], logit[0][nt][2 + j]);
#pragma unroll
        for (int mt = 1; mt < R / 16; ++mt)
          mx[j] = fmaxf(mx[j], fmaxf(logit[mt][nt][j], logit[mt][nt][2 + j]));
      }
      if (__any_sync(0xffffffffu, mx[0] > m[nt][0] + kLag / kLog2E ||
                                      mx[1] > m[nt][1] + kLag / kLog2E)) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          mx[j] = fmaxf(mx[j], __shfl_xor_sync(0xffffffffu, mx[j], 4));
          mx[j] = fmaxf(mx[j], __shfl_xor_sync(0xffffffffu, mx[j], 8));
          mx[j] = fmaxf(mx[j], __shfl_xor_sync(0xffffffffu, mx[j], 16));
          const float top = fmaxf(m[nt][j], mx[j]);
          const float alpha = exp2_of((m[nt][j] - finite_or_zero(top)) * kLog2E);
          m[nt][j] = top;
          l[nt][j] *= alpha;
#pragma unroll
          for (int dt = 0; dt < D / 16; ++dt) {
            o[dt][nt][j] *= alpha;
            o[dt][nt][2 + j] *= alpha;
          }
        }
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float ref = finite_or_zero(m[nt][j]);
#pragma unroll
        for (int mt = 0; mt < R / 16; ++mt)
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            float& x = logit[mt][nt][2 * half + j];
            x = exp2_of(fmaf(x - ref, kLog2E, kBoost));
            l[nt][j] += x;
          }
      }
    }
  }

  // A row's part ends: its sums without the boost (exact).
  static __device__ __forceinline__ void settle(Columns l, Outputs o) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      l[nt][0] *= kUnboost;
      l[nt][1] *= kUnboost;
#pragma unroll
      for (int dt = 0; dt < D / 16; ++dt)
#pragma unroll
        for (int c = 0; c < 4; ++c) o[dt][nt][c] *= kUnboost;
    }
  }

  static __device__ __forceinline__ void weigh(uint8_t* at, uint32_t tile, Logits weights, Outputs o,
                                               const Seen& seen, uint32_t scratch, int lane,
                                               const PagedParams& p) {
    if (!seen.all(R)) {
      // Rows that are not visible may hold anything: scales of zero make their
      // channels zero (codes are finite).
      uint16_t* scales = reinterpret_cast<uint16_t*>(at + R * kRow);
      for (int i = lane; i < R * kScales / 2; i += 32) {
        if (!seen.row(i / (kScales / 2))) scales[i] = 0;
      }
      __syncwarp();
    }
    // Weights below kLeast have fewer than 11 bits in fp16, or none, and they count where the
    // values of the greater ones are zero.  bf16 queries: a tile that has such weights has
    // them in a second operand, kStep times as large.  What the operands cut off of a tile's
    // weights goes through by itself where it can matter.  16 sequences of 32K tokens: 141
    // to 144 us where fp16 holds all weights, 165 to 182 with logits that spread by 3.5 to 7
    // (standard deviation), 255 by 14, 222 with biases of up to 0.84 a token (without any
    // of this 141, and 176 with the biases).
    const uint32_t least = least_of(weights);
    const auto some_below = [&](float bound) {
      return __any_sync(0xffffffffu, least < __float_as_uint(bound) - 1u);
    };
    const bool small = some_below(kLeast);
    if (!p.query_f32 && !small) {
      weigh_terms<1, 1>(tile, weights, o, scratch, lane);
      return;
    }
    // The weights below this are cut off, at 2^-11 of it (2^-22: fp32 queries) at the most.
    const float bound = p.query_f32 ? kLeast : kLeast / kStep;
    const bool cut = p.query_f32 ? small : some_below(bound);
    volatile float held[R / 16][NT][4];
    if (cut) hold(weights, held);
    if (p.query_f32) weigh_terms<2, 1>(tile, weights, o, scratch, lane);
    else weigh_terms<1, 2>(tile, weights, o, scratch, lane);
    if (!cut || negligible(tile, o, bound / kFine / (p.query_f32 ? kFine : 1.f), lane, p)) return;
    weigh_rest(tile, held, o, scratch, lane, p, [&](float w) {
      if (!(w < bound)) return 0.f;
      const float up = p.query_f32 ? 1.f : kStep;
      const float rest = w - __half2float(__float2half_rn(w * up)) / up;
      if (!p.query_f32) return rest;
      return rest - __half2float(__float2half_rn(rest * kFine)) * (1.f / kFine);
    });
  }

  // Puts a tile's weights aside: local memory, since nothing else has room, and it is seldom
  // read back.
  static __device__ __forceinline__ void hold(Logits weights, volatile float (&held)[R / 16][NT][4]) {
#pragma unroll
    for (int mt = 0; mt < R / 16; ++mt)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 4; ++c) held[mt][nt][c] = weights[mt][nt][c];
  }

  // Whether a tile's weights may be off by this much each: where every channel's sum is by now
  // so large that all tiles together would change it by less than 2^-18 of its size (2^-21:
  // fp32 queries).
  static __device__ __forceinline__ bool negligible(uint32_t tile, Outputs o, float off, int lane,
                                                    const PagedParams& p) {
    uint32_t words[D / 32], most = 0;  // the greatest scale
    lds_words(tile + R * kRow + lane * (D / 8), words);
#pragma unroll
    for (int i = 0; i < D / 32; ++i) most = __vmaxu4(most, words[i]);
    most = __vmaxu4(most, most >> 16);
    most = __reduce_max_sync(0xffffffffu, max(most & 0xffu, most >> 8 & 0xffu));
    float least = INFINITY;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int dt = 0; dt < D / 16; ++dt)
#pragma unroll
        for (int c = 0; c < 4; ++c) least = fminf(least, fabsf(o[dt][nt][c]));
    off *= 6.f * fp4_scale_value(most) * static_cast<float>(p.capacity + R);
    return __all_sync(0xffffffffu, least >= off * (p.query_f32 ? 2097152.f : 262144.f));
  }

  // The least of a lane's weights that are not zero (those of rows that are not visible are), as
  // an integer less 1.
  static __device__ __forceinline__ uint32_t least_of(Logits weights) {
    uint32_t least = 0xffffffffu;
#pragma unroll
    for (int mt = 0; mt < R / 16; ++mt)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 4; ++c) least = min(least, __float_as_uint(weights[mt][nt][c]) - 1u);
    return least;
  }

  // The fp16 terms of a lane's four weights of 16 rows, as operands.
  template <int Terms>
  static __device__ __forceinline__ void split(float (&w)[4], uint32_t (*frag)[2]) {
#pragma unroll
    for (int term = 0; term < Terms; ++term)
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        float& a = w[2 * half];
        float& b = w[2 * half + 1];
        const __half2 part = __floats2half2_rn(a, b);
        if (term + 1 < Terms) {
          a = (a - __low2float(part)) * kFine;
          b = (b - __high2float(part)) * kFine;
        }
        frag[term][half] = movmatrix_trans(*reinterpret_cast<const uint32_t*>(&part));
      }
  }

  // o += V^T r with the part r = rest(w) of each weight that its operands do not hold, numbers of
  // any size (the exponential gives nothing below fp32's normal ones): those within 2^28 of
  // the greatest as many times as large as brings that one to 2^14 or more, in two terms, and
  // their products added by as little of them; then the ones below these, and so on until
  // what is left is negligible, five times at most.
  template <typename Rest>
  static __device__ __forceinline__ void weigh_rest(uint32_t tile,
                                                    volatile float (&held)[R / 16][NT][4], Outputs o,
                                                    uint32_t scratch, int lane, const PagedParams& p,
                                                    Rest rest) {
    // They wait in shared memory, as the logits did, until they are done with.
    const uint32_t kept = scratch + lane * kLane;
    const auto put = [&](int mt, int nt, const float (&w)[4]) {
      asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(kept + mt * 32 * kLane + 16 * nt),
                   "f"(w[0]), "f"(w[1]), "f"(w[2]), "f"(w[3]));
    };
    const auto get = [&](int mt, int nt, float (&w)[4]) {
      asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
                   : "=f"(w[0]), "=f"(w[1]), "=f"(w[2]), "=f"(w[3])
                   : "r"(kept + mt * 32 * kLane + 16 * nt));
    };
#pragma unroll
    for (int mt = 0; mt < R / 16; ++mt)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float w[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) w[c] = rest(held[mt][nt][c]);
        put(mt, nt, w);
      }
#pragma unroll 1
    for (int time = 0; time < 5; ++time) {
      float greatest = 0.f;
#pragma unroll
      for (int mt = 0; mt < R / 16; ++mt)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float w[4];
          get(mt, nt, w);
#pragma unroll
          for (int c = 0; c < 4; ++c) greatest = fmaxf(greatest, fabsf(w[c]));
        }
      const uint32_t most = __reduce_max_sync(0xffffffffu, __float_as_uint(greatest));
      // 2^k brings the greatest into [2^14, 2^15), or as near as a normal number 2^-k allows;
      // this is 2^-k, found again wherever it is needed: registers are short here.
      const auto down = [most] {
        uint32_t again = most;
        asm volatile("" : "+r"(again));
        return __int_as_float((127 - min(126, 141 - static_cast<int>(again >> 23))) << 23);
      };
      if (most == 0 || negligible(tile, o, __uint_as_float(most), lane, p)) return;
      weigh_rows<2, 1, true>(tile, o, lane, down, [&](int mt, uint32_t (&frag)[NT][2][2]) {
        const float unit = down(), up = 1.f / unit, least = kLeast * unit;  // exact, if subnormal
        bool some = false;
        float w[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float all[4];
          get(mt, nt, all);
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const bool now = fabsf(all[c]) >= least;
            w[nt][c] = now ? all[c] * up : 0.f;
            if (now) all[c] = 0.f;
            some = some || now;
          }
          put(mt, nt, all);
        }
        if (!__any_sync(0xffffffffu, some)) return false;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) split<2>(w[nt], frag[nt]);
        return true;
      });
    }
  }

  // o += V^T p, the weights of each of `Sizes` sizes in `Terms` fp16 terms.
  template <int Terms, int Sizes>
  static __device__ __forceinline__ void weigh_terms(uint32_t tile, Logits weights, Outputs o,
                                                     uint32_t scratch, int lane) {
    constexpr int kOperands = Terms * Sizes;
    static_assert(kOperands <= 2, "8 bytes each of a lane's 16");
    const uint32_t kept = scratch + lane * kLane;
#pragma unroll
    for (int mt = 0; mt < R / 16; ++mt)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        uint32_t frag[kOperands][2];
        float(&w)[4] = weights[mt][nt];
        if constexpr (Sizes > 1) {
          float low[4];
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            low[c] = w[c] < kLeast ? w[c] * kStep : 0.f;
            if (w[c] < kLeast) w[c] = 0.f;  // a NaN stays
          }
          split<1>(low, &frag[1]);
        }
        split<Terms>(w, &frag[0]);
        const uint32_t to = kept + mt * 32 * kLane + 16 * nt;
#pragma unroll
        for (int k = 0; k < kOperands; ++k) {
          asm volatile("st.shared.v2.u32 [%0], {%1, %2};" ::"r"(to + 8 * k), "r"(frag[k][0]),
                       "r"(frag[k][1]));
        }
      }
    const auto load = [&](int mt, uint32_t (&frag)[NT][kOperands][2]) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int k = 0; k < kOperands; ++k) {
          asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];"
                       : "=r"(frag[nt][k][0]), "=r"(frag[nt][k][1])
                       : "r"(kept + mt * 32 * kLane + 16 * nt + 8 * k));
        }
      return true;
    };
    weigh_rows<Terms, Sizes, false>(tile, o, lane, [] { return 1.f; }, load);
  }

  // o += V^T p (factor() times, where Scaled), 16 rows at a time; load(i, frag) gets the
  // operands of the i-th 16 weights, or says that there is nothing to add.  With two
  // terms 16 rows' products are summed apart and added by a rounded addition, since the
  // tensor cores cut their sums off.  Codes are taken kChunk bytes at a time.
  template <int Terms, int Sizes, bool Scaled, typename Factor, typename Load>
  static __device__ __forceinline__ void weigh_rows(uint32_t tile, Outputs o, int lane, Factor factor,
                                                    Load load) {
    constexpr int kOperands = Terms * Sizes;
    const int g = lane >> 2, j = lane & 3;
    const int first = 2 * j + (j & 1), second = 2 * j + 1 - (j & 1);  // swapped(2j), swapped(2j + 1)
    // Channels are taken by units of 8 (a word), or 4 where a lane's part is no whole words.
    constexpr int kUnit = kBytes % 4 == 0 ? 4 : 2;
    constexpr int kChunk = Terms == 1 && kBytes % 8 == 0 ? 8 : kUnit;
    constexpr int kUnits = kChunk / kUnit;
    constexpr uint32_t kLow = 0x0f0f0f0fu;
    uint32_t codes_at[2] = {tile + first * kRow + g * kBytes, tile + second * kRow + g * kBytes};
    uint32_t scales_at[2] = {tile + R * kRow + first * kScales, tile + R * kRow + second * kScales};
#pragma unroll 1
    for (int mt = 0; mt < R / 16; ++mt) {
      const uint32_t codes_16 = mt * 16 * kRow, scales_16 = mt * 16 * kScales;
      uint32_t frag[NT][kOperands][2];
      if (!load(mt, frag)) continue;
#pragma unroll
      for (int chunk = 0; chunk < kBytes / kChunk; ++chunk) {
        uint32_t codes[4][kUnits], scale[4];
        [[maybe_unused]] const float by = factor();
        // Two units of a chunk lie in one block of 16 channels.
        const int block = (g * (kBytes / kUnit) + chunk * kUnits) / (kUnit == 4 ? 2 : 4);
#pragma unroll
        for (int t = 0; t < 4; ++t) {  // tokens first, second, first + 8, second + 8
          const uint32_t at = codes_at[t & 1] + codes_16 + (t >> 1) * 8 * kRow + chunk * kChunk;
          if constexpr (kUnit == 4) {
            lds_words(at, codes[t]);
          } else {
            codes[t][0] = lds<2>(at);
          }
          scale[t] = lds<1>(scales_at[t & 1] + scales_16 + block + (t >> 1) * 8 * kScales);
        }
        // The scales of tokens 0 and 1, and 2 and 3.
        const uint32_t near = fp4_scales(__byte_perm(scale[0], scale[1], 0x0040));
        const uint32_t far = fp4_scales(__byte_perm(scale[2], scale[3], 0x0040));
#pragma unroll
        for (int u = 0; u < kUnits; ++u) {
          // A byte has two channels of a token; exchanged, one channel of two tokens: the
          // even channels' and the odd ones' of tokens 0 and 1, and of 2 and 3.
          const uint32_t mixed[4] = {
              (codes[0][u] & kLow) | (codes[1][u] << 4 & ~kLow),
              (codes[0][u] >> 4 & kLow) | (codes[1][u] & ~kLow),
              (codes[2][u] & kLow) | (codes[3][u] << 4 & ~kLow),
              (codes[2][u] >> 4 & kLow) | (codes[3][u] & ~kLow)};
          uint32_t x[4][4];
#pragma unroll
          for (int t = 0; t < 4; ++t) fp4_decode(mixed[t], x[t]);
#pragma unroll
          for (int i = 0; i < kUnit; ++i) {
            const uint32_t a[4] = {times(x[0][i], near), times(x[1][i], near), times(x[2][i], far),
                                   times(x[3][i], far)};
            const int dt = chunk * kChunk + u * kUnit + i;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              if constexpr (Terms == 1) {
                if constexpr (Sizes > 1) {
                  float sum[4];
                  mma_f16_first(sum, a, frag[nt][1][0], frag[nt][1][1]);
#pragma unroll
                  for (int c = 0; c < 4; ++c) {
                    o[dt][nt][c] = fmaf(sum[c], 1.f / kStep, o[dt][nt][c]);
                  }
                }
                mma_f16(o[dt][nt], a, frag[nt][0][0], frag[nt][0][1]);
              } else {
                float sum[4];
                mma_f16_first(sum, a, frag[nt][1][0], frag[nt][1][1]);
#pragma unroll
                for (int c = 0; c < 4; ++c) sum[c] *= 1.f / kFine;
                mma_f16(sum, a, frag[nt][0][0], frag[nt][0][1]);
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                  if constexpr (Scaled) o[dt][nt][c] = fmaf(sum[c], by, o[dt][nt][c]);
                  else o[dt][nt][c] += sum[c];
                }
              }
            }
          }
        }
      }
    }
  }
};

// f(pool) for the pool of a head dim.
template <int NT, typename F>
auto by_dim(int64_t dim, F&& f) {
  switch (dim) {
    case 32: return f(Fp4Pool<32, NT>{});
    case 64: return f(Fp4Pool<64, NT>{});
    case 96: return f(Fp4Pool<96, NT>{});
    case 128: return f(Fp4Pool<128, NT>{});
    case 160: return f(Fp4Pool<160, NT>{});
    case 192: return f(Fp4Pool<192, NT>{});
    case 224: return f(Fp4Pool<224, NT>{});
    default: return f(Fp4Pool<256, NT>{});
  }
}

template <int NT>
cudaError_t launch_fp4(const Fp4Pages& pages, const PagedParams& p, int ctas, cudaStream_t stream) {
  return by_dim<NT>(p.dim, [&](auto pool) {
    return launch_pool<decltype(pool), true>(pages, p, ctas, stream);
  });
}

}  // namespace
}  // namespace rkv
