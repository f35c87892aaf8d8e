// Pools of bf16 for paged_kernel: tiles fetched by TMA through a 4-D map of the
// pool, scored and weighed by mma.sync with the tokens on M and the group on N.
#pragma once

#include "rkv_paged.cu"

namespace rkv {
namespace {

// Tokens per tile: 64 for head dims up to 64, else 32, so that a K and V tile
// is 16 KB at D 64 and 128.
constexpr int tile_rows(int D) { return D <= 64 ? 64 : 32; }
// One stage (a K and a V tile) per warp, up to eight warps.  Eight against six:
// one sequence of 2K tokens 9.4 us against 11.3, one of 128K 87.3 against 88.0, a
// ragged batch of 43 51.0 against 53.5, D 64 23.4 against 25.1; only 16 sequences of
// 32K are faster with six, 313 against 326.  Two CTAs of four warps per SM cost 2
// to 4 us on every batch (more parts to join).
constexpr int paged_warps(int D) { return D <= 192 ? 8 : 6; }

// Query B fragments: rows at `q`, p.q_head elements apart.
template <int D, int NT>
__device__ __forceinline__ void load_queries(uint32_t (&qb)[D / 16][NT][2], const PagedParams& p,
                                             int seq, int head, int lane) {
  const int64_t base = seq * p.q_seq + static_cast<int64_t>(head) * p.group * p.q_head;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int g = nt * 8 + (lane >> 2);
    const int64_t row = base + min(g, p.group - 1) * p.q_head;
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks)
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int d = ks * 16 + half * 8 + 2 * (lane & 3);
        const int64_t at = row + min(d, p.dim - 2);
        uint32_t bits;
        if (p.query_f32) {
          const float2 x = *reinterpret_cast<const float2*>(static_cast<const float*>(p.query) + at);
          bits = pack_bf16(x.x, x.y);
        } else {
          bits = *reinterpret_cast<const uint32_t*>(
              static_cast<const __nv_bfloat16*>(p.query) + at);
        }
        qb[ks][nt][half] = g < p.group && d < p.dim ? bits : 0u;
      }
  }
}

// o += V^T p for a tile's weights p (C layout), held in `Terms` bf16 terms: two
// for bf16 queries (2^-16 at most, far within the output's own rounding: the
// error against 64 bits is the output's 1.66e-3; one term, 2^-8, made it 2.0 to
// 2.3e-3 and took 7.9 instead of 8.3 us for 333 tokens, 319 instead of 322 for 16
// sequences of 32K, 46 instead of 50 for D 256 with 16 queries a KV head), three
// for fp32 queries, which hold all 24 bits of p.  The further
// terms may be negative or zero, so they meet V with its infinities clamped:
// an infinite value times p is infinite, whatever p's bits are.  For fp32 queries
// a tile's products are summed apart and added to o by a rounded addition: the
// tensor cores cut their sums off, which over a long row would cost fp32 digits.
// A bf16 output does not see them (the same error with both), and the second
// set of sums would spill: 68 us instead of 50 for that D 256 batch.
template <int R, int D, int NT, int Terms>
__device__ __forceinline__ void weigh_values(uint32_t tile, float (&p)[R / 16][NT][4],
                                             float (&o)[D / 16][NT][4], int lane) {
  uint32_t frag[Terms][R / 16][NT][2];
#pragma unroll
  for (int term = 0; term < Terms; ++term)
#pragma unroll
    for (int mt = 0; mt < R / 16; ++mt)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          float& a = p[mt][nt][2 * half];
          float& b = p[mt][nt][2 * half + 1];
          const __nv_bfloat162 part = __floats2bfloat162_rn(a, b);
          a -= __low2float(part);
          b -= __high2float(part);
          frag[term][mt][nt][half] = movmatrix_trans(*reinterpret_cast<const uint32_t*>(&part));
        }
  const int trow = (lane & 7) + ((lane >> 4) & 1) * 8;
  const int cadd = (lane >> 3) & 1;
#pragma unroll
  for (int dt = 0; dt < D / 16; ++dt) {
    float sum[NT][4];  // of the tile
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) sum[nt][0] = sum[nt][1] = sum[nt][2] = sum[nt][3] = 0.f;
    float(&to)[NT][4] = Terms > 2 ? sum : o[dt];
#pragma unroll
    for (int kt = 0; kt < R / 16; ++kt) {
      uint32_t a[4];
      ldsm_x4_trans(tile + swz(kt * 16 + trow, dt * 2 + cadd, R), a);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) mma_bf16(to[nt], a, frag[0][kt][nt][0], frag[0][kt][nt][1]);
      if constexpr (Terms > 1) {
        const __nv_bfloat162 most = __halves2bfloat162(__ushort_as_bfloat16(0x7f7f),
                                                       __ushort_as_bfloat16(0x7f7f));
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          __nv_bfloat162& v = *reinterpret_cast<__nv_bfloat162*>(&a[i]);
          v = __hmax2(__hmin2(v, most), __hneg2(most));
        }
#pragma unroll
        for (int term = 1; term < Terms; ++term)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
            mma_bf16(to[nt], a, frag[term][kt][nt][0], frag[term][kt][nt][1]);
      }
    }
    if constexpr (Terms > 2) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 4; ++c) o[dt][nt][c] += sum[nt][c];
    }
  }
}

template <int D_, int NT_>
struct Bf16Pool {
  static constexpr int D = D_, NT = NT_, R = tile_rows(D), W = paged_warps(D);
  static constexpr int kTile = R * D * 2;
  static constexpr bool kFirstInSmem = D <= 128;
  static __device__ __forceinline__ int range_of(int warp) { return warp; }
  // The most CTAs that a row is worth: those that give every warp a tile (2K tokens, 8
  // heads: a microsecond less than with two tiles a warp), one for a row of up to two tiles
  // a warp (333 tokens: 8.3 us against 8.9 with a tile a warp and a join across CTAs).
  static __device__ __forceinline__ unsigned ctas_of(unsigned tiles, unsigned rows) {
    return tiles <= 2 * W * rows ? 1 : (tiles / rows + W - 1) / W;
  }
  static constexpr int kScratch = 0;
  // Kept scores: by shape_logits (16 x 8K tokens 56 us; by keep_scores 61).
  static constexpr bool kBareScores = false;
  static constexpr int kJoinBatch = D > 192 && NT > 1 ? 4 : 8, kLongBatch = 20;
  using Source = PagedMaps;
  struct Query {
    uint32_t frags[D / 16][NT][2];
  };
  using Logits = float (&)[R / 16][NT][4];
  using Columns = float (&)[NT][2];
  using Outputs = float (&)[D / 16][NT][4];

  static __device__ __forceinline__ void prefetch(const Source& maps) {
    tma_prefetch_desc(&maps.keys);
    tma_prefetch_desc(&maps.values);
  }
  static __device__ __forceinline__ int box_bytes(int rows) { return rows * D * 2; }
  static constexpr int kPieces = 1;
  struct Lane {  // the box that a lane fetches
    int offset;
    __device__ Lane(int lane, int, int box_rows) : offset(lane * box_rows * 128) {}
  };
  static __device__ __forceinline__ void fetch(const Source& maps, const Lane& own, int which,
                                               uint8_t* tile, uint64_t* bar, int row, int head,
                                               int page, uint64_t policy) {
    uint8_t* to = tile + own.offset;
    const CUtensorMap* map = which ? &maps.values : &maps.keys;
#pragma unroll
    for (int i = 0; i < D / 64; ++i) {
      tma_load_4d_hint(to + i * R * 128, map, bar, i * 64, row, head, page, policy);
    }
  }
  static __device__ __forceinline__ void load_queries(Query& q, const PagedParams& p, int seq,
                                                      int head, int lane) {
    rkv::load_queries<D, NT>(q.frags, p, seq, head, lane);
  }
  // What the products of column (nt, col) of a lane are multiplied by.
  static __device__ __forceinline__ float column_scale(const Query&, const PagedParams& p, int nt,
                                                       int col, int lane) {
    return p.scale;
  }
  // The row of a tile whose logits a lane holds.
  static __device__ __forceinline__ int token_of(int mt, int half, int lane) {
    return mt * 16 + (lane >> 2) + half * 8;
  }
  // The channel that a lane's sums belong to.
  static __device__ __forceinline__ int channel(int dt, int half, int lane) {
    return dt * 16 + half * 8 + (lane >> 2);
  }
  static __device__ __forceinline__ void score(uint32_t tile, const Query& q, Logits logit, uint32_t,
                                               int lane, const PagedParams&) {
    score_tile<R, D, NT>(tile, q.frags, logit, lane);
  }
  static __device__ __forceinline__ void softmax(Logits logit, Columns m, Columns l, Outputs o) {
    softmax_update<R, D, NT>(logit, m, l, o);
  }
  static __device__ __forceinline__ void settle(Columns, Outputs) {}
  static __device__ __forceinline__ void weigh(uint8_t* tile, uint32_t at, Logits weights, Outputs o,
                                               const Seen& seen, uint32_t, int lane,
                                               const PagedParams& p) {
    if (!seen.all(R)) {
      // Rows that are not visible may hold anything: a weight of zero
      // would not silence a NaN, so they are zeroed.
      for (int i = lane; i < R * (D / 8); i += 32) {
        const int r = i / (D / 8), c16 = i - r * (D / 8);
        if (!seen.row(r)) {
          *reinterpret_cast<uint4*>(tile + swz(r, c16, R)) = make_uint4(0, 0, 0, 0);
        }
      }
      fence_proxy_async();
      __syncwarp();
    }
    if (p.query_f32) {
      weigh_values<R, D, NT, 3>(at, weights, o, lane);
    } else {
      weigh_values<R, D, NT, 2>(at, weights, o, lane);
    }
  }
};

template <bool More>
cudaError_t launch_bf16(const PagedMaps& maps, const PagedParams& p, int D, int ctas,
                        cudaStream_t stream) {
  const auto by_group = [&](auto one, auto two) {
    return p.group <= 8 ? launch_pool<decltype(one), More>(maps, p, ctas, stream)
                        : launch_pool<decltype(two), More>(maps, p, ctas, stream);
  };
  switch (D) {
    case 64: return by_group(Bf16Pool<64, 1>{}, Bf16Pool<64, 2>{});
    case 128: return by_group(Bf16Pool<128, 1>{}, Bf16Pool<128, 2>{});
    case 192: return by_group(Bf16Pool<192, 1>{}, Bf16Pool<192, 2>{});
    case 256: return by_group(Bf16Pool<256, 1>{}, Bf16Pool<256, 2>{});
  }
  return cudaErrorInvalidValue;
}

}  // namespace
}  // namespace rkv
