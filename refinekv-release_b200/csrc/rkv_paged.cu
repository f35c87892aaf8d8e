// Dense attention of one new token per sequence over a page pool, in one launch.
//
// Mathematics.  Per sequence s and KV head h a row of `group` queries attends
// to the visible tokens of its sequence: an online softmax over tiles of R
// tokens keeps (m, l, o) per query, and partial results over parts of the
// tokens join exactly as l = sum l_i e^(m_i - m), o = sum o_i e^(m_i - m).
//
// Bound: HBM on long sequences.  Each visible K and V row is read once (4 D
// bytes for 4 G D flop, G <= 16).  mma.sync with the tokens on M and the group
// on N keeps the tensor pipe 13 % active at the streaming rate, so tcgen05
// (M = 64 at least, operands from shared-memory descriptors) would not move
// the bound.  Measured on B200 (graph replay): 16 sequences of 32K tokens, 8 KV
// heads, D 128: 320-326 us for 2.15 GB, 6.6-6.7 TB/s, what a plain copy reaches or
// a little more; one of 128K: 87 us for 537 MB (6.2 TB/s; the SMs that stream
// slowest, about a fifth of them, end 10 us after the mean, and equal shares
// cannot follow that); a ragged batch of 43, 270 MB: 52 us.  About 5 us before
// the stream is up and 4 to 6 for the joins at its end are what short calls
// consist of: one sequence of 333 tokens takes 8.3 us.  Sixteen queries a KV head
// of D 192 or 256 spill a little (200 and 292 bytes of stores a thread): 8
// sequences of 32K tokens, 2 KV heads, D 256: 103 us for 537 MB, against 97 with
// eight queries; D 192: 82 us for 403 MB, against 72 with four.
//
// Split.  The tiles of all rows, sequence-major then head, form one list that
// is cut into equal contiguous ranges, one per CTA, and each CTA's range into
// equal contiguous ranges, one per warp: every warp streams the same number
// of tiles whatever the lengths are.  A warp streams through its own
// shared-memory stage by TMA with one barrier each for K and V (K of the next
// tile is requested as soon as this one's scores are done).  Rows that lie
// within one warp's range are written from registers; a row cut by a range
// end leaves a partial, at most two per warp; the CTA joins its warps'
// partials, and a row cut by CTA ranges is joined by whichever of its CTAs
// arrives last at a counter -- nobody waits.  All joins run in token order, so
// results repeat bit for bit.
//
// The lengths and the page table are read on the device (graphs replay with
// growing sequences): every CTA scans the lengths itself.
#include <algorithm>
#include <string>

#include "refinekv_b200.h"
#include "rkv_device.cuh"
#include "rkv_drain.h"
#include "rkv_kernels.h"

namespace rkv {
void set_last_error(const std::string& message);

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
constexpr int stage_bytes(int D) { return 2 * tile_rows(D) * D * 2; }

// A row's CTAs are joined in one level up to this many, else in groups of about
// the square root.  24 against 32: three ragged D 256 sequences (24 to 39 parts)
// 37.5 against 44.3 us, 8K tokens of one head (32 parts) 11.4 against 11.7; 16: 128K
// tokens of eight heads (18 parts) 88.2 against 87.3, 21 and 24 parts the same;
// 80 and 160: up to 18 us more.
constexpr int kFlatJoin = 24;

// Workspace: status word, counters (at the same place for every geometry;
// they are zero between calls), then the partials.
constexpr size_t kCounterBytes = 256;
constexpr int kMostCtas = 512;  // two counters per CTA and one per row that begins in it
constexpr size_t kHeader = 8192;

// A warp's partial is o[G8][D + 4] (the pad spreads the fragments' rows over
// the shared-memory banks), its m and l wait in shared memory; a CTA's is
// m[G8], l[G8], o[G8][D].
// A warp's first partial, left while its stage is in use, has its own place in
// shared memory where that fits, else in the workspace.
constexpr int kPad = 4;
constexpr bool first_in_smem(int D) { return D <= 128; }
constexpr int warp_partial_floats(int D, int NT) { return NT * 8 * (D + kPad); }
constexpr int partial_floats(int D, int NT) { return NT * 8 * (D + 2); }
// Dynamic shared memory: the stages, the warps' first partials, then the
// table of the sequences' first tiles.
constexpr size_t table_offset(int D, int NT) {
  return static_cast<size_t>(paged_warps(D)) *
         (stage_bytes(D) + (first_in_smem(D) ? warp_partial_floats(D, NT) * 4 : 0));
}
constexpr size_t paged_smem(int D, int NT, int64_t sequences) {
  return kSmemSlack + table_offset(D, NT) + static_cast<size_t>(sequences + 1) * 4;
}

struct Cursor {
  int seq, head, tile, tiles;  // tile of `tiles` of the row
  int first;                   // the row's first tile, in tiles from the sequence's start
  int low, length;             // visible tokens [low, length)
};

template <int D, int NT>
struct Paged {
  static constexpr int R = tile_rows(D);
  static constexpr int W = paged_warps(D);
  static constexpr int G8 = NT * 8;
  static constexpr int kTile = R * D * 2;
  static constexpr int kThreads = W * 32;
  static constexpr int kPartial = partial_floats(D, NT);
  static constexpr int kWarpPartial = warp_partial_floats(D, NT);
};

// A length that the page table cannot hold counts as zero: nothing of its row
// is read, and the row is NaN.
__device__ __forceinline__ int clamp_length(const PagedParams& p, int seq) {
  const int length = p.lengths[seq];
  return length > p.capacity ? 0 : max(0, length);
}

constexpr int kNoPage = -1, kBadPage = -2;  // of a box: nothing visible; not in the pool

__device__ __forceinline__ int first_visible(const PagedParams& p, int length) {
  return p.window > 0 && length > p.window ? length - p.window : 0;
}

// Tiles of a sequence: those that hold its visible tokens.
template <int R>
__device__ __forceinline__ int tiles_of(const PagedParams& p, int seq) {
  const int length = clamp_length(p, seq);
  return (length + R - 1) / R - first_visible(p, length) / R;
}

template <int R>
__device__ __forceinline__ void enter_row(const PagedParams& p, const int* start, Cursor& c) {
  c.tiles = start[c.seq + 1] - start[c.seq];
  c.length = clamp_length(p, c.seq);
  c.low = first_visible(p, c.length);
  c.first = c.low / R;
}

// The cursor at global tile x.
template <int R>
__device__ __forceinline__ Cursor seek(const PagedParams& p, const int* start, unsigned x) {
  int a = 0, b = p.sequences;  // start[a] * heads <= x < start[b] * heads
  while (b - a > 1) {
    const int mid = (a + b) >> 1;
    if (static_cast<unsigned>(start[mid]) * p.heads <= x) a = mid; else b = mid;
  }
  Cursor c;
  c.seq = a;
  enter_row<R>(p, start, c);
  const unsigned y = x - static_cast<unsigned>(start[a]) * p.heads;
  c.head = static_cast<int>(y / c.tiles);
  c.tile = static_cast<int>(y - static_cast<unsigned>(c.head) * c.tiles);
  return c;
}

// `total` things in `parts` equal contiguous ranges: the k-th begins at
// bound(k), and x lies in range owner(x).
struct Ranges {
  unsigned each, rest, parts;
  __device__ Ranges(unsigned total, unsigned n) : each(total / n), rest(total % n), parts(n) {}
  // rest < parts <= 512, so the product stays small.
  __device__ unsigned bound(unsigned k) const { return each * k + rest * k / parts; }
  __device__ unsigned owner(unsigned x) const {
    unsigned k = min(parts - 1, x / max(1u, each));  // at or past the owner
    while (bound(k) > x) --k;
    return k;
  }
};

// A row cut by the CTA's range: slot 0 began before it, slot 1 within it.  Its
// parts are the partials of the CTAs from first_cta on, each CTA's in slot 1 if
// the row begins there and slot 0 otherwise.  `members` of them from CTA
// `first` on, this CTA's among them, are joined by the last of those to
// arrive; where they are not all of the row's, the `groups` results, `fan` CTAs
// apart, are joined in turn.
struct Cut {
  int row;  // -1: none
  int first_cta, first, members, groups, fan;
  __device__ int slot_at(int cta) const { return 2 * cta + (cta == first_cta ? 1 : 0); }
};

__device__ __forceinline__ Cut cut_row(const Ranges& ranges, int cta, int row, unsigned begin,
                                       unsigned tiles) {
  Cut c;
  c.row = row;
  c.first_cta = ranges.owner(begin);
  const int parts = ranges.owner(begin + tiles - 1) - c.first_cta + 1;
  c.fan = parts;
  if (parts > kFlatJoin) {
    c.fan = 1;
    while (c.fan * c.fan < parts) ++c.fan;
  }
  const int group = (cta - c.first_cta) / c.fan;
  c.first = c.first_cta + group * c.fan;
  c.members = min(c.fan, parts - group * c.fan);
  c.groups = (parts + c.fan - 1) / c.fan;
  return c;
}

__device__ __forceinline__ int arrive_add(int* counter) {
  int seen;
  asm volatile("atom.add.acq_rel.gpu.global.s32 %0, [%1], 1;" : "=r"(seen) : "l"(counter) : "memory");
  return seen;
}

// The next tile of the list (there must be one).
template <int R>
__device__ __forceinline__ void advance(const PagedParams& p, const int* start, Cursor& c) {
  if (++c.tile < c.tiles) return;
  c.tile = 0;
  if (++c.head < p.heads) return;
  c.head = 0;
  do ++c.seq; while (start[c.seq + 1] == start[c.seq]);
  enter_row<R>(p, start, c);
}

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

// One normalised output value; an all -inf row is 0 / 0, as the formula has it.
__device__ __forceinline__ void put(const PagedParams& p, int64_t at, float x) {
  if (p.query_f32) static_cast<float*>(p.out)[at] = x;
  else static_cast<__nv_bfloat16*>(p.out)[at] = __float2bfloat16_rn(x);
}

__device__ __forceinline__ void put4(const PagedParams& p, int64_t at, float4 x) {
  if (p.query_f32) {
    *reinterpret_cast<float4*>(static_cast<float*>(p.out) + at) = x;
  } else {
    *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(p.out) + at) =
        make_uint2(pack_bf16(x.x, x.y), pack_bf16(x.z, x.w));
  }
}

__device__ __forceinline__ void fma4(float4& acc, float w, const float4& x) {
  acc.x += w * x.x;
  acc.y += w * x.y;
  acc.z += w * x.z;
  acc.w += w * x.w;
}

__device__ __forceinline__ float finite_or_zero(float m) { return m == -INFINITY ? 0.f : m; }

// Joins the parts k of the bit set `members` for one query: m_of(k) and l_of(k)
// give part k's m and l, o_of(k, d) its channels d .. d + 3, and put(d, m, l, o)
// takes the joined ones of d = 4 lane, 4 (lane + kLanes), ...  Every load of
// kBatch parts is in flight at once.  Each thread finds the weights for
// itself: an exponential a part instead of a barrier for the CTA.  The batches
// are short because this code runs once and cold: twenty parts unrolled cost a
// batch of two or three 0.8 us.
template <int D, int kLanes, int kBatch, typename M, typename L, typename O, typename Put>
__device__ __forceinline__ void join(unsigned members, int lane, M m_of, L l_of, O o_of, Put put) {
  constexpr int kCols = (D / 4 + kLanes - 1) / kLanes;
  float top = -INFINITY, sum = 0.f;
  float4 acc[kCols];
#pragma unroll
  for (int c = 0; c < kCols; ++c) acc[c] = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int base = 0; base < 32; base += kBatch) {
    const unsigned set = members >> base;
    if (set == 0) break;
    float m[kBatch], l[kBatch];
    float4 o[kCols][kBatch];
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      m[u] = -INFINITY;
      if (set >> u & 1) {
        m[u] = m_of(base + u);
        l[u] = l_of(base + u);
#pragma unroll
        for (int c = 0; c < kCols; ++c) {
          const int d = 4 * (lane + c * kLanes);
          if (d < D) o[c][u] = o_of(base + u, d);
        }
      }
    }
    float next = top;
#pragma unroll
    for (int u = 0; u < kBatch; ++u) next = fmaxf(next, m[u]);
    const float ref = finite_or_zero(next);
    if (base > 0) {
      const float keep = __expf(top - ref);
      sum *= keep;
#pragma unroll
      for (int c = 0; c < kCols; ++c) {
        acc[c] = make_float4(acc[c].x * keep, acc[c].y * keep, acc[c].z * keep, acc[c].w * keep);
      }
    }
    top = next;
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      if (set >> u & 1) {
        const float w = __expf(m[u] - ref);
        sum += w * l[u];
#pragma unroll
        for (int c = 0; c < kCols; ++c) {
          if (4 * (lane + c * kLanes) < D) fma4(acc[c], w, o[c][u]);
        }
      }
    }
  }
#pragma unroll
  for (int c = 0; c < kCols; ++c) {
    const int d = 4 * (lane + c * kLanes);
    if (d < D) put(d, top, sum, acc[c]);
  }
}

// Four joined channels of query g of a row and, with the first of them, its m
// and l: finished, or into the partial `to`.
template <int D, int G8>
__device__ __forceinline__ void put_joined(const PagedParams& p, int row, int g, int d, float* to,
                                           float m, float l, const float4& o) {
  if (to != nullptr) {
    *reinterpret_cast<float4*>(to + 2 * G8 + g * D + d) = o;
    if (d == 0) {
      to[g] = m;
      to[G8 + g] = l;
    }
  } else if (d < p.dim) {
    const int64_t at = static_cast<int64_t>(row) * p.group + g;
    const float inverse = 1.f / l;
    put4(p, at * p.dim + d,
         make_float4(o.x * inverse, o.y * inverse, o.z * inverse, o.w * inverse));
    if (d == 0 && p.lse != nullptr) p.lse[at] = finite_or_zero(m) + logf(l);
  }
}

template <int D, int NT>
__global__ void __launch_bounds__(paged_warps(D) * 32, 1)
    paged_kernel(const __grid_constant__ PagedMaps maps, const __grid_constant__ PagedParams p) {
  using K = Paged<D, NT>;
  constexpr int R = K::R, W = K::W, G8 = K::G8, kTile = K::kTile;
  constexpr int kThreads = K::kThreads, kPartial = K::kPartial, kWarpPartial = K::kWarpPartial;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* ring = align_smem(smem_raw);  // [warp][K | V]
  __shared__ __align__(8) uint64_t bars[W][2];
  __shared__ int warp_sum[W];
  // The CTA's partials, two per warp, in token order: the row (or -1), and each
  // query's m and l.
  __shared__ int seg_row[2 * W];
  __shared__ float seg_m[2 * W][G8], seg_l[2 * W][G8];
  __shared__ Cut cuts[2];
  __shared__ int last_arrival[2];
  __shared__ int busy;  // sequences that are not empty
  int* start = reinterpret_cast<int*>(ring + table_offset(D, NT));  // tiles before each sequence
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (lane == 0) {
    mbar_init(&bars[warp][0], 1);
    mbar_init(&bars[warp][1], 1);
    mbar_fence_init();
    seg_row[2 * warp] = seg_row[2 * warp + 1] = -1;
  }
  if (threadIdx.x == 0) {
    busy = 0;
    tma_prefetch_desc(&maps.keys);
    tma_prefetch_desc(&maps.values);
  }
  // The lengths and the page table's lines come to L2 before the dependency wait
  // (hints: they return no data, so what the previous kernel still writes is
  // read correctly after it): 6.9 -> 6.6 us for 128 tokens, whose table was last
  // read a layer's worth of traffic ago.
  {
    const int64_t bytes =
        ((p.sequences - 1) * p.page_table_stride + (p.capacity >> p.block_shift)) * 4;
    const int64_t at = (blockIdx.x + static_cast<int64_t>(lane) * gridDim.x) * 128;
    if (warp == 0 && at < bytes) prefetch_l2(reinterpret_cast<const char*>(p.page_table) + at);
    if (warp == 1 && lane * 32 < p.sequences) prefetch_l2(p.lengths + lane * 32);
  }
  pdl_wait();
  pdl_launch_dependents();

  // start[s] = tiles of the sequences before s, by a scan over the CTA.
  {
    const int per = (p.sequences + W * 32 - 1) / (W * 32);
    const int s0 = min(p.sequences, static_cast<int>(threadIdx.x) * per);
    const int s1 = min(p.sequences, s0 + per);
    int sum = 0, some = 0;
    for (int s = s0; s < s1; ++s) {
      if (blockIdx.x == 0 && (p.lengths[s] < 0 || p.lengths[s] > p.capacity)) {
        atomicOr(p.status, kStatusBadInput);
      }
      const int tiles = tiles_of<R>(p, s);
      start[s] = tiles;
      sum += tiles;
      some += tiles > 0;
    }
    int scan = sum;
#pragma unroll
    for (int step = 1; step < 32; step <<= 1) {
      const int other = __shfl_up_sync(0xffffffffu, scan, step);
      if (lane >= step) scan += other;
    }
    if (lane == 31) warp_sum[warp] = scan;
    __syncthreads();
    int before = scan - sum;
    for (int w = 0; w < warp; ++w) before += warp_sum[w];
    some = __reduce_add_sync(0xffffffffu, some);
    if (lane == 0 && some > 0) atomicAdd(&busy, some);
    for (int s = s0; s < s1; ++s) {
      const int tiles = start[s];
      start[s] = before;
      before += tiles;
    }
    if (s1 == p.sequences && s0 < s1) start[p.sequences] = before;
    __syncthreads();
  }
  const unsigned T = static_cast<unsigned>(start[p.sequences]) * p.heads;
  // Idle slots: zero rows; lengths past the table: NaN.
  for (int s = blockIdx.x; s < p.sequences; s += gridDim.x) {
    if (start[s + 1] != start[s]) continue;
    const bool past = p.lengths[s] > p.capacity;
    const int queries = p.heads * p.group;
    const int64_t row = static_cast<int64_t>(s) * queries;
    for (int i = threadIdx.x; i < queries * p.dim; i += blockDim.x) {
      put(p, row * p.dim + i, past ? NAN : 0.f);
    }
    if (p.lse != nullptr) {
      for (int i = threadIdx.x; i < queries; i += blockDim.x) {
        p.lse[row + i] = past ? NAN : -INFINITY;
      }
    }
  }
  // How many CTAs share the tiles.  Many rows: every SM, but a tile a warp at
  // least.  Few rows: whole CTAs per row where that leaves few SMs idle, since a
  // CTA with one row has one join less (three D 256 sequences 37.5 us against 40.5
  // with every SM, two of 60K tokens 79.7 against 80.3, one of 128K 87.3 against
  // 87.5), and no more of them than give every warp a tile (2K tokens, 8 heads: a
  // microsecond less than with two tiles a warp), one for a row of up to two tiles a
  // warp (333 tokens: 8.3 us against 8.9 with a tile a warp and a join across CTAs).
  const unsigned rows = static_cast<unsigned>(busy) * p.heads, grid = gridDim.x;
  unsigned C = min(grid, (T + W - 1) / W);
  if (rows > 0 && rows <= grid) {
    const unsigned fit = grid / rows, worth = T <= 2 * W * rows ? 1 : (T / rows + W - 1) / W;
    if (worth < fit) C = rows * worth;
    else if (fit * rows * 16 >= grid * 15) C = fit * rows;
    C = min(C, T);
  }
  const unsigned cta = blockIdx.x;
  if (cta >= C) return;
  const Ranges ranges(T, C);
  const unsigned lo = ranges.bound(cta), hi = ranges.bound(cta + 1);
  const Ranges shares(hi - lo, W);
  const unsigned wlo = lo + shares.bound(warp), whi = lo + shares.bound(warp + 1);

  uint8_t* stage = ring + warp * 2 * kTile;
  const uint32_t k_tile = smem_addr(stage), v_tile = k_tile + kTile;
  // Where partial i of the CTA keeps its o: a warp's last row waits in the
  // warp's own idle stage, an earlier one (cut by the range's start) apart.
  float* firsts = first_in_smem(D)
                      ? reinterpret_cast<float*>(ring + W * 2 * kTile)
                      : p.warp_partials + static_cast<size_t>(cta) * W * kWarpPartial;
  const auto segment = [&](int i) {
    return i & 1 ? reinterpret_cast<float*>(ring + (i >> 1) * 2 * kTile)
                 : firsts + (i >> 1) * kWarpPartial;
  };
  const uint64_t policy = l2_evict_first_policy();
  const int page_rows = 1 << p.block_shift;
  const int box_rows = min(R, page_rows), boxes = R / box_rows;

  // Lane i of the first `boxes` lanes looks up the page of the tile's i-th box.
  auto page_of = [&](const Cursor& c) {
    if (lane >= boxes) return kNoPage;
    const int token = (c.first + c.tile) * R + lane * box_rows;
    if (token >= c.length || token + box_rows <= c.low) return kNoPage;
    const int page = p.page_table[c.seq * p.page_table_stride + (token >> p.block_shift)];
    if (page >= 0 && page < p.pool_pages) return page;
    atomicOr(p.status, kStatusBadInput);
    return kBadPage;
  };
  // Requests the tile's boxes; a bad page's are left out, and its row is NaN.
  auto issue = [&](int which, const Cursor& c, int page) {
    uint64_t* bar = &bars[warp][which];
    const unsigned used = __ballot_sync(0xffffffffu, page >= 0);
    if (lane == 0) mbar_expect_tx(bar, __popc(used) * box_rows * D * 2);
    fence_proxy_async();
    __syncwarp();
    if (page >= 0) {
      const int token = (c.first + c.tile) * R + lane * box_rows;
      uint8_t* to = stage + which * kTile + lane * box_rows * 128;
      const CUtensorMap* map = which ? &maps.values : &maps.keys;
#pragma unroll
      for (int i = 0; i < D / 64; ++i) {
        tma_load_4d_hint(to + i * R * 128, map, bar, i * 64, token & (page_rows - 1), c.head, page,
                         policy);
      }
    }
  };

  // The rows that the range's two ends cut: known from the start, so worked out
  // while the first tiles are on their way.
  const auto find_cuts = [&] {
    if (warp >= 2) return;
    const Cursor c = seek<R>(p, start, warp == 0 ? lo : hi - 1);
    const unsigned begin = (warp == 0 ? lo : hi - 1) - c.tile;
    const bool cut = warp == 0 ? begin < lo : begin >= lo && begin + c.tiles > hi;
    Cut found;
    found.row = -1;
    if (cut) found = cut_row(ranges, cta, c.seq * p.heads + c.head, begin, c.tiles);
    if (lane == 0) cuts[warp] = found;
  };
  if (wlo >= whi) find_cuts();
  if (wlo < whi) {
    uint32_t qb[D / 16][NT][2];
    float m[NT][2], l[NT][2], o[D / 16][NT][4];
    Cursor cur = seek<R>(p, start, wlo), next = cur;
    int page = page_of(cur);
    issue(0, cur, page);
    issue(1, cur, page);
    // Whether a tile lacks a page: this one, the next, any so far of the row.
    bool bad = __any_sync(0xffffffffu, page == kBadPage), next_bad = false, spoilt = false;
    find_cuts();
    const int count = static_cast<int>(whi - wlo);
    int seg_first = cur.tile;  // the segment's first tile of its row
    bool fresh = true, aborted = false;
    const auto again = [&](int which, int parity) { warp_wait(&bars[warp][which], parity); };
    if (count > 1) {
      advance<R>(p, start, next);
      page = page_of(next);
    }
    for (int j = 0; j < count; ++j) {
      if (fresh) {
        load_queries<D, NT>(qb, p, cur.seq, cur.head, lane);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          m[nt][0] = m[nt][1] = -INFINITY;
          l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
          for (int dt = 0; dt < D / 16; ++dt)
            o[dt][nt][0] = o[dt][nt][1] = o[dt][nt][2] = o[dt][nt][3] = 0.f;
        }
        fresh = spoilt = false;
      }
      spoilt = spoilt || bad;
      const bool more = j + 1 < count;
      const int token = (cur.first + cur.tile) * R;
      const int row_lo = max(0, cur.low - token), row_hi = min(R, cur.length - token);
      // A wait that runs out leaves the rest of the warp's range out (the
      // status word says so, and its rows are NaN); nothing is in flight after
      // its drain.
      if (!aborted && !warp_wait(&bars[warp][0], j & 1)) {
        if (lane == 0) atomicOr(p.status, kStatusTimeout);
        drain_keys_and_values(j, again);
        aborted = true;
      }
      if (!aborted) {
        float logit[R / 16][NT][4];
        score_tile<R, D, NT>(k_tile, qb, logit, lane);
#pragma unroll
        for (int mt = 0; mt < R / 16; ++mt)
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const int r = mt * 16 + (lane >> 2) + (c >> 1) * 8;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
              logit[mt][nt][c] =
                  r >= row_lo && r < row_hi ? logit[mt][nt][c] * p.scale : -INFINITY;
          }
        __syncwarp();
        if (more) {
          issue(0, next, page);
          next_bad = __any_sync(0xffffffffu, page == kBadPage);
        }
        softmax_update<R, D, NT>(logit, m, l, o);
        if (!warp_wait(&bars[warp][1], j & 1)) {
          if (lane == 0) atomicOr(p.status, kStatusTimeout);
          drain_values(j, more, again);
          aborted = true;
        } else {
          if (row_lo > 0 || row_hi < R) {
            // Rows that are not visible may hold anything: a weight of zero
            // would not silence a NaN, so they are zeroed.
            for (int i = lane; i < R * (D / 8); i += 32) {
              const int r = i / (D / 8), c16 = i - r * (D / 8);
              if (r < row_lo || r >= row_hi) {
                *reinterpret_cast<uint4*>(stage + kTile + swz(r, c16, R)) = make_uint4(0, 0, 0, 0);
              }
            }
            fence_proxy_async();
            __syncwarp();
          }
          if (p.query_f32) {
            weigh_values<R, D, NT, 3>(v_tile, logit, o, lane);
          } else {
            weigh_values<R, D, NT, 2>(v_tile, logit, o, lane);
          }
          __syncwarp();
          if (more) issue(1, next, page);
        }
      }
      const bool row_done = cur.tile + 1 == cur.tiles;
      if (row_done || !more) {
        reduce_l<NT>(l);
        if (spoilt || aborted) {  // a sum of NaN spreads through every join
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) l[nt][0] = l[nt][1] = NAN;
        }
        const int row = cur.seq * p.heads + cur.head;
        const bool whole = row_done && seg_first == 0;
        if (whole) {
          const int64_t out_row = static_cast<int64_t>(row) * p.group;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              const int g = nt * 8 + 2 * (lane & 3) + c;
              if (g >= p.group) continue;
              const float inv = 1.f / l[nt][c];
#pragma unroll
              for (int dt = 0; dt < D / 16; ++dt)
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                  const int d = dt * 16 + half * 8 + (lane >> 2);
                  if (d < p.dim) put(p, (out_row + g) * p.dim + d, o[dt][nt][2 * half + c] * inv);
                }
              if (p.lse != nullptr && lane < 4) {
                const float ref = m[nt][c] == -INFINITY ? 0.f : m[nt][c];
                p.lse[out_row + g] = ref + logf(l[nt][c]);
              }
            }
        } else {
          const int i = 2 * warp + (more ? 0 : 1);
          float* to = segment(i);
          if (lane == 0) seg_row[i] = row;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              const int g = nt * 8 + 2 * (lane & 3) + c;
              if (g >= p.group) continue;
              if (lane < 4) {
                seg_m[i][g] = m[nt][c];
                seg_l[i][g] = l[nt][c];
              }
#pragma unroll
              for (int dt = 0; dt < D / 16; ++dt)
#pragma unroll
                for (int half = 0; half < 2; ++half)
                  to[g * (D + kPad) + dt * 16 + half * 8 + (lane >> 2)] = o[dt][nt][2 * half + c];
            }
        }
        seg_first = 0;
        fresh = true;
      }
      if (more) {
        cur = next;
        bad = next_bad;
        if (j + 2 < count) {
          advance<R>(p, start, next);
          page = page_of(next);
        }
      }
    }
  }
  __syncthreads();

  // Join the CTA's partials.  A row that began and ended within the CTA is
  // written; one that began before it goes to the CTA's slot 0, one that only
  // goes on after it to slot 1.  kLanes threads share the channels of a query.
  constexpr int kLanes = D / 4 < kThreads / G8 ? D / 4 : kThreads / G8;
  constexpr int kBatch = D > 192 && NT > 1 ? 4 : 8;
  {
    const int mine = lane < 2 * W ? seg_row[lane] : -1;
    const unsigned used = __ballot_sync(0xffffffffu, mine >= 0);
    const unsigned below = used & ((1u << lane) - 1);
    const int previous = __shfl_sync(0xffffffffu, mine, below ? 31 - __clz(below) : 0);
    // The first partial of each row.
    const unsigned heads =
        __ballot_sync(0xffffffffu, mine >= 0 && (below == 0 || previous != mine));
    for (int x = threadIdx.x; x < __popc(heads) * p.group * kLanes; x += kThreads) {
      const int k = x / kLanes / p.group, g = x / kLanes - k * p.group;
      unsigned rest = heads;
      for (int skip = 0; skip < k; ++skip) rest &= rest - 1;
      const int head = __ffs(rest) - 1, row = seg_row[head];
      rest &= rest - 1;
      // The row's partials: from its first to the next row's first.
      const unsigned members =
          used & ~((1u << head) - 1) & (rest ? (rest & -rest) - 1 : 0xffffffffu);
      const int slot = row == cuts[0].row ? 0 : row == cuts[1].row ? 1 : -1;
      float* to = slot < 0 ? nullptr
                           : p.cta_partials + (static_cast<size_t>(cta) * 2 + slot) * kPartial;
      join<D, kLanes, kBatch>(
          members, x % kLanes, [&](int j) { return seg_m[j][g]; },
          [&](int j) { return seg_l[j][g]; },
          [&](int j, int d) {
            return *reinterpret_cast<const float4*>(segment(j) + g * (D + kPad) + d);
          },
          [&](int d, float m, float l, const float4& o) {
            put_joined<D, G8>(p, row, g, d, to, m, l, o);
          });
    }
  }

  // Rows cut by CTA ranges: the last of a row's CTAs to arrive joins them; a
  // row over many CTAs is joined in groups first, so that no CTA reads more
  // than a few partials.  arrive() says whether this is the last of `expected`
  // arrivals, and then leaves the counter at zero.
  const auto arrive = [](int* counter, int expected) {
    const bool last = arrive_add(counter) == expected - 1;
    if (last) *counter = 0;
    return last;
  };
  __syncthreads();
  if (lane == 0 && warp < 2) {  // both slots at once
    const Cut cut = cuts[warp];
    last_arrival[warp] =
        cut.row >= 0 && arrive(p.counters + cut.slot_at(cut.first), cut.members);
  }
  __syncthreads();
  // Joins the rows whose last arrival was this CTA's: its members' partials
  // or, once those are joined, the groups'.
  const auto join_arrived = [&](const bool grouped) {
    const int all = p.group * kLanes;
    const int from = last_arrival[0] ? 0 : all, to = last_arrival[1] ? 2 * all : all;
    for (int x = from + threadIdx.x; x < to; x += kThreads) {
      const int slot = x >= all ? 1 : 0, g = x / kLanes - slot * p.group;
      const Cut cut = cuts[slot];
      const auto part = [&](int k) -> const float* {
        return grouped
                   ? p.group_partials +
                         static_cast<size_t>(cut.slot_at(cut.first_cta + k * cut.fan)) * kPartial
                   : p.cta_partials + static_cast<size_t>(cut.slot_at(cut.first + k)) * kPartial;
      };
      float* target = grouped || cut.groups == 1
                          ? nullptr
                          : p.group_partials + static_cast<size_t>(cut.slot_at(cut.first)) * kPartial;
      const unsigned members = 0xffffffffu >> (32 - (grouped ? cut.groups : cut.members));
      const auto m_of = [&](int k) { return __ldcg(part(k) + g); };
      const auto l_of = [&](int k) { return __ldcg(part(k) + G8 + g); };
      const auto o_of = [&](int k, int d) {
        return __ldcg(reinterpret_cast<const float4*>(part(k) + 2 * G8 + g * D + d));
      };
      const auto put = [&](int d, float m, float l, const float4& o) {
        put_joined<D, G8>(p, cut.row, g, d, target, m, l, o);
      };
      // More than one batch's parts, up to 24 (kFlatJoin) or a group's: in twenties.
      // A row of 18 parts (128K tokens, eight heads) 87.3 us against 87.9 in eights,
      // 21 and 24 parts (16K tokens, seven and six heads) 18.8 and 17.2 against 18.6
      // and 17.0.
      if (kLanes == D / 4 && members >> kBatch) {
        join<D, kLanes, 20>(members, x % kLanes, m_of, l_of, o_of, put);
      } else {
        join<D, kLanes, kBatch>(members, x % kLanes, m_of, l_of, o_of, put);
      }
    }
  };
  join_arrived(false);
  if (!(cuts[0].row >= 0 && cuts[0].groups > 1) && !(cuts[1].row >= 0 && cuts[1].groups > 1)) {
    return;
  }
  __syncthreads();
  if (lane == 0 && warp < 2) {
    const Cut cut = cuts[warp];
    last_arrival[warp] = last_arrival[warp] && cut.groups > 1 &&
                         arrive(p.counters + 2 * kMostCtas + cut.first_cta, cut.groups);
  }
  __syncthreads();
  join_arrived(true);
}

template <int D, int NT>
cudaError_t launch_t(const PagedMaps& maps, const PagedParams& p, int ctas, cudaStream_t stream) {
  const size_t smem = paged_smem(D, NT, p.sequences);
  // One limit for every batch: the largest this kernel takes.
  cudaError_t err = ensure_smem_limit(reinterpret_cast<const void*>(&paged_kernel<D, NT>),
                                      paged_smem(D, NT, kMostSequences));
  if (err != cudaSuccess) return err;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(paged_warps(D) * 32);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, paged_kernel<D, NT>, maps, p);
}

template <int D>
cudaError_t launch_d(const PagedMaps& maps, const PagedParams& p, int ctas, cudaStream_t stream) {
  return p.group <= 8 ? launch_t<D, 1>(maps, p, ctas, stream)
                      : launch_t<D, 2>(maps, p, ctas, stream);
}

int reject(int code, const char* message) {
  set_last_error(message);
  return code;
}

int padded(int64_t dim) { return static_cast<int>((dim + 63) / 64 * 64); }

struct Layout {
  size_t warp_partials, cta_partials, group_partials, bytes;
  Layout(int64_t group, int64_t dim, int sms) {
    const int D = padded(dim), NT = group <= 8 ? 1 : 2;
    const size_t one = static_cast<size_t>(partial_floats(D, NT)) * 4;
    size_t off = kHeader;
    warp_partials = off;
    if (!first_in_smem(D)) {
      off += static_cast<size_t>(warp_partial_floats(D, NT)) * 4 * sms * paged_warps(D);
    }
    cta_partials = off;
    off += one * sms * 2;
    group_partials = off;
    off += one * sms * 2;
    bytes = (off + 255) & ~static_cast<size_t>(255);
  }
};

}  // namespace

}  // namespace rkv

extern "C" {

size_t rkv_paged_workspace_size(int64_t group, int64_t head_dim) {
  using namespace rkv;
  int sms = 0;
  if (group < 1 || group > kMaxGroup || head_dim < 32 || head_dim > 256 || head_dim % 32 ||
      device_sms(&sms) != RKV_OK || sms > kMostCtas) {
    return 0;
  }
  return Layout(group, head_dim, sms).bytes;
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
  const int D = padded(a->head_dim), R = tile_rows(D);
  const int64_t tiles = a->sequences * a->kv_heads * ((a->table_blocks * a->block_size + R - 1) / R);
  if (tiles > (1LL << 31) - 1) {  // a product below 2^13 * 2^12 * 2^25
    return reject(RKV_ERR_UNSUPPORTED, "the page table covers more rows than are counted");
  }
  if (a->sequences == 0) return RKV_OK;
  if (!a->query || !a->output || !a->lengths || !a->key_pool || !a->value_pool ||
      !a->page_table) {
    return reject(RKV_ERR_INVALID_ARGUMENT,
                  "query, output, pools, page_table and lengths must be non-null");
  }
  if (a->pool_pages < 1) return reject(RKV_ERR_INVALID_ARGUMENT, "the pool has no pages");
  if (a->workspace == nullptr || a->workspace_size < static_cast<int64_t>(kHeader)) {
    return reject(RKV_ERR_WORKSPACE, "workspace is missing or too small");
  }
  const int width = a->query_dtype == RKV_DTYPE_F32 ? 4 : 2;
  uintptr_t bits = reinterpret_cast<uintptr_t>(a->query) | reinterpret_cast<uintptr_t>(a->output);
  bits |= reinterpret_cast<uintptr_t>(a->key_pool) | reinterpret_cast<uintptr_t>(a->value_pool);
  for (int64_t s : a->query_strides) bits |= static_cast<uintptr_t>(s * width);
  for (int64_t s : a->key_pool_strides) bits |= static_cast<uintptr_t>(s * 2);
  for (int64_t s : a->value_pool_strides) bits |= static_cast<uintptr_t>(s * 2);
  if (bits & 15u) {
    return reject(RKV_ERR_ALIGNMENT, "pointers and strides must be 16-byte aligned");
  }
  if (!aligned_to(4, {a->page_table, a->lengths, a->lse})) {
    return reject(RKV_ERR_ALIGNMENT,
                  "page_table, lengths and lse must be aligned to their elements");
  }
  int rc = RKV_OK, sms = 0;
  PagedMaps maps;
  const int box_rows = static_cast<int>(std::min<int64_t>(R, a->block_size));
  const int64_t *ks = a->key_pool_strides, *vs = a->value_pool_strides;
  if ((rc = pool_map(&maps.keys, a->key_pool, a->head_dim, a->block_size, box_rows, a->kv_heads,
                     a->pool_pages, ks[2], ks[1], ks[0], "key_pool")) != RKV_OK ||
      (rc = pool_map(&maps.values, a->value_pool, a->head_dim, a->block_size, box_rows,
                     a->kv_heads, a->pool_pages, vs[2], vs[1], vs[0], "value_pool")) != RKV_OK ||
      (rc = device_sms(&sms)) != RKV_OK) {
    return rc;
  }
  if (sms > kMostCtas) return reject(RKV_ERR_UNSUPPORTED, "more SMs than the workspace counts");
  const Layout layout(a->group, a->head_dim, sms);
  if (a->workspace_size < static_cast<int64_t>(layout.bytes) ||
      (reinterpret_cast<uintptr_t>(a->workspace) & 255u) != 0) {
    return reject(RKV_ERR_WORKSPACE, "workspace is too small or not 256-byte aligned");
  }
  char* ws = static_cast<char*>(a->workspace);
  PagedParams p = {};
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
  const int ctas = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(sms, tiles)));
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t err = cudaErrorInvalidValue;
  switch (D) {
    case 64: err = launch_d<64>(maps, p, ctas, st); break;
    case 128: err = launch_d<128>(maps, p, ctas, st); break;
    case 192: err = launch_d<192>(maps, p, ctas, st); break;
    case 256: err = launch_d<256>(maps, p, ctas, st); break;
  }
  if (err != cudaSuccess) {
    set_last_error(std::string("paged attention launch: ") + cudaGetErrorString(err));
    return RKV_ERR_CUDA;
  }
  return RKV_OK;
}

}  // extern "C"
