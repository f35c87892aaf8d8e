// Dense attention of one new token per sequence over a page pool, in one launch:
// the kernel, included by the files that instantiate it for pools of bf16
// (rkv_paged_api.cu, rkv_paged_more.cu) and of 4 bits (rkv_paged_fp4.cu).
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
// of D 192 or 256 spill a little (200 and 332 bytes of stores a thread): 8
// sequences of 32K tokens, 2 KV heads, D 256: 102 us for 537 MB, against 94 with
// eight queries; D 192: 81 us for 403 MB, against 72 with four.
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
#ifndef RKV_PAGED_CU_
#define RKV_PAGED_CU_

#include <algorithm>

#include "refinekv_b200.h"
#include "rkv_device.cuh"
#include "rkv_drain.h"
#include "rkv_kernels.h"

namespace rkv {
namespace {

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
constexpr int warp_partial_floats(int D, int NT) { return NT * 8 * (D + kPad); }
constexpr int partial_floats(int D, int NT) { return NT * 8 * (D + 2); }
// Dynamic shared memory: the stages, the warps' first partials, what else a pool
// keeps for a warp, then the table of the sequences' first tiles.
template <typename Pool>
constexpr size_t scratch_offset() {
  return static_cast<size_t>(Pool::W) *
         (2 * Pool::kTile + (Pool::kFirstInSmem ? warp_partial_floats(Pool::D, Pool::NT) * 4 : 0));
}
template <typename Pool>
constexpr size_t table_offset() {
  return scratch_offset<Pool>() + static_cast<size_t>(Pool::W) * Pool::kScratch;
}
template <typename Pool>
constexpr size_t paged_smem(int64_t sequences) {
  return kSmemSlack + table_offset<Pool>() + static_cast<size_t>(sequences + 1) * 4;
}

struct Cursor {
  int seq, head, tile, tiles;  // tile of `tiles` of the row
  int token;                   // the tile's first
  int first;                   // the row's first tile, in tiles from the sequence's start
  int low, length;             // visible tokens [low, length)
  int prefix, prefix_tiles;    // and [0, prefix), whose tiles come first
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

// Tiles of a sequence: those that hold its visible tokens.  With a prefix
// (`More`) these are the prefix's and, behind it, the window's.
template <int R, bool More>
__device__ __forceinline__ void enter_tokens(const PagedParams& p, int length, Cursor& c) {
  c.length = length;
  c.low = first_visible(p, length);
  c.first = c.low / R;
  c.prefix = c.prefix_tiles = 0;
  if (More && p.prefix > 0) {
    c.prefix = min(p.prefix, c.low);
    c.prefix_tiles = (c.prefix + R - 1) / R;
    // Tiles from here on are `first` behind their place in the row.
    c.first = max(c.first, c.prefix_tiles) - c.prefix_tiles;
  }
}

template <int R, bool More>
__device__ __forceinline__ int tiles_of(const PagedParams& p, int seq) {
  Cursor c;
  enter_tokens<R, More>(p, clamp_length(p, seq), c);
  return (c.length + R - 1) / R - c.first;
}

template <int R, bool More>
__device__ __forceinline__ void enter_row(const PagedParams& p, const int* start, Cursor& c) {
  c.tiles = start[c.seq + 1] - start[c.seq];
  enter_tokens<R, More>(p, clamp_length(p, c.seq), c);
}

// The first token of the cursor's tile.
template <int R, bool More>
__device__ __forceinline__ int tile_token(const Cursor& c) {
  return (More && c.tile < c.prefix_tiles ? c.tile : c.first + c.tile) * R;
}

// The cursor at global tile x.
template <int R, bool More>
__device__ __forceinline__ Cursor seek(const PagedParams& p, const int* start, unsigned x) {
  int a = 0, b = p.sequences;  // start[a] * heads <= x < start[b] * heads
  while (b - a > 1) {
    const int mid = (a + b) >> 1;
    if (static_cast<unsigned>(start[mid]) * p.heads <= x) a = mid; else b = mid;
  }
  Cursor c;
  c.seq = a;
  enter_row<R, More>(p, start, c);
  const unsigned y = x - static_cast<unsigned>(start[a]) * p.heads;
  c.head = static_cast<int>(y / c.tiles);
  c.tile = static_cast<int>(y - static_cast<unsigned>(c.head) * c.tiles);
  c.token = tile_token<R, More>(c);
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
template <int R, bool More>
__device__ __forceinline__ void advance(const PagedParams& p, const int* start, Cursor& c) {
  if (++c.tile < c.tiles) {
    c.token += R;
    if (More && c.tile == c.prefix_tiles) c.token = tile_token<R, More>(c);
    return;
  }
  c.tile = 0;
  if (++c.head == p.heads) {
    c.head = 0;
    do ++c.seq; while (start[c.seq + 1] == start[c.seq]);
    enter_row<R, More>(p, start, c);
  }
  c.token = tile_token<R, More>(c);
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

// What a KV head's values are multiplied by (pools of 4 bits).
__device__ __forceinline__ float value_factor(const PagedParams& p, int head) {
  return p.value_scale != nullptr ? p.value_scale[head] : 1.f;
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
template <int D, int G8, bool More>
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
    float inverse = 1.f / l;
    if (More) inverse *= value_factor(p, row % p.heads);
    put4(p, at * p.dim + d,
         make_float4(o.x * inverse, o.y * inverse, o.z * inverse, o.w * inverse));
    if (d == 0 && p.lse != nullptr) p.lse[at] = finite_or_zero(m) + logf(l);
  }
}

// The rows of a tile that are visible: [low, high) and [0, prefix).
struct Seen {
  int low, high, prefix;
  __device__ bool row(int r) const { return r < high && (r >= low || r < prefix); }
  __device__ bool all(int rows) const { return high == rows && (low == 0 || prefix >= rows); }
};

// The logits of a tile that is visible as a whole, for the weights' sums.
template <typename Pool>
__device__ __forceinline__ void keep_scores(const float (&logit)[Pool::R / 16][Pool::NT][4],
                                            const Cursor& cur, int token, int lane,
                                            const PagedParams& p) {
#pragma unroll
  for (int nt = 0; nt < Pool::NT; ++nt)
#pragma unroll
    for (int col = 0; col < 2; ++col) {
      const int g = nt * 8 + 2 * (lane & 3) + col;
      if (g >= p.group) continue;
      float* keep = p.scores + (static_cast<int64_t>(cur.seq * p.heads + cur.head) * p.group + g) *
                                   p.capacity + token;
#pragma unroll
      for (int mt = 0; mt < Pool::R / 16; ++mt)
#pragma unroll
        for (int half = 0; half < 2; ++half)
          keep[Pool::token_of(mt, half, lane)] = logit[mt][nt][2 * half + col];
    }
}

// A tile's products to logits: scaled, capped, biased by distance, -inf where the
// row is not visible; and kept for the weights' sums where these are wanted.
//   x = c tanh(scale q.k / c) + slope (j - (L - 1))
template <typename Pool>
__device__ __forceinline__ void shape_logits(float (&logit)[Pool::R / 16][Pool::NT][4],
                                             const typename Pool::Query& query, const Seen& seen,
                                             const Cursor& cur, int token, int lane,
                                             const PagedParams& p) {
  const float cap = p.softcap, inverse = 1.f / cap;
  const int from = token - (cur.length - 1);
#pragma unroll
  for (int nt = 0; nt < Pool::NT; ++nt)
#pragma unroll
    for (int col = 0; col < 2; ++col) {
      const int g = nt * 8 + 2 * (lane & 3) + col;
      const float scale = Pool::column_scale(query, p, nt, col, lane);
      const int head = cur.head * p.group + g;
      const float slope = p.slopes != nullptr && g < p.group ? p.slopes[head] : 0.f;
      float* keep = p.scores != nullptr && g < p.group
                        ? p.scores + (static_cast<int64_t>(cur.seq) * p.heads * p.group + head) *
                                         p.capacity + token
                        : nullptr;
#pragma unroll
      for (int mt = 0; mt < Pool::R / 16; ++mt)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const int r = Pool::token_of(mt, half, lane);
          float& x = logit[mt][nt][2 * half + col];
          x *= scale;
          if (cap > 0.f) x = cap * tanhf(x * inverse);
          if (p.slopes != nullptr) x += slope * static_cast<float>(from + r);
          const bool visible = seen.row(r);
          if (keep != nullptr && visible) keep[r] = x;
          if (!visible) x = -INFINITY;
        }
    }
}

// The pool says how a tile is fetched, scored and weighed (Bf16Pool, Fp4Pool).
// More: a cap, a bias, a prefix, factors and the logits for the weights' sums,
// each looked up in the parameters; without it the kernel gives the same results in
// the same time as before these (D 256 with sixteen queries spills 332 bytes a thread
// instead of 292: 101.5 us against 101.8).
template <typename Pool, bool More>
__global__ void __launch_bounds__(Pool::W * 32, 1)
    paged_kernel(const __grid_constant__ typename Pool::Source source,
                 const __grid_constant__ PagedParams p) {
  constexpr int D = Pool::D, NT = Pool::NT, R = Pool::R, W = Pool::W, kTile = Pool::kTile;
  constexpr int G8 = NT * 8, kThreads = W * 32;
  constexpr int kPartial = partial_floats(D, NT), kWarpPartial = warp_partial_floats(D, NT);
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
  int* start = reinterpret_cast<int*>(ring + table_offset<Pool>());  // tiles before each sequence
  // A warp's place in the order of ranges and partials.
  const int warp = Pool::range_of(threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (lane == 0) {
    mbar_init(&bars[warp][0], 1);
    mbar_init(&bars[warp][1], 1);
    mbar_fence_init();
    seg_row[2 * warp] = seg_row[2 * warp + 1] = -1;
  }
  if (threadIdx.x == 0) {
    busy = 0;
    Pool::prefetch(source);
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
      const int tiles = tiles_of<R, More>(p, s);
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
    const int scan_warp = threadIdx.x >> 5;
    if (lane == 31) warp_sum[scan_warp] = scan;
    __syncthreads();
    int before = scan - sum;
    for (int w = 0; w < scan_warp; ++w) before += warp_sum[w];
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
  // 87.5), and no more of them than the pool finds worth while.
  const unsigned rows = static_cast<unsigned>(busy) * p.heads, grid = gridDim.x;
  unsigned C = min(grid, (T + W - 1) / W);
  if (rows > 0 && rows <= grid) {
    const unsigned fit = grid / rows, worth = Pool::ctas_of(T, rows);
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
  const uint32_t scratch = smem_addr(ring) + scratch_offset<Pool>() + warp * Pool::kScratch;
  // Where partial i of the CTA keeps its o: a warp's last row waits in the
  // warp's own idle stage, an earlier one (cut by the range's start) apart.
  float* firsts = Pool::kFirstInSmem
                      ? reinterpret_cast<float*>(ring + W * 2 * kTile)
                      : p.warp_partials + static_cast<size_t>(cta) * W * kWarpPartial;
  const auto segment = [&](int i) {
    return i & 1 ? reinterpret_cast<float*>(ring + (i >> 1) * 2 * kTile)
                 : firsts + (i >> 1) * kWarpPartial;
  };
  const uint64_t policy = l2_evict_first_policy();
  const int page_rows = 1 << p.block_shift;
  const int box_rows = min(R, page_rows), boxes = R / box_rows;

  // Lane i of the first `boxes` lanes looks up the page of the tile's i-th box (and,
  // where a box is fetched in pieces, so do the lanes of its other ones).
  const typename Pool::Lane own(lane, boxes, box_rows);
  auto page_of = [&](const Cursor& c) {
    if (lane >= boxes * Pool::kPieces) return kNoPage;
    const int token = c.token + (lane & (boxes - 1)) * box_rows;
    if (token >= c.length) return kNoPage;
    if (token + box_rows <= c.low && !(More && token < c.prefix)) return kNoPage;
    const int page = p.page_table[c.seq * p.page_table_stride + (token >> p.block_shift)];
    if (page >= 0 && page < p.pool_pages) return page;
    atomicOr(p.status, kStatusBadInput);
    return kBadPage;
  };
  // Requests the tile's boxes; a bad page's are left out, and its row is NaN.
  auto issue = [&](int which, const Cursor& c, int page) {
    uint64_t* bar = &bars[warp][which];
    const unsigned used = __ballot_sync(0xffffffffu, page >= 0);
    if (lane == 0) mbar_expect_tx(bar, __popc(used) / Pool::kPieces * Pool::box_bytes(box_rows));
    fence_proxy_async();
    __syncwarp();
    if (page >= 0) {
      const int token = c.token + (lane & (boxes - 1)) * box_rows;
      Pool::fetch(source, own, which, stage + which * kTile, bar, token & (page_rows - 1), c.head,
                  page, policy);
    }
  };

  // The rows that the range's two ends cut: known from the start, so worked out
  // while the first tiles are on their way.
  const auto find_cuts = [&] {
    if (warp >= 2) return;
    const Cursor c = seek<R, More>(p, start, warp == 0 ? lo : hi - 1);
    const unsigned begin = (warp == 0 ? lo : hi - 1) - c.tile;
    const bool cut = warp == 0 ? begin < lo : begin >= lo && begin + c.tiles > hi;
    Cut found;
    found.row = -1;
    if (cut) found = cut_row(ranges, cta, c.seq * p.heads + c.head, begin, c.tiles);
    if (lane == 0) cuts[warp] = found;
  };
  if (wlo >= whi) find_cuts();
  if (wlo < whi) {
    typename Pool::Query query;
    float m[NT][2], l[NT][2], o[D / 16][NT][4];
    Cursor cur = seek<R, More>(p, start, wlo), next = cur;
    int page = page_of(cur);
    issue(0, cur, page);
    issue(1, cur, page);
    // Whether a tile lacks a page: this one, the next, any so far of the row.
    bool bad = __any_sync(0xffffffffu, page == kBadPage), next_bad = false, spoilt = false;
    find_cuts();
    const int count = static_cast<int>(whi - wlo);
    // Nothing to be done to the logits of a tile that is visible as a whole.
    const bool bare = More && p.softcap == 0.f && p.slopes == nullptr &&
                      (Pool::kBareScores || p.scores == nullptr);
    int seg_first = cur.tile;  // the segment's first tile of its row
    bool fresh = true, aborted = false;
    const auto again = [&](int which, int parity) { warp_wait(&bars[warp][which], parity); };
    if (count > 1) {
      advance<R, More>(p, start, next);
      page = page_of(next);
    }
    for (int j = 0; j < count; ++j) {
      if (fresh) {
        Pool::load_queries(query, p, cur.seq, cur.head, lane);
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
      const int token = cur.token;
      Seen seen;
      seen.low = max(0, cur.low - token);
      seen.high = min(R, cur.length - token);
      seen.prefix = More ? max(0, cur.prefix - token) : 0;
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
        Pool::score(k_tile, query, logit, scratch, lane, p);
        if (More && bare && seen.all(R)) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              const float scale = Pool::column_scale(query, p, nt, c & 1, lane);
#pragma unroll
              for (int mt = 0; mt < R / 16; ++mt) logit[mt][nt][c] *= scale;
            }
          if constexpr (Pool::kBareScores) {
            if (p.scores != nullptr) keep_scores<Pool>(logit, cur, token, lane, p);
          }
        } else if constexpr (More) {
          shape_logits<Pool>(logit, query, seen, cur, token, lane, p);
        } else {
#pragma unroll
          for (int mt = 0; mt < R / 16; ++mt)
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              const int r = mt * 16 + (lane >> 2) + (c >> 1) * 8;
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
                logit[mt][nt][c] =
                    r >= seen.low && r < seen.high ? logit[mt][nt][c] * p.scale : -INFINITY;
            }
        }
        __syncwarp();
        if (more) {
          issue(0, next, page);
          next_bad = __any_sync(0xffffffffu, page == kBadPage);
        }
        Pool::softmax(logit, m, l, o);
        if (!warp_wait(&bars[warp][1], j & 1)) {
          if (lane == 0) atomicOr(p.status, kStatusTimeout);
          drain_values(j, more, again);
          aborted = true;
        } else {
          Pool::weigh(stage + kTile, v_tile, logit, o, seen, scratch, lane, p);
          __syncwarp();
          if (more) issue(1, next, page);
        }
      }
      const bool row_done = cur.tile + 1 == cur.tiles;
      if (row_done || !more) {
        reduce_l<NT>(l);
        Pool::settle(l, o);
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
              float inv = 1.f / l[nt][c];
              if (More) inv *= value_factor(p, cur.head);
#pragma unroll
              for (int dt = 0; dt < D / 16; ++dt)
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                  const int d = Pool::channel(dt, half, lane);
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
                  to[g * (D + kPad) + Pool::channel(dt, half, lane)] = o[dt][nt][2 * half + c];
            }
        }
        seg_first = 0;
        fresh = true;
      }
      if (more) {
        cur = next;
        bad = next_bad;
        if (j + 2 < count) {
          advance<R, More>(p, start, next);
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
  constexpr int kBatch = Pool::kJoinBatch;
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
            put_joined<D, G8, More>(p, row, g, d, to, m, l, o);
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
        put_joined<D, G8, More>(p, cut.row, g, d, target, m, l, o);
      };
      // More than one batch's parts, up to 24 (kFlatJoin) or a group's: in twenties.
      // A row of 18 parts (128K tokens, eight heads) 87.3 us against 87.9 in eights,
      // 21 and 24 parts (16K tokens, seven and six heads) 18.8 and 17.2 against 18.6
      // and 17.0.
      if (kLanes == D / 4 && members >> kBatch) {
        join<D, kLanes, Pool::kLongBatch>(members, x % kLanes, m_of, l_of, o_of, put);
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

template <typename Pool, bool More>
cudaError_t launch_pool(const typename Pool::Source& source, const PagedParams& p, int ctas,
                        cudaStream_t stream) {
  // One limit for every batch: the largest this kernel takes.
  cudaError_t err = ensure_smem_limit(reinterpret_cast<const void*>(&paged_kernel<Pool, More>),
                                      paged_smem<Pool>(kMostSequences));
  if (err != cudaSuccess) return err;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(Pool::W * 32);
  cfg.dynamicSmemBytes = paged_smem<Pool>(p.sequences);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, paged_kernel<Pool, More>, source, p);
}

// Where a workspace keeps an instance's partials.
template <typename Pool>
PagedLayout pool_layout(int sms) {
  const size_t one = static_cast<size_t>(partial_floats(Pool::D, Pool::NT)) * 4;
  PagedLayout l;
  size_t off = kHeader;
  l.warp_partials = off;
  if (!Pool::kFirstInSmem) {
    off += static_cast<size_t>(warp_partial_floats(Pool::D, Pool::NT)) * 4 * sms * Pool::W;
  }
  l.cta_partials = off;
  off += one * sms * 2;
  l.group_partials = off;
  off += one * sms * 2;
  l.bytes = (off + 255) & ~static_cast<size_t>(255);
  return l;
}

}  // namespace
}  // namespace rkv

#endif  // RKV_PAGED_CU_
