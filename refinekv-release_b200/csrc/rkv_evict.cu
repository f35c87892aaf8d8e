// Eviction from a page pool by what weight its tokens got.
//
// Mathematics.  Per sequence and KV head with n > budget rows: a row counts by
// its weight (NaN least), the `recent` newest before all; the `budget` rows that
// count most are kept, of equal ones the first.  Kept rows behind the budget
// move into the places of dropped rows before it, the i-th of the ones into the
// i-th of the others, so a row moves once at most and nothing that is read is
// written: sources lie behind the budget, targets before it.
//
// Bound: the weights are read once (4 bytes a row) and only the rows that move are
// touched, 2 x 2 rows of 2 dim bytes (bf16); a step that drops one row a head is
// latency alone.
//
// Two launches.  select_kernel: a cluster of CTAs for each row (as many as the device has
// room for); the budget-th greatest is found from the weights as ordered integers, kept
// in shared memory, eleven bits at a time, until all rows that share the bits found are
// kept (two passes for weights of many values); the cluster's histograms and counts are
// added through distributed shared memory, and the moves listed in the workspace.
// move_kernel makes them with the whole device: in the select kernel's few CTAs a row
// they took twice as long (161 against 82 us for eight prompts of up to 32K tokens).  Now
// 73 us: 25 and 46 for 158 MB.
#include <cooperative_groups.h>

#include <algorithm>
#include <string>

#include "refinekv_b200.h"
#include "rkv_device.cuh"
#include "rkv_fp4.cuh"
#include "rkv_kernels.h"

namespace rkv {
void set_last_error(const std::string& message);

namespace {

namespace cg = cooperative_groups;

struct EvictParams {
  uint8_t* pool[2];                      // keys, values
  int64_t page[2], head[2], row[2];      // byte strides
  const int32_t* page_table;
  int64_t page_table_stride;
  const int32_t* lengths;
  int32_t* lengths_out;
  float* weights;
  int64_t weight_seq, weight_head;
  int32_t* positions;
  int64_t position_seq, position_head;
  int sequences, heads, dim, block_shift, capacity, pool_pages;
  int budget, recent;
  int fp4;
  int slice;   // rows of a CTA that its shared memory holds; 0: they are read again each time
  int most;    // entries of a row's list
  int* status;
  int* counts;  // (rows): moves
  int2* moves;  // (rows, most): from, to
};

constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr int kMostCluster = 8;
constexpr int kSliceBytes = 160 * 1024;
constexpr int kBins = 2048;  // of the widest digit
static_assert(kBins / kThreads == 4, "a thread reads four bins at once, or two of 1024");
constexpr int kFlying = 2;   // moves that a lane has in flight

// Weights in their order as unsigned integers: NaN 0, then -inf .. inf; a
// protected row above all.
__device__ __forceinline__ uint32_t rank_of(float weight) {
  const uint32_t bits = __float_as_uint(weight + 0.f);  // -0 as 0
  if ((bits & 0x7fffffffu) > 0x7f800000u) return 0;
  return bits ^ (bits >> 31 ? 0xffffffffu : 0x80000000u);
}
constexpr uint32_t kProtected = 0xffffffffu;

__global__ void __launch_bounds__(kThreads, 2)
    select_kernel(const __grid_constant__ EvictParams p) {
  extern __shared__ uint32_t ranks[];
  __shared__ __align__(16) unsigned hist[2][kBins];
  __shared__ unsigned totals[3];  // of this CTA, for the cluster: equal ones, holes, movers
  __shared__ int newest;          // of this CTA
  __shared__ unsigned long long least;
  __shared__ unsigned warp_counts[2][kWarps];
  __shared__ uint32_t found;
  __shared__ unsigned found_rest, found_equal;
  const cg::cluster_group cluster = cg::this_cluster();
  const int size = cluster.num_blocks(), part = cluster.block_rank();
  const int row = blockIdx.x / size, seq = row / p.heads, head = row - seq * p.heads;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const auto meet = [&] {
    if (size > 1) cluster.sync();
    else __syncthreads();
  };
  pdl_wait();
  pdl_launch_dependents();
  const int length = p.lengths[seq];
  if (threadIdx.x == 0 && part == 0 && head == 0) {
    if (length < 0 || length > p.capacity) atomicOr(p.status, kStatusBadInput);
    p.lengths_out[seq] = length > p.capacity ? length : min(max(length, 0), p.budget);
  }
  if (length <= p.budget || length > p.capacity) {  // the whole cluster
    if (threadIdx.x == 0 && part == 0) p.counts[row] = 0;
    return;
  }
  const int each = (length + size * kThreads - 1) / (size * kThreads) * kThreads;
  const int lo = min(length, part * each), hi = min(length, lo + each);
  float* weights = p.weights + seq * p.weight_seq + head * p.weight_head;
  const int32_t* positions =
      p.positions != nullptr ? p.positions + seq * p.position_seq + head * p.position_head : nullptr;

  int last = length - 1;
  if (positions != nullptr && p.recent > 0) {
    if (threadIdx.x == 0) newest = INT_MIN;
    __syncthreads();
    int mine = INT_MIN;
    for (int i = lo + threadIdx.x; i < hi; i += kThreads) mine = max(mine, positions[i]);
    mine = __reduce_max_sync(0xffffffffu, mine);
    if (lane == 0) atomicMax(&newest, mine);
    meet();
    last = lane < size ? *cluster.map_shared_rank(&newest, lane) : INT_MIN;
    last = __reduce_max_sync(0xffffffffu, last);
  }
  const auto fresh_rank = [&](int i) {
    // Differences of positions in 64 bits: any two of them.
    const int64_t age = static_cast<int64_t>(last) - (positions != nullptr ? positions[i] : i);
    return p.recent > 0 && age < p.recent ? kProtected : rank_of(weights[i]);
  };
  int2* moves = p.moves + static_cast<int64_t>(row) * p.most;
  if (length - p.budget == 1) {
    // One row goes, as in every step of a full cache: the one of least weight, of equal
    // ones the last (32 sequences of 4097 tokens, 8 KV heads: 8 us against 20 with the
    // search below).
    if (threadIdx.x == 0) least = ~0ull;
    __syncthreads();
    unsigned long long mine = ~0ull;
    for (int i = lo + threadIdx.x; i < hi; i += kThreads) {
      mine = min(mine, static_cast<unsigned long long>(fresh_rank(i)) << 32 |
                           static_cast<uint32_t>(~i));
    }
#pragma unroll
    for (int step = 16; step > 0; step >>= 1) {
      mine = min(mine, __shfl_xor_sync(0xffffffffu, mine, step));
    }
    if (lane == 0) atomicMin(&least, mine);
    meet();
    if (part == 0 && threadIdx.x == 0) {
      for (int c = 1; c < size; ++c) mine = min(mine, *cluster.map_shared_rank(&least, c));
      mine = min(mine, least);
      const int gone = static_cast<int>(~static_cast<uint32_t>(mine));
      p.counts[row] = gone < p.budget;
      if (gone < p.budget) moves[0] = make_int2(p.budget, gone);
      else weights[gone] = 0.f;
    }
    if (size > 1) cluster.sync();  // no CTA leaves while another reads its least
    return;
  }
  // Sums over the warps before this one, and over the CTAs before this one.
  const auto before_warp = [&](int which) {
    return __reduce_add_sync(0xffffffffu, lane < warp ? warp_counts[which][lane] : 0u);
  };
  const auto before_cta = [&](int which) {
    const unsigned theirs = lane < part ? *cluster.map_shared_rank(&totals[which], lane) : 0u;
    return __reduce_add_sync(0xffffffffu, theirs);
  };
  // A CTA's own total, by its first warp.
  const auto add_warps = [&](int which, int total) {
    const unsigned sum =
        __reduce_add_sync(0xffffffffu, lane < kWarps ? warp_counts[which][lane] : 0u);
    if (lane == 0) totals[total] = sum;
  };
  const bool held = p.slice > 0;
  if (held) {
    for (int i = lo + threadIdx.x; i < hi; i += kThreads) ranks[i - lo] = fresh_rank(i);
  }
  const auto rank_at = [&](int i) { return held ? ranks[i - lo] : fresh_rank(i); };

  // The budget-th greatest, from its highest bits down: 11, 11 and 10 of them.
  uint32_t prefix = 0;
  unsigned want = p.budget, equal = 0;
  int shift = 32;
  for (int pass = 0; pass < 3 && (pass == 0 || want < equal); ++pass) {
    const int above = shift;
    shift = pass < 2 ? above - 11 : 0;
    const int bins = 1 << (above - shift);
    unsigned* mine = hist[pass & 1];
    // The other one may still be read by the cluster; this one was two passes ago.
    for (int b = threadIdx.x; b < bins; b += kThreads) mine[b] = 0;
    __syncthreads();
#pragma unroll 4
    for (int base = lo; base < hi; base += kThreads) {  // whole warps
      const int i = base + threadIdx.x;
      const uint32_t x = i < hi ? rank_at(i) : 0;
      const bool counts = i < hi && (pass == 0 || x >> above == prefix);
      const unsigned bin = x >> shift & (bins - 1);
      // Equal weights would all add to one place: a warp of one bin adds once.
      int same;
      __match_all_sync(0xffffffffu, counts ? bin : kBins, &same);
      if (!same) {
        if (counts) atomicAdd(&mine[bin], 1u);
      } else if (lane == 0 && counts) {
        atomicAdd(&mine[bin], 32u);
      }
    }
    meet();
    // Thread 0 has the highest bins, four or two each; the CTAs' are all requested at once.
    const int own_bins = bins / kThreads;
    const int first = bins - own_bins * (static_cast<int>(threadIdx.x) + 1);
    unsigned count[4] = {0, 0, 0, 0};
    uint4 theirs[kMostCluster];
#pragma unroll
    for (int c = 0; c < kMostCluster; ++c) {
      theirs[c] = make_uint4(0, 0, 0, 0);
      if (c >= size) continue;
      const unsigned* at = cluster.map_shared_rank(mine + first, c);
      if (own_bins == 4) {
        theirs[c] = *reinterpret_cast<const uint4*>(at);
      } else {
        const uint2 two = *reinterpret_cast<const uint2*>(at);
        theirs[c].z = two.x, theirs[c].w = two.y;
      }
    }
#pragma unroll
    for (int c = 0; c < kMostCluster; ++c) {
      count[0] += theirs[c].w, count[1] += theirs[c].z;
      count[2] += theirs[c].y, count[3] += theirs[c].x;
    }
    const unsigned sum = count[0] + count[1] + count[2] + count[3];
    unsigned scan = sum;
#pragma unroll
    for (int step = 1; step < 32; step <<= 1) {
      const unsigned other = __shfl_up_sync(0xffffffffu, scan, step);
      if (lane >= step) scan += other;
    }
    if (lane == 31) warp_counts[0][warp] = scan;
    __syncthreads();
    unsigned before = scan - sum + before_warp(0);
    if (before < want && want <= before + sum) {  // one thread
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (before < want && want <= before + count[k]) {
          found = (pass == 0 ? 0 : prefix << (above - shift)) |
                  static_cast<uint32_t>(bins - 1 - static_cast<int>(threadIdx.x) * own_bins - k);
          found_rest = want - before;
          found_equal = count[k];
          before = want;  // done
        } else if (before < want) {
          before += count[k];
        }
      }
    }
    __syncthreads();
    prefix = found;
    want = found_rest;
    equal = found_equal;
  }
  // Rows above the prefix are kept, and of the `equal` ones with it the first `want`.

  // Counts before this CTA and this warp; a warp's rows are contiguous.
  const int span = (each / kWarps + 31) / 32 * 32;
  const int from = min(hi, lo + warp * span), to = min(hi, from + span);
  unsigned equal_before = 0;
  if (want < equal) {
    unsigned mine = 0;
    for (int i = from + lane; i < to; i += 32) mine += rank_at(i) >> shift == prefix;
    mine = __reduce_add_sync(0xffffffffu, mine);
    if (lane == 0) warp_counts[0][warp] = mine;
    __syncthreads();
    if (warp == 0) add_warps(0, 0);
    meet();
    equal_before = before_cta(0) + before_warp(0);
    __syncthreads();
  }
  // Walks the warp's rows: visit(i, there, hole, mover).
  const auto walk = [&](auto visit) {
    unsigned seen = equal_before;
    for (int base = from; base < to; base += 32) {
      const int i = base + lane;
      const bool there = i < to;
      const uint32_t x = there ? rank_at(i) >> shift : 0;
      const bool same = there && x == prefix;
      const unsigned sames = __ballot_sync(0xffffffffu, same);
      const unsigned order = seen + __popc(sames & ((1u << lane) - 1));
      seen += __popc(sames);
      const bool kept = there && (x > prefix || (same && order < want));
      visit(i, there, there && !kept && i < p.budget, kept && i >= p.budget);
    }
  };
  // The first walk leaves a word of holes and one of movers for each 32 rows, in place of
  // the ranks it has read (whose first two of 32 they replace).
  unsigned holes = 0, movers = 0;
  walk([&](int i, bool, bool hole, bool mover) {
    const unsigned all_holes = __ballot_sync(0xffffffffu, hole);
    const unsigned all_movers = __ballot_sync(0xffffffffu, mover);
    holes += __popc(all_holes);
    movers += __popc(all_movers);
    if (held && lane < 2) ranks[i - lo] = lane == 0 ? all_holes : all_movers;
  });
  if (lane == 0) {
    warp_counts[0][warp] = holes;
    warp_counts[1][warp] = movers;
  }
  __syncthreads();
  if (warp < 2) add_warps(warp, 1 + warp);
  meet();
  holes = before_cta(1);
  movers = before_cta(2);
  if (threadIdx.x == 0 && part == size - 1) p.counts[row] = static_cast<int>(movers + totals[2]);
  holes += before_warp(0);
  movers += before_warp(1);
  // A dropped row's weight ends with it; a mover's goes along.
  if (held) {
    // A lane takes the words of 32 rows and lists their bits.
    for (int base = from; base < to; base += 1024) {
      const int at = base + 32 * lane;
      unsigned hole = at < to ? ranks[at - lo] : 0, mover = at < to ? ranks[at - lo + 1] : 0;
      // How many of each the lanes before have: both counts, below 2^16, in one word.
      const unsigned own = __popc(hole) | __popc(mover) << 16;
      unsigned scan = own;
#pragma unroll
      for (int step = 1; step < 32; step <<= 1) {
        const unsigned other = __shfl_up_sync(0xffffffffu, scan, step);
        if (lane >= step) scan += other;
      }
      const unsigned total = __shfl_sync(0xffffffffu, scan, 31);
      unsigned hole_at = holes + (scan - own & 0xffffu), mover_at = movers + (scan - own >> 16);
      for (; hole != 0; hole &= hole - 1) moves[hole_at++].y = at + __ffs(hole) - 1;
      for (; mover != 0; mover &= mover - 1) moves[mover_at++].x = at + __ffs(mover) - 1;
      holes += total & 0xffffu;
      movers += total >> 16;
    }
    for (int base = max(from, p.budget / 32 * 32); base < to; base += 32) {
      const int i = base + lane;
      if (i < to && i >= p.budget && !(ranks[base - lo + 1] >> lane & 1)) weights[i] = 0.f;
    }
  } else {
    walk([&](int i, bool there, bool hole, bool mover) {
      const unsigned below = (1u << lane) - 1;
      const unsigned all_holes = __ballot_sync(0xffffffffu, hole);
      const unsigned all_movers = __ballot_sync(0xffffffffu, mover);
      if (mover) moves[movers + __popc(all_movers & below)].x = i;
      if (hole) moves[holes + __popc(all_holes & below)].y = i;
      holes += __popc(all_holes);
      movers += __popc(all_movers);
      if (there && i >= p.budget && !mover) weights[i] = 0.f;
    });
  }
  if (size > 1) cluster.sync();  // no CTA leaves while another reads its counts
}

// A unit is what a lane copies at once: 16 bytes of a row, or two of its scales'.  A warp
// takes as many moves as it has lanes for, kFlying times.
constexpr int kMoveThreads = 256;

__global__ void __launch_bounds__(kMoveThreads, 6)
    move_kernel(const __grid_constant__ EvictParams p, unsigned parts) {
  const int row = static_cast<int>(blockIdx.x / parts);
  const int part = static_cast<int>(blockIdx.x - static_cast<unsigned>(row) * parts);
  const int seq = row / p.heads, head = row - seq * p.heads;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int units = p.fp4 ? p.dim / 16 : p.dim / 8;  // of a key or a value
  const int wide = p.fp4 ? p.dim / 32 : units;       // of them, 16 bytes each
  const int all = 2 * units, per = all <= 32 ? 32 / all : 1;
  const int slot = all <= 32 ? lane / all : 0, mine = all <= 32 ? lane - slot * all : lane;
  const int stride = static_cast<int>(parts) * (kMoveThreads / 32) * per;
  pdl_wait();
  pdl_launch_dependents();
  if (slot >= per) return;
  const int count = p.counts[row];
  const int2* moves = p.moves + static_cast<int64_t>(row) * p.most;
  const int32_t* table = p.page_table + seq * p.page_table_stride;
  const int mask = (1 << p.block_shift) - 1;
  const auto page_of = [&](int token) {
    const int page = table[token >> p.block_shift];
    return page >= 0 && page < p.pool_pages ? page : -1;
  };
  for (int u = mine; u < all; u += 32) {
    // Where the lane's unit is, but for the page and the row.
    const int which = u >= units ? 1 : 0, unit = u - which * units;
    const bool is_wide = unit < wide;
    uint8_t* unit_base =
        p.pool[which] + head * p.head[which] +
        (is_wide ? 16 * unit : (p.dim / 2 << p.block_shift) + 2 * (unit - wide));
    const int64_t page_bytes = p.page[which];
    const int64_t row_bytes = !p.fp4 ? p.row[which] : is_wide ? p.dim / 2 : p.dim / 16;
    // A row whose page is outside the pool is NaN where it goes.
    const uint32_t nan = is_wide ? 0x7fc07fc0u : kFp4NanScale << 8 | kFp4NanScale;
    for (int base = (part * (kMoveThreads / 32) + warp) * per + slot; base < count;
         base += stride * kFlying) {
      int2 move[kFlying];
      uint8_t* target[kFlying];
      uint4 data[kFlying];
#pragma unroll
      for (int f = 0; f < kFlying; ++f) {
        const int at = base + f * stride;
        move[f] = at < count ? __ldcg(&moves[at]) : make_int2(-1, -1);
      }
#pragma unroll
      for (int f = 0; f < kFlying; ++f) {
        target[f] = nullptr;
        if (move[f].x < 0) continue;
        const int from = page_of(move[f].x), to = page_of(move[f].y);
        if ((from < 0 || to < 0) && u == 0) atomicOr(p.status, kStatusBadInput);
        if (to >= 0) target[f] = unit_base + to * page_bytes + (move[f].y & mask) * row_bytes;
        data[f] = make_uint4(nan, nan, nan, nan);
        if (from < 0) continue;
        const uint8_t* source = unit_base + from * page_bytes + (move[f].x & mask) * row_bytes;
        if (is_wide) data[f] = *reinterpret_cast<const uint4*>(source);
        else data[f].x = *reinterpret_cast<const uint16_t*>(source);
      }
#pragma unroll
      for (int f = 0; f < kFlying; ++f) {
        if (target[f] == nullptr) continue;
        if (is_wide) *reinterpret_cast<uint4*>(target[f]) = data[f];
        else *reinterpret_cast<uint16_t*>(target[f]) = static_cast<uint16_t>(data[f].x);
      }
      if (u == 0) {
        float* weights = p.weights + seq * p.weight_seq + head * p.weight_head;
#pragma unroll
        for (int f = 0; f < kFlying; ++f) {
          if (move[f].x < 0) continue;
          weights[move[f].y] = weights[move[f].x];
          weights[move[f].x] = 0.f;
          if (p.positions != nullptr) {
            int32_t* positions = p.positions + seq * p.position_seq + head * p.position_head;
            positions[move[f].y] = positions[move[f].x];
          }
        }
      }
    }
  }
}

int reject(int code, const char* message) {
  set_last_error(message);
  return code;
}

constexpr size_t kEvictHeader = 256;

int64_t list_entries(int64_t capacity, int64_t budget) {
  return std::max<int64_t>(0, std::min(budget, capacity - budget));
}

// Bytes of a workspace: the status word, a count a row, a list a row.
int64_t evict_bytes(int64_t rows, int64_t capacity, int64_t budget, int64_t* lists) {
  *lists = static_cast<int64_t>(kEvictHeader) + (rows * 4 + 255) / 256 * 256;
  return *lists + rows * list_entries(capacity, budget) * 8;
}

template <typename Kernel, typename... Args>
cudaError_t launch(Kernel kernel, unsigned grid, int threads, size_t smem, int cluster,
                   cudaStream_t stream, const Args&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

}  // namespace
}  // namespace rkv

extern "C" {

size_t rkv_paged_evict_workspace_size(int64_t sequences, int64_t kv_heads, int64_t tokens,
                                      int64_t budget) {
  using namespace rkv;
  if (sequences < 0 || sequences > kMostSequences || kv_heads < 1 || kv_heads > kMostPagedHeads ||
      tokens < 0 || tokens > kMostPagedTokens || budget < 1) {
    return 0;
  }
  int64_t lists;
  return static_cast<size_t>(evict_bytes(sequences * kv_heads, tokens, budget, &lists));
}

int rkv_paged_evict(const rkv_evict_args* a, void* stream) {
  using namespace rkv;
  set_last_error("");
  if (a == nullptr) return reject(RKV_ERR_INVALID_ARGUMENT, "args is null");
  if (a->head_dim < 32 || a->head_dim > 256 || a->head_dim % 32 != 0) {
    return reject(RKV_ERR_UNSUPPORTED, "head_dim must be a multiple of 32 in [32, 256]");
  }
  if (a->block_size != 16 && a->block_size != 32 && a->block_size != 64) {
    return reject(RKV_ERR_UNSUPPORTED, "block_size must be 16, 32 or 64");
  }
  if (a->sequences < 0 || a->sequences > kMostSequences || a->kv_heads < 1 ||
      a->kv_heads > kMostPagedHeads) {
    return reject(RKV_ERR_UNSUPPORTED, "at most 4096 sequences and 4096 KV heads");
  }
  const bool fp4 = a->pool_dtype == RKV_DTYPE_FP4;
  if (!fp4 && a->pool_dtype != RKV_DTYPE_BF16) {
    return reject(RKV_ERR_INVALID_ARGUMENT, "pools are bf16 or fp4");
  }
  if (a->table_blocks < 0 || a->table_blocks > kMostPagedTokens / a->block_size ||
      a->page_table_stride < 0 || a->pool_pages < 0 || a->pool_pages > (1LL << 31) - 1) {
    return reject(RKV_ERR_INVALID_ARGUMENT, "page table or pool sizes are out of range");
  }
  if (a->budget < 1 || a->recent < 0 || a->recent > a->budget) {
    return reject(RKV_ERR_INVALID_ARGUMENT, "budget must be positive and recent at most budget");
  }
  const int64_t capacity = a->table_blocks * a->block_size;
  if (a->weight_width < capacity || (a->positions != nullptr && a->position_width < capacity)) {
    return reject(RKV_ERR_INVALID_ARGUMENT,
                  "rows of weights and positions must hold as many tokens as the page table");
  }
  if (a->sequences == 0) return RKV_OK;
  if (!a->key_pool || !a->value_pool || !a->page_table || !a->lengths || !a->lengths_out ||
      !a->weights) {
    return reject(RKV_ERR_INVALID_ARGUMENT,
                  "pools, page_table, lengths, lengths_out and weights must be non-null");
  }
  const int width = fp4 ? 1 : 2;
  uintptr_t bits = reinterpret_cast<uintptr_t>(a->key_pool) | reinterpret_cast<uintptr_t>(a->value_pool);
  for (int i = 0; i < (fp4 ? 2 : 3); ++i) {
    bits |= static_cast<uintptr_t>(a->key_pool_strides[i] * width);
    bits |= static_cast<uintptr_t>(a->value_pool_strides[i] * width);
  }
  if (bits & 15u) {
    return reject(RKV_ERR_ALIGNMENT, "pools and their strides must be multiples of 16 bytes");
  }
  if (a->lengths == a->lengths_out) {
    return reject(RKV_ERR_INVALID_ARGUMENT, "lengths_out must not be lengths");
  }
  if (!aligned_to(4, {a->page_table, a->lengths, a->lengths_out, a->weights, a->positions})) {
    return reject(RKV_ERR_ALIGNMENT, "page_table, lengths, weights and positions must be aligned to "
                                     "their elements");
  }
  const int64_t rows = a->sequences * a->kv_heads;
  int64_t lists;
  if (a->workspace == nullptr ||
      a->workspace_size < evict_bytes(rows, capacity, a->budget, &lists) ||
      (reinterpret_cast<uintptr_t>(a->workspace) & 255u) != 0) {
    return reject(RKV_ERR_WORKSPACE, "workspace is missing, too small or not 256-byte aligned");
  }
  int sms = 0;
  const int rc = device_sms(&sms);
  if (rc != RKV_OK) return rc;
  EvictParams p = {};
  p.pool[0] = static_cast<uint8_t*>(a->key_pool);
  p.pool[1] = static_cast<uint8_t*>(a->value_pool);
  for (int i = 0; i < 2; ++i) {
    const int64_t* strides = i ? a->value_pool_strides : a->key_pool_strides;
    p.page[i] = strides[0] * width;
    p.head[i] = strides[1] * width;
    p.row[i] = fp4 ? 0 : strides[2] * width;
  }
  p.page_table = a->page_table;
  p.page_table_stride = a->page_table_stride;
  p.lengths = a->lengths;
  p.lengths_out = a->lengths_out;
  p.weights = a->weights;
  p.weight_seq = a->weight_strides[0];
  p.weight_head = a->weight_strides[1];
  p.positions = a->positions;
  p.position_seq = a->position_strides[0];
  p.position_head = a->position_strides[1];
  p.sequences = static_cast<int>(a->sequences);
  p.heads = static_cast<int>(a->kv_heads);
  p.dim = static_cast<int>(a->head_dim);
  p.block_shift = a->block_size == 16 ? 4 : a->block_size == 32 ? 5 : 6;
  p.capacity = static_cast<int>(capacity);
  p.pool_pages = static_cast<int>(a->pool_pages);
  p.budget = static_cast<int>(std::min<int64_t>(a->budget, kMostPagedTokens));
  p.recent = static_cast<int>(std::min<int64_t>(a->recent, kMostPagedTokens));
  p.fp4 = fp4;
  p.most = static_cast<int>(list_entries(capacity, a->budget));
  char* ws = static_cast<char*>(a->workspace);
  p.status = reinterpret_cast<int*>(ws);
  p.counts = reinterpret_cast<int*>(ws + kEvictHeader);
  p.moves = reinterpret_cast<int2*>(ws + lists);
  // A row is shared by as many CTAs as the device has room for, of 4096 tokens at
  // least, and by eight where its ranks fit in shared memory only so.
  int size = 1;
  while (size < kMostCluster && ((rows * size < sms && capacity > 4096 * size) ||
                                 capacity * 4 > static_cast<int64_t>(kSliceBytes) * size)) {
    size *= 2;
  }
  const int64_t whole = static_cast<int64_t>(size) * kThreads;
  const int64_t slice = (capacity + whole - 1) / whole * kThreads;
  p.slice = slice * 4 <= kSliceBytes ? static_cast<int>(slice) : 0;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t err = ensure_smem_limit(reinterpret_cast<const void*>(&select_kernel), kSliceBytes);
  if (err == cudaSuccess) {
    err = launch(select_kernel, static_cast<unsigned>(rows * size), kThreads,
                 static_cast<size_t>(p.slice) * 4, size, st, p);
  }
  if (err == cudaSuccess && p.most > 0) {
    // More CTAs than are resident at once: rows that move nothing leave theirs idle.
    const int64_t lanes = static_cast<int64_t>(p.most) * 2 * (fp4 ? p.dim / 16 : p.dim / 8);
    const unsigned parts = static_cast<unsigned>(std::max<int64_t>(
        1, std::min((lanes + kMoveThreads - 1) / kMoveThreads, (16 * sms + rows - 1) / rows)));
    err = launch(move_kernel, static_cast<unsigned>(rows * parts), kMoveThreads, 0, 1, st, p, parts);
  }
  if (err != cudaSuccess) {
    set_last_error(std::string("eviction launch: ") + cudaGetErrorString(err));
    return RKV_ERR_CUDA;
  }
  return RKV_OK;
}

}  // extern "C"
