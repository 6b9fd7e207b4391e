// Changes of a paged key/value cache on B200 (sm_100a): rows appended, and
// slots evicted by the attention weight that they gathered.

#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cstdint>
#include <type_traits>

#include "fa_host.h"
#include "fa_sm100.h"
#include "paged_cache.cuh"

namespace cg = cooperative_groups;

namespace fa {
namespace cache {

// ------------------------------------------------------------------ append
//
// Row path[b][i] (or row i) of the new keys and values becomes slot
// lengths[b] + i of sequence b, i < counts[b].  A copy: bound by HBM when long
// and by its launch when short.  4 x 8 x 2048 rows of 64 that no cache holds: 10.2
// us a call, 3.3 TB/s, half the copy rate, as the loads of a thread wait for the
// length and the table.  One 16-byte vector of K and one of V per thread;
// the eight or sixteen threads of a row are neighbours, and a block holds whole rows.
//
// A path's rows end before its first entry that names none: the slots below the
// new length are then all written.  Each block looks at the entries up to its own
// last one, the block that writes the length at all of them.

constexpr int kAppendThreads = 256;

struct AppendParams {
  Pages pages;
  const uint4* key;            // [batch, kv_heads, rows, dim], strides in vectors
  const uint4* value;
  int64_t ks[3], vs[3];        // batch, head, row
  uint4* k_pages;
  uint4* v_pages;
  const int* path;             // [batch][rows] or null
  const int* counts;           // [batch] or null: all rows
  const int* new_positions;    // [batch][rows] or null
  float* weights;              // [batch][kv_heads][slots] or null
  int* positions;              // the same
  int* lengths_out;            // [batch]
  int batch, rows, vectors;    // vectors of 16 bytes in a row
};

__global__ void __launch_bounds__(kAppendThreads) append_kernel(const AppendParams p) {
  const int64_t at = static_cast<int64_t>(blockIdx.x) * kAppendThreads + threadIdx.x;
  const int b = static_cast<int>(blockIdx.z), h = static_cast<int>(blockIdx.y);
  const int i = static_cast<int>(at / p.vectors);
  const int vec = static_cast<int>(at - static_cast<int64_t>(i) * p.vectors);
  const int slots = p.pages.slots();
  const int length = cache_length(p.pages, b);
  int count = p.counts == nullptr ? p.rows : p.counts[b];
  if (count < 0 || count > p.rows || count > slots - length) {
    atomicOr(p.pages.status, kStatusCache);
    count = max(0, min(min(count, p.rows), slots - length));
  }
  const int* path = p.path == nullptr ? nullptr : p.path + static_cast<int64_t>(b) * p.rows;
  if (path != nullptr) {
    __shared__ int first_bad;
    const int last = static_cast<int>((static_cast<int64_t>(blockIdx.x) + 1) * kAppendThreads / p.vectors);
    const int looked = blockIdx.x == 0 && h == 0 ? count : min(count, last);
    int bad = INT32_MAX;
    for (int j = static_cast<int>(threadIdx.x); j < looked && bad == INT32_MAX; j += kAppendThreads)
      if (static_cast<unsigned>(path[j]) >= static_cast<unsigned>(p.rows)) bad = j;
    if (__syncthreads_or(bad != INT32_MAX)) {
      if (threadIdx.x == 0) {
        first_bad = INT32_MAX;
        atomicOr(p.pages.status, kStatusCache);
      }
      __syncthreads();
      atomicMin(&first_bad, bad);
      __syncthreads();
      count = min(count, first_bad);
    }
  }
  if (i == 0 && h == 0 && vec == 0) p.lengths_out[b] = length + count;
  if (i >= count) return;
  const int from = path == nullptr ? i : path[i];
  const int slot = length + i;
  const int64_t row = cache_row(p.pages, b, h, slot);
  if (row < 0) return;
  const int64_t to = row / 8 + vec;  // eight elements in a vector
  p.k_pages[to] = p.key[b * p.ks[0] + h * p.ks[1] + from * p.ks[2] + vec];
  p.v_pages[to] = p.value[b * p.vs[0] + h * p.vs[1] + from * p.vs[2] + vec];
  if (vec == 0) {
    const int64_t meta = (static_cast<int64_t>(b) * p.pages.kv_heads + h) * slots + slot;
    if (p.weights != nullptr) p.weights[meta] = 0.0f;
    if (p.positions != nullptr)
      p.positions[meta] = p.new_positions[static_cast<int64_t>(b) * p.rows + from];
  }
}

// The new lengths of a call that has no rows or no heads to change: those that
// append_kernel (limit: none) or select_kernel (limit: the budget) would write.
__global__ void __launch_bounds__(kAppendThreads)
    lengths_kernel(const Pages pages, const int* counts, int rows, int limit, int batch, int* lengths_out) {
  const int b = static_cast<int>(blockIdx.x) * kAppendThreads + static_cast<int>(threadIdx.x);
  if (b >= batch) return;
  const int length = cache_length(pages, b), given = counts == nullptr ? rows : counts[b];
  const int count = max(0, min(min(given, rows), pages.slots() - length));
  if (count != given) atomicOr(pages.status, kStatusCache);
  lengths_out[b] = min(length + count, limit);
}

cudaError_t launch_lengths(const Pages& pages, const int* counts, int rows, int limit, int64_t batch,
                           int* lengths_out, cudaStream_t stream) {
  const unsigned blocks = static_cast<unsigned>((batch + kAppendThreads - 1) / kAppendThreads);
  lengths_kernel<<<blocks, kAppendThreads, 0, stream>>>(pages, counts, rows, limit, static_cast<int>(batch),
                                                        lengths_out);
  return cudaGetLastError();
}

// ------------------------------------------------------------------- evict
//
// Of each (sequence, kv head) `budget` slots stay: the first `sinks`
// positions, the last `recent` ones, then those of largest weight, the lowest
// slot first among equals.  A kept slot behind the budget moves into a dropped
// slot before it, the i-th into the i-th: attention over the cache does not
// ask for the order of slots, so only what must move does, and as sources lie
// behind the budget and destinations before it, all moves are independent.
//
// select_kernel finds which: a radix selection (11 + 11 + 10 bits) over the
// weights' bits in an order-preserving form, one block or cluster of blocks per
// (b, h), each block on a contiguous part of the slots held in shared memory;
// histograms and prefix counts cross the cluster through distributed shared
// memory.  It is bound by the latency of its passes and barriers: blocks of 512
// threads, two per SM, so that one's barriers run under the other's passes.
// move_kernel then copies rows, bound by HBM; each move is two trips to memory.
// 32 x 8 lists from 4352 to 4096 slots at dimension 64: 20.5 us a call, in a graph
// too; 8 of 65536 to 16384 at dimension 128: 45 us a call, 43 in a graph, 18 of
// them for the selection.

constexpr int kSelectThreads = 512;
constexpr int kWarps = kSelectThreads / 32;
constexpr int kBins = 2048;
constexpr int kMoveThreads = 256;
constexpr int kMaxKeys = 24 * 1024;  // slots that a block holds in shared memory: key and position

struct EvictParams {
  Pages pages;
  uint4* k_pages;
  uint4* v_pages;
  const float* weights;  // [batch][kv_heads][slots]
  const int* positions;  // the same
  float* weights_out;
  int* positions_out;
  int* lengths_out;      // [batch]
  int* n_moves;          // [batch * kv_heads]
  int* to;               // [batch * kv_heads][max_moves]: slots
  int* from;
  int max_moves;
  int budget, recent, sinks;
  int room;              // slots in a block's shared memory
  int vectors;
};

// A weight as an unsigned number of the same order; NaN is below everything,
// both zeros are one value.
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (w != w) return 0u;
  const uint32_t u = __float_as_uint(w + 0.0f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// Exclusive prefix of one value per warp over the block (a value per warp in
// `mine`, the same in every lane); returns the prefix, and the block's sum
// through `total`.  Uses `scratch` (one int per warp).
__device__ __forceinline__ int warps_prefix(int mine, int* scratch, int* total) {
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  __syncthreads();
  if (lane == 0) scratch[warp] = mine;
  __syncthreads();
  const int v = lane < kWarps ? scratch[lane] : 0;
  int s = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, s, o);
    if (lane >= o) s += u;
  }
  *total = __shfl_sync(0xffffffffu, s, 31);
  return __shfl_sync(0xffffffffu, s - v, warp);
}

template <bool kCluster>
__global__ void __launch_bounds__(kSelectThreads, 2) select_kernel(const EvictParams p) {
  extern __shared__ uint4 held_keys[];  // room keys, room positions
  __shared__ __align__(16) int hist[3][kBins];
  __shared__ __align__(16) int all_ranks[kCluster ? kBins : 4];
  __shared__ int scratch[kWarps];
  __shared__ int shared_max, found_bin, found_above, found_count, block_holes, block_movers;

  cg::cluster_group cluster = cg::this_cluster();
  const int rank = kCluster ? static_cast<int>(cluster.block_rank()) : 0;
  const int ranks = kCluster ? static_cast<int>(cluster.num_blocks()) : 1;
  auto sync = [&]() {
    if (kCluster)
      cluster.sync();
    else
      __syncthreads();
  };
  auto of_rank = [&](int& x, int r) -> int { return kCluster ? *cluster.map_shared_rank(&x, r) : x; };
  // move_kernel's blocks may take their places; they wait for this kernel's end
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  const int bh = static_cast<int>(blockIdx.x) / ranks;
  const int b = bh / p.pages.kv_heads, h = bh - b * p.pages.kv_heads;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int slots = p.pages.slots();
  const int n = cache_length(p.pages, b);
  const int64_t base = static_cast<int64_t>(bh) * slots;
  const float* w = p.weights + base;
  const int* pos = p.positions + base;
  const int n_new = min(n, p.budget);
  if (threadIdx.x == 0 && rank == 0 && h == 0) p.lengths_out[b] = n_new;

  // slots behind the new length are empty
  for (int i = n_new + rank * kSelectThreads + static_cast<int>(threadIdx.x); i < slots;
       i += ranks * kSelectThreads) {
    p.weights_out[base + i] = 0.0f;
    p.positions_out[base + i] = -1;
  }

  // This warp's slots: [s0, s1), in steps of 128, four neighbours in a lane.
  const int per_rank = (n + ranks - 1) / ranks;
  const int seg = ((per_rank + kWarps - 1) / kWarps + 127) & ~127;
  const int64_t first = (static_cast<int64_t>(rank) * kWarps + warp) * seg;
  const int s0 = static_cast<int>(first < n ? first : n);
  const int s1 = static_cast<int>(first + seg < n ? first + seg : n);
  const int key0 = rank * kWarps * seg;  // the first slot that is held
  const bool held = kWarps * seg <= p.room;
  uint32_t* keys = reinterpret_cast<uint32_t*>(held_keys);
  int* places = reinterpret_cast<int*>(keys + p.room);

  for (int i = threadIdx.x; i < 3 * kBins; i += kSelectThreads) (&hist[0][0])[i] = 0;
  if (threadIdx.x == 0) shared_max = INT32_MIN;
  __syncthreads();
  // One pass over memory: keys into shared memory, the last position, and what
  // lies before the budget to the outputs, where move_kernel will put another
  // slot's into the dropped ones.  (A row of slots is a multiple of 16 long.)
  int top = INT32_MIN;
#pragma unroll 4
  for (int i = s0 + 4 * lane; i < s1; i += 128) {
    const int4 at = *reinterpret_cast<const int4*>(pos + i);
    const float4 x = *reinterpret_cast<const float4*>(w + i);
    if (held) {
      *reinterpret_cast<uint4*>(keys + (i - key0)) =
          make_uint4(weight_key(x.x), weight_key(x.y), weight_key(x.z), weight_key(x.w));
      *reinterpret_cast<int4*>(places + (i - key0)) = at;
    }
    if (i + 3 < n_new) {
      *reinterpret_cast<int4*>(p.positions_out + base + i) = at;
      *reinterpret_cast<float4*>(p.weights_out + base + i) = x;
    } else {
      const int ats[4] = {at.x, at.y, at.z, at.w};
      const float xs[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (i + j < n_new) {
          p.positions_out[base + i + j] = ats[j];
          p.weights_out[base + i + j] = xs[j];
        }
      }
    }
    top = max(top, at.x);
    if (i + 1 < s1) top = max(top, at.y);
    if (i + 2 < s1) top = max(top, at.z);
    if (i + 3 < s1) top = max(top, at.w);
  }
  if (n <= p.budget) {  // the same in every block of the cluster
    if (threadIdx.x == 0 && rank == 0) p.n_moves[bh] = 0;
    return;
  }

  top = __reduce_max_sync(0xffffffffu, top);
  if (lane == 0) atomicMax(&shared_max, top);
  sync();
  top = __reduce_max_sync(0xffffffffu, lane < ranks ? of_rank(shared_max, lane) : INT32_MIN);
  const int64_t last_unsafe = static_cast<int64_t>(top) - p.recent;
  // positions above it are among the last; below every int where all of them are
  const int recent_from = static_cast<int>(last_unsafe < INT32_MIN ? INT32_MIN : last_unsafe);
  const bool all_recent = last_unsafe < INT32_MIN;
  auto safe = [&](int at) { return at > recent_from || all_recent || at < p.sinks; };

  // Keys of slots i .. i + 3 (those from s1 on are not to be used).
  auto keys_at = [&](int i, uint32_t (&k)[4]) {
    if (held) {
      const uint4 v = *reinterpret_cast<const uint4*>(keys + (i - key0));
      k[0] = v.x;
      k[1] = v.y;
      k[2] = v.z;
      k[3] = v.w;
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) k[j] = i + j < s1 ? (safe(pos[i + j]) ? 0xffffffffu : weight_key(w[i + j])) : 0u;
    }
  };

  // the budget-th largest key, digit by digit from the top
  uint32_t threshold = 0;
  int need = p.budget;
  auto digit_pass = [&](auto which) {
    constexpr int d = decltype(which)::value;
    constexpr int shift = d == 0 ? 21 : d == 1 ? 10 : 0;
    constexpr uint32_t mask = d == 2 ? 1023u : 2047u;
    constexpr int above_shift = d == 1 ? 21 : 10;
    const uint32_t prefix = threshold >> above_shift;
    for (int i0 = s0; i0 < s1; i0 += 128) {
      const int i = i0 + 4 * lane;
      uint32_t k[4];
      keys_at(i, k);
      if (d == 0 && held) {
        const int4 at = *reinterpret_cast<const int4*>(places + (i - key0));
        k[0] = safe(at.x) ? 0xffffffffu : k[0];
        k[1] = safe(at.y) ? 0xffffffffu : k[1];
        k[2] = safe(at.z) ? 0xffffffffu : k[2];
        k[3] = safe(at.w) ? 0xffffffffu : k[3];
        *reinterpret_cast<uint4*>(keys + (i - key0)) = make_uint4(k[0], k[1], k[2], k[3]);
      }
      if (i0 + 128 <= s1) {
        // equal weights would be 128 additions to one place: they are one
        const uint32_t one = __shfl_sync(0xffffffffu, k[0], 0);
        if (__all_sync(0xffffffffu, k[0] == one && k[1] == one && k[2] == one && k[3] == one)) {
          if (lane == 0 && (d == 0 || (one >> above_shift) == prefix)) atomicAdd(&hist[d][(one >> shift) & mask], 128);
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (d == 0 || (k[j] >> above_shift) == prefix) atomicAdd(&hist[d][(k[j] >> shift) & mask], 1);
        }
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (i + j < s1 && (d == 0 || (k[j] >> above_shift) == prefix)) atomicAdd(&hist[d][(k[j] >> shift) & mask], 1);
      }
    }
    sync();
    if (kCluster) {  // each block adds up its share of the bins for all
      for (int bin = rank * (kBins / ranks) + static_cast<int>(threadIdx.x); bin < (rank + 1) * (kBins / ranks);
           bin += kSelectThreads) {
        int x[8];
#pragma unroll
        for (int r = 0; r < 8; ++r) x[r] = r < ranks ? of_rank(hist[d][bin], r) : 0;
        const int all = ((x[0] + x[1]) + (x[2] + x[3])) + ((x[4] + x[5]) + (x[6] + x[7]));
#pragma unroll
        for (int r = 0; r < 8; ++r)
          if (r < ranks) *cluster.map_shared_rank(&all_ranks[bin], r) = all;
      }
      sync();
    }
    // bins from the top, neighbours in a thread
    constexpr int kPer = kBins / kSelectThreads;
    static_assert(kPer == 4, "a thread's bins are one vector");
    const int top_bin = kBins - 1 - kPer * static_cast<int>(threadIdx.x);
    const int4 four = *reinterpret_cast<const int4*>((kCluster ? all_ranks : hist[d]) + top_bin - 3);
    const int c[kPer] = {four.w, four.z, four.y, four.x};
    const int sum = (c[0] + c[1]) + (c[2] + c[3]);
    int incl = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += u;
    }
    int total;
    int above = warps_prefix(__shfl_sync(0xffffffffu, incl, 31), scratch, &total) + incl - sum;
    if (above < need && need <= above + sum) {  // one thread
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        if (above < need && need <= above + c[j]) {
          found_bin = top_bin - j;
          found_above = above;
          found_count = c[j];
        }
        above += c[j];
      }
    }
    __syncthreads();
    threshold |= static_cast<uint32_t>(found_bin) << shift;
    need -= found_above;
  };
  digit_pass(std::integral_constant<int, 0>());
  digit_pass(std::integral_constant<int, 1>());
  digit_pass(std::integral_constant<int, 2>());

  // Of the slots equal to the threshold the first `need` stay; mostly that is all
  // of them, and none has to be counted.
  const bool some_ties = need < found_count;
  int left = INT32_MAX;  // of this warp's ties, those that may stay
  if (some_ties) {
    const int last_digit = static_cast<int>(threshold & 1023u);
    int before = 0;
    if (kCluster) before = __reduce_add_sync(0xffffffffu, lane < rank ? of_rank(hist[2][last_digit], lane) : 0);
    int mine = 0, total;
    for (int i0 = s0; i0 < s1; i0 += 128) {
      const int i = i0 + 4 * lane;
      uint32_t k[4];
      keys_at(i, k);
#pragma unroll
      for (int j = 0; j < 4; ++j) mine += i + j < s1 && k[j] == threshold;
    }
    left = need - before - warps_prefix(__reduce_add_sync(0xffffffffu, mine), scratch, &total);
  }

  // Which of slots i .. i + 3 stay (bit j: slot i + j); `ties` may still stay.
  auto kept_of = [&](int i0, int& ties_left) -> uint32_t {
    const int i = i0 + 4 * lane;
    uint32_t k[4], kept = 0;
    keys_at(i, k);
#pragma unroll
    for (int j = 0; j < 4; ++j) kept |= (k[j] >= threshold ? 1u : 0u) << j;
    if (some_ties) {
      uint32_t ties = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) ties |= (k[j] == threshold && i + j < s1 ? 1u : 0u) << j;
      int incl = __popc(ties);
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += u;
      }
      int before = incl - __popc(ties);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if ((ties >> j) & 1) {
          if (before >= ties_left) kept &= ~(1u << j);
          ++before;
        }
      }
      ties_left -= __shfl_sync(0xffffffffu, incl, 31);
    }
    return kept;
  };
  // holes (dropped, before the budget) and movers (kept, behind it)
  auto sides = [&](int i0, uint32_t kept, uint32_t& hole, uint32_t& mover) {
    const int i = i0 + 4 * lane;
    const uint32_t valid = (1u << min(max(s1 - i, 0), 4)) - 1u, in = (1u << min(max(p.budget - i, 0), 4)) - 1u;
    hole = valid & ~kept & in;
    mover = valid & kept & ~in;
  };
  // a warp of a block that holds its slots has at most 16 steps: their bits stay
  // in a register for the second time
  uint64_t remembered = 0;
  int holes = 0, movers = 0, ties_left = left;
  for (int i0 = s0, n_step = 0; i0 < s1; i0 += 128, ++n_step) {
    const uint32_t kept = kept_of(i0, ties_left);
    if (n_step < 16) remembered |= static_cast<uint64_t>(kept) << (4 * n_step);
    uint32_t hole, mover;
    sides(i0, kept, hole, mover);
    holes += __popc(hole);
    movers += __popc(mover);
  }
  int all_holes, all_movers;
  static_assert(kMaxKeys <= 16 * 128 * kWarps, "sixteen steps of a warp");
  int hole_at = warps_prefix(__reduce_add_sync(0xffffffffu, holes), scratch, &all_holes);
  int mover_at = warps_prefix(__reduce_add_sync(0xffffffffu, movers), scratch, &all_movers);
  int moves = all_holes;
  if (kCluster) {
    if (threadIdx.x == 0) {
      block_holes = all_holes;
      block_movers = all_movers;
    }
    sync();
    const int hr = lane < ranks ? of_rank(block_holes, lane) : 0;
    const int mr = lane < rank ? of_rank(block_movers, lane) : 0;
    moves = __reduce_add_sync(0xffffffffu, hr);
    hole_at += __reduce_add_sync(0xffffffffu, lane < rank ? hr : 0);
    mover_at += __reduce_add_sync(0xffffffffu, mr);
  }
  if (threadIdx.x == 0 && rank == 0) p.n_moves[bh] = moves;
  int* to = p.to + static_cast<int64_t>(bh) * p.max_moves;
  int* from = p.from + static_cast<int64_t>(bh) * p.max_moves;
  ties_left = left;
  for (int i0 = s0, n_step = 0; i0 < s1; i0 += 128, ++n_step) {
    const uint32_t kept = held ? static_cast<uint32_t>(remembered >> (4 * n_step)) & 15u : kept_of(i0, ties_left);
    uint32_t hole, mover;
    sides(i0, kept, hole, mover);
    if (!__any_sync(0xffffffffu, (hole | mover) != 0)) continue;
    const int both = __popc(hole) | __popc(mover) << 16;  // 128 at most of each
    int incl = both;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += u;
    }
    const int sum = __shfl_sync(0xffffffffu, incl, 31), i = i0 + 4 * lane;
    int* t = to + hole_at + ((incl - both) & 0xffff);
    int* f = from + mover_at + ((incl - both) >> 16);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if ((hole >> j) & 1) *t++ = i + j;
      if ((mover >> j) & 1) *f++ = i + j;
    }
    hole_at += sum & 0xffff;
    mover_at += sum >> 16;
  }
  if (kCluster) sync();  // no block leaves while another still reads its shared memory
}

__global__ void __launch_bounds__(kMoveThreads) move_kernel(const EvictParams p) {
  const int bh = static_cast<int>(blockIdx.y);
  const int rows = kMoveThreads / p.vectors;  // of a block and step
  const int row = static_cast<int>(threadIdx.x) / p.vectors;
  const int vec = static_cast<int>(threadIdx.x) - row * p.vectors;
  const int64_t base = static_cast<int64_t>(bh) * p.pages.slots();
  const int* tos = p.to + static_cast<int64_t>(bh) * p.max_moves;
  const int* froms = p.from + static_cast<int64_t>(bh) * p.max_moves;
  const int b = bh / p.pages.kv_heads, h = bh - b * p.pages.kv_heads;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  // One move in flight per thread, all threads of the GPU: two or four per thread
  // took longer (23 against 21 us for 256 moves in each of 256 lists).
  const int n = p.n_moves[bh];
  for (int m = static_cast<int>(blockIdx.x) * rows + row; m < p.max_moves;
       m += static_cast<int>(gridDim.x) * rows) {
    const int to = tos[m], from = froms[m];  // the lists have max_moves entries, n of them written
    if (m >= n) break;
    const int64_t dst = cache_row(p.pages, b, h, to), src = cache_row(p.pages, b, h, from);
    // A row that no page holds moves nowhere, its weight and position neither: the
    // destination keeps its own, which select_kernel has copied.
    if (dst < 0 || src < 0) continue;
    if (vec == 0) {
      p.weights_out[base + to] = p.weights[base + from];
      p.positions_out[base + to] = p.positions[base + from];
    }
    const uint4 k = p.k_pages[src / 8 + vec], v = p.v_pages[src / 8 + vec];
    p.k_pages[dst / 8 + vec] = k;
    p.v_pages[dst / 8 + vec] = v;
  }
}

}  // namespace cache
}  // namespace fa

using fa::host::set_error;

extern "C" int fa_cache_append_sm100(const fa_paged_cache* cache, const fa_rows* key,
                                     const fa_rows* value, int64_t rows, const int* path,
                                     const int* counts, float* weights, int* positions,
                                     const int* new_positions, int* lengths_out, void* cuda_stream) {
  fa::cache::AppendParams p;
  int rc = fa::check_pages(cache, &p.pages);
  if (rc != FA_OK) return rc;
  if (rows < 0) return set_error(FA_ERR_INVALID, "negative size");
  if (rows > (1ll << 30)) return set_error(FA_ERR_INVALID, "size too large");
  if (cache->batch == 0) return FA_OK;
  if (lengths_out == nullptr || (positions != nullptr && rows > 0 && new_positions == nullptr))
    return set_error(FA_ERR_INVALID, "null pointer");
  if (cache->lengths == lengths_out)
    return set_error(FA_ERR_INVALID, "lengths cannot be changed in place");
  cudaStream_t stream = static_cast<cudaStream_t>(cuda_stream);
  fa::host::Device d;
  if (rows == 0 || cache->kv_heads == 0) {
    if ((rc = fa::host::current_device(&d)) != FA_OK) return rc;
    p.pages.status = d.status;
    const cudaError_t e = fa::cache::launch_lengths(p.pages, counts, static_cast<int>(rows), INT32_MAX,
                                                    cache->batch, lengths_out, stream);
    if (e != cudaSuccess) return set_error(FA_ERR_CUDA, "kernel launch: %s", cudaGetErrorString(e));
    return FA_OK;
  }
  const fa_rows* sides[2] = {key, value};
  for (const fa_rows* r : sides) {
    if (r == nullptr || r->data == nullptr) return set_error(FA_ERR_INVALID, "null pointer");
    if ((reinterpret_cast<uintptr_t>(r->data) & 15) ||
        (r->batch_stride | r->head_stride | r->row_stride) % 8 != 0)
      return set_error(FA_ERR_INVALID, "rows of key and value must be 16-byte aligned");
  }
  if (cache->v_pages == nullptr) return set_error(FA_ERR_INVALID, "null pointer");
  if ((rc = fa::host::current_device(&d)) != FA_OK) return rc;
  p.pages.status = d.status;
  p.key = static_cast<const uint4*>(key->data);
  p.value = static_cast<const uint4*>(value->data);
  for (int i = 0; i < 2; ++i) {
    int64_t* s = i == 0 ? p.ks : p.vs;
    s[0] = sides[i]->batch_stride / 8;
    s[1] = sides[i]->head_stride / 8;
    s[2] = sides[i]->row_stride / 8;
  }
  p.k_pages = static_cast<uint4*>(cache->k_pages);
  p.v_pages = static_cast<uint4*>(cache->v_pages);
  p.path = path;
  p.counts = counts;
  p.new_positions = new_positions;
  p.weights = weights;
  p.positions = positions;
  p.lengths_out = lengths_out;
  p.batch = static_cast<int>(cache->batch);
  p.rows = static_cast<int>(rows);
  p.vectors = p.pages.dim / 8;
  const int64_t blocks = (rows * p.vectors + fa::cache::kAppendThreads - 1) / fa::cache::kAppendThreads;
  fa::cache::append_kernel<<<dim3(static_cast<unsigned>(blocks), static_cast<unsigned>(p.pages.kv_heads),
                                  static_cast<unsigned>(p.batch)),
                             fa::cache::kAppendThreads, 0, stream>>>(p);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return set_error(FA_ERR_CUDA, "kernel launch: %s", cudaGetErrorString(e));
  return FA_OK;
}

namespace {

// Moves a (sequence, kv head) can need: no more slots than lie on either side
// of the budget.
int64_t max_moves(const fa_paged_cache* c, int64_t budget) {
  const int64_t slots = c->max_pages * c->page_size;
  return std::max<int64_t>(0, std::min(budget, slots - budget));
}

int64_t counts_bytes(const fa_paged_cache* c) {
  return (c->batch * c->kv_heads * static_cast<int64_t>(sizeof(int)) + 255) & ~255ll;
}

}  // namespace

extern "C" int64_t fa_cache_evict_workspace(const fa_paged_cache* cache, int64_t budget) {
  fa::Pages pages;
  if (fa::check_pages(cache, &pages) != FA_OK) return -1;
  return counts_bytes(cache) +
         2 * cache->batch * cache->kv_heads * max_moves(cache, budget) * static_cast<int64_t>(sizeof(int));
}

extern "C" int fa_cache_evict_sm100(const fa_paged_cache* cache, const float* weights,
                                    const int* positions, float* weights_out, int* positions_out,
                                    int* lengths_out, int64_t budget, int64_t recent, int64_t sinks,
                                    void* workspace, int64_t workspace_bytes, void* cuda_stream) {
  namespace fc = fa::cache;
  fc::EvictParams p;
  int rc = fa::check_pages(cache, &p.pages);
  if (rc != FA_OK) return rc;
  if (budget < 1 || recent < 0 || sinks < 0 || recent > budget || sinks > budget - recent)
    return set_error(FA_ERR_INVALID,
                     "budget must be positive and hold the recent and the first positions");
  if (budget > 0x7fffffffll) return set_error(FA_ERR_INVALID, "size too large");
  const int64_t bh = cache->batch * cache->kv_heads;
  if (cache->batch == 0) return FA_OK;
  if (lengths_out == nullptr || (bh > 0 && workspace == nullptr) ||
      (bh > 0 && p.pages.slots() > 0 && (weights == nullptr || positions == nullptr || weights_out == nullptr ||
                               positions_out == nullptr || cache->v_pages == nullptr)))
    return set_error(FA_ERR_INVALID, "null pointer");
  if ((weights == weights_out && weights != nullptr) || (positions == positions_out && positions != nullptr) ||
      cache->lengths == lengths_out)
    return set_error(FA_ERR_INVALID, "weights, positions and lengths cannot be changed in place");
  if ((reinterpret_cast<uintptr_t>(weights) | reinterpret_cast<uintptr_t>(positions) |
       reinterpret_cast<uintptr_t>(weights_out) | reinterpret_cast<uintptr_t>(positions_out)) & 15)
    return set_error(FA_ERR_INVALID, "weights and positions must be 16-byte aligned");
  if (workspace_bytes < fa_cache_evict_workspace(cache, budget))
    return set_error(FA_ERR_INVALID, "workspace too small");
  if (reinterpret_cast<uintptr_t>(workspace) & 255)
    return set_error(FA_ERR_INVALID, "workspace must be 256-byte aligned");
  fa::host::Device d;
  if ((rc = fa::host::current_device(&d)) != FA_OK) return rc;
  cudaStream_t stream = static_cast<cudaStream_t>(cuda_stream);
  p.pages.status = d.status;
  cudaError_t e;
  if (bh == 0) {
    e = fc::launch_lengths(p.pages, nullptr, 0, static_cast<int>(budget), cache->batch, lengths_out, stream);
    if (e != cudaSuccess) return set_error(FA_ERR_CUDA, "kernel launch: %s", cudaGetErrorString(e));
    return FA_OK;
  }
  p.k_pages = static_cast<uint4*>(cache->k_pages);
  p.v_pages = static_cast<uint4*>(cache->v_pages);
  p.weights = weights;
  p.positions = positions;
  p.weights_out = weights_out;
  p.positions_out = positions_out;
  p.lengths_out = lengths_out;
  p.n_moves = static_cast<int*>(workspace);
  p.max_moves = static_cast<int>(max_moves(cache, budget));
  p.to = reinterpret_cast<int*>(static_cast<uint8_t*>(workspace) + counts_bytes(cache));
  p.from = p.to + bh * p.max_moves;
  p.budget = static_cast<int>(budget);
  p.recent = static_cast<int>(recent);
  p.sinks = static_cast<int>(sinks);
  p.vectors = p.pages.dim / 8;

  // Blocks per (b, h): as many as the SMs have room for, two each, up to the
  // portable cluster size of 8, while each still has four slots per thread.
  int ranks = 1;
  while (ranks < 8 && bh * ranks <= d.sms && p.pages.slots() > ranks * 4 * fc::kSelectThreads) ranks *= 2;
  // a block's slots are its share rounded up to whole steps of its warps
  const int share = (p.pages.slots() + ranks - 1) / ranks;
  p.room = std::min((share + 128 * fc::kWarps + 127) & ~127, fc::kMaxKeys);
  const void* kernel = ranks > 1 ? reinterpret_cast<const void*>(&fc::select_kernel<true>)
                                 : reinterpret_cast<const void*>(&fc::select_kernel<false>);
  static std::atomic<uint64_t> allowed[2];  // zero: static
  e = fa::host::allow_smem(kernel, fc::kMaxKeys * 2 * static_cast<int>(sizeof(int)), d.index,
                                       allowed[ranks > 1 ? 1 : 0]);
  if (e != cudaSuccess) return set_error(FA_ERR_CUDA, "cudaFuncSetAttribute: %s", cudaGetErrorString(e));
  cudaLaunchAttribute attr[1];
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(bh * ranks));
  cfg.blockDim = dim3(fc::kSelectThreads);
  cfg.dynamicSmemBytes = static_cast<size_t>(p.room) * 2 * sizeof(int);
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = ranks > 1 ? 1 : 0;
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(ranks);
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  e = ranks > 1 ? cudaLaunchKernelEx(&cfg, fc::select_kernel<true>, p)
                : cudaLaunchKernelEx(&cfg, fc::select_kernel<false>, p);
  if (e != cudaSuccess) return set_error(FA_ERR_CUDA, "kernel launch: %s", cudaGetErrorString(e));
  if (p.max_moves > 0) {
    const int rows = fc::kMoveThreads / p.vectors;
    const int64_t want = (p.max_moves + rows - 1) / rows;
    const int64_t fill = std::max<int64_t>(1, 32ll * d.sms / bh);
    cfg.gridDim = dim3(static_cast<unsigned>(std::min(want, fill)), static_cast<unsigned>(bh));
    cfg.blockDim = dim3(fc::kMoveThreads);
    cfg.dynamicSmemBytes = 0;
    cfg.numAttrs = 1;
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    e = cudaLaunchKernelEx(&cfg, fc::move_kernel, p);
    if (e != cudaSuccess) return set_error(FA_ERR_CUDA, "kernel launch: %s", cudaGetErrorString(e));
  }
  return FA_OK;
}
