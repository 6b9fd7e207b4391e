// Changes of a paged key/value cache on B200 (sm_100a): rows appended, and
// slots evicted by the attention weight that they gathered.

#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>

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
// and by its launch when short.  One 16-byte vector of K and one of V per
// thread; the eight or sixteen threads of a row are neighbours.

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
  if (i >= p.rows) return;
  const int slots = p.pages.slots();
  const int length = cache_length(p.pages, b);
  int count = p.counts == nullptr ? p.rows : p.counts[b];
  if (count < 0 || count > p.rows || count > slots - length) {
    atomicOr(p.pages.status, kStatusCache);
    count = max(0, min(min(count, p.rows), slots - length));
  }
  if (i == 0 && h == 0 && vec == 0) p.lengths_out[b] = length + count;
  if (i >= count) return;
  int from = i;
  if (p.path != nullptr) {
    from = p.path[static_cast<int64_t>(b) * p.rows + i];
    if (static_cast<unsigned>(from) >= static_cast<unsigned>(p.rows)) {
      atomicOr(p.pages.status, kStatusCache);
      return;
    }
  }
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
// weights' bits in an order-preserving form, one cluster of blocks per (b, h),
// each block on a contiguous part of the slots; histograms and prefix counts
// cross the cluster through distributed shared memory.  It is bound by the
// latency of its passes and barriers.  move_kernel then copies rows, bound by
// HBM.

constexpr int kSelectThreads = 1024;
constexpr int kWarps = kSelectThreads / 32;
constexpr int kBins = 2048;
constexpr int kMoveThreads = 256;
constexpr int kMaxKeys = 48 * 1024;  // keys in a block's shared memory

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
  int2* moves;           // [batch * kv_heads][max_moves]: (to, from)
  int max_moves;
  int budget, recent, sinks;
  int key_room;          // keys that fit into a block's shared memory
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
  const int v = scratch[lane];
  int s = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, s, o);
    if (lane >= o) s += u;
  }
  *total = __shfl_sync(0xffffffffu, s, 31);
  return __shfl_sync(0xffffffffu, s - v, warp);
}

__global__ void __launch_bounds__(kSelectThreads) select_kernel(const EvictParams p) {
  extern __shared__ uint32_t keys[];
  __shared__ int hist[3][kBins];
  __shared__ int scratch[kWarps];
  __shared__ int shared_max, found_bin, found_above, block_holes, block_movers;
  static_assert(kWarps == 32, "one warp scans the warps' values");

  cg::cluster_group cluster = cg::this_cluster();
  const int rank = static_cast<int>(cluster.block_rank());
  const int ranks = static_cast<int>(cluster.num_blocks());
  const int bh = static_cast<int>(blockIdx.x) / ranks;
  const int b = bh / p.pages.kv_heads;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const uint32_t below = (1u << lane) - 1u;
  const int slots = p.pages.slots();
  const int n = cache_length(p.pages, b);
  const int64_t base = static_cast<int64_t>(bh) * slots;
  const float* w = p.weights + base;
  const int* pos = p.positions + base;
  const int n_new = min(n, p.budget);
  if (threadIdx.x == 0 && rank == 0 && bh % p.pages.kv_heads == 0) p.lengths_out[b] = n_new;

  // slots behind the new length are empty
  for (int i = n_new + rank * kSelectThreads + static_cast<int>(threadIdx.x); i < slots;
       i += ranks * kSelectThreads) {
    p.weights_out[base + i] = 0.0f;
    p.positions_out[base + i] = -1;
  }
  if (n <= p.budget) {  // the same in every block of the cluster
    for (int i = rank * kSelectThreads + static_cast<int>(threadIdx.x); i < n;
         i += ranks * kSelectThreads) {
      p.weights_out[base + i] = w[i];
      p.positions_out[base + i] = pos[i];
    }
    if (threadIdx.x == 0 && rank == 0) p.n_moves[bh] = 0;
    return;
  }

  // this warp's slots: [s0, s1), steps of 32
  const int per_rank = (n + ranks - 1) / ranks;
  const int seg = ((per_rank + kWarps - 1) / kWarps + 31) & ~31;
  const int64_t first = (static_cast<int64_t>(rank) * kWarps + warp) * seg;
  const int s0 = static_cast<int>(first < n ? first : n);
  const int s1 = static_cast<int>(first + seg < n ? first + seg : n);
  const int key0 = rank * kWarps * seg;  // slot of keys[0]
  const bool in_shared = kWarps * seg <= p.key_room;

  // the last position
  for (int i = threadIdx.x; i < 3 * kBins; i += kSelectThreads) (&hist[0][0])[i] = 0;
  if (threadIdx.x == 0) shared_max = INT32_MIN;
  __syncthreads();
  int top = INT32_MIN;
  for (int i = s0 + lane; i < s1; i += 32) top = max(top, pos[i]);
  top = __reduce_max_sync(0xffffffffu, top);
  if (lane == 0) atomicMax(&shared_max, top);
  cluster.sync();
  top = INT32_MIN;
  for (int r = 0; r < ranks; ++r) top = max(top, *cluster.map_shared_rank(&shared_max, r));
  const int64_t recent_from = static_cast<int64_t>(top) - p.recent;

  auto key_of = [&](int i) -> uint32_t {
    const int at = pos[i];
    return (at > recent_from || at < p.sinks) ? 0xffffffffu : weight_key(w[i]);
  };
  auto key_at = [&](int i) -> uint32_t { return in_shared ? keys[i - key0] : key_of(i); };

  // the budget-th largest key, digit by digit from the top
  uint32_t threshold = 0;
  int need = p.budget;
#pragma unroll 1
  for (int d = 0; d < 3; ++d) {
    const int shift = d == 0 ? 21 : d == 1 ? 10 : 0;
    const uint32_t mask = d == 2 ? 1023u : 2047u;
    const int above_shift = d == 1 ? 21 : 10;
    for (int i0 = s0; i0 < s1; i0 += 32) {
      const int i = i0 + lane;
      int digit = -1;
      if (i < s1) {
        const uint32_t k = d == 0 ? key_of(i) : key_at(i);
        if (d == 0 && in_shared) keys[i - key0] = k;
        if (d == 0 || (k >> above_shift) == (threshold >> above_shift))
          digit = static_cast<int>((k >> shift) & mask);
      }
      // equal digits of a warp (protected slots, zero weights) add up first
      const uint32_t same = __match_any_sync(0xffffffffu, digit);
      if (digit >= 0 && (same & below) == 0) atomicAdd(&hist[d][digit], __popc(same));
    }
    cluster.sync();
    // bins from the top, two per thread
    int c[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int bin = kBins - 1 - (2 * static_cast<int>(threadIdx.x) + j);
      c[j] = 0;
      for (int r = 0; r < ranks; ++r) c[j] += *cluster.map_shared_rank(&hist[d][bin], r);
    }
    int sum = c[0] + c[1], incl = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += u;
    }
    int total;
    const int before = warps_prefix(__shfl_sync(0xffffffffu, incl, 31), scratch, &total);
    int above = before + incl - sum;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      if (above < need && need <= above + c[j]) {
        found_bin = kBins - 1 - (2 * static_cast<int>(threadIdx.x) + j);
        found_above = above;
      }
      above += c[j];
    }
    __syncthreads();
    threshold |= static_cast<uint32_t>(found_bin) << shift;
    need -= found_above;
    __syncthreads();
  }

  // of the slots equal to the threshold the first `need` stay
  const int last_digit = static_cast<int>(threshold & 1023u);
  int equal_before = 0;
  for (int r = 0; r < rank; ++r) equal_before += *cluster.map_shared_rank(&hist[2][last_digit], r);
  int mine = 0, total;
  for (int i0 = s0; i0 < s1; i0 += 32) {
    const int i = i0 + lane;
    mine += __popc(__ballot_sync(0xffffffffu, i < s1 && key_at(i) == threshold));
  }
  equal_before += warps_prefix(mine, scratch, &total);

  // holes (dropped, before the budget) and movers (kept, behind it)
  auto walk = [&](auto&& visit) {
    int eq = equal_before;
    for (int i0 = s0; i0 < s1; i0 += 32) {
      const int i = i0 + lane;
      const bool valid = i < s1;
      const uint32_t k = valid ? key_at(i) : 0u;
      const uint32_t ties = __ballot_sync(0xffffffffu, valid && k == threshold);
      const bool kept = valid && (k > threshold || (k == threshold && eq + __popc(ties & below) < need));
      eq += __popc(ties);
      visit(i, valid, kept);
    }
  };
  int holes = 0, movers = 0;
  walk([&](int i, bool valid, bool kept) {
    holes += __popc(__ballot_sync(0xffffffffu, valid && !kept && i < p.budget));
    movers += __popc(__ballot_sync(0xffffffffu, kept && i >= p.budget));
  });
  int all_holes, all_movers;
  int hole_at = warps_prefix(holes, scratch, &all_holes);
  int mover_at = warps_prefix(movers, scratch, &all_movers);
  if (threadIdx.x == 0) {
    block_holes = all_holes;
    block_movers = all_movers;
  }
  cluster.sync();
  int moves = 0;
  for (int r = 0; r < ranks; ++r) {
    const int hr = *cluster.map_shared_rank(&block_holes, r);
    if (r < rank) {
      hole_at += hr;
      mover_at += *cluster.map_shared_rank(&block_movers, r);
    }
    moves += hr;
  }
  if (threadIdx.x == 0 && rank == 0) p.n_moves[bh] = moves;
  int2* list = p.moves + static_cast<int64_t>(bh) * p.max_moves;
  walk([&](int i, bool valid, bool kept) {
    const bool hole = valid && !kept && i < p.budget, mover = kept && i >= p.budget;
    const uint32_t hb = __ballot_sync(0xffffffffu, hole), mb = __ballot_sync(0xffffffffu, mover);
    if (hole) list[hole_at + __popc(hb & below)].x = i;
    if (mover) list[mover_at + __popc(mb & below)].y = i;
    hole_at += __popc(hb);
    mover_at += __popc(mb);
    if (kept && i < p.budget) {
      p.weights_out[base + i] = w[i];
      p.positions_out[base + i] = pos[i];
    }
  });
  cluster.sync();  // no block leaves while another still reads its shared memory
}

__global__ void __launch_bounds__(kMoveThreads) move_kernel(const EvictParams p) {
  const int bh = static_cast<int>(blockIdx.y);
  const int b = bh / p.pages.kv_heads, h = bh - b * p.pages.kv_heads;
  const int n = p.n_moves[bh];
  const int rows = kMoveThreads / p.vectors;  // of a block and step
  const int row = static_cast<int>(threadIdx.x) / p.vectors;
  const int vec = static_cast<int>(threadIdx.x) - row * p.vectors;
  const int64_t base = static_cast<int64_t>(bh) * p.pages.slots();
  for (int m = static_cast<int>(blockIdx.x) * rows + row; m < n; m += static_cast<int>(gridDim.x) * rows) {
    const int2 move = p.moves[static_cast<int64_t>(bh) * p.max_moves + m];
    if (vec == 0) {
      p.weights_out[base + move.x] = p.weights[base + move.y];
      p.positions_out[base + move.x] = p.positions[base + move.y];
    }
    const int64_t to = cache_row(p.pages, b, h, move.x), from = cache_row(p.pages, b, h, move.y);
    if (to < 0 || from < 0) continue;
    const uint4 k = p.k_pages[from / 8 + vec], v = p.v_pages[from / 8 + vec];
    p.k_pages[to / 8 + vec] = k;
    p.v_pages[to / 8 + vec] = v;
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
  if (cache->batch == 0 || cache->kv_heads == 0) return FA_OK;
  if (lengths_out == nullptr || (positions != nullptr && rows > 0 && new_positions == nullptr))
    return set_error(FA_ERR_INVALID, "null pointer");
  if (cache->lengths == lengths_out)
    return set_error(FA_ERR_INVALID, "lengths cannot be changed in place");
  cudaStream_t stream = static_cast<cudaStream_t>(cuda_stream);
  fa::host::Device d;
  if (rows == 0) {
    if ((rc = fa::host::current_device(&d)) != FA_OK) return rc;
    const cudaError_t e = cudaMemcpyAsync(lengths_out, cache->lengths, cache->batch * sizeof(int),
                                          cudaMemcpyDeviceToDevice, stream);
    if (e != cudaSuccess) return set_error(FA_ERR_CUDA, "lengths copy: %s", cudaGetErrorString(e));
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
         cache->batch * cache->kv_heads * max_moves(cache, budget) * static_cast<int64_t>(sizeof(int2));
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
  if (bh == 0) return FA_OK;
  if (lengths_out == nullptr || workspace == nullptr ||
      (p.pages.slots() > 0 && (weights == nullptr || positions == nullptr || weights_out == nullptr ||
                               positions_out == nullptr || cache->v_pages == nullptr)))
    return set_error(FA_ERR_INVALID, "null pointer");
  if (weights == weights_out || positions == positions_out || cache->lengths == lengths_out)
    return set_error(FA_ERR_INVALID, "weights, positions and lengths cannot be changed in place");
  if (workspace_bytes < fa_cache_evict_workspace(cache, budget))
    return set_error(FA_ERR_INVALID, "workspace too small");
  if (reinterpret_cast<uintptr_t>(workspace) & 255)
    return set_error(FA_ERR_INVALID, "workspace must be 256-byte aligned");
  fa::host::Device d;
  if ((rc = fa::host::current_device(&d)) != FA_OK) return rc;
  cudaStream_t stream = static_cast<cudaStream_t>(cuda_stream);
  p.pages.status = d.status;
  p.k_pages = static_cast<uint4*>(cache->k_pages);
  p.v_pages = static_cast<uint4*>(cache->v_pages);
  p.weights = weights;
  p.positions = positions;
  p.weights_out = weights_out;
  p.positions_out = positions_out;
  p.lengths_out = lengths_out;
  p.n_moves = static_cast<int*>(workspace);
  p.moves = reinterpret_cast<int2*>(static_cast<uint8_t*>(workspace) + counts_bytes(cache));
  p.max_moves = static_cast<int>(max_moves(cache, budget));
  p.budget = static_cast<int>(budget);
  p.recent = static_cast<int>(recent);
  p.sinks = static_cast<int>(sinks);
  p.vectors = p.pages.dim / 8;

  // Blocks per (b, h): as many as the SMs have room for, up to the portable
  // cluster size of 8, while each still has two slots per thread to look at.
  int ranks = 1;
  while (ranks < 8 && bh * ranks * 2 <= d.sms && p.pages.slots() > ranks * 2 * fc::kSelectThreads)
    ranks *= 2;
  const int per_block = ((p.pages.slots() + ranks - 1) / ranks + fc::kSelectThreads) & ~31;
  p.key_room = std::min(per_block + fc::kSelectThreads, fc::kMaxKeys);
  const int smem = p.key_room * static_cast<int>(sizeof(uint32_t));
  cudaError_t e = cudaFuncSetAttribute(reinterpret_cast<const void*>(&fc::select_kernel),
                                       cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       fc::kMaxKeys * static_cast<int>(sizeof(uint32_t)));
  if (e != cudaSuccess) return set_error(FA_ERR_CUDA, "cudaFuncSetAttribute: %s", cudaGetErrorString(e));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(bh * ranks));
  cfg.blockDim = dim3(fc::kSelectThreads);
  cfg.dynamicSmemBytes = static_cast<size_t>(smem);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(ranks);
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  e = cudaLaunchKernelEx(&cfg, fc::select_kernel, p);
  if (e != cudaSuccess) return set_error(FA_ERR_CUDA, "kernel launch: %s", cudaGetErrorString(e));
  if (p.max_moves > 0) {
    const int rows = fc::kMoveThreads / p.vectors;
    const int64_t want = (p.max_moves + rows - 1) / rows;
    const int64_t fill = std::max<int64_t>(1, 8ll * d.sms / bh);
    fc::move_kernel<<<dim3(static_cast<unsigned>(std::min(want, fill)), static_cast<unsigned>(bh)),
                      fc::kMoveThreads, 0, stream>>>(p);
    e = cudaGetLastError();
    if (e != cudaSuccess) return set_error(FA_ERR_CUDA, "kernel launch: %s", cudaGetErrorString(e));
  }
  return FA_OK;
}
