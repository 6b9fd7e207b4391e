// The line of key tiles that the blocks of a tree attention share, and what its
// kernels have in common.
//
// A unit is one (sequence, kv head, tile of rows) with all of its key tiles.
// Units lie one behind the other on a line that is cut into equal parts, one
// per block: however unequal the sequences are, every SM streams the same
// number of bytes, and the plan needs the lengths only on the device.  Where a
// unit is cut, each block leaves the sums of its part, which combine_kernel
// joins in the order of the keys, so results do not depend on timing.
#pragma once

#include <cstdint>

#include "mma_sm80.cuh"
#include "paged_cache.cuh"

namespace fa {
namespace tree {

using namespace warp;

struct Params {
  Pages pages;
  const void* k_pages;
  const void* v_pages;
  Rows q, k_tree, v_tree;
  const unsigned char* mask;  // null: key j <= token
  int64_t mask_batch, mask_row;
  const int* sizes;           // null: tokens
  void* out;
  float* lse;
  float* part_o;   // [2 * blocks][tile rows][dim]
  float2* part_ml; // [2 * blocks][tile rows]: maximum (log2), sum
  int batch, heads, group, tokens;
  int tree;        // the tree has keys of its own
  int rows;        // group * tokens
  int row_tiles;   // of a (sequence, kv head)
  int blocks;      // that share the line
  int tile;        // keys of a tile on the line
  int unit_rows;   // rows that a unit has room for
  int row_threads; // combine_kernel: threads of a row
  int box_rows;    // tile_kernel: rows of a page that one copy brings
  unsigned long long limit_ns;  // of a wait in tile_kernel
  float scale_log2;
};

__device__ __forceinline__ int tree_size(const Params& p, int b) {
  if (p.sizes == nullptr) return p.tokens;
  const int n = p.sizes[b];
  if (n < 0 || n > p.tokens) {
    atomicOr(p.pages.status, kStatusCache);
    return n < 0 ? 0 : p.tokens;
  }
  return n;
}

__device__ __forceinline__ int cache_tiles(const Params& p, int b) {
  return (cache_length(p.pages, b) + p.tile - 1) / p.tile;
}

// Tiles of one unit of sequence b; at least one, so that a unit which sees
// nothing still has its zeros written.
__device__ __forceinline__ int unit_tiles(const Params& p, int b) {
  const int own = p.tree ? (tree_size(p, b) + p.tile - 1) / p.tile : 0;
  const int n = cache_tiles(p, b) + own;
  return n < 1 ? 1 : n;
}

// The line of all tiles: sequence by sequence, unit by unit.
struct Line {
  int64_t per;      // tiles of a block
  int64_t total;
  int b;            // the sequence asked for
  int64_t begin;    // where it begins on the line
};

// Lays out the line with the whole block of kWarps warps; then finds either the
// sequence at which block `at_block` begins, or (at_block < 0) sequence `b`.
template <int kWarps>
__device__ __forceinline__ Line lay_out(const Params& p, int64_t at_block, int b) {
  __shared__ int64_t warp_sum[kWarps];
  __shared__ int64_t found_begin;
  __shared__ int found_b;
  const int lane = threadIdx.x % 32, w = threadIdx.x / 32;
  constexpr int kThreads = 32 * kWarps;
  const int units = p.pages.kv_heads * p.row_tiles;
  const int each = (p.batch + kThreads - 1) / kThreads;
  const int b0 = min(static_cast<int>(threadIdx.x) * each, p.batch), b1 = min(b0 + each, p.batch);
  int64_t mine = 0;
  for (int i = b0; i < b1; ++i) mine += static_cast<int64_t>(unit_tiles(p, i)) * units;
  int64_t incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t u = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += u;
  }
  if (lane == 31) warp_sum[w] = incl;
  __syncthreads();
  Line line;
  int64_t before = incl - mine;
  line.total = 0;
#pragma unroll
  for (int i = 0; i < kWarps; ++i) {
    if (i < w) before += warp_sum[i];
    line.total += warp_sum[i];
  }
  line.per = (line.total + p.blocks - 1) / p.blocks;
  const int64_t at = at_block * line.per;
  if (at_block >= 0 ? (before <= at && at < before + mine) : (b0 <= b && b < b1)) {
    int i = b0;
    while (at_block >= 0 ? at >= before + static_cast<int64_t>(unit_tiles(p, i)) * units : i < b) {
      before += static_cast<int64_t>(unit_tiles(p, i)) * units;
      ++i;
    }
    found_b = i;
    found_begin = before;
  }
  __syncthreads();
  line.b = found_b;
  line.begin = found_begin;
  return line;
}

// Partial or final rows of a unit: row r of the tile, elements [4 i, 4 i + 4).
template <typename T, int kDim>
__device__ __forceinline__ void write_row(const Params& p, int b, int head, int64_t row, bool padding,
                                          int i, float m, float l, float4 o) {
  const bool nothing = padding || l == 0.0f;
  const float inv = nothing ? 0.0f : 1.0f / l;
  if (nothing) o = make_float4(0.f, 0.f, 0.f, 0.f);
  const int64_t at = (static_cast<int64_t>(b) * p.heads + static_cast<int64_t>(head) * p.group) * p.tokens + row;
  uint2 v;
  v.x = pack2<T>(o.x * inv, o.y * inv);
  v.y = pack2<T>(o.z * inv, o.w * inv);
  reinterpret_cast<uint2*>(static_cast<T*>(p.out) + at * kDim)[i] = v;
  if (i == 0) p.lse[at] = nothing ? -INFINITY : 0.69314718055994531f * (m + log2f(l));
}

}  // namespace tree
}  // namespace fa
