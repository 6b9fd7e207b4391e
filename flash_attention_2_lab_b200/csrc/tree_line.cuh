// The line of key tiles that the blocks of a tree attention share, and what its
// kernels have in common.
//
// A unit is one (sequence, kv head, tile of rows) with all of its key tiles.
// Units lie one behind the other on a line that is cut into equal parts, one
// per block: however unequal the sequences are, every SM has the same work, and
// the plan needs the lengths only on the device.  Before its key tiles each unit
// has `extra` places for what beginning one costs a block that has others too.  Where a
// unit is cut, each block leaves the sums of its part, which combine_kernel
// joins in the order of the keys, so results do not depend on timing.
#pragma once

#include <cstdint>

#include "mma_sm80.cuh"
#include "paged_cache.cuh"

namespace fa {
namespace tree {

using namespace warp;

// Division of numbers below 2^31 by a divisor that the host knows (Granlund and
// Montgomery's multiplication by a scaled reciprocal).
struct FastDiv {
  uint32_t by, multiplier, shift;
  FastDiv() = default;
  __host__ explicit FastDiv(uint32_t d) : by(d), multiplier(0), shift(0) {
    while ((1ull << shift) < d) ++shift;
    multiplier = static_cast<uint32_t>(((1ull << 32) * ((1ull << shift) - d)) / d + 1);
  }
  __device__ __forceinline__ int div(int n) const {
    const uint32_t u = static_cast<uint32_t>(n);
    return static_cast<int>((__umulhi(u, multiplier) + u) >> shift);
  }
  __device__ __forceinline__ int mod(int n) const { return n - div(n) * static_cast<int>(by); }
};

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
  float4* part_o;  // [2 * blocks][dim / 4][unit_rows]: lanes of a warp are rows
  float2* part_ml; // [2 * blocks][unit_rows]: maximum (log2), sum
  int batch, heads, group, tokens;
  int tree;        // the tree has keys of its own
  int rows;        // group * tokens
  int row_tiles;   // units of a (sequence, kv head)
  int units;       // of a sequence
  int blocks;      // that share the line
  int tile_shift;  // log2 of the keys of a tile
  int extra;       // places of a unit on the line beyond its tiles
  int unit_rows;   // rows that a unit has room for
  int box_rows;    // tile_kernel: rows of a page that one copy brings
  FastDiv by_tokens, by_page, by_row_tiles, by_blocks;
  unsigned long long limit_ns;  // of a wait in tile_kernel
  int device;      // for the host
  float scale_log2;
};

// What the device says about a sequence.  At least one tile, so that a unit
// which sees nothing still has its zeros written.
struct Sequence {
  int n_cache, n_own;   // cached keys; tokens that are there (queries, tree keys)
  int c_tiles, tiles;   // tiles of cached keys; all tiles of a unit
  int places;           // of a unit on the line
};

__device__ __forceinline__ Sequence look_at(const Params& p, int b) {
  Sequence s;
  s.n_cache = p.pages.lengths[b];
  s.n_own = p.sizes == nullptr ? p.tokens : p.sizes[b];
  if (static_cast<unsigned>(s.n_cache) > static_cast<unsigned>(p.pages.slots()) ||
      static_cast<unsigned>(s.n_own) > static_cast<unsigned>(p.tokens)) {
    atomicOr(p.pages.status, kStatusCache);
    s.n_cache = min(max(s.n_cache, 0), p.pages.slots());
    s.n_own = min(max(s.n_own, 0), p.tokens);
  }
  const int round = (1 << p.tile_shift) - 1;
  s.c_tiles = (s.n_cache + round) >> p.tile_shift;
  s.tiles = max(1, s.c_tiles + (p.tree ? (s.n_own + round) >> p.tile_shift : 0));
  s.places = s.tiles + p.extra;
  return s;
}

// The line of all tiles: sequence by sequence, unit by unit.  The host has
// checked that it is shorter than 2^30.
struct Line {
  int per;       // places of a block
  int total;
  int b;         // the sequence asked for; < 0: the line ends before
  int begin;     // where it begins on the line
  Sequence seq;
};

// Laid out by each warp for itself (all lanes together): no barrier, one trip
// to memory.  Finds the sequence at which block `at_block` begins, or
// (at_block < 0) sequence `b`.
__device__ __forceinline__ Line lay_out(const Params& p, int at_block, int b) {
  const int lane = threadIdx.x % 32;
  const int each = (p.batch + 31) / 32;
  const int b0 = min(lane * each, p.batch), b1 = min(b0 + each, p.batch);
  Sequence s = {};
  int mine = 0;
  for (int i = b0; i < b1; ++i) {
    s = look_at(p, i);
    mine += s.places * p.units;
  }
  int incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += u;
  }
  Line line;
  line.total = __shfl_sync(0xffffffffu, incl, 31);
  line.per = p.by_blocks.div(line.total + p.blocks - 1);
  int begin = incl - mine;
  const int at = at_block * line.per;
  const bool hit = at_block >= 0 ? (begin <= at && at < incl) : (b0 <= b && b < b1);
  const unsigned int who = __ballot_sync(0xffffffffu, hit);
  int i = b0;
  if (hit && each > 1) {
    s = look_at(p, i);
    while (at_block >= 0 ? at >= begin + s.places * p.units : i < b) {
      begin += s.places * p.units;
      s = look_at(p, ++i);
    }
  }
  __syncwarp();
  const int from = who == 0 ? 0 : __ffs(who) - 1;
  line.b = who == 0 ? -1 : __shfl_sync(0xffffffffu, i, from);
  line.begin = __shfl_sync(0xffffffffu, begin, from);
  line.seq.n_cache = __shfl_sync(0xffffffffu, s.n_cache, from);
  line.seq.n_own = __shfl_sync(0xffffffffu, s.n_own, from);
  line.seq.c_tiles = __shfl_sync(0xffffffffu, s.c_tiles, from);
  line.seq.tiles = __shfl_sync(0xffffffffu, s.tiles, from);
  line.seq.places = line.seq.tiles + p.extra;
  return line;
}

// One part of a unit: key tiles [tile0, tile0 + n) for the rows from row0 on.
struct Segment {
  int b, head, row0;
  int tile0, n;
  int n_cache, c_tiles, n_own;  // of the sequence
  int part;                     // its place among the parts
  bool whole;                   // the unit has no other
};

// Walks the parts of a block.
struct Walk {
  int at, end, off, b;  // places; off: within sequence b
  Sequence seq;

  __device__ __forceinline__ Walk(const Params& p, const Line& line) {
    at = static_cast<int>(blockIdx.x) * line.per;
    end = min(at + line.per, line.total);
    off = at - line.begin;
    b = line.b;
    seq = line.seq;
  }
  __device__ __forceinline__ bool next(const Params& p, Segment& s) {
    while (at < end) {
      if (off == seq.places * p.units) {
        seq = look_at(p, ++b);
        off = 0;
      }
      const int unit = off / seq.places;
      const int place = off - unit * seq.places;
      const int n = min(seq.places - place, end - at);  // places of the unit that are the block's
      at += n;
      off += n;
      s.tile0 = max(place - p.extra, 0);
      s.n = place + n - p.extra - s.tile0;
      if (s.n <= 0) continue;  // nothing but the unit's beginning
      s.b = b;
      s.n_cache = seq.n_cache;
      s.c_tiles = seq.c_tiles;
      s.n_own = seq.n_own;
      s.head = p.by_row_tiles.div(unit);
      s.row0 = (unit - s.head * p.row_tiles) * p.unit_rows;
      s.whole = s.n == seq.tiles;
      // of a block's parts one at most begins within a unit, and one ends there
      s.part = 2 * static_cast<int>(blockIdx.x) + (s.tile0 == 0 ? 1 : 0);
      return true;
    }
    return false;
  }
};

// Final rows: row `row` of (b, head), elements [4 i, 4 i + 4), sums o and l over
// exponentials against m (log2).
template <typename T, int kDim>
__device__ __forceinline__ void write_row(const Params& p, int b, int head, int row, int n_own, int i, float m,
                                          float l, float4 o) {
  const bool nothing = l == 0.0f || p.by_tokens.mod(row) >= n_own;
  const float inv = 1.0f / l;
  const int64_t at = (static_cast<int64_t>(b) * p.heads + static_cast<int64_t>(head) * p.group) * p.tokens + row;
  const uint2 v = nothing ? make_uint2(0u, 0u) : make_uint2(pack2<T>(o.x * inv, o.y * inv), pack2<T>(o.z * inv, o.w * inv));
  reinterpret_cast<uint2*>(static_cast<T*>(p.out) + at * kDim)[i] = v;
  if (i == 0) p.lse[at] = nothing ? -INFINITY : 0.69314718055994531f * (m + log2f(l));
}

}  // namespace tree
}  // namespace fa
