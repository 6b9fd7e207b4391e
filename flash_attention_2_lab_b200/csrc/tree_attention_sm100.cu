// Attention for a tree of drafted tokens over a paged cache, B200 (sm_100a).
//
// Query t of a sequence sees all of its cached keys and, of the tree's own
// keys, those that the tree mask shows (its ancestors and itself).  The rows of
// one (sequence, kv head) are the `group` query heads that share the kv head
// times the tokens, row = head_in_group * tokens + token: K and V are read
// once for all of them.
//
// rows_kernel: bound by HBM (2 * 2 * dim bytes per cached key and kv head).
// The key ranges of all (sequence, kv head, row tile) units, in tiles of 64
// keys, form one line that is cut into equal parts, one per block: however
// unequal the sequences are, every SM streams the same number of bytes, and
// the plan needs the lengths only on the device.  A block walks its part;
// where a unit is cut, it leaves partial sums that combine_kernel joins in
// order of the keys, so results do not depend on timing.  Within a block each
// warp takes 16 keys of every tile with an online softmax of its own, fed by
// its own ring of asynchronous copies: no barrier among warps until the unit
// ends.  The sums are fp32; P is rounded to the type of V for the product, whose
// operands are of one type, and added to the row's sum unrounded.

#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstdint>
#include <utility>

#include "fa_host.h"
#include "fa_sm100.h"
#include "mma_sm80.cuh"
#include "paged_cache.cuh"
#include "sm100_ptx.cuh"
#include "tree_line.cuh"
#include "tree_tiles_sm100.cuh"

namespace fa {
namespace tree {

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr int kStep = 16;             // keys of a warp's step; pages hold whole steps
constexpr int kRowsTile = kStep * kWarps;  // keys of a block's step

template <int kDim, int kMt>
struct Shape {
  static constexpr int kRows = 16 * kMt;                // rows of a unit
  static constexpr int kStepBytes = kStep * kDim * 2;   // K or V of a step
  static constexpr int kStages = kDim == 64 ? 3 : 2;
  static constexpr int kWarpBytes = kStages * 2 * kStepBytes;
  static constexpr int kSmem = kWarps * kWarpBytes;
  static constexpr int kMergeStride = kDim + 4;         // floats
  static_assert(kRows * kMergeStride * 4 <= kWarpBytes, "the merge reuses the ring");
  static_assert(16 * kStep * 4 <= kStepBytes, "P of a row tile fits a consumed K");
};

// Blocks of an SM, by registers (128 a thread at dimension 64 with 16 rows, 168 at
// 128) and rings of 48 or 64 KiB.  More warps are worth more than longer rings
// (times of variants beside one another; a call of the first takes 146 us, 135 in a
// graph): 32 sequences of 8192 to 16384 keys took 128 us with 4 blocks and 3 steps a ring, 136
// with 3 and 4, 171 with 2 and 6; at dimension 128 64 of 256 to 512 keys 28 us with
// 3 and 2, 30 with 2 and 3, 47 with 4 and 2, whose registers spill.
template <int kDim, int kMt>
constexpr int kResident = kDim == 128 ? 3 : kMt == 1 ? 4 : 2;

template <typename T, int kDim, int kMt>
__global__ void __launch_bounds__(kThreads, kResident<kDim, kMt>) rows_kernel(const Params p) {
  using S = Shape<kDim, kMt>;
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ int step_keys[kWarps][S::kStages];
  __shared__ float2 merge_ml[kWarps][S::kRows];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  const int lane = threadIdx.x % 32, w = threadIdx.x / 32;
  const int g = lane / 4, q4 = lane % 4;
  const uint32_t ring = ptx::smem_u32(smem) + w * S::kWarpBytes;
  // ldmatrix rows: K as [key][d], two key groups x two d groups; V transposed
  const int k_row = (lane & 7) + ((lane >> 4) << 3), k_vec = (lane >> 3) & 1;
  const int v_row = (lane & 7) + (((lane >> 3) & 1) << 3), v_vec = lane >> 4;

  Walk walk(p, lay_out(p, static_cast<int>(blockIdx.x), 0));
  Segment seg;
  while (walk.next(p, seg)) {
    const int b = seg.b, head = seg.head, row0 = seg.row0;
    const int n_cache = seg.n_cache, c_tiles = seg.c_tiles, n_own = seg.n_own;
    const int tile0 = seg.tile0, tile1 = seg.tile0 + seg.n;

    // K and V of a step, 16 bytes per lane and copy; rows without a key are zeros
    auto load = [&](int tile, int stage) {
      const T *k, *v;
      int64_t k_row_stride, v_row_stride;
      int keys;
      if (tile < c_tiles) {
        const int slot = tile * kRowsTile + w * kStep;
        keys = min(max(n_cache - slot, 0), kStep);
        const int64_t row = keys > 0 ? cache_row(p.pages, b, head, slot) : -1;
        if (row < 0) keys = 0;
        k = static_cast<const T*>(p.k_pages) + (row < 0 ? 0 : row);
        v = static_cast<const T*>(p.v_pages) + (row < 0 ? 0 : row);
        k_row_stride = v_row_stride = kDim;
      } else {
        const int j = (tile - c_tiles) * kRowsTile + w * kStep;
        keys = p.tree ? min(max(n_own - j, 0), kStep) : 0;
        const int from = keys > 0 ? j : 0;
        k = static_cast<const T*>(p.k_tree.data) + b * p.k_tree.batch + head * p.k_tree.head + from * p.k_tree.row;
        v = static_cast<const T*>(p.v_tree.data) + b * p.v_tree.batch + head * p.v_tree.head + from * p.v_tree.row;
        k_row_stride = p.k_tree.row;
        v_row_stride = p.v_tree.row;
      }
      const uint32_t dst = ring + stage * 2 * S::kStepBytes;
      constexpr int kVecs = kDim / 8;
      if (keys > 0) {
#pragma unroll
        for (int i = 0; i < kStep * kVecs / 32; ++i) {
          const int r = (i * 32 + lane) / kVecs, vec = (i * 32 + lane) % kVecs;
          const bool valid = r < keys;
          const int from = valid ? r : 0;
          copy16(dst + tile_at<kDim>(r, vec), k + from * k_row_stride + vec * 8, valid);
          copy16(dst + S::kStepBytes + tile_at<kDim>(r, vec), v + from * v_row_stride + vec * 8, valid);
        }
      }
      if (lane == 0) step_keys[w][stage] = keys;
    };

#pragma unroll
    for (int s = 0; s < S::kStages - 1; ++s) {
      if (tile0 + s < tile1) load(tile0 + s, s);
      copy_commit();
    }

    // Q of the unit in the A layout of the product
    uint32_t q[kMt][kDim / 16][4];
#pragma unroll
    for (int mi = 0; mi < kMt; ++mi) {
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int row = row0 + mi * 16 + half * 8 + g;
        const int hg = p.by_tokens.div(row), t = row - hg * p.tokens;
        const bool valid = row < p.rows && t < n_own;
        const T* src = static_cast<const T*>(p.q.data) + b * p.q.batch +
                       (static_cast<int64_t>(head) * p.group + (valid ? hg : 0)) * p.q.head +
                       (valid ? t : 0) * p.q.row;
#pragma unroll
        for (int kk = 0; kk < kDim / 16; ++kk) {
          const uint32_t* s32 = reinterpret_cast<const uint32_t*>(src + kk * 16);
          q[mi][kk][half] = valid ? s32[q4] : 0u;
          q[mi][kk][2 + half] = valid ? s32[q4 + 4] : 0u;
        }
      }
    }

    float o[kMt][kDim / 8][4];
    float m[kMt][2], l[kMt][2];
#pragma unroll
    for (int mi = 0; mi < kMt; ++mi) {
#pragma unroll
      for (int n = 0; n < kDim / 8; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[mi][n][e] = 0.0f;
      m[mi][0] = m[mi][1] = -INFINITY;
      l[mi][0] = l[mi][1] = 0.0f;
    }

    // whether row r of the tile sees tree key j < n_own
    auto sees = [&](int r, int j) {
      const int row = row0 + r;
      if (row >= p.rows) return false;
      const int t = p.by_tokens.mod(row);
      return p.mask == nullptr ? j <= t : p.mask[b * p.mask_batch + t * p.mask_row + j] != 0;
    };

    int stage = 0;
    for (int tile = tile0; tile < tile1; ++tile) {
      copy_wait<S::kStages - 2>();
      __syncwarp();
      const int keys = step_keys[w][stage];
      const int ahead = tile + S::kStages - 1;
      if (ahead < tile1) load(ahead, stage == 0 ? S::kStages - 1 : stage - 1);
      copy_commit();
      if (keys > 0) {
        const uint32_t k_at = ring + stage * 2 * S::kStepBytes, v_at = k_at + S::kStepBytes;
        float s[kMt][2][4];
#pragma unroll
        for (int mi = 0; mi < kMt; ++mi)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[mi][0][e] = s[mi][1][e] = 0.0f;
#pragma unroll
        for (int kk = 0; kk < kDim / 16; ++kk) {
          uint32_t kb[4];
          ldmatrix4(kb, k_at + tile_at<kDim>(k_row, kk * 2 + k_vec));
#pragma unroll
          for (int mi = 0; mi < kMt; ++mi) {
            mma<T>(s[mi][0], q[mi][kk], kb[0], kb[1]);
            mma<T>(s[mi][1], q[mi][kk], kb[2], kb[3]);
          }
        }
        const bool own = tile >= c_tiles;
        const int j0 = (tile - c_tiles) * kRowsTile + w * kStep;
        if (own || keys < kStep) {
#pragma unroll
          for (int mi = 0; mi < kMt; ++mi)
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const int c = n * 8 + q4 * 2 + (e & 1), r = mi * 16 + g + (e >> 1) * 8;
                if (c >= keys || (own && !sees(r, j0 + c))) s[mi][n][e] = -INFINITY;
              }
        }
        uint32_t pa[kMt][4];
#pragma unroll
        for (int mi = 0; mi < kMt; ++mi) {
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            float top = fmaxf(fmaxf(s[mi][0][2 * half], s[mi][0][2 * half + 1]),
                              fmaxf(s[mi][1][2 * half], s[mi][1][2 * half + 1]));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            const float now = fmaxf(m[mi][half], top * p.scale_log2);
            const float ref = now == -INFINITY ? 0.0f : now;
            if (now != m[mi][half]) {
              const float shrink = ptx::ex2_approx(m[mi][half] - ref);
              m[mi][half] = now;
              l[mi][half] *= shrink;
#pragma unroll
              for (int n = 0; n < kDim / 8; ++n) {
                o[mi][n][2 * half] *= shrink;
                o[mi][n][2 * half + 1] *= shrink;
              }
            }
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                float& x = s[mi][n][2 * half + e];
                x = ptx::ex2_approx(fmaf(x, p.scale_log2, -ref));
                l[mi][half] += x;
              }
          }
          pa[mi][0] = pack2<T>(s[mi][0][0], s[mi][0][1]);
          pa[mi][1] = pack2<T>(s[mi][0][2], s[mi][0][3]);
          pa[mi][2] = pack2<T>(s[mi][1][0], s[mi][1][1]);
          pa[mi][3] = pack2<T>(s[mi][1][2], s[mi][1][3]);
        }
        // A tree value that is infinite or NaN must not reach the rows that do
        // not see it, as 0 * inf would: such a step is summed key by key.
        bool odd = false;
        if (own) {
          for (int i = lane; i < S::kStepBytes / 4; i += 32) {
            uint32_t v;
            asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(v_at + i * 4));
            odd = odd || not_finite2<T>(v);
          }
        }
        if (own && __any_sync(0xffffffffu, odd)) {
          float* pw = reinterpret_cast<float*>(smem + (k_at - ptx::smem_u32(smem)));
          const unsigned char* vw = smem + (v_at - ptx::smem_u32(smem));
          __syncwarp();  // K of the step has been read by every lane
          // P of one row tile at a time lies in K's place
#pragma unroll
          for (int mi = 0; mi < kMt; ++mi) {
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
              for (int e = 0; e < 4; ++e)
                pw[(g + (e >> 1) * 8) * kStep + n * 8 + q4 * 2 + (e & 1)] = s[mi][n][e];
            __syncwarp();
#pragma unroll 1
            for (int c = 0; c < keys; ++c) {
#pragma unroll
              for (int half = 0; half < 2; ++half) {
                if (!sees(mi * 16 + g + half * 8, j0 + c)) continue;
                const float pc = pw[(g + half * 8) * kStep + c];
#pragma unroll
                for (int n = 0; n < kDim / 8; ++n) {
                  const float2 v = unpack2<T>(
                      reinterpret_cast<const uint32_t*>(vw + tile_at<kDim>(c, n))[q4]);
                  o[mi][n][2 * half] = fmaf(pc, v.x, o[mi][n][2 * half]);
                  o[mi][n][2 * half + 1] = fmaf(pc, v.y, o[mi][n][2 * half + 1]);
                }
              }
            }
            __syncwarp();
          }
        } else {
#pragma unroll
          for (int n = 0; n < kDim / 16; ++n) {
            uint32_t vb[4];
            ldmatrix4_trans(vb, v_at + tile_at<kDim>(v_row, n * 2 + v_vec));
#pragma unroll
            for (int mi = 0; mi < kMt; ++mi) {
              mma<T>(o[mi][2 * n], pa[mi], vb[0], vb[1]);
              mma<T>(o[mi][2 * n + 1], pa[mi], vb[2], vb[3]);
            }
          }
        }
      }
      stage = stage + 1 == S::kStages ? 0 : stage + 1;
    }

    // join the warps: rows of fp32 sums in the ring's memory
    copy_wait<0>();
    __syncthreads();
    float* mine = reinterpret_cast<float*>(smem + w * S::kWarpBytes);
#pragma unroll
    for (int mi = 0; mi < kMt; ++mi) {
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        float sum = l[mi][half];
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        const int r = mi * 16 + half * 8 + g;
        if (q4 == 0) merge_ml[w][r] = make_float2(m[mi][half], sum);
#pragma unroll
        for (int n = 0; n < kDim / 8; ++n)
          *reinterpret_cast<float2*>(mine + r * S::kMergeStride + n * 8 + q4 * 2) =
              make_float2(o[mi][n][2 * half], o[mi][n][2 * half + 1]);
      }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < S::kRows * kDim / 4; i += kThreads) {
      // a final row is written along its elements, a part's along the rows
      const int r = seg.whole ? i / (kDim / 4) : i % S::kRows;
      const int vec = seg.whole ? i % (kDim / 4) : i / S::kRows;
      const int row = row0 + r;
      if (row >= p.rows) continue;
      float top = -INFINITY, sum = 0.0f;
#pragma unroll
      for (int k = 0; k < kWarps; ++k) top = fmaxf(top, merge_ml[k][r].x);
      const float ref = top == -INFINITY ? 0.0f : top;
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int k = 0; k < kWarps; ++k) {
        const float f = ptx::ex2_approx(merge_ml[k][r].x - ref);
        sum += f * merge_ml[k][r].y;
        const float4 v = *reinterpret_cast<const float4*>(
            reinterpret_cast<const float*>(smem + k * S::kWarpBytes) + r * S::kMergeStride + vec * 4);
        acc.x = fmaf(f, v.x, acc.x);
        acc.y = fmaf(f, v.y, acc.y);
        acc.z = fmaf(f, v.z, acc.z);
        acc.w = fmaf(f, v.w, acc.w);
      }
      if (seg.whole) {
        write_row<T, kDim>(p, b, head, row, n_own, vec, top, sum, acc);
      } else {
        p.part_o[(static_cast<int64_t>(seg.part) * (kDim / 4) + vec) * S::kRows + r] = acc;
        if (vec == 0) p.part_ml[static_cast<int64_t>(seg.part) * S::kRows + r] = make_float2(top, sum);
      }
    }
    __syncthreads();
  }
}

// Joins the parts of the units that lie in more than one block.  Lanes are rows
// (32 of a unit, or its 16 twice), and each takes kVecs vectors of four elements.
//   kSplit: units of many parts; the block's eight warps take every eighth part
//           of the same vectors and their sums are joined at the end: a few
//           trips to memory however many the parts are.
//   kUnits: units of few parts; the warps take vectors of their own, all parts.
//   kCuts:  the same where the line has fewer cuts than units: a block for each
//           cut, whose unit it joins if the unit has no cut before.  Of 8192 units
//           of 256 to 512 keys, a block for each took 240 us of 575.
enum class Join { kSplit, kUnits, kCuts };
constexpr int kJoinWarps = 8;

template <typename T, int kDim, int kVecs, Join kJoin>
__global__ void __launch_bounds__(32 * kJoinWarps) combine_kernel(const Params p) {
  const int w = threadIdx.x / 32, lane = threadIdx.x % 32;
  constexpr bool kSplit = kJoin == Join::kSplit, kCuts = kJoin == Join::kCuts;
  const int x = static_cast<int>(blockIdx.x), b = kCuts ? 0 : x / p.units;
  const Line line = lay_out(p, kCuts ? x + 1 : -1, b);
  const int unit = kCuts ? ((x + 1) * line.per - line.begin) / max(line.seq.places, 1) : x - b * p.units;
  const int first = line.begin + unit * line.seq.places + p.extra;  // the unit's first tile
  const int c0 = first / line.per, c1 = (first + line.seq.tiles - 1) / line.per;
  // every block waits, so that this kernel cannot end before the one that leaves the parts
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (c0 == c1) return;                                    // one part: written there
  if (kCuts && (line.b < 0 || c0 != x || c1 < c0)) return;  // no unit, or one that begins elsewhere
  const int head = p.by_row_tiles.div(unit), row0 = (unit - head * p.row_tiles) * p.unit_rows;
  const int rows = min(p.unit_rows, 32);  // of the block: all lanes, or half of them twice
  const int r = static_cast<int>(blockIdx.y) * 32 + lane % rows, row = row0 + r;
  const int group = kSplit ? static_cast<int>(blockIdx.z) : static_cast<int>(blockIdx.z) * kJoinWarps + w;
  const int vec0 = (group * (32 / rows) + lane / rows) * kVecs;
  const int n_parts = c1 - c0 + 1;
  const float2* ml = p.part_ml + r;
  const float4* po = p.part_o + static_cast<int64_t>(vec0) * p.unit_rows + r;
  const int64_t part_vecs = static_cast<int64_t>(kDim / 4) * p.unit_rows;
  auto part = [&](int i) { return 2 * (c0 + i) + (i == 0 ? 1 : 0); };

  // up to kAhead parts under way at a time, sums kept against the running maximum
  constexpr int kAhead = kVecs <= 2 ? 4 : 2, kStride = kSplit ? kJoinWarps : 1;
  float top = -INFINITY, sum = 0.0f;
  float4 acc[kVecs];
#pragma unroll
  for (int k = 0; k < kVecs; ++k) acc[k] = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int i0 = kSplit ? w : 0; i0 < n_parts; i0 += kStride * kAhead) {
    float2 m[kAhead];
    float4 v[kAhead][kVecs];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const int i = i0 + j * kStride;
      m[j] = make_float2(-INFINITY, 0.0f);
      if (i < n_parts) {
        m[j] = __ldcg(ml + static_cast<int64_t>(part(i)) * p.unit_rows);
#pragma unroll
        for (int k = 0; k < kVecs; ++k) v[j][k] = __ldcg(po + part(i) * part_vecs + k * p.unit_rows);
      }
    }
    float now = top;
#pragma unroll
    for (int j = 0; j < kAhead; ++j) now = fmaxf(now, m[j].x);
    const float ref = now == -INFINITY ? 0.0f : now;
    const float shrink = ptx::ex2_approx(top - ref);
    top = now;
    sum *= shrink;
#pragma unroll
    for (int k = 0; k < kVecs; ++k)
      acc[k] = make_float4(acc[k].x * shrink, acc[k].y * shrink, acc[k].z * shrink, acc[k].w * shrink);
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      if (i0 + j * kStride >= n_parts) break;
      const float f = ptx::ex2_approx(m[j].x - ref);
      sum = fmaf(f, m[j].y, sum);
#pragma unroll
      for (int k = 0; k < kVecs; ++k) {
        acc[k].x = fmaf(f, v[j][k].x, acc[k].x);
        acc[k].y = fmaf(f, v[j][k].y, acc[k].y);
        acc[k].z = fmaf(f, v[j][k].z, acc[k].z);
        acc[k].w = fmaf(f, v[j][k].w, acc[k].w);
      }
    }
  }
  if constexpr (!kSplit) {
    if (row >= p.rows) return;
#pragma unroll
    for (int k = 0; k < kVecs; ++k)
      write_row<T, kDim>(p, kCuts ? line.b : b, head, row, line.seq.n_own, vec0 + k, top, sum, acc[k]);
  } else {
    __shared__ float4 sums[kJoinWarps][kVecs][32];
    __shared__ float2 tops[kJoinWarps][32];
    tops[w][lane] = make_float2(top, sum);
#pragma unroll
    for (int k = 0; k < kVecs; ++k) sums[w][k][lane] = acc[k];
    __syncthreads();
    // thread (k, lane) joins the warps' sums of its vector
    const int k = w;
    if (k >= kVecs || row >= p.rows) return;
    top = -INFINITY;
#pragma unroll
    for (int i = 0; i < kJoinWarps; ++i) top = fmaxf(top, tops[i][lane].x);
    const float ref = top == -INFINITY ? 0.0f : top;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    sum = 0.0f;
#pragma unroll
    for (int i = 0; i < kJoinWarps; ++i) {
      const float f = ptx::ex2_approx(tops[i][lane].x - ref);
      sum = fmaf(f, tops[i][lane].y, sum);
      const float4 x = sums[i][k][lane];
      o.x = fmaf(f, x.x, o.x);
      o.y = fmaf(f, x.y, o.y);
      o.z = fmaf(f, x.z, o.z);
      o.w = fmaf(f, x.w, o.w);
    }
    write_row<T, kDim>(p, b, head, row, line.seq.n_own, vec0 + k, top, sum, o);
  }
}

struct Plan {
  bool tiles;      // tile_kernel; else rows_kernel
  bool pair;       // tile_kernel with two row tiles in a unit
  int unit_rows;
  int row_tiles;   // units of a (sequence, kv head)
  int tile_shift;  // log2 of the keys of a tile
  int blocks;
  int extra;        // places of a unit beyond its tiles
  int64_t longest;  // tiles that the line can have, and places
  int64_t places;
  int64_t part_rows, ml_bytes, workspace;
};

Plan make_plan(const Pages& pages, int64_t batch, int64_t rows, int64_t tokens, bool tree, int sms) {
  Plan plan;
  // tile_kernel for many rows, unless there are so few pairs of a row and a key that
  // its longer start decides.  64 rows of each of 8 heads over 2048 keys (1 M pairs)
  // took 12.2 us by rows_kernel and 13.2 by tile_kernel, of each of 64 heads over 512
  // keys (2 M) 16.9 and 19.2, over 1024 keys 22.1 and 20.9; at dimension 128, whose
  // rows_kernel has 16 rows in a unit, 14.0 and 14.6, 22.5 and 21.7; 256 rows of each
  // of 8 heads over 512 keys (1.2 M) 16.9 and 18.4, over 1024 keys 21.6 and 19.3.  Up
  // to 16 rows rows_kernel is faster at any length (32 caches of 4096 to 8192 keys: 40
  // us against 64, and 71 against 83 at dimension 128); at 17 to 32 rows and dimension
  // 64 the two are alike.
  const double pairs = static_cast<double>(batch) * pages.kv_heads * rows *
                       (static_cast<double>(pages.slots()) + (tree ? tokens : 0));
  plan.tiles = rows > (pages.dim == 64 ? 32 : 16) && pairs > (pages.dim == 64 ? 2.0e6 : 1.6e6);
  plan.pair = plan.tiles && rows > 128;
  plan.unit_rows = plan.tiles ? (plan.pair ? 256 : 128) : pages.dim == 64 && rows > 16 ? 32 : 16;
  plan.row_tiles = static_cast<int>((rows + plan.unit_rows - 1) / plan.unit_rows);
  plan.tile_shift = plan.tiles ? 7 : 6;
  static_assert(tiles::kKeys == 128 && kRowsTile == 64, "tile_shift");
  // as many blocks as the GPU holds
  const int64_t resident = static_cast<int64_t>(sms) *
                           (plan.tiles ? 1 : pages.dim == 128 ? kResident<128, 1> : plan.unit_rows == 16 ? kResident<64, 1> : kResident<64, 2>);
  const int64_t round = (1 << plan.tile_shift) - 1;
  plan.longest = batch * pages.kv_heads * plan.row_tiles *
                 (((pages.slots() + round) >> plan.tile_shift) + (tree ? (tokens + round) >> plan.tile_shift : 0) + 1);
  // Beginning a unit and leaving its sums costs a block about as much as 6 tiles
  // of tile_kernel: 8 x 8 units of 16 to 64 tiles at dimension 128 took 66 us with
  // it in the plan, 71 without, 69 with 16; of rows_kernel some 2 small ones.
  plan.extra = plan.tiles ? 6 : 2;
  plan.places = plan.longest + batch * pages.kv_heads * plan.row_tiles * plan.extra;
  // at most 256 parts a unit: joining 592 took longer than reading with fewer
  // blocks saved (one kv head of 65536 keys: 14.3 against 18.7 us; 128: 14.4,
  // and 62 against 44 us at 524288 keys)
  const int64_t units = batch * pages.kv_heads * plan.row_tiles;
  plan.blocks = static_cast<int>(std::max<int64_t>(1, std::min({resident, plan.places, 256 * units})));
  plan.part_rows = 2ll * plan.blocks * plan.unit_rows;
  plan.ml_bytes = (plan.part_rows * static_cast<int64_t>(sizeof(float2)) + 255) & ~255ll;
  plan.workspace = plan.ml_bytes + plan.part_rows * pages.dim * static_cast<int64_t>(sizeof(float));
  return plan;
}

template <typename T, int kDim, int kVecs, Join kJoin>
cudaError_t launch_combine(const Params& p, cudaStream_t stream) {
  const int rows = std::min(p.unit_rows, 32);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(kJoin == Join::kCuts ? p.blocks - 1 : p.batch * p.units),
                     static_cast<unsigned>((std::min(p.unit_rows, p.rows) + 31) / 32),
                     static_cast<unsigned>(kDim / 4 * rows / 32 / kVecs / (kJoin == Join::kSplit ? 1 : kJoinWarps)));
  cfg.blockDim = dim3(32 * kJoinWarps);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, combine_kernel<T, kDim, kVecs, kJoin>, p);
}

template <typename T, int kDim>
cudaError_t launch_combine(const Params& p, cudaStream_t stream) {
  if (p.blocks == 1) return cudaSuccess;  // the line has no cuts
  // more than four parts a unit, were all alike
  if (p.blocks > 4 * p.batch * p.units) return launch_combine<T, kDim, 2, Join::kSplit>(p, stream);
  constexpr int kFew = kDim / 64, kMany = kDim / 32;  // vectors of a thread
  if (p.blocks <= p.batch * p.units)
    return p.unit_rows == 16 ? launch_combine<T, kDim, kFew, Join::kCuts>(p, stream)
                             : launch_combine<T, kDim, kMany, Join::kCuts>(p, stream);
  return p.unit_rows == 16 ? launch_combine<T, kDim, kFew, Join::kUnits>(p, stream)
                           : launch_combine<T, kDim, kMany, Join::kUnits>(p, stream);
}

template <typename T, int kDim, int kMt>
cudaError_t launch_rows(Params& p, cudaStream_t stream) {
  using S = Shape<kDim, kMt>;
  static std::atomic<uint64_t> allowed{0};
  cudaError_t e = host::allow_smem(reinterpret_cast<const void*>(&rows_kernel<T, kDim, kMt>), S::kSmem, p.device, allowed);
  if (e != cudaSuccess) return e;
  rows_kernel<T, kDim, kMt><<<p.blocks, kThreads, S::kSmem, stream>>>(p);
  if ((e = cudaGetLastError()) != cudaSuccess) return e;
  return launch_combine<T, kDim>(p, stream);
}

template <typename T, int kDim, bool kPair>
cudaError_t launch_tiles(Params& p, const tiles::Maps& maps, cudaStream_t stream) {
  using S = tiles::Shape<kDim, kPair>;
  static std::atomic<uint64_t> allowed{0};
  cudaError_t e = host::allow_smem(reinterpret_cast<const void*>(&tiles::tile_kernel<T, kDim, kPair>), S::kSmem,
                                   p.device, allowed);
  if (e != cudaSuccess) return e;
  tiles::tile_kernel<T, kDim, kPair><<<p.blocks, tiles::kThreads, S::kSmem, stream>>>(maps.k, maps.v, p);
  if ((e = cudaGetLastError()) != cudaSuccess) return e;
  return launch_combine<T, kDim>(p, stream);
}

template <typename T>
cudaError_t launch_type(Params& p, const Plan& plan, const tiles::Maps& maps, cudaStream_t stream) {
  if (plan.tiles) {
    if (p.pages.dim == 64)
      return plan.pair ? launch_tiles<T, 64, true>(p, maps, stream) : launch_tiles<T, 64, false>(p, maps, stream);
    return plan.pair ? launch_tiles<T, 128, true>(p, maps, stream) : launch_tiles<T, 128, false>(p, maps, stream);
  }
  if (p.pages.dim == 128) return launch_rows<T, 128, 1>(p, stream);
  return plan.unit_rows == 16 ? launch_rows<T, 64, 1>(p, stream) : launch_rows<T, 64, 2>(p, stream);
}

}  // namespace tree
}  // namespace fa

using fa::host::set_error;

extern "C" int64_t fa_tree_attention_workspace(const fa_paged_cache* cache, int64_t heads,
                                               int64_t tokens, int has_tree) {
  fa::Pages pages;
  if (fa::check_pages(cache, &pages) != FA_OK) return -1;
  if (fa::check_queries(pages, cache->batch, heads, tokens, FA_FP16, 1.0f) != FA_OK) return -1;
  if (cache->batch == 0 || heads == 0 || tokens == 0) return 0;
  fa::host::Device d;
  if (fa::host::current_device(&d) != FA_OK) return -1;
  return fa::tree::make_plan(pages, cache->batch, heads / pages.kv_heads * tokens, tokens,
                             has_tree != 0, d.sms)
      .workspace;
}

extern "C" int fa_tree_attention_sm100(const fa_paged_cache* cache, const fa_rows* query,
                                       int64_t heads, int64_t tokens, const fa_rows* k_tree,
                                       const fa_rows* v_tree, const unsigned char* tree_mask,
                                       int64_t mask_batch_stride, int64_t mask_row_stride,
                                       const int* tree_sizes, int dtype, float scale, void* out,
                                       float* lse, void* workspace, int64_t workspace_bytes,
                                       void* cuda_stream) {
  namespace ft = fa::tree;
  ft::Params p = {};
  int rc = fa::check_pages(cache, &p.pages);
  if (rc != FA_OK) return rc;
  if ((rc = fa::check_queries(p.pages, cache->batch, heads, tokens, dtype, scale)) != FA_OK) return rc;
  if ((k_tree == nullptr) != (v_tree == nullptr))
    return set_error(FA_ERR_INVALID, "k_tree and v_tree go together");
  if (k_tree == nullptr && tree_mask != nullptr)
    return set_error(FA_ERR_INVALID, "a tree mask needs k_tree and v_tree");
  if (cache->batch == 0 || heads == 0 || tokens == 0) return FA_OK;
  if ((rc = fa::check_rows(query, "query", &p.q)) != FA_OK) return rc;
  p.tree = k_tree != nullptr;
  if (p.tree) {
    if ((rc = fa::check_rows(k_tree, "k_tree", &p.k_tree)) != FA_OK) return rc;
    if ((rc = fa::check_rows(v_tree, "v_tree", &p.v_tree)) != FA_OK) return rc;
  }
  if (out == nullptr || lse == nullptr || workspace == nullptr ||
      (p.pages.slots() > 0 && p.pages.num_pages > 0 && cache->v_pages == nullptr))
    return set_error(FA_ERR_INVALID, "null pointer");
  if (reinterpret_cast<uintptr_t>(out) & 15)
    return set_error(FA_ERR_INVALID, "out must be 16-byte aligned");
  if (reinterpret_cast<uintptr_t>(workspace) & 255)
    return set_error(FA_ERR_INVALID, "workspace must be 256-byte aligned");
  fa::host::Device d;
  if ((rc = fa::host::current_device(&d)) != FA_OK) return rc;
  p.pages.status = d.status;
  p.k_pages = cache->k_pages;
  p.v_pages = cache->v_pages;
  p.mask = tree_mask;
  p.mask_batch = mask_batch_stride;
  p.mask_row = mask_row_stride;
  p.sizes = tree_sizes;
  p.out = out;
  p.lse = lse;
  p.batch = static_cast<int>(cache->batch);
  p.heads = static_cast<int>(heads);
  p.group = p.heads / p.pages.kv_heads;
  p.tokens = static_cast<int>(tokens);
  p.rows = p.group * p.tokens;
  p.scale_log2 = scale * 1.4426950408889634f;
  const ft::Plan plan = ft::make_plan(p.pages, p.batch, p.rows, tokens, p.tree != 0, d.sms);
  if (plan.places > (1ll << 30)) return set_error(FA_ERR_INVALID, "size too large");
  if (workspace_bytes < plan.workspace) return set_error(FA_ERR_INVALID, "workspace too small");
  p.row_tiles = plan.row_tiles;
  p.blocks = plan.blocks;
  p.tile_shift = plan.tile_shift;
  p.extra = plan.extra;
  p.units = p.pages.kv_heads * p.row_tiles;
  p.by_tokens = ft::FastDiv(static_cast<uint32_t>(p.tokens));
  p.by_page = ft::FastDiv(static_cast<uint32_t>(p.pages.page_size));
  p.by_row_tiles = ft::FastDiv(static_cast<uint32_t>(p.row_tiles));
  p.by_blocks = ft::FastDiv(static_cast<uint32_t>(plan.blocks));
  p.unit_rows = plan.unit_rows;
  p.part_ml = static_cast<float2*>(workspace);
  p.part_o = reinterpret_cast<float4*>(static_cast<uint8_t*>(workspace) + plan.ml_bytes);
  p.limit_ns = fa::host::wait_limit_ns();
  p.device = d.index;
  ft::tiles::Maps maps = {};
  p.box_rows = 16;  // of a page, a power of two that divides its size
  while (p.box_rows < ft::tiles::kKeys && p.pages.page_size % (2 * p.box_rows) == 0) p.box_rows *= 2;
  if (plan.tiles && p.pages.slots() > 0 && p.pages.num_pages > 0) {
    const int64_t slices = cache->num_pages * cache->kv_heads;
    for (auto [map, base] : {std::pair{&maps.k, p.k_pages}, std::pair{&maps.v, p.v_pages}})
      if ((rc = fa::host::encode_rows_map(map, base, dtype == FA_BF16, cache->head_dim, cache->page_size,
                                          slices, static_cast<uint32_t>(p.box_rows))) != FA_OK)
        return rc;
  }
  cudaStream_t stream = static_cast<cudaStream_t>(cuda_stream);
  const cudaError_t e = dtype == FA_FP16 ? ft::launch_type<__half>(p, plan, maps, stream)
                                         : ft::launch_type<__nv_bfloat16>(p, plan, maps, stream);
  if (e != cudaSuccess) return set_error(FA_ERR_CUDA, "kernel launch: %s", cudaGetErrorString(e));
  return FA_OK;
}
