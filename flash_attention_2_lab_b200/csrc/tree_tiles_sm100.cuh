// Tree attention on tcgen05 tiles, for units of many rows.
//
// One block of twelve warps per SM walks its part of the line.  Warp 8 brings K
// and V tiles of 128 keys into a ring of swizzled shared memory, one TMA box
// per piece of a page; warp 9 issues S_t = Q K^T and O_t += P_t V with all
// three in tensor memory; warps 0-3 and 4-7 are the softmax of two slots t,
// one thread per row, which alternate on the exponential unit: while one slot
// is at its exponentials the other's products run.
//   kPair: a unit is 256 rows, the slots are its two tiles of 128 rows, and
//          both see every key tile.
//   else:  a unit is 128 rows; slot t takes every second key tile with sums of
//          its own, joined when the unit's part ends.
// P overwrites S_t in place (16-bit, half the columns), so S_t of the next tile
// is issued behind the product that reads P; its completion then also says that
// O_t is at rest, and the rare rescale of O_t needs no barrier of its own.  The
// exponent's maximum moves only when a row's maximum grows by more than 2^8.
//
// Bound by HBM up to 128 rows at dimension 128 (64 KiB per key tile and SM
// against 1024 clocks of exponentials), by the exponentials (16 per clock and
// SM) from there on.
//
// Keys behind a sequence's length, in pages that do not exist, and tree keys
// that a row does not see are hidden by selection on S; their V rows are zeros
// in shared memory, whatever memory holds, because P = 0 times NaN is NaN.  A
// tree value that is infinite or NaN is zeroed there too and added at the end,
// key by key, to the rows that see it.
//
// Every wait is bounded; one that runs out sets a status bit and an abort flag
// that releases the others, and the block drains its copies and products, frees
// tensor memory and returns.
#pragma once

#include <cuda.h>

#include <type_traits>

#include "mma_sm80.cuh"
#include "paged_cache.cuh"
#include "sm100_ptx.cuh"
#include "tree_line.cuh"

namespace fa {
namespace tree {
namespace tiles {

using namespace ptx;

constexpr int kKeys = 128;    // of a tile
constexpr int kWarps = 12;      // the last two only complete the third warpgroup
constexpr int kThreads = 32 * kWarps;
constexpr int kProducer = 8, kIssuer = 9;
constexpr int kInfo = 16;     // key tiles described at a time, more than the ring holds
constexpr int kSegments = 8;  // parts of units described at a time

struct Maps {
  CUtensorMap k, v;
};

// Status bits, as in the forward kernel.
constexpr unsigned int kTimeoutProducer = 1u, kTimeoutMma = 2u, kTimeoutSoftmax = 4u, kTimeoutDrain = 8u;
constexpr unsigned long long kDrainNs = 200000000ull;

struct Control {
  uint64_t q_full, fix, sync, drain;
  uint64_t kv_full[12], kv_empty[12];
  uint64_t s_full[2], p_full[2], o_done[2];
  uint32_t tmem;
  int abort;
  int keys[kInfo];            // valid keys of a key tile
  unsigned int boxes[kInfo];  // which of its boxes are there
  int odd[kSegments];         // a tree value of the part is not finite
};

template <int kDim, bool kPair>
struct Shape {
  static constexpr int kTileBytes = kKeys * kDim * 2;  // K, V, and 128 rows of Q
  static constexpr int kQBytes = (kPair ? 2 : 1) * kTileBytes;
  static constexpr int kSlots = kDim == 64 ? 10 : 5;
  static constexpr int kRing = kQBytes;
  static constexpr int kControl = kRing + kSlots * kTileBytes;
  static constexpr int kMl = kControl + static_cast<int>(sizeof(Control));  // float2 [2][128], one row tile only
  static constexpr int kSmem = kMl + (kPair ? 0 : 2048) + 1024;             // + alignment
  static constexpr int kRows = kPair ? 256 : 128;
  static_assert(kSmem <= 227 * 1024 - 256, "shared memory of a block, lay_out's included");
  static_assert(kSlots <= 12, "control block");
};

// One part of a unit, the same for every role.
struct Segment {
  int b, head, row0;       // row0: first row of the unit
  int tile0, n;            // key tiles [tile0, tile0 + n) of the unit
  int n_cache, c_tiles;    // cached keys and their tiles
  int n_own;               // tokens that are there (queries, tree keys)
  bool whole;
  int64_t part;
};

// Walks the parts of this block.
struct Walk {
  int64_t start, at, end, off;
  int b, units;

  __device__ __forceinline__ Walk(const Params& p, const Line& line) {
    start = blockIdx.x * line.per;
    at = start;
    end = min(start + line.per, line.total);
    off = start - line.begin;
    b = line.b;
    units = p.pages.kv_heads * p.row_tiles;
  }
  __device__ __forceinline__ bool next(const Params& p, Segment& s) {
    if (at >= end) return false;
    const int tiles = unit_tiles(p, b);
    s.b = b;
    s.n_cache = cache_length(p.pages, b);
    s.c_tiles = cache_tiles(p, b);
    s.n_own = tree_size(p, b);
    const int unit = static_cast<int>(off / tiles);
    s.tile0 = static_cast<int>(off - static_cast<int64_t>(unit) * tiles);
    s.n = static_cast<int>(min(static_cast<int64_t>(tiles), s.tile0 + (end - at))) - s.tile0;
    s.head = unit / p.row_tiles;
    s.row0 = (unit - s.head * p.row_tiles) * p.unit_rows;
    s.whole = s.n == tiles;
    s.part = 2 * static_cast<int64_t>(blockIdx.x) + (at != start ? 1 : 0);
    at += s.n;
    off += s.n;
    if (off == static_cast<int64_t>(tiles) * units) {
      ++b;
      off = 0;
    }
    return true;
  }
};

// Whether row `row` of (b, head) sees tree key j < n_own.
__device__ __forceinline__ bool sees(const Params& p, int b, int row, int j) {
  if (row >= p.rows) return false;
  const int t = row % p.tokens;
  return p.mask == nullptr ? j <= t : p.mask[b * p.mask_batch + t * p.mask_row + j] != 0;
}

template <int kDim>
__device__ __forceinline__ uint32_t swizzled(int row, int vec) {  // of a tile, 64 elements wide halves
  return static_cast<uint32_t>((vec >> 3) * (kKeys * 128) + row * 128 + (((vec & 7) ^ (row & 7)) << 4));
}

template <typename T, int kDim, bool kPair>
struct Block {
  using S = Shape<kDim, kPair>;
  static constexpr int kVecs = kDim / 8;
  const Params& p;
  Control* ctl;
  unsigned char* smem;  // aligned
  uint32_t base;        // the same as a shared address
  uint32_t tmem;
  int lane;

  __device__ __forceinline__ uint32_t slot_at(uint32_t i) const {
    return base + S::kRing + (i % S::kSlots) * S::kTileBytes;
  }
  __device__ __forceinline__ uint32_t full(uint32_t i) const { return smem_u32(&ctl->kv_full[i % S::kSlots]); }
  __device__ __forceinline__ uint32_t empty(uint32_t i) const { return smem_u32(&ctl->kv_empty[i % S::kSlots]); }
  static __device__ __forceinline__ uint32_t parity(uint32_t i) { return (i / S::kSlots) & 1; }

  // ------------------------------------------------------------- producer
  // `count`: ring entries begun, so that a block that gives up can wait for them.
  __device__ bool produce(const CUtensorMap* mk, const CUtensorMap* mv, Walk walk, uint32_t& count) {
    uint32_t tile_no = 0, fixes = 0, segment = 0;
    Segment s = {};
    auto wait = [&](uint32_t bar, uint32_t par) {
      return mbar_wait_warp(bar, par, &ctl->abort, p.pages.status, kTimeoutProducer, p.limit_ns);
    };
    const int row_boxes = kKeys / p.box_rows, n_boxes = row_boxes * (kDim / 64);
    const uint32_t box_bytes = static_cast<uint32_t>(p.box_rows) * 128;

    // K or V of key tile `i` of the segment into the next ring entry
    auto bring = [&](int i, bool is_v, uint32_t info) -> bool {
      if (count >= S::kSlots && !wait(empty(count), parity(count) ^ 1)) return false;
      const uint32_t dst = slot_at(count), bar = full(count);
      const int tile = s.tile0 + i;
      if (tile < s.c_tiles) {
        const int slot0 = tile * kKeys, keys = min(s.n_cache - slot0, kKeys);
        // lane l: box l % row_boxes, column half l / row_boxes
        const int box = lane % row_boxes, half = lane / row_boxes;
        const int slot = slot0 + box * p.box_rows;
        int64_t row = -1;
        if (lane < n_boxes && slot < s.n_cache) row = cache_row(p.pages, s.b, s.head, slot);
        const unsigned int have = __ballot_sync(0xffffffffu, row >= 0);
        const unsigned int here = have & ((1u << row_boxes) - 1u);  // at most 8
        const bool all = keys == kKeys && here == (1u << row_boxes) - 1u;
        const uint32_t to = is_v && !all ? smem_u32(&ctl->fix) : bar;
        const uint32_t bytes = __popc(have) * box_bytes;
        if (lane == 0) {
          if (!is_v) {
            ctl->keys[info % kInfo] = keys;
            ctl->boxes[info % kInfo] = here;
          }
          if (bytes > 0 || to == bar) mbar_arrive_expect_tx(to, bytes);
        }
        __syncwarp();
        if (row >= 0) {
          const int in_page = static_cast<int>((row / kDim) % p.pages.page_size);
          const int slice = static_cast<int>((row / kDim) / p.pages.page_size);
          tma_load_3d(dst + half * (kKeys * 128) + box * box_bytes, is_v ? mv : mk, to, half * 64, in_page, slice);
        }
        if (to != bar) {
          // a tile that is not full: rows without a key become zeros
          if (bytes > 0) {
            if (!wait(to, fixes & 1)) {  // the copies land all the same
              if (lane == 0) mbar_wait(to, fixes & 1, nullptr, p.pages.status, kTimeoutDrain, kDrainNs);
              return false;
            }
            ++fixes;
          }
          for (int v = lane; v < kKeys * kVecs; v += 32) {
            const int r = v / kVecs;
            if (r < keys && ((here >> (r / p.box_rows)) & 1)) continue;
            *reinterpret_cast<uint4*>(smem + (dst - base) + swizzled<kDim>(r, v % kVecs)) = make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(bar);
        }
      } else {
        // keys of the tree: strided rows, copied 16 bytes at a time
        const int j0 = (tile - s.c_tiles) * kKeys;
        const int keys = p.tree ? max(0, min(s.n_own - j0, kKeys)) : 0;
        const Rows& src = is_v ? p.v_tree : p.k_tree;
        // without keys nothing is read, but every copy names an address
        const T* from = keys > 0 ? static_cast<const T*>(src.data) + s.b * src.batch + s.head * src.head
                                 : static_cast<const T*>(p.q.data);
        for (int v = lane; v < kKeys * kVecs; v += 32) {
          const int r = v / kVecs, vec = v % kVecs;
          copy16(dst + swizzled<kDim>(r, vec), from + (r < keys ? (j0 + r) * src.row : 0) + vec * 8, r < keys);
        }
        copy_commit();
        copy_wait<0>();
        __syncwarp();
        if (is_v) {
          bool any = false;
          for (int v0 = 0; v0 < keys * kVecs; v0 += 32) {
            const int v = v0 + lane, r = v / kVecs;
            uint4* at = reinterpret_cast<uint4*>(smem + (dst - base) + swizzled<kDim>(r, v % kVecs));
            bool bad = false;
            if (r < keys) {
              const uint4 x = *at;
              bad = not_finite2<T>(x.x) || not_finite2<T>(x.y) || not_finite2<T>(x.z) || not_finite2<T>(x.w);
            }
            // the lanes of a row are neighbours: 8 or 16 of them
            const unsigned int bits = __ballot_sync(0xffffffffu, bad);
            const unsigned int mine = (bits >> (lane / kVecs * kVecs)) & ((1u << kVecs) - 1u);
            if (r < keys && mine != 0) *at = make_uint4(0, 0, 0, 0);
            any = any || bits != 0;
          }
          if (lane == 0 && any) ctl->odd[segment % kSegments] = 1;
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          if (!is_v) {
            ctl->keys[info % kInfo] = keys;
            ctl->boxes[info % kInfo] = ~0u;
          }
          mbar_arrive(bar);
        }
      }
      __syncwarp();
      ++count;
      return true;
    };

    while (walk.next(p, s)) {
      if (lane == 0) ctl->odd[segment % kSegments] = 0;
      if (kPair) {
        for (int i = 0; i < s.n; ++i) {
          if (!bring(i, false, tile_no + i) || !bring(i, true, tile_no + i)) return false;
        }
      } else {  // K runs two tiles ahead: one for each slot
        if (!bring(0, false, tile_no)) return false;
        if (s.n > 1 && !bring(1, false, tile_no + 1)) return false;
        for (int i = 0; i < s.n; ++i) {
          if (!bring(i, true, tile_no + i)) return false;
          if (i + 2 < s.n && !bring(i + 2, false, tile_no + i + 2)) return false;
        }
      }
      tile_no += s.n;
      ++segment;
    }
    return true;
  }

  // --------------------------------------------------------------- issuer
  __device__ bool issue(Walk walk) {
    constexpr uint32_t kType = std::is_same<T, __nv_bfloat16>::value ? (1u << 7) | (1u << 10) : 0u;
    constexpr uint32_t kIdS = idesc_f16_f32(128, kKeys, false) | kType;
    constexpr uint32_t kIdO = idesc_f16_f32(128, 64, true) | kType;
    uint32_t count = 0, segment = 0, p_count[2] = {0, 0};
    Segment s = {};
    auto wait = [&](uint32_t bar, uint32_t par) {
      return mbar_wait_warp(bar, par, &ctl->abort, p.pages.status, kTimeoutMma, p.limit_ns);
    };
    auto scores = [&](int t, uint32_t k) {  // S_t = Q K^T
      if (elect_one()) {
        const uint32_t q = base + (kPair ? t * S::kTileBytes : 0);
#pragma unroll
        for (int kk = 0; kk < kDim / 16; ++kk) {  // 16 elements are 32 bytes; 64 are a half
          const uint32_t at = (kk / 4) * (kKeys * 128) + (kk % 4) * 32;
          mma_ss_f16(tmem + t * 128, smem_desc_sw128(q + at, 16, 1024),
                     smem_desc_sw128(slot_at(k) + at, 16, 1024), kIdS, kk > 0);
        }
        tc_commit(smem_u32(&ctl->s_full[t]));
      }
      __syncwarp();
    };
    auto values = [&](int t, uint32_t v, bool more) {  // O_t (+)= P_t V
      if (elect_one()) {
#pragma unroll
        for (int half = 0; half < kDim / 64; ++half)
#pragma unroll
          for (int kk = 0; kk < kKeys / 16; ++kk)  // 16 keys: 8 columns of P, 2 KiB of V
            mma_ts_f16(tmem + 256 + t * kDim + half * 64, tmem + t * 128 + kk * 8,
                       smem_desc_sw128(slot_at(v) + half * (kKeys * 128) + kk * 2048, 16, 1024), kIdO,
                       (more || kk > 0) ? 1u : 0u);
      }
      __syncwarp();
    };
    auto release = [&](uint32_t bar) {
      if (elect_one()) tc_commit(bar);
      __syncwarp();
    };
    auto wait_p = [&](int t) {
      if (!wait(smem_u32(&ctl->p_full[t]), p_count[t] & 1)) return false;
      ++p_count[t];
      tc_fence_after();
      return true;
    };
    auto wait_kv = [&](uint32_t i) {
      if (!wait(full(i), parity(i))) return false;
      tc_fence_after();
      return true;
    };

    while (walk.next(p, s)) {
      if (!wait(smem_u32(&ctl->q_full), segment & 1)) return false;
      ++segment;
      tc_fence_after();
      if (kPair) {  // the ring holds K_0 V_0 K_1 V_1 ...
        for (int i = 0; i <= s.n; ++i) {
          const uint32_t k = count + 2 * i, v = k - 1;  // V of the tile before
          if (i < s.n && !wait_kv(k)) return false;
          if (i > 0 && !wait_kv(v)) return false;
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            if (i > 0) {
              if (!wait_p(t)) return false;
              values(t, v, i > 1);
              if (i == s.n) release(smem_u32(&ctl->o_done[t]));
            }
            if (i < s.n) scores(t, k);
          }
          if (i > 0) release(empty(v));
          if (i < s.n) release(empty(k));
        }
      } else {  // K_0 K_1 V_0 K_2 V_1 K_3 ...
        uint32_t at = count;
        for (int i = 0; i < 2 && i < s.n; ++i, ++at) {
          if (!wait_kv(at)) return false;
          scores(i, at);
          release(empty(at));
        }
        for (int i = 0; i < s.n; ++i) {
          const int t = i & 1;
          if (!wait_kv(at) || !wait_p(t)) return false;
          values(t, at, i > 1);
          release(empty(at));
          if (i + 2 >= s.n) release(smem_u32(&ctl->o_done[t]));
          ++at;
          if (i + 2 < s.n) {
            if (!wait_kv(at)) return false;
            scores(t, at);
            release(empty(at));
            ++at;
          }
        }
      }
      count += 2 * s.n;
    }
    return true;
  }

  // -------------------------------------------------------------- softmax
  // The tree values that are not finite, added to 32 columns of a row's sums.
  __device__ __noinline__ void add_odd(const Segment& s, int row, int col0, float ref, float* o) {
    const int j0 = max(s.tile0 - s.c_tiles, 0) * kKeys;
    const int j1 = min((s.tile0 + s.n - s.c_tiles) * kKeys, s.n_own);
    const int hg = row / p.tokens, t = row - hg * p.tokens;
    if (row >= p.rows || t >= s.n_own) return;
    const T* q = static_cast<const T*>(p.q.data) + s.b * p.q.batch +
                 (static_cast<int64_t>(s.head) * p.group + hg) * p.q.head + t * p.q.row;
    for (int j = j0; j < j1; ++j) {
      const T* k = static_cast<const T*>(p.k_tree.data) + s.b * p.k_tree.batch + s.head * p.k_tree.head + j * p.k_tree.row;
      const T* v = static_cast<const T*>(p.v_tree.data) + s.b * p.v_tree.batch + s.head * p.v_tree.head + j * p.v_tree.row;
      const uint32_t* v32 = reinterpret_cast<const uint32_t*>(v);
      bool bad = false;
      for (int i = 0; i < kDim / 2; ++i) bad = bad || not_finite2<T>(v32[i]);
      if (!bad || !sees(p, s.b, row, j)) continue;
      float score = 0.0f;
      for (int i = 0; i < kDim / 2; ++i) {
        const float2 a = unpack2<T>(reinterpret_cast<const uint32_t*>(q)[i]);
        const float2 c = unpack2<T>(reinterpret_cast<const uint32_t*>(k)[i]);
        score = fmaf(a.x, c.x, fmaf(a.y, c.y, score));
      }
      const float w = ex2_approx(fmaf(score, p.scale_log2, -ref));
      for (int i = 0; i < 16; ++i) {
        const float2 x = unpack2<T>(v32[col0 / 2 + i]);
        o[2 * i] = fmaf(w, x.x, o[2 * i]);
        o[2 * i + 1] = fmaf(w, x.y, o[2 * i + 1]);
      }
    }
  }

  // 32 columns of a row's sums: final, or as this part's share.
  __device__ __forceinline__ void write(const Segment& s, int row, int col0, float m, float l, const float* o) {
    if (row >= p.rows) return;
    const int64_t at = (static_cast<int64_t>(s.b) * p.heads + static_cast<int64_t>(s.head) * p.group) * p.tokens + row;
    const int r = row - s.row0;
    if (s.whole) {
      const bool nothing = l == 0.0f || row % p.tokens >= s.n_own;
      const float inv = 1.0f / l;
      uint4* out = reinterpret_cast<uint4*>(static_cast<T*>(p.out) + at * kDim + col0);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e)
          w[e] = nothing ? 0u : pack2<T>(o[8 * i + 2 * e] * inv, o[8 * i + 2 * e + 1] * inv);
        out[i] = make_uint4(w[0], w[1], w[2], w[3]);
      }
      if (col0 == 0) p.lse[at] = nothing ? -INFINITY : 0.69314718055994531f * (m + log2f(l));
    } else {
      float4* out = reinterpret_cast<float4*>(p.part_o + (s.part * S::kRows + r) * kDim + col0);
#pragma unroll
      for (int i = 0; i < 8; ++i) out[i] = make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
      if (col0 == 0) p.part_ml[s.part * S::kRows + r] = make_float2(m, l);
    }
  }

  __device__ bool soften(Walk walk, int t, int warp_in_slot) {
    const int r = warp_in_slot * 32 + lane;  // row of the slot's tile
    const uint32_t lanes = static_cast<uint32_t>(warp_in_slot * 32) << 16;
    const uint32_t t_s = tmem + lanes + t * 128, t_o = tmem + lanes + 256 + t * kDim;
    uint32_t s_count = 0, o_count = 0, syncs = 0, segment = 0, tile_no = 0;
    Segment s = {};
    auto wait = [&](uint32_t bar, uint32_t par) {
      return mbar_wait_warp(bar, par, &ctl->abort, p.pages.status, kTimeoutSoftmax, p.limit_ns);
    };
    auto sync = [&]() {  // the eight softmax warps
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&ctl->sync));
      return wait(smem_u32(&ctl->sync), syncs++ & 1);
    };

    while (walk.next(p, s)) {
      // ---- Q: rows of the unit, zeros where there is none
      for (int v = t * 128 + warp_in_slot * 32 + lane; v < S::kRows * kVecs; v += 256) {
        const int qr = v / kVecs, vec = v % kVecs, row = s.row0 + qr;
        const int hg = row / p.tokens, tok = row - hg * p.tokens;
        const bool there = row < p.rows && tok < s.n_own;
        const T* src = static_cast<const T*>(p.q.data) + s.b * p.q.batch +
                       (static_cast<int64_t>(s.head) * p.group + (there ? hg : 0)) * p.q.head + (there ? tok : 0) * p.q.row;
        copy16(base + (qr / 128) * S::kTileBytes + swizzled<kDim>(qr % 128, vec), src + vec * 8, there);
      }
      copy_commit();
      copy_wait<0>();
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&ctl->q_full));

      const int row = s.row0 + (kPair ? t * 128 : 0) + r;
      // a warp without rows passes its turns; what it leaves reaches only its own rows
      const bool idle = s.row0 + (kPair ? t * 128 : 0) + warp_in_slot * 32 >= p.rows;
      float m = -INFINITY, l = 0.0f;
      bool first = true;
      for (int i = kPair ? 0 : t; i < s.n; i += kPair ? 1 : 2) {
        if (!wait(smem_u32(&ctl->s_full[t]), s_count++ & 1)) return false;
        tc_fence_after();
        if (!idle) {
          const int tile = s.tile0 + i;
          const int keys = *static_cast<volatile int*>(&ctl->keys[(tile_no + i) % kInfo]);
          const unsigned int boxes = *static_cast<volatile unsigned int*>(&ctl->boxes[(tile_no + i) % kInfo]);
          const bool own = tile >= s.c_tiles;
          uint32_t x[128];
#pragma unroll
          for (int c = 0; c < 4; ++c) tmem_ld32(t_s + c * 32, x + c * 32);
#pragma unroll
          for (int c = 0; c < 4; ++c) tc_wait_ld32(x + c * 32);
          const unsigned int all = p.box_rows >= kKeys ? 1u : (1u << (kKeys / p.box_rows)) - 1u;
          if (own || keys < kKeys || (boxes & all) != all) {
            const int j0 = (tile - s.c_tiles) * kKeys;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              // bit e: this row sees key 32 c + e
              uint32_t seen = 0;
              for (int e = 0; e < 32; ++e) {
                const int key = c * 32 + e;
                if (key >= keys) break;
                if (own ? sees(p, s.b, row, j0 + key) : ((boxes >> (key / p.box_rows)) & 1) != 0) seen |= 1u << e;
              }
#pragma unroll
              for (int e = 0; e < 32; ++e)
                if (!((seen >> e) & 1)) x[c * 32 + e] = 0xff800000u;  // -inf
            }
            __syncwarp();
          }
          float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int e = 0; e < 128; e += 8)
#pragma unroll
            for (int c = 0; c < 4; ++c)
              top[c] = max3f(top[c], __uint_as_float(x[e + 2 * c]), __uint_as_float(x[e + 2 * c + 1]));
          const float now = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * p.scale_log2;
          const bool grow = now > m + 8.0f;
          if (first) {
            m = now;
          } else if (__any_sync(0xffffffffu, grow)) {
            const float to = grow ? now : m;
            const float shrink = grow ? ex2_approx(m - to) : 1.0f;
            m = to;
            l *= shrink;
#pragma unroll
            for (int c = 0; c < kDim / 32; ++c) {
              uint32_t o[32];
              tmem_ld32(t_o + c * 32, o);
              tc_wait_ld32(o);
#pragma unroll
              for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * shrink);
              tmem_st32(t_o + c * 32, o);
            }
          }
          const float ref = m == -INFINITY ? 0.0f : m;
          float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            uint32_t packed[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              float a, b;
              ffma2(a, b, __uint_as_float(x[c * 32 + 2 * e]), __uint_as_float(x[c * 32 + 2 * e + 1]),
                    p.scale_log2, p.scale_log2, -ref, -ref);
              a = ex2_approx(a);
              b = ex2_approx(b);
              fadd2(sum[(e & 1) * 2], sum[(e & 1) * 2 + 1], sum[(e & 1) * 2], sum[(e & 1) * 2 + 1], a, b);
              packed[e] = pack2<T>(a, b);
            }
            tmem_st16(t_s + c * 16, packed);
          }
          l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
          tc_wait_st();
        }
        first = false;
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&ctl->p_full[t]));
      }
      tile_no += s.n;

      // ---- the part's sums
      if (!first) {
        if (!wait(smem_u32(&ctl->o_done[t]), o_count++ & 1)) return false;
        tc_fence_after();
      }
      const bool odd = s.tile0 + s.n > s.c_tiles &&
                       *static_cast<volatile int*>(&ctl->odd[segment % kSegments]) != 0;
      if (kPair) {
        if (!idle) {
#pragma unroll 1
          for (int c = 0; c < kDim / 32; ++c) {
            uint32_t o[32];
            __syncwarp();
            tmem_ld32(t_o + c * 32, o);
            tc_wait_ld32(o);
            if (odd) add_odd(s, row, c * 32, m == -INFINITY ? 0.0f : m, reinterpret_cast<float*>(o));
            write(s, row, c * 32, m, l, reinterpret_cast<const float*>(o));
          }
        }
        tc_fence_before();
      } else {
        float2* ml = reinterpret_cast<float2*>(smem + S::kMl);  // a slot's maximum and sum of each row
        ml[t * 128 + r] = make_float2(m, l);
        tc_fence_before();
        if (!sync()) return false;
        tc_fence_after();
        if (!idle) {
          const float2 a = ml[r], b = ml[128 + r];
          const float top = fmaxf(a.x, b.x), ref = top == -INFINITY ? 0.0f : top;
          const float fa = ex2_approx(a.x - ref), fb = ex2_approx(b.x - ref);
          const float sum = fa * a.y + fb * b.y;
#pragma unroll 1
          for (int c = t * (kDim / 64); c < (t + 1) * (kDim / 64); ++c) {
            uint32_t o0[32], o1[32];
            const uint32_t from = tmem + lanes + 256 + c * 32;
            __syncwarp();
            tmem_ld32(from, o0);
            if (s.n > 1) tmem_ld32(from + kDim, o1);  // else slot 1 has no sums
            tc_wait_ld32(o0);
            if (s.n > 1) {
              tc_wait_ld32(o1);
#pragma unroll
              for (int e = 0; e < 32; ++e)
                o0[e] = __float_as_uint(fa * __uint_as_float(o0[e]) + fb * __uint_as_float(o1[e]));
            } else {
#pragma unroll
              for (int e = 0; e < 32; ++e) o0[e] = __float_as_uint(fa * __uint_as_float(o0[e]));
            }
            if (odd) add_odd(s, row, c * 32, ref, reinterpret_cast<float*>(o0));
            write(s, row, c * 32, top, sum, reinterpret_cast<const float*>(o0));
          }
        }
        tc_fence_before();
      }
      __syncwarp();
      // Q and O of both slots are at rest before the next part overwrites them
      if (!sync()) return false;
      tc_fence_after();
      ++segment;
    }
    return true;
  }
};

template <typename T, int kDim, bool kPair>
__global__ void __launch_bounds__(kThreads, 1)
    tile_kernel(const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mv, const Params p) {
  using S = Shape<kDim, kPair>;
  extern __shared__ unsigned char smem_raw[];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const uint32_t raw = smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
  unsigned char* smem = smem_raw + (base - raw);
  Control* ctl = reinterpret_cast<Control*>(smem + S::kControl);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;

  if (threadIdx.x == 0) {
    mbar_init(smem_u32(&ctl->q_full), 8);
    mbar_init(smem_u32(&ctl->fix), 1);
    mbar_init(smem_u32(&ctl->sync), 8);
    mbar_init(smem_u32(&ctl->drain), 1);
    for (int i = 0; i < S::kSlots; ++i) {
      mbar_init(smem_u32(&ctl->kv_full[i]), 1);
      mbar_init(smem_u32(&ctl->kv_empty[i]), 1);
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(smem_u32(&ctl->s_full[t]), 1);
      mbar_init(smem_u32(&ctl->p_full[t]), 4);
      mbar_init(smem_u32(&ctl->o_done[t]), 1);
    }
    ctl->abort = 0;
    fence_mbar_init();
  }
  if (warp == kIssuer) {
    tmem_alloc(smem_u32(&ctl->tmem), 512);
    tmem_relinquish();
  }
  tc_fence_before();
  const Line line = lay_out<kWarps>(p, blockIdx.x, 0);  // with barriers of its own
  __syncthreads();
  tc_fence_after();
  Block<T, kDim, kPair> block{p, ctl, smem, base, ctl->tmem, lane};
  const Walk walk(p, line);

  // the softmax warps take registers that the third warpgroup gives up:
  // 2 x 128 x 208 + 128 x 88 = 384 x 168, the launch's allocation
  if (warp < 8)
    asm volatile("setmaxnreg.inc.sync.aligned.u32 208;" ::: "memory");
  else
    asm volatile("setmaxnreg.dec.sync.aligned.u32 88;" ::: "memory");
  if (warp < 8) {
    block.soften(walk, warp / 4, warp % 4);
  } else if (warp == kProducer) {
    uint32_t count = 0;
    if (!block.produce(&mk, &mv, walk, count)) {
      // the copies that were begun land before the block leaves
      if (lane == 0) {
        for (uint32_t i = 0; i < count && i < S::kSlots; ++i)
          mbar_wait(block.full(count - 1 - i), block.parity(count - 1 - i), nullptr, p.pages.status, kTimeoutDrain, kDrainNs);
      }
    }
    __syncwarp();
  } else if (warp == kIssuer) {
    block.issue(walk);
    // products and the arrivals that follow them end before memory is freed
    if (lane == 0) {
      tc_commit(smem_u32(&ctl->drain));
      mbar_wait(smem_u32(&ctl->drain), 0, nullptr, p.pages.status, kTimeoutDrain, kDrainNs);
    }
    __syncwarp();
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kIssuer) {
    tc_fence_after();
    tmem_dealloc(ctl->tmem, 512);
  }
}

}  // namespace tiles
}  // namespace tree
}  // namespace fa
