// Tree attention on tcgen05 tiles, for units of many rows.
//
// One block of twelve warps per SM walks its part of the line.  Two warps bring
// K and V tiles of 128 keys into a ring of swizzled shared memory, one TMA box
// per piece of a page; one or two issue S_t = Q K^T and O_t += P_t V, with S, P
// and O in tensor memory; one brings the queries of the next part; warps 0-3 and
// 4-7 are the softmax of two slots t, one thread per row, so that one slot's
// products run while the other is at its exponentials.
//   kPair: a unit is 256 rows, the slots are its two tiles of 128 rows, and
//          both see every key tile.
//   else:  a unit is 128 rows; slot t takes every second key tile with sums of
//          its own, joined when the unit's part ends.
// The exponent's maximum moves, and O_t is rescaled, only when a row's maximum
// grows by more than 2^8, which keeps P below 2^8.
//
// Bound by HBM up to 128 rows at dimension 128 (64 KiB per key tile and SM
// against 1024 clocks of exponentials), by the exponentials (16 per clock and
// SM) from there on.  A call in a graph of twelve takes 66 us for 116 rows over 8 x
// 8 caches of 5700 to 8192 keys at dimension 128 (3.6 TB/s) and 68 us for 512 rows
// over 4 of 65500 at dimension 64 (507 TFLOP/s), some 30 us of either whatever the
// length: a key tile more costs a block 1.42 us (6.8 TB/s) and 1.67 us (3280
// clocks, 2048 of them exponentials).  Start, tree tile and the ends of parts are
// what lies above the bounds.  (Differences of variants below: the same calls,
// measured beside one another.)
//
// P is rounded to 16 bits for the product, whose operands are of one type; the
// row's sum adds it unrounded.
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
constexpr int kWarps = 12;
constexpr int kThreads = 32 * kWarps;
constexpr int kProducer = 8, kIssuer = 9, kIssuerV = 10, kBringer = 11;
constexpr int kInfo = 16;     // key tiles described at a time, more than the ring holds
constexpr int kSegments = 8;  // parts of units described at a time

struct Maps {
  CUtensorMap k, v;
};

// Status bits, as in the forward kernel.
constexpr unsigned int kTimeoutProducer = 1u, kTimeoutMma = 2u, kTimeoutSoftmax = 4u, kTimeoutDrain = 8u;
constexpr unsigned long long kDrainNs = 200000000ull;

struct Control {
  uint64_t q_full[2], q_empty[2], fix, sync, drain;
  uint64_t kv_full[12], kv_empty[12];
  uint64_t s_full[2], s_empty[2], p_full[2], o_done[2];
  uint64_t drain_v, turn[8];
  uint32_t tmem;
  int abort;
  int keys[kInfo];            // valid keys of a key tile
  unsigned int boxes[kInfo];  // which of its boxes are there
  int odd[kSegments];         // a tree value of the part is not finite
  uint32_t begun[12];         // uses of a ring entry that were begun
};

template <int kDim, bool kPair>
struct Shape {
  static constexpr int kTileBytes = kKeys * kDim * 2;  // K, V, and 128 rows of Q
  static constexpr int kQBytes = (kPair ? 2 : 1) * kTileBytes;
  // Q of the next part is brought while this one runs, where two fit
  static constexpr int kQBufs = kPair && kDim == 128 ? 1 : 2;
  static constexpr int kSlots = kDim == 64 ? 10 : 5;
  static constexpr int kRing = kQBufs * kQBytes;
  static constexpr int kControl = kRing + kSlots * kTileBytes;
  static constexpr int kMl = kControl + static_cast<int>(sizeof(Control));  // a slot's (maximum, sum) of each row
  static constexpr int kSmem = kMl + (kPair ? 0 : 2 * 128 * 8);
  static constexpr int kRows = kPair ? 256 : 128;
  // Tensor memory, 512 columns: S_t at 128 t, O_t behind both.  At dimension 64
  // there is room for P_t beside S_t, so the next S_t is made while P_t is; at
  // 128 P_t overwrites S_t.
  static constexpr bool kOwnP = kDim == 64;
  static constexpr int kColO = 256, kColP = kOwnP ? 256 + 2 * kDim : 0;
  static constexpr int kStrideP = kOwnP ? 64 : 128;
  static_assert(kSmem <= 227 * 1024, "shared memory of a block");
  static_assert(kSlots <= 12, "control block");
};

// Whether row `row` of (b, head) sees tree key j < n_own.
__device__ __forceinline__ bool sees(const Params& p, int b, int row, int j) {
  if (row >= p.rows) return false;
  const int t = p.by_tokens.mod(row);
  return p.mask == nullptr ? j <= t : p.mask[b * p.mask_batch + t * p.mask_row + j] != 0;
}

// Steps of 16 keys that the product with V takes; one at least, which makes zeros.
__device__ __forceinline__ int value_steps(int keys) { return max(1, (keys + 15) / 16); }

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
  // a page's part that one copy brings: 2^box_shift rows; this lane's of a tile
  int box_shift;
  unsigned int every_row;  // the boxes of a tile's rows
  int my_row, my_half;     // my_half < 0: none
  uint32_t my_dst;

  __device__ __forceinline__ uint32_t slot_at(uint32_t i) const {
    return base + S::kRing + (i % S::kSlots) * S::kTileBytes;
  }
  __device__ __forceinline__ uint32_t full(uint32_t i) const { return smem_u32(&ctl->kv_full[i % S::kSlots]); }
  __device__ __forceinline__ uint32_t empty(uint32_t i) const { return smem_u32(&ctl->kv_empty[i % S::kSlots]); }
  static __device__ __forceinline__ uint32_t parity(uint32_t i) { return (i / S::kSlots) & 1; }

  // ------------------------------------------------------------- producer
  // Two producers, one for K and one for V: a tile takes a warp some 1000 clocks,
  // and at dimension 64 the bytes of both take 1400.  Lane l brings box
  // l % row_boxes, column half l / row_boxes.
  struct Spot {  // what a lane has to look up for its box, a tile before it is needed
    int page;    // as the table has it
    int row;     // first row of the box in the page; < 0: no box
  };

  __device__ __forceinline__ Spot look_up(const Segment& s, const int* table, int i) const {
    Spot spot = {0, -1};
    const int tile = s.tile0 + i, slot = tile * kKeys + my_row;
    if (i < s.n && tile < s.c_tiles && my_half >= 0 && slot < s.n_cache) {
      const int in_table = p.by_page.div(slot);
      spot.page = __ldg(table + in_table);
      spot.row = slot - in_table * p.pages.page_size;
    }
    return spot;
  }

  // Ring entries of a segment of n tiles: K_0 V_0 K_1 V_1 ... where a unit is a
  // pair; else K runs two tiles ahead, one for each slot: K_0 K_1 V_0 K_2 V_1 ...
  // V_{n-1}, two entries per V until K ends.
  static __device__ __forceinline__ uint32_t v_entry(int i, int n) {
    if (kPair) return static_cast<uint32_t>(2 * i + 1);
    return static_cast<uint32_t>((n > 1 ? 2 : 1) + (i + 2 < n ? 2 * i : i + min(i, max(n - 2, 0))));
  }
  static __device__ __forceinline__ uint32_t k_entry(int i, int n) {
    if (kPair) return static_cast<uint32_t>(2 * i);
    return i < 2 ? static_cast<uint32_t>(i) : v_entry(i - 2, n) + 1u;
  }

  // K or V of the segment's tile i into ring entry `entry`.
  template <bool kIsV>
  __device__ __forceinline__ bool bring(const Segment& s, int i, const Spot& spot, const CUtensorMap* map,
                                        uint32_t entry, uint32_t info, uint32_t segment, uint32_t& fixes) const {
    auto wait = [&](uint32_t bar, uint32_t par) {
      return mbar_wait_warp(bar, par, &ctl->abort, p.pages.status, kTimeoutProducer, p.limit_ns);
    };
    const uint32_t slot = entry % S::kSlots, use = entry / S::kSlots;
    const uint32_t bar = smem_u32(&ctl->kv_full[slot]), dst = base + S::kRing + slot * S::kTileBytes;
    if (use > 0 && !wait(smem_u32(&ctl->kv_empty[slot]), (use - 1) & 1)) return false;
    if (lane == 0) ctl->begun[slot] = use + 1;
    const int tile = s.tile0 + i;
    if (tile < s.c_tiles) {
      const int keys = min(s.n_cache - tile * kKeys, kKeys);
      const bool there = static_cast<unsigned>(spot.page) < static_cast<unsigned>(p.pages.num_pages);
      if (spot.row >= 0 && !there) atomicOr(p.pages.status, kStatusCache);
      const unsigned int have = __ballot_sync(0xffffffffu, spot.row >= 0 && there);
      const unsigned int here = have & every_row;
      const bool all = !kIsV || (keys == kKeys && here == every_row);
      const uint32_t to = all ? bar : smem_u32(&ctl->fix);
      const uint32_t bytes = __popc(have) << (box_shift + 7);
      if (lane == 0) {
        if (!kIsV) {
          ctl->keys[info % kInfo] = keys;
          ctl->boxes[info % kInfo] = here;
        }
        if (bytes > 0 || all) mbar_arrive_expect_tx(to, bytes);
      }
      __syncwarp();
      if ((have >> lane) & 1)
        tma_load_3d(dst + my_dst, map, to, my_half * 64, spot.row, spot.page * p.pages.kv_heads + s.head);
      if (!all) {
        // a tile that is not full: rows without a key become zeros, as far as the product reads
        if (bytes > 0) {
          if (!wait(to, fixes & 1)) {  // the copies land all the same
            if (lane == 0) {
              mbar_wait(to, fixes & 1, nullptr, p.pages.status, kTimeoutDrain, kDrainNs);
              mbar_arrive(bar);
            }
            return false;
          }
          ++fixes;
        }
        for (int v = lane; v < 16 * value_steps(keys) * kVecs; v += 32) {
          const int r = v / kVecs;
          if (r < keys && ((here >> (r >> box_shift)) & 1)) continue;
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
      const Rows& src = kIsV ? p.v_tree : p.k_tree;
      // a lane keeps its vector and goes down the rows, 2 or 4 at a time
      constexpr int kRowsAtOnce = 32 / kVecs;
      const int vec = lane % kVecs, r0 = lane / kVecs;
      const T* from = static_cast<const T*>(src.data) + s.b * src.batch + s.head * src.head +
                      static_cast<int64_t>(j0 + r0) * src.row + vec * 8;
#pragma unroll 4
      for (int r = r0; r < keys; r += kRowsAtOnce, from += kRowsAtOnce * src.row)
        copy16(dst + swizzled<kDim>(r, vec), from, true);
      // V behind the last key, as far as the product reads it; K there is hidden by selection
      if (kIsV)
        for (int r = keys + r0; r < 16 * value_steps(keys); r += kRowsAtOnce)
          *reinterpret_cast<uint4*>(smem + (dst - base) + swizzled<kDim>(r, vec)) = make_uint4(0, 0, 0, 0);
      copy_commit();
      copy_wait<0>();
      __syncwarp();
      if (kIsV) {
        unsigned int any = 0;
#pragma unroll 4
        for (int r = r0; r - r0 < keys; r += kRowsAtOnce) {  // the same steps in every lane
          uint4* at = reinterpret_cast<uint4*>(smem + (dst - base) + swizzled<kDim>(r, vec));
          bool bad = false;
          if (r < keys) {
            const uint4 x = *at;
            bad = not_finite2<T>(x.x) || not_finite2<T>(x.y) || not_finite2<T>(x.z) || not_finite2<T>(x.w);
          }
          // the lanes of a row are neighbours: 8 or 16 of them
          const unsigned int bits = __ballot_sync(0xffffffffu, bad);
          if (bits != 0) {
            any |= bits;
            const unsigned int mine = (bits >> (lane / kVecs * kVecs)) & ((1u << kVecs) - 1u);
            if (mine != 0) *at = make_uint4(0, 0, 0, 0);
          }
        }
        if (lane == 0 && any != 0) ctl->odd[segment % kSegments] = 1;
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        if (!kIsV) {
          ctl->keys[info % kInfo] = keys;
          ctl->boxes[info % kInfo] = ~0u;
        }
        mbar_arrive(bar);
      }
    }
    __syncwarp();
    return true;
  }

  // kWithQ: this warp brings the queries of the next part too, behind its last
  // tile of a part: the ring holds some tiles more while it does.
  template <bool kIsV, bool kWithQ>
  __device__ __forceinline__ bool produce(const CUtensorMap* map, Walk walk) const {
    uint32_t count = 0, tile_no = 0, fixes = 0, segment = 0;
    Segment s = {};
    Walk coming = walk;
    if (kWithQ) coming.next(p, s);  // the first part's come by the softmax warps
    while (walk.next(p, s)) {
      if (kIsV && lane == 0) ctl->odd[segment % kSegments] = 0;
      const int* table = p.pages.table + s.b * p.pages.table_stride;
      Spot spot = look_up(s, table, 0);
#pragma unroll 1
      for (int i = 0; i < s.n; ++i) {
        const Spot ahead = look_up(s, table, i + 1);
        if (!bring<kIsV>(s, i, spot, map, count + (kIsV ? v_entry(i, s.n) : k_entry(i, s.n)), tile_no + i, segment,
                         fixes))
          return false;
        spot = ahead;
      }
      count += 2 * s.n;
      tile_no += s.n;
      ++segment;
      if (kWithQ && coming.next(p, s) && !bring_queries(s, segment)) return false;
    }
    return true;
  }

  // Once all roles are through and one of them gave up: the copies that were begun land
  // before the block leaves, whether their producer gave up or had no more to bring.  Every
  // use that was begun fills its barrier.
  __device__ __forceinline__ void drain() const {
#pragma unroll 1
    for (int slot = 0; slot < S::kSlots; ++slot)
      if (ctl->begun[slot] != 0)
        mbar_wait(smem_u32(&ctl->kv_full[slot]), (ctl->begun[slot] - 1) & 1, nullptr, p.pages.status, kTimeoutDrain,
                  kDrainNs);
  }

  // Q of a part: rows of the unit, zeros where there is none, by threads
  // `first`, `first` + 1 ... of `threads`.
  __device__ __forceinline__ void bring_q(const Segment& s, uint32_t buf, int first, int threads) const {
#pragma unroll 4
    for (int v = first; v < S::kRows * kVecs; v += threads) {
      const int r = v / kVecs, vec = v % kVecs, row = s.row0 + r;
      const int hg = p.by_tokens.div(row), t = row - hg * p.tokens;
      const bool there = row < p.rows && t < s.n_own;
      const T* src = static_cast<const T*>(p.q.data) + s.b * p.q.batch +
                     (static_cast<int64_t>(s.head) * p.group + (there ? hg : 0)) * p.q.head + (there ? t : 0) * p.q.row;
      copy16(base + buf * S::kQBytes + (r / 128) * S::kTileBytes + swizzled<kDim>(r % 128, vec), src + vec * 8, there);
    }
    copy_commit();
    copy_wait<0>();
    fence_proxy_async_smem();
    __syncwarp();
  }

  // Those of part `segment` > 0, by one warp.
  __device__ __forceinline__ bool bring_queries(const Segment& s, uint32_t segment) const {
    const uint32_t buf = segment % S::kQBufs, use = segment / S::kQBufs;
    if (use > 0 && !mbar_wait_warp(smem_u32(&ctl->q_empty[buf]), (use - 1) & 1, &ctl->abort, p.pages.status,
                                   kTimeoutProducer, p.limit_ns))
      return false;
    bring_q(s, buf, lane, 32);
    if (lane == 0)
      for (int i = 0; i < 8; ++i) mbar_arrive(smem_u32(&ctl->q_full[buf]));
    return true;
  }

  __device__ __forceinline__ void bring_all_queries(Walk walk) const {
    Segment s = {};
    for (uint32_t segment = 0; walk.next(p, s); ++segment)
      if (segment > 0 && !bring_queries(s, segment)) return;
  }

  // --------------------------------------------------------------- issuer
  // kS, kV: which products this warp issues.  With room for P beside S they have
  // a warp each, so that neither waits for what the other waits for; else one
  // warp issues both and their order in the tensor pipe keeps S_t's next product
  // behind the one that reads P_t.
  template <bool kS, bool kV>
  __device__ __forceinline__ bool issue(Walk walk) const {
    constexpr uint32_t kType = std::is_same<T, __nv_bfloat16>::value ? (1u << 7) | (1u << 10) : 0u;
    constexpr uint32_t kIdS = idesc_f16_f32(128, kKeys, false) | kType;
    constexpr uint32_t kIdO = idesc_f16_f32(128, kDim, true) | kType;
    uint32_t count = 0, segment = 0, p_count[2] = {0, 0}, s_count[2] = {0, 0};
    Segment s = {};
    auto wait = [&](uint32_t bar, uint32_t par) {
      return mbar_wait_warp(bar, par, &ctl->abort, p.pages.status, kTimeoutMma, p.limit_ns);
    };
    auto wait_kv = [&](uint32_t i) {
      if (!wait(full(i), parity(i))) return false;
      tc_fence_after();
      return true;
    };
    // S_t = Q K^T; `last`: Q is not needed after the slots' last product
    auto scores = [&](int t, uint32_t k, bool last) {
      if (S::kOwnP) {
        if (!wait(smem_u32(&ctl->s_empty[t]), (s_count[t] & 1) ^ 1)) return false;
        ++s_count[t];
        tc_fence_after();
      }
      if (elect_one()) {
        const uint32_t q = base + ((segment - 1) % S::kQBufs) * S::kQBytes + (kPair ? t * S::kTileBytes : 0);
#pragma unroll
        for (int kk = 0; kk < kDim / 16; ++kk) {  // 16 elements are 32 bytes; 64 are a half
          const uint32_t at = (kk / 4) * (kKeys * 128) + (kk % 4) * 32;
          mma_ss_f16(tmem + t * 128, smem_desc_sw128(q + at, 16, 1024),
                     smem_desc_sw128(slot_at(k) + at, 16, 1024), kIdS, kk > 0);
        }
        tc_commit(smem_u32(&ctl->s_full[t]));
        if (last) tc_commit(smem_u32(&ctl->q_empty[(segment - 1) % S::kQBufs]));
      }
      __syncwarp();
      return true;
    };
    auto values = [&](int t, uint32_t v, int i, bool more, bool last) {  // O_t (+)= P_t V of tile i
      const int tile = s.tile0 + i;
      const int steps = value_steps(tile < s.c_tiles ? min(s.n_cache - tile * kKeys, kKeys)
                                    : p.tree ? min(s.n_own - (tile - s.c_tiles) * kKeys, kKeys)
                                             : 0);
      if (!wait(smem_u32(&ctl->p_full[t]), p_count[t] & 1)) return false;
      ++p_count[t];
      tc_fence_after();
      if (elect_one()) {
        // V lies with the elements along its rows: column halves of 64 are one
        // tile half apart (leading offset), eight keys 1 KiB (stride offset).  One
        // product over all kDim columns: two of 64 take as long each.
#pragma unroll
        for (int kk = 0; kk < kKeys / 16; ++kk)  // 16 keys: 8 columns of P, 2 KiB of V
          if (kk < steps)
            mma_ts_f16(tmem + S::kColO + t * kDim, tmem + S::kColP + t * S::kStrideP + kk * 8,
                     smem_desc_sw128(slot_at(v) + kk * 2048, kKeys * 128, 1024), kIdO, (more || kk > 0) ? 1u : 0u);
        if (S::kOwnP || last) tc_commit(smem_u32(&ctl->o_done[t]));
      }
      __syncwarp();
      return true;
    };
    auto release = [&](uint32_t i) {
      if (elect_one()) tc_commit(empty(i));
      __syncwarp();
    };

    while (walk.next(p, s)) {
      if (kS) {
        if (!wait(smem_u32(&ctl->q_full[segment % S::kQBufs]), (segment / S::kQBufs) & 1)) return false;
        ++segment;
        tc_fence_after();
      }
      if (kPair) {
        for (int i = 0; i <= s.n; ++i) {
          const uint32_t k = count + k_entry(i, s.n), v = count + v_entry(i - 1, s.n);  // V of the tile before
          if (kS && i < s.n && !wait_kv(k)) return false;
          if (kV && i > 0 && !wait_kv(v)) return false;
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            if (kV && i > 0 && !values(t, v, i - 1, i > 1, i == s.n)) return false;
            if (kS && i < s.n && !scores(t, k, t == 1 && i == s.n - 1)) return false;
          }
          if (kV && i > 0) release(v);
          if (kS && i < s.n) release(k);
        }
      } else {
        for (int i = -2; i < s.n; ++i) {
          const int t = i & 1, j = i + 2;
          if (kV && i >= 0) {
            const uint32_t v = count + v_entry(i, s.n);
            if (!wait_kv(v) || !values(t, v, i, i > 1, j >= s.n)) return false;
            release(v);
          }
          if (kS && j < s.n) {
            const uint32_t k = count + k_entry(j, s.n);
            if (!wait_kv(k) || !scores(t, k, j == s.n - 1)) return false;
            release(k);
          }
        }
      }
      count += 2 * s.n;
    }
    return true;
  }

  // -------------------------------------------------------------- softmax
  // Which keys of a tile that is not plain row `row` sees: bit e of words[c] for
  // key 32 c + e.  own_tile: the tile's number among those of the tree, < 0 for
  // cached keys.
  __device__ __forceinline__ void seen_keys(int b, int own_tile, int row, int keys, unsigned int boxes,
                                            uint64_t (&words)[2]) const {
    words[0] = words[1] = 0;
    const int t = row < p.rows ? p.by_tokens.mod(row) : -1;
#pragma unroll 1
    for (int c = 0; c < 4; ++c) {
      const int key0 = c * 32, n = min(keys - key0, 32);
      if (n <= 0) break;
      uint32_t seen = 0;
      if (own_tile < 0) {
#pragma unroll
        for (int e = 0; e < 32; e += 16)  // a box has at least 16 rows
          if ((boxes >> ((key0 + e) >> box_shift)) & 1) seen |= 0xffffu << e;
      } else if (t >= 0) {
        const int j = own_tile * kKeys + key0;
        if (p.mask == nullptr) {
          const int last = t - j;  // the last one seen
          seen = last < 0 ? 0u : last >= 31 ? ~0u : (2u << last) - 1u;
        } else {
          const unsigned char* m = p.mask + b * p.mask_batch + t * p.mask_row + j;
          if (n == 32 && (reinterpret_cast<uintptr_t>(m) & 3) == 0) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {  // four truth values: bytes 0 or 1 to neighbouring bits
              const uint32_t x = __vsetne4(__ldg(reinterpret_cast<const uint32_t*>(m) + e), 0u);
              seen |= ((x * 0x01020408u) >> 24) << (4 * e);
            }
          } else {
#pragma unroll 8
            for (int e = 0; e < n; ++e) seen |= (m[e] != 0 ? 1u : 0u) << e;
          }
        }
      }
      if (n < 32) seen &= (1u << n) - 1u;
      const uint64_t word = static_cast<uint64_t>(seen) << (32 * (c & 1));
      words[0] |= c < 2 ? word : 0;
      words[1] |= c < 2 ? 0 : word;
    }
  }

  // The tree values that are not finite, added to 16 columns of a row's sums.
  __device__ __forceinline__ void add_odd(const Segment& s, int row, int col0, float ref, uint32_t (&o)[16]) const {
    const int j0 = max(s.tile0 - s.c_tiles, 0) * kKeys;  // tree keys of the part
    const int j1 = min((s.tile0 + s.n - s.c_tiles) * kKeys, s.n_own);
    const int hg = p.by_tokens.div(row), t = row - hg * p.tokens;
    if (row >= p.rows || t >= s.n_own) return;
    const uint32_t* q = reinterpret_cast<const uint32_t*>(
        static_cast<const T*>(p.q.data) + s.b * p.q.batch + (static_cast<int64_t>(s.head) * p.group + hg) * p.q.head +
        t * p.q.row);
#pragma unroll 1
    for (int j = j0; j < j1; ++j) {
      const uint32_t* k = reinterpret_cast<const uint32_t*>(
          static_cast<const T*>(p.k_tree.data) + s.b * p.k_tree.batch + s.head * p.k_tree.head + j * p.k_tree.row);
      const uint32_t* v = reinterpret_cast<const uint32_t*>(
          static_cast<const T*>(p.v_tree.data) + s.b * p.v_tree.batch + s.head * p.v_tree.head + j * p.v_tree.row);
      bool bad = false;
#pragma unroll 1
      for (int i = 0; i < kDim / 2; ++i) bad = bad || not_finite2<T>(v[i]);
      if (!bad || !sees(p, s.b, row, j)) continue;
      float score = 0.0f;
#pragma unroll 1
      for (int i = 0; i < kDim / 2; ++i) {
        const float2 a = unpack2<T>(q[i]), c = unpack2<T>(k[i]);
        score = fmaf(a.x, c.x, fmaf(a.y, c.y, score));
      }
      const float w = ex2_approx(fmaf(score, p.scale_log2, -ref));
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float2 x = unpack2<T>(v[col0 / 2 + i]);
        o[2 * i] = __float_as_uint(fmaf(w, x.x, __uint_as_float(o[2 * i])));
        o[2 * i + 1] = __float_as_uint(fmaf(w, x.y, __uint_as_float(o[2 * i + 1])));
      }
    }
  }

  // 16 columns of a row's sums: final, or as this part's share.  Short pieces, as
  // what runs once a part is fetched anew each time: 256 units of 64 rows over 256
  // to 512 keys at dimension 128 took 39 us with 32 columns at a time, 36 with 16.
  __device__ __forceinline__ void write(const Segment& s, int row, int col0, float m, float l, const float* o) const {
    if (row >= p.rows) return;
    const int64_t at = (static_cast<int64_t>(s.b) * p.heads + static_cast<int64_t>(s.head) * p.group) * p.tokens + row;
    const int r = row - s.row0;
    if (s.whole) {
      const bool nothing = l == 0.0f || p.by_tokens.mod(row) >= s.n_own;
      const float inv = 1.0f / l;
      uint4* out = reinterpret_cast<uint4*>(static_cast<T*>(p.out) + at * kDim + col0);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        uint32_t w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e)
          w[e] = nothing ? 0u : pack2<T>(o[8 * i + 2 * e] * inv, o[8 * i + 2 * e + 1] * inv);
        out[i] = make_uint4(w[0], w[1], w[2], w[3]);
      }
      if (col0 == 0) p.lse[at] = nothing ? -INFINITY : 0.69314718055994531f * (m + log2f(l));
    } else {
      // lanes are rows: 512 bytes of a warp lie together
      float4* out = p.part_o + (static_cast<int64_t>(s.part) * (kDim / 4) + col0 / 4) * S::kRows + r;
#pragma unroll
      for (int i = 0; i < 4; ++i) out[i * S::kRows] = make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
      if (col0 == 0) p.part_ml[static_cast<int64_t>(s.part) * S::kRows + r] = make_float2(m, l);
    }
  }

  __device__ __forceinline__ bool soften(Walk walk, int t, int warp_in_slot) const {
    const int r = warp_in_slot * 32 + lane;  // row of the slot's tile
    const uint32_t lanes = static_cast<uint32_t>(warp_in_slot * 32) << 16;
    const uint32_t t_s = tmem + lanes + t * 128, t_o = tmem + lanes + S::kColO + t * kDim;
    const uint32_t t_p = tmem + lanes + S::kColP + t * S::kStrideP;
    uint32_t s_count = 0, o_count = 0, syncs = 0, segment = 0, tile_no = 0, turns = 0;
    Segment s = {};
    auto wait = [&](uint32_t bar, uint32_t par) {
      return mbar_wait_warp(bar, par, &ctl->abort, p.pages.status, kTimeoutSoftmax, p.limit_ns);
    };
    auto sync = [&]() {  // the eight softmax warps
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&ctl->sync));
      return wait(smem_u32(&ctl->sync), syncs++ & 1);
    };

    // The two warps of a scheduler, one of each slot, take turns at its exponential
    // unit, so that one's load of S, maximum and store of P run under the other's
    // exponentials.  Only where both slots see every tile: else a slot's own chain
    // from S to P is what bounds it, and waiting for turns took 52 us for 47.
    const uint32_t my_turn = smem_u32(&ctl->turn[t * 4 + warp_in_slot]);
    const uint32_t their_turn = smem_u32(&ctl->turn[(t ^ 1) * 4 + warp_in_slot]);
    auto take_turn = [&]() { return !kPair || wait(my_turn, (turns++ & 1) ^ (t == 0 ? 1u : 0u)); };
    auto pass_turn = [&]() {
      if (!kPair) return;
      __syncwarp();
      if (lane == 0) mbar_arrive(their_turn);
    };

    while (walk.next(p, s)) {
      if (segment == 0) {  // the first Q by all eight warps, the others ahead of time
        bring_q(s, 0, t * 128 + warp_in_slot * 32 + lane, 256);
        if (lane == 0) mbar_arrive(smem_u32(&ctl->q_full[0]));
      }

      const int row = s.row0 + (kPair ? t * 128 : 0) + r;
      // a warp without rows passes its turns; what it leaves reaches only its own rows
      const bool idle = s.row0 + (kPair ? t * 128 : 0) + warp_in_slot * 32 >= p.rows;
      // the row of the mask that the part's last tile will need, to be there by then
      if (!idle && p.mask != nullptr && s.tile0 + s.n > s.c_tiles && row < p.rows) {
        const unsigned char* at = p.mask + s.b * p.mask_batch + p.by_tokens.mod(row) * p.mask_row +
                                  (s.tile0 + s.n - 1 - s.c_tiles) * kKeys;
        asm volatile("prefetch.global.L1 [%0];" ::"l"(at));
      }
      float m = -INFINITY, l = 0.0f;
      bool first = true;
      for (int i = kPair ? 0 : t; i < s.n; i += kPair ? 1 : 2) {
        if (!wait(smem_u32(&ctl->s_full[t]), s_count++ & 1)) return false;
        tc_fence_after();
        if (!idle) {
          const int tile = s.tile0 + i;
          const int keys = *static_cast<volatile int*>(&ctl->keys[(tile_no + i) % kInfo]);
          const unsigned int boxes = *static_cast<volatile unsigned int*>(&ctl->boxes[(tile_no + i) % kInfo]);
          const unsigned int all = p.box_rows >= kKeys ? 1u : (1u << (kKeys / p.box_rows)) - 1u;
          const bool plain = tile < s.c_tiles && keys == kKeys && (boxes & all) == all;
          uint64_t seen[2] = {0, 0};
          if (!plain) {
            seen_keys(s.b, tile - s.c_tiles, row, keys, boxes, seen);
            __syncwarp();
          }
          uint32_t x[128];
#pragma unroll
          for (int c = 0; c < 4; ++c) tmem_ld32(t_s + c * 32, x + c * 32);
#pragma unroll
          for (int c = 0; c < 4; ++c) tc_wait_ld32(x + c * 32);
          if (S::kOwnP) {  // S_t may be made anew
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&ctl->s_empty[t]));
          }
          if (!plain) {
#pragma unroll
            for (int c = 0; c < 4; ++c)
#pragma unroll
              for (int e = 0; e < 32; ++e)
                if (!((seen[c >> 1] >> (32 * (c & 1) + e)) & 1)) x[c * 32 + e] = 0xff800000u;  // -inf
          }
          float top[8];
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            top[k] = __uint_as_float(x[16 * k]);
#pragma unroll
            for (int e = 1; e + 1 < 16; e += 2)
              top[k] = max3f(top[k], __uint_as_float(x[16 * k + e]), __uint_as_float(x[16 * k + e + 1]));
            top[k] = fmaxf(top[k], __uint_as_float(x[16 * k + 15]));
          }
          const float now = max3f(max3f(top[0], top[1], top[2]), max3f(top[3], top[4], top[5]),
                                  fmaxf(top[6], top[7])) * p.scale_log2;
          const bool grow = now > m + 8.0f;
          float shrink = 1.0f;
          if (first) {
            m = now;
          } else if (grow) {
            shrink = ex2_approx(m - now);
            m = now;
            l *= shrink;
          }
          const float ref = m == -INFINITY ? 0.0f : m;
          if (!take_turn()) return false;
          uint32_t packed[64];
          float sum[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
          for (int e = 0; e < 64; ++e) {
            if (e == 48) pass_turn();  // the other's first ones are under way when these end
            float a, b;
            ffma2(a, b, __uint_as_float(x[2 * e]), __uint_as_float(x[2 * e + 1]), p.scale_log2, p.scale_log2, -ref,
                  -ref);
            a = ex2_approx(a);
            b = ex2_approx(b);
            fadd2(sum[(e & 3) * 2], sum[(e & 3) * 2 + 1], sum[(e & 3) * 2], sum[(e & 3) * 2 + 1], a, b);
            packed[e] = pack2<T>(a, b);
          }
          l += ((sum[0] + sum[1]) + (sum[2] + sum[3])) + ((sum[4] + sum[5]) + (sum[6] + sum[7]));
          // The product with the last P_t is done: its own barrier says so, or S_t's,
          // which is made behind it.
          if (S::kOwnP && !first) {
            if (!wait(smem_u32(&ctl->o_done[t]), o_count++ & 1)) return false;
            tc_fence_after();
          }
          if (!first && __any_sync(0xffffffffu, grow)) {
#pragma unroll 1
            for (int c = 0; c < kDim / 32; ++c) {
              uint32_t o[32];
              tmem_ld32(t_o + c * 32, o);
              tc_wait_ld32(o);
#pragma unroll
              for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * shrink);
              tmem_st32(t_o + c * 32, o);
            }
          }
          tmem_st32(t_p, packed);
          tmem_st32(t_p + 32, packed + 32);
          tc_wait_st();
        } else {
          if (!take_turn()) return false;
          pass_turn();
          if (S::kOwnP) {
            if (lane == 0) mbar_arrive(smem_u32(&ctl->s_empty[t]));
            if (!first && !wait(smem_u32(&ctl->o_done[t]), o_count++ & 1)) return false;
          }
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
      // known once the part's last product is done, which one slot alone does not know
      auto any_odd = [&]() {
        return s.tile0 + s.n > s.c_tiles && *static_cast<volatile int*>(&ctl->odd[segment % kSegments]) != 0;
      };
      if (kPair) {
        const bool odd = any_odd();
        if (!idle) {
#pragma unroll 1
          for (int c = 0; c < kDim / 16; ++c) {
            uint32_t o[16];
            __syncwarp();
            tmem_ld16(t_o + c * 16, o);
            tc_wait_ld16(o);
            if (odd) add_odd(s, row, c * 16, m == -INFINITY ? 0.0f : m, o);
            write(s, row, c * 16, m, l, reinterpret_cast<const float*>(o));
          }
        }
        tc_fence_before();
      } else {
        float2* ml = reinterpret_cast<float2*>(smem + S::kMl);
        ml[t * 128 + r] = make_float2(m, l);
        tc_fence_before();
        if (!sync()) return false;
        tc_fence_after();
        const bool odd = any_odd();
        if (!idle) {
          const float2 a = ml[r], b = ml[128 + r];
          const float top = fmaxf(a.x, b.x), ref = top == -INFINITY ? 0.0f : top;
          const float fa = ex2_approx(a.x - ref), fb = ex2_approx(b.x - ref);
          const float sum = fa * a.y + fb * b.y;
#pragma unroll 1
          for (int c = t * (kDim / 32); c < (t + 1) * (kDim / 32); ++c) {
            uint32_t o0[16], o1[16];
            const uint32_t from = tmem + lanes + S::kColO + c * 16;
            __syncwarp();
            tmem_ld16(from, o0);
            if (s.n > 1) tmem_ld16(from + kDim, o1);  // else slot 1 has no sums
            tc_wait_ld16(o0);
            if (s.n > 1) {
              tc_wait_ld16(o1);
#pragma unroll
              for (int e = 0; e < 16; ++e)
                o0[e] = __float_as_uint(fa * __uint_as_float(o0[e]) + fb * __uint_as_float(o1[e]));
            } else {
#pragma unroll
              for (int e = 0; e < 16; ++e) o0[e] = __float_as_uint(fa * __uint_as_float(o0[e]));
            }
            if (odd) add_odd(s, row, c * 16, ref, o0);
            write(s, row, c * 16, top, sum, reinterpret_cast<const float*>(o0));
          }
        }
        tc_fence_before();
        // both slots' O have been read before the next part's products
        if (!sync()) return false;
        tc_fence_after();
      }
      ++segment;
    }
    return true;
  }
};

template <typename T, int kDim, bool kPair>
__global__ void __launch_bounds__(kThreads, 1)
    tile_kernel(const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mv, const Params p) {
  using S = Shape<kDim, kPair>;
  extern __shared__ __align__(1024) unsigned char smem[];  // swizzled tiles begin at multiples of 1 KiB
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const uint32_t base = smem_u32(smem);
  if ((base & 1023u) != 0) {  // the same in every thread
    if (threadIdx.x == 0) atomicOr(p.pages.status, kTimeoutProducer);
    return;
  }
  Control* ctl = reinterpret_cast<Control*>(smem + S::kControl);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&ctl->q_full[i]), 8);
      mbar_init(smem_u32(&ctl->q_empty[i]), 1);
    }
    for (int i = 0; i < 8; ++i) mbar_init(smem_u32(&ctl->turn[i]), 1);
    mbar_init(smem_u32(&ctl->fix), 1);
    mbar_init(smem_u32(&ctl->sync), 8);
    mbar_init(smem_u32(&ctl->drain), 1);
    mbar_init(smem_u32(&ctl->drain_v), 1);
    for (int i = 0; i < S::kSlots; ++i) {
      mbar_init(smem_u32(&ctl->kv_full[i]), 1);
      mbar_init(smem_u32(&ctl->kv_empty[i]), 1);
      ctl->begun[i] = 0;
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(smem_u32(&ctl->s_full[t]), 1);
      mbar_init(smem_u32(&ctl->s_empty[t]), 4);
      mbar_init(smem_u32(&ctl->p_full[t]), 4);
      mbar_init(smem_u32(&ctl->o_done[t]), 1);
    }
    ctl->abort = 0;
    fence_mbar_init();
  }
  if (warp == kProducer && lane == 0 && p.pages.slots() > 0 && p.pages.num_pages > 0) {  // else there are no maps
    tma_prefetch_desc(&mk);
    tma_prefetch_desc(&mv);
  }
  if (warp == kIssuer) {
    tmem_alloc(smem_u32(&ctl->tmem), 512);
    tmem_relinquish();
  }
  const Walk walk(p, lay_out(p, static_cast<int>(blockIdx.x), 0));
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const int box_shift = 31 - __clz(p.box_rows), row_boxes = kKeys >> box_shift;  // at most 8
  const int half = lane / row_boxes, my_row = (lane - half * row_boxes) << box_shift;
  const Block<T, kDim, kPair> block{p,         ctl,    smem,
                                    base,      ctl->tmem, lane,
                                    box_shift, (1u << row_boxes) - 1u, my_row,
                                    half < kDim / 64 ? half : -1, static_cast<uint32_t>(half * (kKeys * 128) + my_row * 128)};

  // the softmax warps take registers that the third warpgroup gives up:
  // 2 x 128 x 208 + 128 x 88 = 384 x 168, the launch's allocation
  if (warp < 8)
    asm volatile("setmaxnreg.inc.sync.aligned.u32 208;" ::: "memory");
  else
    asm volatile("setmaxnreg.dec.sync.aligned.u32 88;" ::: "memory");
  if (warp < 8) {
    block.soften(walk, warp / 4, warp % 4);
  } else if (warp == kProducer) {
    block.template produce<false, false>(&mk, walk);
  } else if (warp == (S::kOwnP ? kBringer : kIssuerV)) {
    block.template produce<true, S::kOwnP>(&mv, walk);
  } else if (warp == kBringer) {
    block.bring_all_queries(walk);
  } else if (warp == kIssuer || (S::kOwnP && warp == kIssuerV)) {
    if (!S::kOwnP)
      block.template issue<true, true>(walk);
    else if (warp == kIssuer)
      block.template issue<true, false>(walk);
    else
      block.template issue<false, true>(walk);
    // products and the arrivals that follow them end before memory is freed
    if (lane == 0) {
      const uint32_t drain = smem_u32(warp == kIssuer ? &ctl->drain : &ctl->drain_v);
      tc_commit(drain);
      mbar_wait(drain, 0, nullptr, p.pages.status, kTimeoutDrain, kDrainNs);
    }
    __syncwarp();
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (threadIdx.x == 0 && *static_cast<volatile int*>(&ctl->abort) != 0) block.drain();
  if (warp == kIssuer) {
    tc_fence_after();
    tmem_dealloc(ctl->tmem, 512);
  }
}

}  // namespace tiles
}  // namespace tree
}  // namespace fa
