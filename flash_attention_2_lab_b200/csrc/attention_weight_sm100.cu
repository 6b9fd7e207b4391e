// The attention weight that cached keys gather, B200 (sm_100a):
//   weights[b, hk, s] += sum over the rows r of (b, hk) of
//                        exp(scale q_r . k_s - lse_r),
// rows being the query heads of the kv head times the tokens.
//
// Bound by HBM while the rows are few (K is read once, 2 * dim bytes a slot), by
// the exponentials (16 per clock and SM) when they are many: 128 rows take 1024
// clocks of them per 128 keys, whose bytes take 700 (dimension 64) or 1400.
// 4 rows over 32 x 8 caches of 65536 keys at dimension 64, pages of 64: 365 us (6.2
// TB/s); 128 rows over 8 of 262144 at dimension 128: 116 us (4.8 TB/s).  11 to 14 us
// of a call do not depend on the length.
//
// The product is taken as S^T = K Q^T on tcgen05, 128 keys by up to 128 rows:
// in tensor memory a key is a lane and the rows are columns, so one thread adds
// up one key's weight, with no exchange between threads and in one fixed order.
// A block of twelve warps per SM walks its part of the line of key tiles: warps 8
// and 11 bring K tiles into a ring (one TMA box per piece of a page), warp 9 issues the
// products, warp 10 brings the rows of the next part, and warps 0-3 and 4-7 sum
// up even and odd key tiles, each with two tiles of S in tensor memory.
//
// Keys behind a sequence's length or in pages that do not exist are computed on
// whatever shared memory holds and not written; rows that saw nothing are left
// out by selection.

#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cstdint>
#include <type_traits>

#include "fa_host.h"
#include "fa_sm100.h"
#include "mma_sm80.cuh"
#include "paged_cache.cuh"
#include "sm100_ptx.cuh"
#include "tree_line.cuh"

namespace fa {
namespace weight {

using namespace ptx;
using tree::Segment;
using tree::Walk;

constexpr int kKeys = 128;      // of a tile
constexpr int kChunk = 128;     // rows of a product
constexpr int kThreads = 384;   // warps: 8 sum, then producer, issuer, bringer, second producer
constexpr int kProducer = 8, kIssuer = 9, kBringer = 10, kProducer2 = 11;
constexpr int kMaxSlots = 13;
constexpr unsigned int kTimeoutProducer = 1u, kTimeoutMma = 2u, kTimeoutSum = 4u, kTimeoutDrain = 8u;
constexpr unsigned long long kDrainNs = 200000000ull;

struct Params : tree::Params {
  const float* row_lse;  // [batch, heads, tokens]
  float* weights;        // [batch, kv_heads, slots]
  int chunks;            // of rows in shared memory
  int passes;            // over the keys, each with its chunks of rows
  int slots;             // entries of the ring
  int rows_at, ring_at, control_at;  // bytes: log-sum-exps, ring, control block
};

struct Control {
  uint64_t q_full[2], q_empty[2], drain;
  uint64_t k_full[kMaxSlots], k_empty[kMaxSlots];
  uint64_t s_full[4], s_empty[4];
  uint32_t begun[kMaxSlots];  // uses of a ring entry that were begun
  uint32_t tmem;
  int abort;
};

template <int kDim>
struct Sizes {
  static constexpr int kTileBytes = kKeys * kDim * 2;
  static constexpr int kMaxChunks = kDim == 64 ? 4 : 2;  // two buffers of 64 KiB
};

// Where the passes of a part begin: a role's loop over (part, pass).
struct Jobs {
  Walk walk;
  Segment s;
  int pass;
  __device__ __forceinline__ Jobs(const Walk& w) : walk(w), s(), pass(0) {}
  __device__ __forceinline__ bool next(const Params& p) {
    if (pass > 0 && pass < p.passes) {
      ++pass;
      return true;
    }
    pass = 1;
    return walk.next(p, s);
  }
  // rows [first(), first() + count()) of the unit
  __device__ __forceinline__ int first(const Params& p) const { return (pass - 1) * p.chunks * kChunk; }
  __device__ __forceinline__ int count(const Params& p) const { return min(p.rows - first(p), p.chunks * kChunk); }
};

template <typename T, int kDim>
__global__ void __launch_bounds__(kThreads, 1)
    weight_kernel(const __grid_constant__ CUtensorMap mk, const __grid_constant__ Params p) {
  using S = Sizes<kDim>;
  constexpr int kVecs = kDim / 8;
  extern __shared__ __align__(1024) unsigned char smem[];  // swizzled tiles begin at multiples of 1 KiB
  const uint32_t base = smem_u32(smem);
  if ((base & 1023u) != 0) {  // the same in every thread
    if (threadIdx.x == 0) atomicOr(p.pages.status, kTimeoutProducer);
    return;
  }
  Control* ctl = reinterpret_cast<Control*>(smem + p.control_at);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&ctl->q_full[i]), 1);
      mbar_init(smem_u32(&ctl->q_empty[i]), 9);  // the last product, and the warps that read the rows' lse
    }
    mbar_init(smem_u32(&ctl->drain), 1);
    for (int i = 0; i < p.slots; ++i) {
      mbar_init(smem_u32(&ctl->k_full[i]), 1);
      mbar_init(smem_u32(&ctl->k_empty[i]), 1);
      ctl->begun[i] = 0;
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(smem_u32(&ctl->s_full[i]), 1);
      mbar_init(smem_u32(&ctl->s_empty[i]), 4);
    }
    ctl->abort = 0;
    fence_mbar_init();
  }
  if (warp == kProducer && lane == 0 && p.pages.num_pages > 0) tma_prefetch_desc(&mk);
  if (warp == kIssuer) {
    tmem_alloc(smem_u32(&ctl->tmem), 512);
    tmem_relinquish();
  }
  const Walk walk(p, tree::lay_out(p, static_cast<int>(blockIdx.x), 0));
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = ctl->tmem;
  Jobs jobs(walk);
  auto wait = [&](uint32_t bar, uint32_t parity, unsigned int code) {
    return mbar_wait_warp(bar, parity, &ctl->abort, p.pages.status, code, p.limit_ns);
  };
  const uint32_t q_bytes = static_cast<uint32_t>(p.chunks) * S::kTileBytes;
  auto rows_of = [&](uint32_t job) {  // a job's log-sum-exps (-log2), then a bit for each row that counts
    return reinterpret_cast<float*>(smem + p.rows_at) + (job & 1) * p.chunks * (kChunk + kChunk / 32);
  };

  if (warp < 8) {
    // ------------------------------------------------------------------ sums
    const int w = warp / 4, r = (warp % 4) * 32 + lane;  // key of the tile
    const uint32_t lanes = static_cast<uint32_t>((warp % 4) * 32) << 16;
    uint32_t items = 0;
    bool ok = true;
    for (uint32_t job = 0; ok && jobs.next(p); ++job) {
      const Segment& s = jobs.s;
      const int count = jobs.count(p);
      const float* lse = rows_of(job);
      const uint32_t* bits = reinterpret_cast<const uint32_t*>(lse + p.chunks * kChunk);
      ok = wait(smem_u32(&ctl->q_full[job & 1]), (job >> 1) & 1, kTimeoutSum);
      for (int i = w; ok && i < s.n; i += 2) {
        const int slot = (s.tile0 + i) * kKeys + r;
        // a slot whose page does not exist has no weight
        bool there = slot < s.n_cache;
        if (there) {
          const int page = __ldg(p.pages.table + s.b * p.pages.table_stride + p.by_page.div(slot));
          there = static_cast<unsigned>(page) < static_cast<unsigned>(p.pages.num_pages);
        }
        float* at = p.weights + (static_cast<int64_t>(s.b) * p.pages.kv_heads + s.head) * p.pages.slots() + slot;
        const float before = there ? *at : 0.0f;
        float sum0 = 0.0f, sum1 = 0.0f, sum2 = 0.0f, sum3 = 0.0f;
        for (int c = 0; ok && c * kChunk < count; ++c) {
          const uint32_t buf = w * 2 + (items & 1);
          if (!(ok = wait(smem_u32(&ctl->s_full[buf]), (items >> 1) & 1, kTimeoutSum))) break;
          ++items;
          tc_fence_after();
          const int cols = min(count - c * kChunk, kChunk);
          const uint32_t from = tmem + lanes + buf * 128;
          // exp(scale s - lse) of N columns, added up pair by pair; `have`: which count
          auto add_up = [&](auto& x, const float* minus_lse, uint32_t have) {
            constexpr int kCols = static_cast<int>(sizeof(x) / 4);
            const bool all = have == (kCols == 32 ? ~0u : (1u << (kCols & 31)) - 1u);  // of the whole warp
#pragma unroll
            for (int e = 0; e < kCols / 4; ++e) {
              const float4 l = reinterpret_cast<const float4*>(minus_lse)[e];
              float v[4];
              ffma2(v[0], v[1], __uint_as_float(x[4 * e]), __uint_as_float(x[4 * e + 1]), p.scale_log2, p.scale_log2,
                    l.x, l.y);
              ffma2(v[2], v[3], __uint_as_float(x[4 * e + 2]), __uint_as_float(x[4 * e + 3]), p.scale_log2,
                    p.scale_log2, l.z, l.w);
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                v[j] = ex2_approx(v[j]);
                if (!all) v[j] = (have >> (4 * e + j)) & 1 ? v[j] : 0.0f;
              }
              fadd2(sum0, sum1, sum0, sum1, v[0], v[1]);
              fadd2(sum2, sum3, sum2, sum3, v[2], v[3]);
            }
          };
          const float* row = lse + c * kChunk;
          const uint32_t* have = bits + c * (kChunk / 32);
          if (cols <= 16) {
            uint32_t x[16];
            tmem_ld16(from, x);
            tc_wait_ld16(x);
            add_up(x, row, have[0] & 0xffffu);
          } else {
            uint32_t x[2][32];
            tmem_ld32(from, x[0]);
#pragma unroll 2
            for (int g = 0; g * 32 < cols; ++g) {
              tc_wait_ld32(x[g & 1]);
              if ((g + 1) * 32 < cols) tmem_ld32(from + (g + 1) * 32, x[(g + 1) & 1]);
              add_up(x[g & 1], row + g * 32, have[g]);
            }
          }
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_u32(&ctl->s_empty[buf]));
        }
        if (ok && there) *at = before + ((sum0 + sum1) + (sum2 + sum3));
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&ctl->q_empty[job & 1]));
    }
  } else if (warp == kProducer || warp == kProducer2) {
    // -------------------------------------------------------------- K tiles
    // Every other tile each: a tile takes a warp some 700 clocks, as long as its
    // bytes at dimension 64.  Lane l brings box l % row_boxes, column half l / row_boxes of every tile.
    const int box_shift = 31 - __clz(p.box_rows), row_boxes = kKeys >> box_shift;
    const int half = lane / row_boxes, my_row = (lane - half * row_boxes) << box_shift;
    const uint32_t my_dst = static_cast<uint32_t>(half * (kKeys * 128) + my_row * 128);
    struct Spot {
      int page, row;  // row < 0: no box
    };
    auto look_up = [&](const Segment& s, int i) {  // one tile ahead of its use
      Spot spot = {0, -1};
      const int slot = (s.tile0 + i) * kKeys + my_row;
      if (i < s.n && half < kDim / 64 && slot < s.n_cache) {
        const int in_table = p.by_page.div(slot);
        spot.page = __ldg(p.pages.table + s.b * p.pages.table_stride + in_table);
        spot.row = slot - in_table * p.pages.page_size;
      }
      return spot;
    };
    uint32_t count = 0, use = 0;  // of all tiles; this warp brings those of its parity
    const uint32_t mine = warp == kProducer ? 0u : 1u;
    int slot = 0;
    bool ok = true;
    while (ok && jobs.next(p)) {
      const Segment& s = jobs.s;
      Spot spot = look_up(s, static_cast<int>((count ^ mine) & 1));
      for (int i = 0; i < s.n; ++i) {
        if ((count & 1) == mine) {
          const Spot ahead = look_up(s, i + 2);
          if (use > 0 && !(ok = wait(smem_u32(&ctl->k_empty[slot]), (use - 1) & 1, kTimeoutProducer))) break;
          const bool there = static_cast<unsigned>(spot.page) < static_cast<unsigned>(p.pages.num_pages);
          if (spot.row >= 0 && !there) atomicOr(p.pages.status, kStatusCache);
          const unsigned int have = __ballot_sync(0xffffffffu, spot.row >= 0 && there);
          const uint32_t bar = smem_u32(&ctl->k_full[slot]);
          if (lane == 0) {
            ctl->begun[slot] = use + 1;
            mbar_arrive_expect_tx(bar, __popc(have) << (box_shift + 7));
          }
          __syncwarp();
          if ((have >> lane) & 1)
            tma_load_3d(base + p.ring_at + slot * S::kTileBytes + my_dst, &mk, bar, half * 64, spot.row,
                        spot.page * p.pages.kv_heads + s.head);
          __syncwarp();
          spot = ahead;
        }
        ++count;
        if (++slot == p.slots) {
          slot = 0;
          ++use;
        }
      }
    }
    __syncwarp();
  } else if (warp == kIssuer) {
    // ------------------------------------------------------------- products
    constexpr uint32_t kType = std::is_same<T, __nv_bfloat16>::value ? (1u << 7) | (1u << 10) : 0u;
    uint32_t items[2] = {0, 0}, use = 0;
    int slot = 0;
    bool ok = true;
    for (uint32_t job = 0; ok && jobs.next(p); ++job) {
      const Segment& s = jobs.s;
      const int count = jobs.count(p);
      if (!(ok = wait(smem_u32(&ctl->q_full[job & 1]), (job >> 1) & 1, kTimeoutMma))) break;
      tc_fence_after();
      const uint32_t q = base + (job & 1) * q_bytes;
      // two key tiles at a time, one for each half of the sum warps, chunk by chunk
      for (int i = 0; ok && i < s.n; i += 2) {
        const int two = min(s.n - i, 2);
        int at[2] = {slot, slot + 1 == p.slots ? 0 : slot + 1};
        uint32_t round[2] = {use, slot + 1 == p.slots ? use + 1 : use};
        for (int c = 0; ok && c * kChunk < count; ++c) {
          const uint32_t n = static_cast<uint32_t>(min(count - c * kChunk, kChunk) + 15) / 16 * 16;
          const uint32_t idesc = idesc_f16_f32(128, 0, false) | (n >> 3) << 17 | kType;
          const bool last = (c + 1) * kChunk >= count;
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            if (w >= two) break;
            if (c == 0 && !(ok = wait(smem_u32(&ctl->k_full[at[w]]), round[w] & 1, kTimeoutMma))) break;
            const uint32_t buf = w * 2 + (items[w] & 1);
            if (!(ok = wait(smem_u32(&ctl->s_empty[buf]), ((items[w] >> 1) & 1) ^ 1, kTimeoutMma))) break;
            ++items[w];
            tc_fence_after();
            if (elect_one()) {
              const uint32_t k = base + p.ring_at + at[w] * S::kTileBytes;
#pragma unroll
              for (int kk = 0; kk < kDim / 16; ++kk) {  // 16 elements are 32 bytes; 64 are a half
                const uint32_t off = (kk / 4) * (kKeys * 128) + (kk % 4) * 32;
                mma_ss_f16(tmem + buf * 128, smem_desc_sw128(k + off, 16, 1024),
                           smem_desc_sw128(q + c * S::kTileBytes + off, 16, 1024), idesc, kk > 0);
              }
              tc_commit(smem_u32(&ctl->s_full[buf]));
              if (last) tc_commit(smem_u32(&ctl->k_empty[at[w]]));
              if (last && i + w == s.n - 1) tc_commit(smem_u32(&ctl->q_empty[job & 1]));
            }
            __syncwarp();
          }
        }
        slot += two;
        if (slot >= p.slots) {
          slot -= p.slots;
          ++use;
        }
      }
    }
    // products and the arrivals that follow them end before memory is freed
    if (lane == 0) {
      tc_commit(smem_u32(&ctl->drain));
      mbar_wait(smem_u32(&ctl->drain), 0, nullptr, p.pages.status, kTimeoutDrain, kDrainNs);
    }
    __syncwarp();
  } else if (warp == kBringer) {
    // ------------------------------------- rows and their log-sum-exps, ahead
    for (uint32_t job = 0; jobs.next(p); ++job) {
      const Segment& s = jobs.s;
      const int first = jobs.first(p), count = jobs.count(p);
      if (job > 1 && !wait(smem_u32(&ctl->q_empty[job & 1]), ((job >> 1) - 1) & 1, kTimeoutProducer)) break;
      const uint32_t q = base + (job & 1) * q_bytes;
      const T* src = static_cast<const T*>(p.q.data) + s.b * p.q.batch + static_cast<int64_t>(s.head) * p.group * p.q.head;
      const int filled = (count + 15) / 16 * 16;
#pragma unroll 4
      for (int v = lane; v < filled * kVecs; v += 32) {
        const int r = v / kVecs, vec = v % kVecs, row = first + (r < count ? r : 0);
        const int hg = p.by_tokens.div(row), t = row - hg * p.tokens;
        const uint32_t off = (vec >> 3) * (kKeys * 128) + (r % kChunk) * 128 + (((vec & 7) ^ (r & 7)) << 4);
        warp::copy16(q + (r / kChunk) * S::kTileBytes + off, src + hg * p.q.head + t * p.q.row + vec * 8, r < count);
      }
      float* lse = rows_of(job);
      uint32_t* bits = reinterpret_cast<uint32_t*>(lse + p.chunks * kChunk);
      const float* from = p.row_lse + (static_cast<int64_t>(s.b) * p.heads + static_cast<int64_t>(s.head) * p.group) * p.tokens + first;
      for (int r0 = 0; r0 < (filled + 31) / 32 * 32; r0 += 32) {
        const int r = r0 + lane;
        const float x = r < count ? from[r] : -INFINITY;
        lse[r] = x == -INFINITY ? 0.0f : x * -1.4426950408889634f;
        const uint32_t have = __ballot_sync(0xffffffffu, x != -INFINITY);
        if (lane == 0) bits[r0 / 32] = have;
      }
      warp::copy_commit();
      warp::copy_wait<0>();
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&ctl->q_full[job & 1]));
      __syncwarp();
    }
  }
  tc_fence_before();
  __syncthreads();
  if (threadIdx.x == 0 && *static_cast<volatile int*>(&ctl->abort) != 0) {
    // all roles are through and one gave up: the copies that were begun land
    // before the block leaves, whoever has waited for them
#pragma unroll 1
    for (int i = 0; i < p.slots; ++i)
      if (ctl->begun[i] != 0)
        mbar_wait(smem_u32(&ctl->k_full[i]), (ctl->begun[i] - 1) & 1, nullptr, p.pages.status, kTimeoutDrain, kDrainNs);
  }
  if (warp == kIssuer) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

template <typename T, int kDim>
cudaError_t launch(Params& p, const CUtensorMap& mk, cudaStream_t stream) {
  using S = Sizes<kDim>;
  constexpr int kSmem = 227 * 1024;
  const int all = (p.rows + kChunk - 1) / kChunk;
  p.chunks = std::min(all, S::kMaxChunks);
  p.passes = (all + p.chunks - 1) / p.chunks;
  const int rows_bytes = 2 * p.chunks * (kChunk + kChunk / 32) * 4;
  const int fixed = 2 * p.chunks * S::kTileBytes + rows_bytes + static_cast<int>(sizeof(Control)) + 64;
  p.slots = std::min(kMaxSlots, (kSmem - fixed) / S::kTileBytes);
  p.ring_at = 2 * p.chunks * S::kTileBytes;
  p.rows_at = p.ring_at + p.slots * S::kTileBytes;
  p.control_at = (p.rows_at + rows_bytes + 15) & ~15;
  static std::atomic<uint64_t> allowed{0};
  const cudaError_t e =
      host::allow_smem(reinterpret_cast<const void*>(&weight_kernel<T, kDim>), kSmem, p.device, allowed);
  if (e != cudaSuccess) return e;
  const size_t smem = static_cast<size_t>(p.control_at) + sizeof(Control);
  weight_kernel<T, kDim><<<p.blocks, kThreads, smem, stream>>>(mk, p);
  return cudaGetLastError();
}

}  // namespace weight
}  // namespace fa

using fa::host::set_error;

extern "C" int fa_attention_weight_sm100(const fa_paged_cache* cache, const fa_rows* query,
                                         int64_t heads, int64_t tokens, const float* lse,
                                         float* weights, int dtype, float scale,
                                         void* cuda_stream) {
  namespace fw = fa::weight;
  fw::Params p = {};
  int rc = fa::check_pages(cache, &p.pages);
  if (rc != FA_OK) return rc;
  if ((rc = fa::check_queries(p.pages, cache->batch, heads, tokens, dtype, scale)) != FA_OK) return rc;
  if (cache->batch == 0 || heads == 0 || tokens == 0 || p.pages.slots() == 0) return FA_OK;
  if ((rc = fa::check_rows(query, "query", &p.q)) != FA_OK) return rc;
  if (lse == nullptr || weights == nullptr) return set_error(FA_ERR_INVALID, "null pointer");
  const int64_t units = cache->batch * cache->kv_heads;
  const int64_t longest = units * ((p.pages.slots() + fw::kKeys - 1) / fw::kKeys);
  if (longest + units * 4 > (1ll << 30)) return set_error(FA_ERR_INVALID, "size too large");
  fa::host::Device d;
  if ((rc = fa::host::current_device(&d)) != FA_OK) return rc;
  p.pages.status = d.status;
  p.k_pages = cache->k_pages;
  p.row_lse = lse;
  p.weights = weights;
  p.batch = static_cast<int>(cache->batch);
  p.heads = static_cast<int>(heads);
  p.group = p.heads / p.pages.kv_heads;
  p.tokens = static_cast<int>(tokens);
  p.rows = p.group * p.tokens;
  p.row_tiles = 1;
  p.units = p.pages.kv_heads;
  p.extra = 0;  // beginning a unit costs little here: 2, 4 and 8 measured no faster
  p.blocks = static_cast<int>(std::min<int64_t>(d.sms, longest + units * p.extra));
  p.tile_shift = 7;
  static_assert(fw::kKeys == 128, "tile_shift");
  p.unit_rows = p.rows;
  p.by_tokens = fa::tree::FastDiv(static_cast<uint32_t>(p.tokens));
  p.by_page = fa::tree::FastDiv(static_cast<uint32_t>(p.pages.page_size));
  p.by_row_tiles = fa::tree::FastDiv(1);
  p.by_blocks = fa::tree::FastDiv(static_cast<uint32_t>(p.blocks));
  p.limit_ns = fa::host::wait_limit_ns();
  p.device = d.index;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.box_rows = 16;  // of a page, a power of two that divides its size
  while (p.box_rows < fw::kKeys && p.pages.page_size % (2 * p.box_rows) == 0) p.box_rows *= 2;
  CUtensorMap mk = {};
  if (p.pages.num_pages > 0 &&
      (rc = fa::host::encode_rows_map(&mk, cache->k_pages, dtype == FA_BF16, cache->head_dim,
                                      cache->page_size, cache->num_pages * cache->kv_heads,
                                      static_cast<uint32_t>(p.box_rows))) != FA_OK)
    return rc;
  cudaStream_t stream = static_cast<cudaStream_t>(cuda_stream);
  cudaError_t e;
  if (p.pages.dim == 64)
    e = dtype == FA_FP16 ? fw::launch<__half, 64>(p, mk, stream)
                         : fw::launch<__nv_bfloat16, 64>(p, mk, stream);
  else
    e = dtype == FA_FP16 ? fw::launch<__half, 128>(p, mk, stream)
                         : fw::launch<__nv_bfloat16, 128>(p, mk, stream);
  if (e != cudaSuccess) return set_error(FA_ERR_CUDA, "kernel launch: %s", cudaGetErrorString(e));
  return FA_OK;
}
