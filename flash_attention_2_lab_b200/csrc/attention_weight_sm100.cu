// The attention weight that cached keys gather, B200 (sm_100a):
//   weights[b, hk, s] += sum over the rows r of (b, hk) of
//                        exp(scale q_r . k_s - lse_r),
// rows being the query heads of the kv head times the tokens.
//
// Bound by HBM when the rows are few (K is read once, 2 * dim bytes per slot)
// and by the exponentials (16 per clock and SM) when they are many.  The
// product is taken as K Q^T, keys along the rows of the matrix instruction, so
// that a key's sum over the queries stays in the four lanes that hold its row:
// no exchange until the end, and one block, one warp and one order of adding
// for each key.  A block takes 256 keys of one (b, hk), each warp 32, held in
// registers, while the rows go by in shared memory 64 at a time; several
// blocks per SM overlap their loads.

#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>

#include "fa_host.h"
#include "fa_sm100.h"
#include "mma_sm80.cuh"
#include "paged_cache.cuh"
#include "sm100_ptx.cuh"

namespace fa {
namespace weight {

using namespace warp;

constexpr int kThreads = 256;
constexpr int kKeys = 256;   // of a block; a warp has 32
constexpr int kChunk = 64;   // rows in shared memory at a time

struct Params {
  Pages pages;
  const void* k_pages;
  Rows q;
  const float* lse;
  float* weights;
  int heads, group, tokens, rows;
  float scale_log2;
};

template <int kDim>
constexpr int smem_bytes(bool two) {
  return kKeys * kDim * 2 + (two ? 2 : 1) * (kChunk * kDim * 2 + kChunk * 4);
}

template <typename T, int kDim>
__global__ void __launch_bounds__(kThreads) weight_kernel(const Params p) {
  extern __shared__ __align__(128) unsigned char smem[];
  const int b = static_cast<int>(blockIdx.z), head = static_cast<int>(blockIdx.y);
  const int n = cache_length(p.pages, b);
  const int slot0 = static_cast<int>(blockIdx.x) * kKeys;
  if (slot0 >= n) return;
  constexpr int kVecs = kDim / 8;
  const int lane = threadIdx.x % 32, w = threadIdx.x / 32;
  const int g = lane / 4, q4 = lane % 4;
  const uint32_t k_at = ptx::smem_u32(smem);
  constexpr uint32_t kChunkBytes = kChunk * kDim * 2 + kChunk * 4;
  auto chunk_at = [&](int c) { return static_cast<uint32_t>(kKeys * kDim * 2) + (c & 1) * kChunkBytes; };

  // 256 keys: every 16 rows lie in one page; slots without a key are zeros
  for (int i = threadIdx.x; i < kKeys * kVecs; i += kThreads) {
    const int r = i / kVecs, vec = i % kVecs;
    const bool inside = slot0 + r < n;
    const int64_t row = inside ? cache_row(p.pages, b, head, slot0 + r) : -1;
    // without a row nothing is read, but every copy names an address
    const T* from = row >= 0 ? static_cast<const T*>(p.k_pages) + row : static_cast<const T*>(p.q.data);
    copy16(k_at + tile_at<kDim>(r, vec), from + vec * 8, row >= 0);
  }
  auto load_chunk = [&](int c) {
    const uint32_t dst = k_at + chunk_at(c);
    for (int i = threadIdx.x; i < kChunk * kVecs; i += kThreads) {
      const int r = i / kVecs, vec = i % kVecs, row = c * kChunk + r;
      const bool valid = row < p.rows;
      const int hg = valid ? row / p.tokens : 0, t = valid ? row - hg * p.tokens : 0;
      const T* src = static_cast<const T*>(p.q.data) + b * p.q.batch +
                     (static_cast<int64_t>(head) * p.group + hg) * p.q.head + t * p.q.row;
      copy16(dst + tile_at<kDim>(r, vec), src + vec * 8, valid);
    }
    float* lse = reinterpret_cast<float*>(smem + chunk_at(c) + kChunk * kDim * 2);
    for (int r = threadIdx.x; r < kChunk; r += kThreads) {
      const int row = c * kChunk + r;
      const float x = row < p.rows ? p.lse[(static_cast<int64_t>(b) * p.heads +
                                            static_cast<int64_t>(head) * p.group) * p.tokens + row]
                                   : -INFINITY;
      lse[r] = x * 1.4426950408889634f;  // -inf: the row saw nothing
    }
    copy_commit();
  };
  const int chunks = (p.rows + kChunk - 1) / kChunk;
  load_chunk(0);

  uint32_t k[2][kDim / 16][4];
  float sum[2][2] = {{0.0f, 0.0f}, {0.0f, 0.0f}};
  for (int c = 0; c < chunks; ++c) {
    if (c + 1 < chunks) {
      load_chunk(c + 1);
      copy_wait<1>();
    } else {
      copy_wait<0>();
    }
    __syncthreads();
    if (c == 0) {
#pragma unroll
      for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int kk = 0; kk < kDim / 16; ++kk)
          ldmatrix4(k[a][kk], k_at + tile_at<kDim>(w * 32 + a * 16 + (lane & 15), kk * 2 + (lane >> 4)));
    }
    const uint32_t q_at = k_at + chunk_at(c);
    const float* lse = reinterpret_cast<const float*>(smem + chunk_at(c) + kChunk * kDim * 2);
    const int here = min(kChunk, p.rows - c * kChunk);
    for (int r0 = 0; r0 < here; r0 += 8) {
      float s[2][4];
#pragma unroll
      for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[a][e] = 0.0f;
#pragma unroll
      for (int kk = 0; kk < kDim / 32; ++kk) {
        uint32_t q[4];
        ldmatrix4(q, q_at + tile_at<kDim>(r0 + (lane & 7), kk * 4 + (lane >> 3)));
#pragma unroll
        for (int a = 0; a < 2; ++a) {
          mma<T>(s[a], k[a][2 * kk], q[0], q[1]);
          mma<T>(s[a], k[a][2 * kk + 1], q[2], q[3]);
        }
      }
      const float2 l = *reinterpret_cast<const float2*>(lse + r0 + q4 * 2);
#pragma unroll
      for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float le = (e & 1) ? l.y : l.x;
          const float x = ptx::ex2_approx(fmaf(s[a][e], p.scale_log2, -le));
          sum[a][e >> 1] += le == -INFINITY ? 0.0f : x;
        }
    }
    __syncthreads();  // the chunk's buffer is filled again after next
  }
#pragma unroll
  for (int a = 0; a < 2; ++a)
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      float x = sum[a][half];
      x += __shfl_xor_sync(0xffffffffu, x, 1);
      x += __shfl_xor_sync(0xffffffffu, x, 2);
      const int slot = slot0 + w * 32 + a * 16 + half * 8 + g;
      if (q4 == 0 && slot < n && cache_row(p.pages, b, head, slot) >= 0)
        p.weights[(static_cast<int64_t>(b) * p.pages.kv_heads + head) * p.pages.slots() + slot] += x;
    }
}

template <typename T, int kDim>
cudaError_t launch(const Params& p, int batch, cudaStream_t stream) {
  const cudaError_t e =
      cudaFuncSetAttribute(reinterpret_cast<const void*>(&weight_kernel<T, kDim>),
                           cudaFuncAttributeMaxDynamicSharedMemorySize, smem_bytes<kDim>(true));
  if (e != cudaSuccess) return e;
  const dim3 grid((p.pages.slots() + kKeys - 1) / kKeys, p.pages.kv_heads, batch);
  weight_kernel<T, kDim><<<grid, kThreads, smem_bytes<kDim>(p.rows > kChunk), stream>>>(p);
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
  fa::host::Device d;
  if ((rc = fa::host::current_device(&d)) != FA_OK) return rc;
  p.pages.status = d.status;
  p.k_pages = cache->k_pages;
  p.lse = lse;
  p.weights = weights;
  p.heads = static_cast<int>(heads);
  p.group = p.heads / p.pages.kv_heads;
  p.tokens = static_cast<int>(tokens);
  p.rows = p.group * p.tokens;
  p.scale_log2 = scale * 1.4426950408889634f;
  cudaStream_t stream = static_cast<cudaStream_t>(cuda_stream);
  const int batch = static_cast<int>(cache->batch);
  cudaError_t e;
  if (p.pages.dim == 64)
    e = dtype == FA_FP16 ? fw::launch<__half, 64>(p, batch, stream)
                         : fw::launch<__nv_bfloat16, 64>(p, batch, stream);
  else
    e = dtype == FA_FP16 ? fw::launch<__half, 128>(p, batch, stream)
                         : fw::launch<__nv_bfloat16, 128>(p, batch, stream);
  if (e != cudaSuccess) return set_error(FA_ERR_CUDA, "kernel launch: %s", cudaGetErrorString(e));
  return FA_OK;
}
