// Rotary positions for B200 (sm_100a): queries and keys of one attention call
// turned by their positions in one launch.
//
// Of each row the first R elements form R/2 pairs, (i, i + R/2) or (2i, 2i+1);
// pair i of a token at position p turns by the angle a = p * frequency[i]:
//   x' = f * (x cos a - y sin a),   y' = f * (y cos a + x sin a),
// with one factor f; elements from R on are copied.  The transpose of that
// map, which the backward pass needs, is the same with -a.
//
// The angle is taken in 64 bits as a number of turns and reduced to [-1/2,
// 1/2] before it is rounded to 32: at position 2^20 a 32-bit angle is off by
// up to 0.06 rad, this one by 2e-7.  cos and sin of a token's pairs are the
// same for every head, so a thread computes those of its pairs once and walks
// over a group of heads with them.
//
// Bound by HBM: every element is read once and written once.  A thread holds
// two 16-byte vectors of one row (the two halves of its pairs) and relies on the
// number of threads for loads in flight: two or four rows at a time per thread
// measured slower (fp16, 4 x 32 heads x 8191 x 64, queries and keys: 85 us, 6.3
// TB/s, against 91 and 99; from rows of [B, N, H, D]: 94 against 102 and 110).

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cmath>
#include <cstdint>

#include "fa_host.h"
#include "fa_sm100.h"

namespace fa {
namespace rotary {

constexpr int kThreads = 128;

struct Side {
  const void* x;       // [batch, heads, tokens, dim], any strides, elements dense
  void* y;             // the same, contiguous
  int64_t sb, sh, sn;  // strides of x in elements
  int heads;
};

struct Params {
  Side side[2];              // queries, keys
  const void* positions;     // [batch, tokens], 32 or 64 bits
  int64_t pb, pn;            // strides of positions
  const double* frequencies; // radians a position, [pairs]
  int batch, tokens, dim, pairs;
  int slots;                 // threads of a row
  int group;                 // heads of a thread
  int groups0;               // head groups of side 0; those after it belong to side 1
  int wide_positions, interleaved;
  float factor, sign;
};

template <typename T>
__device__ __forceinline__ float to_float(T x);
template <>
__device__ __forceinline__ float to_float(float x) { return x; }
template <>
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
template <>
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T>
__device__ __forceinline__ T from_float(float x);
template <>
__device__ __forceinline__ float from_float(float x) { return x; }
template <>
__device__ __forceinline__ __half from_float(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float(float x) { return __float2bfloat16_rn(x); }

// V elements that move together: 16 bytes, or one element where sizes or
// alignment do not allow that.
template <typename T, int V>
struct alignas(V * sizeof(T)) Vec {
  T e[V];
};

// A slot of a row is two vectors at element offsets `one` and `two` (two < 0:
// there is none), turned as V pairs or, behind the pairs, copied.
template <typename T, int V, bool kInterleaved>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const Params p) {
  using Vt = Vec<T, V>;
  const int64_t at = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  const int64_t row = at / p.slots;
  if (row >= static_cast<int64_t>(p.batch) * p.tokens) return;
  const int slot = static_cast<int>(at - row * p.slots);
  const int b = static_cast<int>(row / p.tokens);
  const int n = static_cast<int>(row - static_cast<int64_t>(b) * p.tokens);

  const bool first = static_cast<int>(blockIdx.y) < p.groups0;
  const Side& s = p.side[first ? 0 : 1];
  const int h0 = (static_cast<int>(blockIdx.y) - (first ? 0 : p.groups0)) * p.group;
  const int h1 = min(h0 + p.group, s.heads);

  const int turned = p.pairs / V;  // slots that turn; the others copy
  int one, two;
  if (slot < turned) {
    one = kInterleaved ? 2 * slot * V : slot * V;
    two = kInterleaved ? one + V : one + p.pairs;
  } else {
    one = 2 * p.pairs + (slot - turned) * 2 * V;
    two = one + V < p.dim ? one + V : -1;
  }

  float c[V], sn[V];
  if (slot < turned) {
    const int64_t pi = b * p.pb + n * p.pn;
    const double pos = p.wide_positions
                           ? static_cast<double>(static_cast<const long long*>(p.positions)[pi])
                           : static_cast<double>(static_cast<const int*>(p.positions)[pi]);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const double turns = pos * (p.frequencies[slot * V + i] * 0.15915494309189533577);  // 1/(2 pi)
      const float t = static_cast<float>(turns - rint(turns));
      sincospif(2.0f * t, &sn[i], &c[i]);
      c[i] *= p.factor;
      sn[i] *= p.factor * p.sign;
    }
  }

  const T* x = static_cast<const T*>(s.x) + b * s.sb + n * s.sn;
  T* y = static_cast<T*>(s.y) + (static_cast<int64_t>(b) * s.heads * p.tokens + n) * p.dim;
  const int64_t yh = static_cast<int64_t>(p.tokens) * p.dim;
  for (int h = h0; h < h1; ++h) {
    const T* r = x + h * s.sh;
    Vt a = *reinterpret_cast<const Vt*>(r + one), d;
    if (two >= 0) d = *reinterpret_cast<const Vt*>(r + two);
    if (slot < turned) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        // pair i of the slot: the two vectors' i-th elements, or neighbours
        T& u = kInterleaved ? (2 * i < V ? a.e[(2 * i) % V] : d.e[(2 * i) % V]) : a.e[i];
        T& w = kInterleaved ? (2 * i + 1 < V ? a.e[(2 * i + 1) % V] : d.e[(2 * i + 1) % V]) : d.e[i];
        const float fu = to_float<T>(u), fw = to_float<T>(w);
        u = from_float<T>(fu * c[i] - fw * sn[i]);
        w = from_float<T>(fw * c[i] + fu * sn[i]);
      }
    }
    T* o = y + h * yh;
    *reinterpret_cast<Vt*>(o + one) = a;
    if (two >= 0) *reinterpret_cast<Vt*>(o + two) = d;
  }
}

template <typename T, int V>
cudaError_t launch(Params& p, int sms, cudaStream_t stream) {
  const int tail = p.dim - 2 * p.pairs;
  p.slots = p.pairs / V + (tail + 2 * V - 1) / (2 * V);
  const int64_t threads = static_cast<int64_t>(p.batch) * p.tokens * p.slots;
  const int64_t blocks = (threads + kThreads - 1) / kThreads;
  // Heads per thread: as many as still leave 8 blocks of 128 threads per SM,
  // so that one token's decoding step uses one head a thread (its time is the
  // latency of one row) and a long batch computes each sine once per 8 heads.
  const int heads = p.side[0].heads + p.side[1].heads;
  int64_t group = blocks * heads / (8 * static_cast<int64_t>(sms));
  group = group < 1 ? 1 : group > 8 ? 8 : group;
  p.group = static_cast<int>(group);
  p.groups0 = (p.side[0].heads + p.group - 1) / p.group;
  const int groups = p.groups0 + (p.side[1].heads + p.group - 1) / p.group;
  const dim3 grid(static_cast<unsigned>(blocks), static_cast<unsigned>(groups));
  if (p.interleaved)
    rotary_kernel<T, V, true><<<grid, kThreads, 0, stream>>>(p);
  else
    rotary_kernel<T, V, false><<<grid, kThreads, 0, stream>>>(p);
  return cudaGetLastError();
}

template <typename T>
cudaError_t launch_type(Params& p, int sms, cudaStream_t stream) {
  constexpr int V = 16 / sizeof(T);
  bool wide = p.pairs % V == 0 && p.dim % V == 0;
  for (const Side& s : p.side) {
    if (s.heads == 0) continue;
    wide = wide && ((reinterpret_cast<uintptr_t>(s.x) | reinterpret_cast<uintptr_t>(s.y)) & 15) == 0;
    // the stride of an axis of one element is never used
    wide = wide && (p.batch == 1 || s.sb % V == 0) && (s.heads == 1 || s.sh % V == 0) &&
           (p.tokens == 1 || s.sn % V == 0);
  }
  return wide ? launch<T, V>(p, sms, stream) : launch<T, 1>(p, sms, stream);
}

}  // namespace rotary
}  // namespace fa

extern "C" int fa_rotary_sm100(const fa_rotary_tensor* query, const fa_rotary_tensor* key,
                               const void* positions, int position_bits,
                               int64_t position_batch_stride, int64_t position_token_stride,
                               const double* frequencies, int64_t batch, int64_t tokens,
                               int64_t head_dim, int64_t rotary_dim, int interleaved, int dtype,
                               float factor, int inverse, void* cuda_stream) {
  using fa::host::set_error;
  if (query == nullptr) return set_error(FA_ERR_INVALID, "null pointer");
  const fa_rotary_tensor none = {nullptr, nullptr, 0, 0, 0, 0};
  const fa_rotary_tensor* sides[2] = {query, key != nullptr ? key : &none};
  const int64_t heads = sides[0]->heads + sides[1]->heads;
  if (batch < 0 || tokens < 0 || sides[0]->heads < 0 || sides[1]->heads < 0)
    return set_error(FA_ERR_INVALID, "negative size");
  if (head_dim < 1 || rotary_dim < 2 || rotary_dim % 2 != 0 || rotary_dim > head_dim)
    return set_error(FA_ERR_INVALID, "rotary dimension must be even, positive and at most the head dimension");
  if (position_bits != 32 && position_bits != 64)
    return set_error(FA_ERR_INVALID, "positions have 32 or 64 bits");
  if (dtype != FA_FP16 && dtype != FA_BF16 && dtype != FA_FP32)
    return set_error(FA_ERR_INVALID, "unknown element type %d", dtype);
  if (batch == 0 || tokens == 0 || heads == 0) return FA_OK;
  if (positions == nullptr || frequencies == nullptr) return set_error(FA_ERR_INVALID, "null pointer");
  // grid limits: blocks of 128 threads along x, head groups along y
  if (batch > (1ll << 30) || tokens > (1ll << 30) || head_dim > 65536 ||
      batch * tokens > (1ll << 37) / head_dim || heads > 65535)
    return set_error(FA_ERR_INVALID, "size too large");
  const uintptr_t element = dtype == FA_FP32 ? 4 : 2;
  fa::rotary::Params p;
  for (int i = 0; i < 2; ++i) {
    const fa_rotary_tensor& t = *sides[i];
    if (t.heads > 0 && (t.x == nullptr || t.y == nullptr))
      return set_error(FA_ERR_INVALID, "null pointer");
    if ((reinterpret_cast<uintptr_t>(t.x) | reinterpret_cast<uintptr_t>(t.y)) % element)
      return set_error(FA_ERR_INVALID, "tensors must be aligned to their elements");
    p.side[i] = {t.x, t.y, t.batch_stride, t.head_stride, t.token_stride, static_cast<int>(t.heads)};
  }
  fa::host::Device d;
  const int rc = fa::host::current_device(&d);
  if (rc != FA_OK) return rc;
  p.positions = positions;
  p.pb = position_batch_stride;
  p.pn = position_token_stride;
  p.frequencies = frequencies;
  p.batch = static_cast<int>(batch);
  p.tokens = static_cast<int>(tokens);
  p.dim = static_cast<int>(head_dim);
  p.pairs = static_cast<int>(rotary_dim / 2);
  p.wide_positions = position_bits == 64;
  p.interleaved = interleaved != 0;
  p.factor = factor;
  p.sign = inverse ? -1.0f : 1.0f;
  cudaStream_t stream = static_cast<cudaStream_t>(cuda_stream);
  const cudaError_t e = dtype == FA_FP16   ? fa::rotary::launch_type<__half>(p, d.sms, stream)
                        : dtype == FA_BF16 ? fa::rotary::launch_type<__nv_bfloat16>(p, d.sms, stream)
                                           : fa::rotary::launch_type<float>(p, d.sms, stream);
  if (e != cudaSuccess) return set_error(FA_ERR_CUDA, "kernel launch: %s", cudaGetErrorString(e));
  return FA_OK;
}
