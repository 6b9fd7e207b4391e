// Addressing of a paged key/value cache, shared by the kernels that read or
// change one.
//
// Pages are [num_pages][kv_heads][page_size][dim] of a 16-bit type, so one
// head's part of a page is contiguous.  Slot s of sequence b is row
// s % page_size of page table[b][s / page_size].  Table entries, lengths,
// counts and paths live on the device and cannot be checked before a launch:
// every kernel checks those that it uses, leaves out the rows they would lead
// to, and reports kStatusCache.
#pragma once

#include <cmath>
#include <cstdint>

#include "fa_host.h"
#include "fa_sm100.h"

namespace fa {

constexpr unsigned int kStatusCache = 1u << 5;

struct Pages {
  const int* table;        // [batch][table_stride]
  const int* lengths;      // [batch]
  int64_t table_stride;
  int max_pages;           // table entries of a sequence
  int num_pages;
  int page_size;           // a multiple of 16
  int kv_heads;
  int dim;
  unsigned int* status;

  __host__ __device__ int slots() const { return max_pages * page_size; }
};

// Length of sequence b, held inside what its table can address.
__device__ __forceinline__ int cache_length(const Pages& p, int b) {
  const int n = p.lengths[b];
  if (n < 0 || n > p.slots()) {
    atomicOr(p.status, kStatusCache);
    return n < 0 ? 0 : p.slots();
  }
  return n;
}

// Element offset of row `slot` of (b, head h) in k_pages and v_pages, or -1
// if the table's entry names no page.  slot must be in [0, slots()).
__device__ __forceinline__ int64_t cache_row(const Pages& p, int b, int h, int slot) {
  const int in_table = slot / p.page_size;
  const int page = p.table[b * p.table_stride + in_table];
  if (static_cast<unsigned>(page) >= static_cast<unsigned>(p.num_pages)) {
    atomicOr(p.status, kStatusCache);
    return -1;
  }
  return ((static_cast<int64_t>(page) * p.kv_heads + h) * p.page_size + (slot - in_table * p.page_size)) *
         p.dim;
}

// What every cache call checks of its pages on the host.
inline int check_pages(const fa_paged_cache* c, Pages* out) {
  using host::set_error;
  if (c == nullptr) return set_error(FA_ERR_INVALID, "null pointer");
  if (c->batch < 0 || c->kv_heads < 0 || c->num_pages < 0 || c->max_pages < 0)
    return set_error(FA_ERR_INVALID, "negative size");
  if (c->page_size < 16 || c->page_size % 16 != 0)
    return set_error(FA_ERR_INVALID, "page size must be a positive multiple of 16");
  if (c->head_dim != 64 && c->head_dim != 128)
    return set_error(FA_ERR_INVALID, "head dimension must be 64 or 128");
  if (c->batch > 65535 || c->kv_heads > 65535 || c->num_pages > 0x7fffffffll ||
      c->page_size > (1 << 30) || c->max_pages > (1ll << 30) / c->page_size ||
      c->batch * c->kv_heads > 65535)
    return set_error(FA_ERR_INVALID, "size too large");
  if (c->batch > 0 && (c->lengths == nullptr || (c->max_pages > 0 && c->block_table == nullptr)))
    return set_error(FA_ERR_INVALID, "null pointer");
  if ((reinterpret_cast<uintptr_t>(c->k_pages) | reinterpret_cast<uintptr_t>(c->v_pages)) & 15)
    return set_error(FA_ERR_INVALID, "pages must be 16-byte aligned");
  if (c->batch > 0 && c->kv_heads > 0 && c->num_pages > 0 && c->k_pages == nullptr)
    return set_error(FA_ERR_INVALID, "null pointer");
  out->table = c->block_table;
  out->lengths = c->lengths;
  out->table_stride = c->table_stride;
  out->max_pages = static_cast<int>(c->max_pages);
  out->num_pages = static_cast<int>(c->num_pages);
  out->page_size = static_cast<int>(c->page_size);
  out->kv_heads = static_cast<int>(c->kv_heads);
  out->dim = static_cast<int>(c->head_dim);
  out->status = nullptr;
  return FA_OK;
}

struct Rows {  // strides in elements
  const void* data;
  int64_t batch, head, row;
};

// Checks that the calls with queries share; rows and their product with the
// batch stay below 2^31.
inline int check_queries(const Pages& pages, int64_t batch, int64_t heads, int64_t tokens, int dtype,
                  float scale) {
  using host::set_error;
  if (heads < 0 || tokens < 0) return set_error(FA_ERR_INVALID, "negative size");
  if (dtype != FA_FP16 && dtype != FA_BF16)
    return set_error(FA_ERR_INVALID, "element type must be fp16 or bf16");
  if (!(scale > 0.f) || !std::isfinite(scale))
    return set_error(FA_ERR_INVALID, "scale must be positive and finite");
  if (heads > 0 && (pages.kv_heads == 0 || heads % pages.kv_heads != 0))
    return set_error(FA_ERR_INVALID, "heads must be a multiple of the cache's heads");
  if (heads > 65536 || tokens > (1 << 20) || batch * heads * tokens > (1ll << 30))
    return set_error(FA_ERR_INVALID, "size too large");
  return FA_OK;
}

inline int check_rows(const fa_rows* r, const char* name, Rows* out) {
  using host::set_error;
  if (r == nullptr || r->data == nullptr) return set_error(FA_ERR_INVALID, "null pointer");
  if ((reinterpret_cast<uintptr_t>(r->data) & 15) ||
      (r->batch_stride | r->head_stride | r->row_stride) % 8 != 0)
    return set_error(FA_ERR_INVALID, "rows of %s must be 16-byte aligned", name);
  *out = {r->data, r->batch_stride, r->head_stride, r->row_stride};
  return FA_OK;
}

}  // namespace fa
