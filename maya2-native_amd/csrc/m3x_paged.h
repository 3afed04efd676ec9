// The paged 16-bit KV cache: what its kernels share (format: include/m3x.h).
//
// Pools k, v [pages][kv_heads][page_size][D], the last three contiguous, pages page_stride elements apart; table
// [slots][width] (int32) names the page of every page_size positions of a slot. An entry outside [0, pages) is no page:
// what would lie there is not written, read as zeros and seen by no row. Sixteen positions of a head always lie next to
// each other (page_size is a power of two, at least 16).
#pragma once
#include "m3x_common.h"

// mirror of M3xPagedKv (include/m3x.h)
struct M3xPagedKv {
  void* k;
  void* v;
  const int32_t* table;
  long page_stride;
  int pages, page_size, kv_heads, head_dim, slots, width, dtype;
};

struct Paged {
  uint16_t* k;
  uint16_t* v;
  const int32_t* table;
  long page_stride;
  int pages, shift, kv_heads, slots, width;

  // element of position p's head kh in the pools, or -1 where the slot, the position or the page is outside the cache
  template <int D> __device__ __forceinline__ long at(long slot, int kh, int p) const {
    if (slot < 0 || slot >= slots || p < 0 || (p >> shift) >= width) return -1;
    const int id = table[slot * width + (p >> shift)];
    if ((unsigned)id >= (unsigned)pages) return -1;
    return id * page_stride + ((((long)kh << shift) + (p & ((1 << shift) - 1))) * D);
  }
};

// the kernels' view of a caller's cache, or a status
static inline int paged_take(const M3xPagedKv* p, Paged& c) {
  if (!p) return M3X_ENULL;
  if (p->pages <= 0 || p->kv_heads <= 0 || p->slots <= 0 || p->width <= 0) return M3X_EINVAL;
  if (p->head_dim != 64 && p->head_dim != 128) return M3X_EUNSUPPORTED;
  if (p->dtype != M3X_BF16 && p->dtype != M3X_F16) return M3X_EUNSUPPORTED;
  int shift = 4;
  while (shift < 8 && 1 << shift != p->page_size) ++shift;
  if (1 << shift != p->page_size) return M3X_EUNSUPPORTED;
  if (((long)p->width << shift) > 1L << 30) return M3X_EINVAL;  // positions are counted past the last in 32 bits
  if (!p->k || !p->v || !p->table) return M3X_ENULL;
  if (p->kv_heads > 65535 || p->page_stride < (long)p->kv_heads * p->page_size * p->head_dim || p->page_stride % 8 ||
      !m3x_aligned16(p->k) || !m3x_aligned16(p->v) || ((uintptr_t)p->table & 3u))
    return M3X_EINVAL;
  c = Paged{(uint16_t*)p->k, (uint16_t*)p->v, p->table, p->page_stride, p->pages, shift, p->kv_heads, p->slots, p->width};
  return M3X_OK;
}
