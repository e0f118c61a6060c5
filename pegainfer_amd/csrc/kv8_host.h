// Host side shared by the entries over the 8-bit paged cache: what a descriptor has to hold, and the choice of an instance.
#pragma once

#include <type_traits>

#include "kv8_core.h"
#include "pegainfer_kernels_blocks.h"

#define PK_BAD ((pegainfer_status_t)hipErrorInvalidValue)

namespace pk {

// of an entry at most 2^30 slots, so that slots and a grid's steps over them stay within 32 bits
constexpr int kKv8MostIds = 1 << 26;

inline bool kv8_ok(const pegainfer_kv8_cache* c) {
  return c && (c->format == kE4m3 || c->format == kInt8) && (c->dim == 64 || c->dim == 128 || c->dim == 256) && c->kv_heads >= 1 && c->kv_heads <= 65535 &&
         c->n_entries >= 0 && c->n_entries <= 65535 && c->n_pages >= 1 && c->n_page_ids >= 0 && c->n_page_ids <= kKv8MostIds &&
         (c->n_entries == 0 || (c->codes && c->scales && c->page_indptr && (c->page_ids || c->n_page_ids == 0) && host_aligned16(c->codes) &&
                                c->code_page_stride % 16 == 0 && c->code_page_stride >= (int64_t)2 * c->kv_heads * kKv8Page * c->dim &&
                                c->scale_page_stride >= (int64_t)2 * c->kv_heads));
}
inline Kv8 kv8_of(const pegainfer_kv8_cache* c) {
  return {static_cast<uint8_t*>(c->codes), c->scales, c->code_page_stride, c->scale_page_stride, c->page_indptr, c->page_ids, c->n_page_ids, c->n_pages, c->kv_heads,
          c->n_entries};
}
// fn(storage type's tag, format, dim), the last two as constants
template <typename F>
inline void kv8_by(int dtype, int format, int dim, F&& fn) {
  by_dtype(dtype, [&](auto* t) {
    auto dims = [&](auto fmt) {
      if (dim == 64) fn(t, fmt, std::integral_constant<int, 64>{});
      else if (dim == 128) fn(t, fmt, std::integral_constant<int, 128>{});
      else fn(t, fmt, std::integral_constant<int, 256>{});
    };
    if (format == kE4m3) dims(std::integral_constant<int, kE4m3>{});
    else dims(std::integral_constant<int, kInt8>{});
  });
}

}  // namespace pk
