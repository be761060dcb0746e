// The paged KV cache's geometry, on the host and in kernels (plain C++, so
// that a host test can walk it over tables that name pages the pool lacks).
#pragma once
#include <cstdint>

#ifdef __HIPCC__
#define PAGED_FN __host__ __device__ __forceinline__
#else
#define PAGED_FN inline
#endif

namespace mdma {

constexpr uint32_t NO_PAGE = 0xffffffffu;

// One layer of a paged cache: K and V rows of `width` f16 in pages of
// 1 << page_shift positions. Page i of sequence s is prefix[i] for
// i < n_prefix, else table[s * max_pages + i]; an id that is not below n_pages names
// no page, and its positions are neither read nor written.
struct PagedView {
  uint16_t *k, *v;
  const uint32_t *table, *lens, *prefix;
  uint32_t n_pages, page_shift, width, n_seqs, max_pages, n_prefix;

  // Positions sequence s holds: a length past the table's end is read as that end.
  PAGED_FN uint32_t length(uint32_t s) const {
    const uint64_t cap = (uint64_t)max_pages << page_shift;
    const uint32_t n = lens[s];
    return n < cap ? n : (uint32_t)cap;
  }
  // Page i of sequence s (i < max_pages), NO_PAGE where the entry names none.
  PAGED_FN uint32_t page(uint32_t s, uint32_t i) const {
    const uint32_t id = i < n_prefix ? prefix[i] : table[(uint64_t)s * max_pages + i];
    return id < n_pages ? id : NO_PAGE;
  }
  // Element offset of position pos's row in k and v, given its page.
  PAGED_FN uint64_t row(uint32_t id, uint32_t pos) const {
    const uint32_t in_page = pos & ((1u << page_shift) - 1);
    return (((uint64_t)id << page_shift) + in_page) * width;
  }
};

}  // namespace mdma
