// Host walk of PagedView (mdma_amd/csrc/paged.h) over tables whose entries and
// lengths are anything: every row it gives lies inside the pool.
#include <cstdio>
#include <random>
#include <vector>

#include "../mdma_amd/csrc/paged.h"

using namespace mdma;

int main() {
  std::mt19937 r(7);
  auto pick = [&](uint32_t n) { return (uint32_t)(r() % n); };
  uint64_t rows = 0, skipped = 0;
  for (int c = 0; c < 400; c++) {
    PagedView v{};
    v.n_pages = 1 + pick(50);
    v.page_shift = 4 + pick(5);
    v.width = 8 * (1 + pick(40));
    v.n_seqs = 1 + pick(6);
    v.max_pages = 1 + pick(20);
    v.n_prefix = pick(v.max_pages + 1);
    auto id = [&] { return pick(3) ? pick(v.n_pages) : pick(2) ? r() : v.n_pages; };
    std::vector<uint32_t> table(v.n_seqs * v.max_pages), lens(v.n_seqs), prefix(v.n_prefix + 1);
    for (auto &x : table) x = id();
    for (auto &x : prefix) x = id();
    for (auto &x : lens) x = pick(2) ? pick(v.max_pages << v.page_shift) : r();
    v.table = table.data(), v.lens = lens.data(), v.prefix = prefix.data();
    const uint64_t pool = ((uint64_t)v.n_pages << v.page_shift) * v.width;
    for (uint32_t s = 0; s < v.n_seqs; s++) {
      const uint32_t n = v.length(s);
      if (n > v.max_pages << v.page_shift) return printf("length %u\n", n), 1;
      for (uint32_t p = 0; p < n; p++) {
        const uint32_t pg = v.page(s, p >> v.page_shift);
        if (pg == NO_PAGE) {
          skipped++;
          continue;
        }
        rows++;
        const uint32_t want = (p >> v.page_shift) < v.n_prefix ? prefix[p >> v.page_shift]
                                                               : table[s * v.max_pages + (p >> v.page_shift)];
        if (pg != want || v.row(pg, p) + v.width > pool || v.row(pg, p) != (((uint64_t)pg << v.page_shift) + p % (1u << v.page_shift)) * v.width)
          return printf("sequence %u position %u page %u\n", s, p, pg), 1;
      }
    }
  }
  // Rows past 2^32 elements.
  PagedView v{};
  v.n_pages = 1u << 20, v.page_shift = 8, v.width = 1024;
  if (v.row((1u << 20) - 1, 255) != (((1ull << 20) - 1) * 256 + 255) * 1024) return printf("row overflow\n"), 1;
  printf("ok: %llu rows, %llu positions without a page\n", (unsigned long long)rows, (unsigned long long)skipped);
  return rows && skipped ? 0 : 1;
}
