// A paged key-value cache: [page][keys, values][kv head][slot][HD] fp16 or fp32, P slots a page (a power of two from 16 on).
// Position n of a sequence is slot n % P of page table[n / P]; an entry outside the cache is no page.
#pragma once
#include "miq_common.h"

namespace miq {

constexpr int kPageMin = 16, kPageMax = 4096;

inline int check_paged(const char* what, int HD, int page, int num_pages, int max_pages) {
  MIQ_REQUIRE(HD == 64 || HD == 128 || HD == 192 || HD == 256, MIQ_ERR_UNSUPPORTED, "%s: HD=%d (64, 128, 192 or 256)", what, HD);
  MIQ_REQUIRE(page >= kPageMin && page <= kPageMax && (page & (page - 1)) == 0, MIQ_ERR_UNSUPPORTED,
              "%s: pages of %d positions (a power of two from %d to %d)", what, page, kPageMin, kPageMax);
  MIQ_REQUIRE((int64_t)max_pages * page <= (1 << 30), MIQ_ERR_UNSUPPORTED, "%s: %d pages of %d positions (at most 2^30 positions)", what, max_pages,
              page);
  MIQ_REQUIRE(num_pages <= (1 << 30), MIQ_ERR_UNSUPPORTED, "%s: %d pages", what, num_pages);
  return MIQ_OK;
}

}  // namespace miq
