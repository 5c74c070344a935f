// Index arithmetic of the paged and packed kernels. Plain arithmetic without the CUDA headers, so that its bounds are tested on
// the host.
#pragma once
#include "ahead.cuh"

namespace djv {

// Where tokens of a paged cache are.
struct PageMap {
  const int *table;  // this sequence's row
  int width, page, pages;
};
constexpr long long NO_PAGE = -1;
// Page of token t >= 0, or NO_PAGE where the table has none for it. slot receives its place in the page.
DJV_HOST_DEVICE long long page_of(const PageMap &m, long long t, int &slot) {
  const long long i = t / m.page;
  slot = (int)(t - i * m.page);
  if (t < 0 || i >= m.width) return NO_PAGE;
  const int entry = m.table[i];
  return entry >= 0 && entry < m.pages ? entry : NO_PAGE;
}

// The sequence that row t of a packed batch belongs to (the last b with cu[b] <= t, if t < cu[b + 1]), or -1.
DJV_HOST_DEVICE int sequence_of(const int *cu, int B, int t) {
  int lo = 0, hi = B;  // cu[lo] <= t < cu[hi], if there is such a pair
  if (t < cu[0] || t >= cu[B]) return -1;
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (cu[mid] <= t) lo = mid;
    else hi = mid;
  }
  return lo;
}

}  // namespace djv
