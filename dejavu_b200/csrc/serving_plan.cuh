// Index arithmetic of the paged and packed kernels. Plain arithmetic without the CUDA headers, so that its bounds are tested on
// the host.
#pragma once
#include "ahead.cuh"

namespace djv {

// Division of numbers below 2^31 by a fixed one from 1 to 2^31 - 1: t / d = (t * times) >> (32 + shift), times = floor(2^(32 + shift) / d) + 1
// with 2^shift < d <= 2^(shift + 1). (times * d exceeds 2^(32 + shift) by at most d <= 2^(shift + 1), which t < 2^31 keeps below one.)
struct Divider {
  unsigned times;
  int shift;  // -1: by 1
};
inline Divider divider_of(unsigned d) {
  Divider v{0, -1};
  if (d == 1) return v;
  while ((2ull << (v.shift + 1)) < d) ++v.shift;
  ++v.shift;
  v.times = (unsigned)((1ull << (32 + v.shift)) / d + 1);
  return v;
}
DJV_HOST_DEVICE unsigned divided(unsigned t, const Divider &v) {
  return v.shift < 0 ? t : (unsigned)(((unsigned long long)t * v.times) >> 32) >> v.shift;
}

// Where tokens of a paged cache are.
struct PageMap {
  const int *table;  // this sequence's row
  int width, page, pages;
  Divider by_page;
};
constexpr long long NO_PAGE = -1;
// Page of token t >= 0, or NO_PAGE where the table has none for it. slot receives its place in the page.
DJV_HOST_DEVICE long long page_of(const PageMap &m, long long t, int &slot) {
  slot = 0;
  if (t < 0 || t >= (long long)m.width * m.page) return NO_PAGE;
  const unsigned i = divided((unsigned)t, m.by_page);  // (a table has room for less than 2^31 tokens)
  slot = (int)((unsigned)t - i * (unsigned)m.page);
  const int entry = m.table[i];
  return entry >= 0 && entry < m.pages ? entry : NO_PAGE;
}

// The sequence that row t of a packed batch belongs to, the last b with cu[b] <= t: a search with 32 probes at a time. `lo` is the answer
// when hi - lo is 1, and always a sequence of the batch, whatever the offsets are.
struct SequenceSearch {
  int lo, hi;
  DJV_HOST_DEVICE bool done() const { return hi - lo <= 1; }
  DJV_HOST_DEVICE int step() const { return (hi - lo + 31) / 32; }
  DJV_HOST_DEVICE int probe(int lane) const { return lo + (lane + 1) * step(); }  // looked at if below hi
  // before: how many lanes there are up to the last one whose probe is not after t
  DJV_HOST_DEVICE void narrow(int before) {
    const int s = step();
    lo += before * s;
    hi = hi < lo + s ? hi : lo + s;
  }
};

// How the cached tokens of a batch are dealt out to blocks: sequence b of n tokens is `share` items (key/value heads times groups of
// query heads), each of units_of(n) units: DECODE_ITEM for its beginning and end, which take about as long as so many times DECODE_UNIT
// tokens do, and one for every DECODE_UNIT tokens. All units stand in a row, sequence by sequence and item by item, and every block
// takes `per` of them, so that an item may begin in one block and end in another.
constexpr int DECODE_UNIT = 64, DECODE_ITEM = 2;
DJV_HOST_DEVICE long long units_of(long long tokens) { return (tokens <= 0 ? 0 : (tokens + DECODE_UNIT - 1) / DECODE_UNIT) + DECODE_ITEM; }
// Tokens of an item in front of its unit u.
DJV_HOST_DEVICE long long tokens_before(long long u, long long tokens) {
  const long long t = u <= DECODE_ITEM ? 0 : (u - DECODE_ITEM) * DECODE_UNIT;
  return t < tokens ? t : (tokens < 0 ? 0 : tokens);
}
DJV_HOST_DEVICE long long units_per_block(long long units, int blocks, int least) {
  const long long per = (units + blocks - 1) / blocks;
  return per < least ? least : per;
}
// Part of an item that a block has: units from .. to - 1 of the item (to > from).
struct DecodePart {
  long long item, from, to;  // item: within its sequence
};
// The part that begins at unit x, for a block whose units end before `end`; base: the sequence's first unit, units: of one of its items.
DJV_HOST_DEVICE DecodePart decode_part(long long x, long long end, long long base, long long units) {
  const long long item = (x - base) / units, from = x - base - item * units, left = end - x;
  return {item, from, from + left < units ? from + left : units};
}

}  // namespace djv
