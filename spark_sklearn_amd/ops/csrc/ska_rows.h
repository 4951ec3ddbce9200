// Row and entry numbers of the grouped-row operators.  They go up to
// 2^31 - 65537 in 32 bits, so that neither the sum of two of them nor one and
// the length of a part may be formed in 32 bits.  (constexpr: for host and
// device alike.)
#pragma once

namespace ska {

// The first position in keys[0, n) whose key is not below g.
template <typename Keys, typename K>
constexpr int lower_bound(const Keys& keys, int n, K g) {
  int lo = 0, hi = n;
  while (lo < hi) {
    const int mid = lo + ((hi - lo) >> 1);
    if (keys[mid] < g)
      lo = mid + 1;
    else
      hi = mid;
  }
  return lo;
}

// Rows first .. last - 1 in parts of 2^shift: how many parts there are, and
// where the one that begins at `at` ends.
constexpr int part_count(int first, int last, int shift) {
  return first < last ? ((last - first - 1) >> shift) + 1 : 0;
}
constexpr int part_end(int at, int last, int shift) {
  const int rest = last - at, whole = 1 << shift;
  return at + (rest < whole ? rest : whole);
}

}  // namespace ska
