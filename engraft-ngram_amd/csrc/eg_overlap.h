// Whether strided matrices share memory: what is written must not be what another workgroup still
// reads or writes.  Host code only, for the library and the torch binding.
#pragma once

#include <stddef.h>
#include <stdint.h>

#include <algorithm>
#include <numeric>
#include <vector>

namespace eg {

// rows x cols elements of `item` bytes, element (i, j) at at + i * step[0] + j * step[1] bytes.
struct Extent {
  int64_t at;
  int64_t count[2], step[2];
  int64_t item;

  Extent(const void* data, int64_t rows, int64_t cols, int64_t row_stride, int64_t col_stride, int64_t item_bytes)
      : at((int64_t)(uintptr_t)data), count{rows, cols}, step{row_stride * item_bytes, col_stride * item_bytes},
        item(item_bytes) {
    for (int d = 0; d < 2; ++d) {
      if (count[d] <= 1) step[d] = 0;
      if (step[d] < 0) {  // the same elements from the other end
        at += (count[d] - 1) * step[d];
        step[d] = -step[d];
      }
    }
    // the longer step first
    if (step[0] < step[1]) {
      std::swap(step[0], step[1]);
      std::swap(count[0], count[1]);
    }
  }
  bool empty() const { return count[0] <= 0 || count[1] <= 0; }
  int64_t end() const { return at + (count[0] - 1) * step[0] + (count[1] - 1) * step[1] + item; }
  // each row one piece of memory, one after the other
  bool rows_whole() const { return (step[1] == item || count[1] == 1) && (count[0] == 1 || step[0] >= row_bytes()); }
  int64_t row_bytes() const { return (count[1] - 1) * step[1] + item; }
};

// Whether two elements of a matrix are the same: i step[0] = j step[1] for some i and j within it.
inline bool overlaps_itself(const Extent& x) {
  if (x.empty()) return false;
  const int64_t g = std::gcd(x.step[0], x.step[1]);
  if (g == 0) return x.count[0] > 1 || x.count[1] > 1;
  if (x.step[1] == 0) return x.count[1] > 1;
  return x.step[1] / g < x.count[0] && x.step[0] / g < x.count[1];
}

// Whether two matrices share a byte.  Exact where they have the same steps or rows that are whole;
// otherwise (columns apart, of different steps) taken to be apart.
inline bool overlap(const Extent& a, const Extent& b) {
  if (a.empty() || b.empty() || a.end() <= b.at || b.end() <= a.at) return false;
  if (a.step[0] == b.step[0] && a.step[1] == b.step[1]) {
    // an element of a at (i, j) and one of b at (k, l): x = (k - i) step[0] + (l - j) step[1] + b.at - a.at
    const int64_t d = b.at - a.at, s0 = a.step[0], s1 = a.step[1];
    auto floor_div = [](int64_t n, int64_t m) { return n / m - (n % m < 0 ? 1 : 0); };
    int64_t first = 1 - a.count[0], last = b.count[0] - 1;
    if (s0 > 0) {
      first = std::max(first, floor_div(-b.item - (b.count[1] - 1) * s1 - d, s0));
      last = std::min(last, floor_div(a.item + (a.count[1] - 1) * s1 - d, s0));
    }
    for (int64_t t = first; t <= last; ++t) {
      const int64_t rest = d + t * s0;
      const int64_t u0 = s1 > 0 ? floor_div(-rest, s1) : 0;
      for (int64_t u = u0; u <= u0 + 1; ++u) {
        if (u < 1 - a.count[1] || u > b.count[1] - 1) continue;
        const int64_t x = rest + u * s1;
        if (x > -b.item && x < a.item) return true;
      }
    }
    return false;
  }
  if (!a.rows_whole() || !b.rows_whole()) return false;
  // b's row of a's row, from the first on that ends behind it: at most one look a row of a
  const Extent &few = a.count[0] <= b.count[0] ? a : b, &many = a.count[0] <= b.count[0] ? b : a;
  for (int64_t i = 0; i < few.count[0]; ++i) {
    const int64_t lo = few.at + i * few.step[0], hi = lo + few.row_bytes();
    const int64_t past = lo - many.at - many.row_bytes();  // rows that start at or before this end before lo
    const int64_t j = past < 0 || many.step[0] == 0 ? (past < 0 ? 0 : 1) : past / many.step[0] + 1;
    if (j < many.count[0] && many.at + j * many.step[0] < hi) return true;
  }
  return false;
}

// What a call reads (grads) or writes (params, momenta) of matrix `matrix`.
struct Operand {
  enum Kind { kParam, kMomentum, kGrad } kind;
  size_t matrix;
  Extent extent;
};

// The first pair that shares memory and must not, or the first operand written that overlaps itself
// (twice the same); false if there is none.  A matrix's own gradient may be its param: it is read whole first.
inline bool find_overlap(std::vector<Operand>& all, const Operand*& x, const Operand*& y) {
  std::sort(all.begin(), all.end(), [](const Operand& p, const Operand& q) { return p.extent.at < q.extent.at; });
  for (size_t i = 0; i < all.size(); ++i) {
    const Operand& p = all[i];
    if (p.kind != Operand::kGrad && overlaps_itself(p.extent)) {
      x = y = &p;
      return true;
    }
    for (size_t j = i + 1; j < all.size() && all[j].extent.at < p.extent.end(); ++j) {
      const Operand& q = all[j];
      if (p.kind == Operand::kGrad && q.kind == Operand::kGrad) continue;
      if (p.matrix == q.matrix && p.kind != Operand::kMomentum && q.kind != Operand::kMomentum) continue;
      if (!overlap(p.extent, q.extent)) continue;
      x = &p;
      y = &q;
      return true;
    }
  }
  return false;
}

inline const char* name_of(Operand::Kind kind) {
  return kind == Operand::kParam ? "params" : kind == Operand::kMomentum ? "momenta" : "grads";
}

}  // namespace eg
