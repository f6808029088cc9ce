// bb_rows.h — whether two strided arrays share memory. Host code, no HIP in it.
#ifndef BB_ROWS_H
#define BB_ROWS_H
#include <stddef.h>
#include <stdint.h>

namespace bb {

// Rows of `len` bytes, n[1] of them stride[1] apart and n[0] such groups stride[0] >= stride[1] apart (bytes).
struct Rows {
  const void* p;
  size_t n[2], stride[2], len;
  size_t extent(int level) const {  // of a group, from its first to past its last byte
    return level == 2 ? len : (n[level] - 1) * stride[level] + extent(level + 1);
  }
};

// n rows of len elements `stride` apart.
inline Rows rows_of(const void* p, size_t n, size_t stride, size_t len, size_t elem) {
  return {p, {1, n}, {0, stride * elem}, len * elem};
}

// Whether rows of a and b, b's first `off` bytes after a's, share a byte (from `level` on). Where the groups of both
// are one stride apart and none is longer than it, a group of a can meet the two of b that begin next to it only;
// other strides are taken to meet where their ends overlap.
inline bool rows_meet(const Rows& a, const Rows& b, int64_t off, int level) {
  const int64_t ea = (int64_t)a.extent(level), eb = (int64_t)b.extent(level);
  if (off >= ea || -off >= eb) return false;
  if (level == 2) return true;
  const int64_t na = (int64_t)a.n[level], nb = (int64_t)b.n[level];
  if (na == 1 && nb == 1) return rows_meet(a, b, off, level + 1);
  const int64_t step = (int64_t)(na > 1 ? a.stride[level] : b.stride[level]);
  if (nb > 1 && step != (int64_t)b.stride[level]) return true;
  if (step < (int64_t)a.extent(level + 1) || step < (int64_t)b.extent(level + 1)) return true;
  const int64_t down = off >= 0 ? off / step : -((step - 1 - off) / step);
  for (const int64_t m : {-down, -down - 1})  // b's group index less a's
    if (m > -na && m < nb && rows_meet(a, b, off + m * step, level + 1)) return true;
  return false;
}

inline bool rows_overlap(const Rows& a, const Rows& b) {
  return rows_meet(a, b, (int64_t)(reinterpret_cast<uintptr_t>(b.p) - reinterpret_cast<uintptr_t>(a.p)), 0);
}

}  // namespace bb
#endif
