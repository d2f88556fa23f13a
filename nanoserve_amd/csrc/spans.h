// Host checks of what a call reads against what it writes, by address range.
#pragma once
#include <stddef.h>
#include <stdint.h>

namespace ns {

struct Bytes {
  uintptr_t lo, hi;  // [lo, hi), empty for a null pointer
};

inline Bytes bytes_of(const void* p, size_t n) {
  const uintptr_t a = reinterpret_cast<uintptr_t>(p);
  return p ? Bytes{a, a + n} : Bytes{0, 0};
}

// `rows` rows of `columns` elements of `size` bytes, `stride` elements apart, with what lies between them
inline Bytes rows_of(const void* p, long long rows, long long stride, long long columns, size_t size) {
  return bytes_of(p, (static_cast<size_t>(rows - 1) * stride + columns) * size);
}

inline bool apart(Bytes a, Bytes b) { return a.lo >= a.hi || b.lo >= b.hi || a.hi <= b.lo || b.hi <= a.lo; }

}  // namespace ns
