// Checks of arguments that describe memory (host side): overlap and alignment.
#pragma once

#include <cstddef>
#include <cstdint>
#include <initializer_list>

namespace frhip {

// Whether [rows][cols] of ld elements a row at a and b (ldb) share memory.  Rows of the same pitch may lie side by side.
inline bool rows_overlap(const void* a, size_t lda, const void* b, size_t ldb, size_t rows, size_t cols_a, size_t cols_b, size_t elem) {
  if (!a || !b || !rows) return false;
  const uintptr_t pa = reinterpret_cast<uintptr_t>(a), pb = reinterpret_cast<uintptr_t>(b);
  const uintptr_t ea = pa + ((rows - 1) * lda + cols_a) * elem, eb = pb + ((rows - 1) * ldb + cols_b) * elem;
  if (ea <= pb || eb <= pa) return false;
  if (lda != ldb) return true;
  const size_t pitch = lda * elem, off = (pa < pb ? pb - pa : pa - pb) % pitch;
  // seen from the lower one, the other begins `off` bytes into a row
  const size_t low = (pa < pb ? cols_a : cols_b) * elem, high = (pa < pb ? cols_b : cols_a) * elem;
  return off < low || off + high > pitch;
}

inline bool spans_clash(const void* a, const void* b, size_t bytes) {  // neither the same nor apart
  const uintptr_t pa = reinterpret_cast<uintptr_t>(a), pb = reinterpret_cast<uintptr_t>(b);
  return pa != pb && pa < pb + bytes && pb < pa + bytes;
}

inline bool spans_meet(const void* a, size_t bytes_a, const void* b, size_t bytes_b) {
  const uintptr_t pa = reinterpret_cast<uintptr_t>(a), pb = reinterpret_cast<uintptr_t>(b);
  return a && b && pa < pb + bytes_b && pb < pa + bytes_a;
}

inline bool off_grid(size_t elem, std::initializer_list<const void*> ptrs) {
  uintptr_t v = 0;
  for (const void* p : ptrs) v |= reinterpret_cast<uintptr_t>(p);
  return v % elem != 0;
}

}  // namespace frhip
