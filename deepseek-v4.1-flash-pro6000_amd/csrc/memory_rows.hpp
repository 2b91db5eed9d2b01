// Rows of memory that a call reads or writes, and whether two of them share a byte: an output over an input would be
// written before the input is read for the last time.
#pragma once

#include <cstddef>
#include <cstdint>

namespace ds41g {

// `rows` rows of `bytes` bytes, `stride` apart (at least `bytes`); at 0: none.
struct MemoryRows {
  uintptr_t at;
  size_t rows, bytes, stride;
  uintptr_t end() const { return at + (rows - 1) * stride + bytes; }
};
inline MemoryRows memory_rows(const void *p, size_t rows, size_t bytes, size_t stride) { return MemoryRows{(uintptr_t)p, rows, bytes, stride}; }
inline MemoryRows memory_block(const void *p, size_t bytes) { return MemoryRows{(uintptr_t)p, 1, bytes, bytes}; }

// Exact, so that columns of one buffer stay usable beside each other. Constant time but for rows of two strides whose extents meet,
// where it is a step for each row of the shorter list.
inline bool memory_meets(MemoryRows a, MemoryRows b) {
  if (!a.at || !b.at || !a.rows || !b.rows || !a.bytes || !b.bytes || a.at >= b.end() || b.at >= a.end()) return false;
  const auto whole = [](const MemoryRows &m) { return m.rows == 1 || m.stride == m.bytes; };
  if (whole(a) && whole(b)) return true;
  if (whole(a)) a = MemoryRows{a.at, 1, a.end() - a.at, b.stride};
  if (whole(b)) b = MemoryRows{b.at, 1, b.end() - b.at, a.stride};
  if (a.rows > b.rows) {
    const MemoryRows c = a;
    a = b;
    b = c;
  }
  if (a.stride == b.stride && a.rows > 1) {
    if (a.at > b.at) {
      const MemoryRows c = a;
      a = b;
      b = c;
    }
    // b's first row stands `in` bytes behind the start of a's row `first`; the row after that is the only other one it can reach
    const size_t first = (b.at - a.at) / a.stride, in = (b.at - a.at) % a.stride;
    return (first < a.rows && in < a.bytes) || (first + 1 < a.rows && in + b.bytes > a.stride);
  }
  for (size_t i = 0; i < a.rows; ++i) {
    const uintptr_t from = a.at + i * a.stride, to = from + a.bytes;
    // the first of b's rows that ends behind `from`
    const size_t j = from < b.at + b.bytes ? 0 : (from - b.at - b.bytes) / b.stride + 1;
    if (j < b.rows && b.at + j * b.stride < to) return true;
  }
  return false;
}

// Whether any of the outputs shares a byte with an input or with another output.
template <size_t O, size_t I>
bool memory_collides(const MemoryRows (&out)[O], const MemoryRows (&in)[I]) {
  for (size_t i = 0; i < O; ++i) {
    for (const MemoryRows &m : in)
      if (memory_meets(out[i], m)) return true;
    for (size_t j = 0; j < i; ++j)
      if (memory_meets(out[i], out[j])) return true;
  }
  return false;
}

}  // namespace ds41g
