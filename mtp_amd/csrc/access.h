// The access width of row copies. Plain C++: no HIP header.
#pragma once

#include <cstdint>

// The widest of 16, 4 and 2 bytes in which rows of row_bytes can be copied from p to q.
inline int copy_access_bytes(int64_t row_bytes, const void* p, const void* q) {
  const uint64_t all = (uint64_t)row_bytes | (uint64_t)(uintptr_t)p | (uint64_t)(uintptr_t)q;
  return all % 16 == 0 ? 16 : all % 4 == 0 ? 4 : 2;
}
