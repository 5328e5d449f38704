// attn_rows.h - where the query rows of the block-sparse attention sit: one
// sequence's consecutive positions (from the host or from device memory), or
// rows of sequences with positions and page tables of their own.
#ifndef G4_ATTN_ROWS_H
#define G4_ATTN_ROWS_H

#include <hip/hip_runtime.h>

#include <cstdint>

namespace g4 {

struct RowSet {
  int kv_base;
  const int* d_pos;               // row r at *d_pos + r
  const int* d_pt;                // position -> arena row (nullptr: the position)
  const int* row_pos;             // row r at row_pos[r] ...
  const int* const* row_pt;       // ... with its own table (row_pt[r] nullptr: the position)
};

__device__ __forceinline__ long long row_position(const RowSet& s, int r) {
  if (s.row_pos != nullptr) return s.row_pos[r];
  return static_cast<long long>(s.d_pos != nullptr ? *s.d_pos : s.kv_base) + r;
}
__device__ __forceinline__ const int* row_table(const RowSet& s, int r) {
  return s.row_pt != nullptr ? s.row_pt[r] : s.d_pt;
}

// The argument rules every entry point over a RowSet shares: row_pos and
// row_pt come together, a host position lies inside max_len.
inline bool row_set_ok(const RowSet& s, int rows, int max_len) {
  return rows > 0 && s.kv_base >= 0 && (s.row_pos == nullptr) == (s.row_pt == nullptr) &&
         (s.d_pos != nullptr || s.row_pos != nullptr ||
          static_cast<long long>(s.kv_base) + rows <= max_len);
}

inline bool block_ok(int block, int stride) {
  return (block == 16 || block == 32 || block == 64 || block == 128) && stride > 0 &&
         stride % block == 0;
}

inline bool aligned(const void* p, unsigned bytes) {
  return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0;
}

}  // namespace g4

#endif  // G4_ATTN_ROWS_H
