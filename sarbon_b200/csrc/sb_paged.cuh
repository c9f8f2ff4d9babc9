// sb_paged.cuh -- what the kernels of the paged memory share: pools, tables and where a state lies.
#pragma once
#include "sb_xattn.cuh"

namespace sb {

// Division of n < 2^31 by a fixed d >= 1 as a product: with 2^s >= d the smallest power and
// m = floor(2^32 (2^s - d) / d) + 1, n / d = (hi32(m n) + n) >> s (Granlund and Montgomery, 1994).
struct FastDiv {
  uint32_t d, m, s;
  SB_DEV uint32_t div(uint32_t n) const { return (__umulhi(m, n) + n) >> s; }
};
inline FastDiv fast_div(uint32_t d) {
  FastDiv f{d, 0, 0};
  while ((1ull << f.s) < d) ++f.s;
  f.m = (uint32_t)((((1ull << f.s) - d) << 32) / d + 1);
  return f;
}

// State j of item b lies in row j % page of the page that table[b * table_row + j / page] names; a number
// outside [0, P) is no page.
struct PageTable {
  const int* table;
  long long table_row;
  FastDiv page;
  int N, P, cap;  // entries an item, pages of the pool, N * page
  SB_DEV int entry(int b, uint32_t j, uint32_t& row) const {
    const uint32_t at = page.div(j);
    row = j - at * page.d;
    return table[b * table_row + at];
  }
  SB_DEV bool has(int p) const { return (uint32_t)p < (uint32_t)P; }
  SB_DEV int clamp(int n) const { return min(max(n, 0), cap); }
};

// A pool of rows, strides in bytes.
struct Pool {
  uint8_t* p;
  long long row, page;
};

inline int page_dtype_bytes(int dt) { return dt == SB_F8 ? 1 : 2; }
inline bool page_dtype_ok(int dt) { return dt == SB_F16 || dt == SB_BF16 || dt == SB_F8; }
inline bool paged_sizes_ok(int B, int Hkv, int dh, int P, int page, int N) {
  return B >= 0 && Hkv >= 1 && (dh == 32 || dh == 64 || dh == 128) && (long long)Hkv * dh <= 65536 && P >= 0 &&
         page >= 1 && N >= 0 && (long long)N * page < (1ll << 30) && (long long)B * Hkv < (1ll << 30);
}
// 16-byte rows, strides in elements of es bytes
inline bool pool_ok(const void* p, long long row, long long page, int es) {
  return p && (reinterpret_cast<uintptr_t>(p) & 15) == 0 && row >= 0 && page >= 0 && row * es % 16 == 0 &&
         page * es % 16 == 0 && row < (1ll << 38) && page < (1ll << 38);
}
inline PageTable page_table(const int* table, long long table_row, int P, int page, int N) {
  return {table, table_row, fast_div((uint32_t)page), N, P, N * page};
}
inline Pool pool_of(const void* p, long long row, long long page, int es) {
  return {static_cast<uint8_t*>(const_cast<void*>(p)), row * es, page * es};
}

}  // namespace sb
