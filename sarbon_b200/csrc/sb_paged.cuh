// sb_paged.cuh -- what the kernels of the paged memory share: pools, tables and where a state lies.
#pragma once
#include <cmath>

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

// A pool of rows, strides in units of 16 bytes (below 2^32: checked).
struct Pool {
  uint8_t* p;
  uint32_t row, page;
  SB_DEV uint64_t row_at(int pg, uint32_t r) const {
    return reinterpret_cast<uint64_t>(p) + (((uint64_t)(uint32_t)pg * page + (uint64_t)r * row) << 4);
  }
};

// 32 bits of another CTA of the cluster, at the place that `p` has in this one.
SB_DEV uint32_t peer_word(const void* p, uint32_t rank) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(mapa_shared(smem_u32(p), rank)) : "memory");
  return v;
}

// 16 bytes of it (at a multiple of 16).
SB_DEV uint4 peer_words(const void* p, uint32_t rank) {
  uint4 v;
  asm volatile("ld.shared::cluster.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(mapa_shared(smem_u32(p), rank))
               : "memory");
  return v;
}

// A launch whose CTAs may start while the kernel before them on the stream ends; they call grid_dep_wait() before they
// read what it wrote.  cluster: CTAs that share their memory (1: none).
template <class Args>
cudaError_t launch_after(void (*kernel)(Args), long long ctas, int threads, size_t smem, cudaStream_t st, const Args& args,
                         int cluster = 1, bool after = true) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)ctas);
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (after) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (cluster > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = (unsigned)cluster;
    attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
    ++n;
  }
  cfg.attrs = attr;
  cfg.numAttrs = (unsigned)n;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args);
  return e != cudaSuccess ? e : cudaGetLastError();
}

inline int page_dtype_bytes(int dt) { return dt == SB_F8 ? 1 : 2; }
inline bool page_dtype_ok(int dt) { return dt == SB_F16 || dt == SB_BF16 || dt == SB_F8; }
inline bool paged_sizes_ok(int B, int Hkv, int dh, int P, int page, int N) {
  return B >= 0 && Hkv >= 1 && (dh == 32 || dh == 64 || dh == 128) && (long long)Hkv * dh <= 65536 && P >= 0 &&
         page >= 1 && N >= 0 && (long long)N * page < (1ll << 30) && (long long)B * Hkv < (1ll << 30);
}
inline bool paged_memory_ok(const sb_paged_memory* m) {
  return m && page_dtype_ok(m->dtype) &&
         paged_sizes_ok(m->B, m->Hkv, m->dh, m->P, m->page, m->N);
}
// 16-byte rows, strides in elements of es bytes
inline bool pool_ok(const void* p, long long row, long long page, int es) {
  return p && (reinterpret_cast<uintptr_t>(p) & 15) == 0 && row >= 0 && page >= 0 && row * es % 16 == 0 &&
         page * es % 16 == 0 && row < (1ll << 35) && page < (1ll << 35);
}
// pools and table of a memory that has places; without them nothing is read
inline bool paged_pools_ok(const sb_paged_memory* m) {
  const int es = page_dtype_bytes(m->dtype);
  return (m->N == 0 || (m->table && m->table_row >= 0)) &&
         (m->N == 0 || m->P == 0 || (pool_ok(m->k, m->k_row, m->k_page, es) && pool_ok(m->v, m->v_row, m->v_page, es)));
}
inline PageTable page_table(const sb_paged_memory* m) {
  return {m->table, m->table_row, fast_div((uint32_t)m->page), m->N, m->P, m->N * m->page};
}
inline Pool k_pool(const sb_paged_memory* m) {
  const int es = page_dtype_bytes(m->dtype);
  return {static_cast<uint8_t*>(m->k), (uint32_t)(m->k_row * es / 16), (uint32_t)(m->k_page * es / 16)};
}
inline Pool v_pool(const sb_paged_memory* m) {
  const int es = page_dtype_bytes(m->dtype);
  return {static_cast<uint8_t*>(m->v), (uint32_t)(m->v_row * es / 16), (uint32_t)(m->v_page * es / 16)};
}
inline bool scales_ok(const sb_paged_memory* m, float k_scale, float v_scale) {
  return k_scale > 0.f && k_scale < INFINITY && v_scale > 0.f && v_scale < INFINITY &&
         (m->dtype == SB_F8 || (k_scale == 1.f && v_scale == 1.f));
}

}  // namespace sb
