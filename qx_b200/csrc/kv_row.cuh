// kv_row.cuh — where a cache row lives in an arena's regions.
#pragma once

namespace qx {

// How a (sequence, layer, slot) finds its cache row in the arena's regions
// (rows of [kv_heads][head_dim]). A contiguous arena keeps each (sequence,
// layer) cache as `capacity` consecutive rows. A paged arena keeps, per
// layer, a pool of pages of 2^shift rows; a sequence's block table (shared
// by all layers, as in vLLM) maps its logical page to a physical page.
struct KvPaging {
  const int* table;  // device [sequences][stride] physical page per logical page; null: contiguous
  int stride;        // logical pages per sequence
  int shift;         // log2 of rows per page (>= 6: a 64-row TMA box never straddles pages)
  int pool;          // physical pages per layer
};

__device__ __forceinline__ long long kv_row(const KvPaging& pg, int capacity, int layers, int seq, int layer,
                                            int slot) {
  if (!pg.table) return ((long long)seq * layers + layer) * capacity + slot;
  const int page = __ldg(pg.table + (long long)seq * pg.stride + (slot >> pg.shift));
  return (((long long)layer * pg.pool + page) << pg.shift) + (slot & ((1 << pg.shift) - 1));
}

}  // namespace qx
