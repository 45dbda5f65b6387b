// A paged cache relation as its kernels see it: the sequences' page tables
// and lengths are read on the device at every launch (a program advances
// them in place between launches), so nothing here is known to the host but
// their sizes.
#pragma once

#include <stdint.h>

#include "tgx_device.h"
#include "tgx_host.h"

namespace tgx {

struct PagedRel {
  const int32_t* table;    // [n_seqs, heads, pages_per_seq] page ids
  int64_t seq_stride;      // elements between the tables of two sequences
  int64_t head_stride;     // and of two heads of one sequence
  const int32_t* lengths;  // [n_seqs] cached tokens
  int n_seqs;
  int heads;               // tables per sequence
  int pages_per_seq;
  int page_size;
  int num_pages;
  int queries;             // newest tokens of a sequence that ask
};

inline PagedRel paged_rel(const tgx_paged& p) {
  return PagedRel{p.page_table_dev, p.seq_stride, p.head_stride, p.lengths_dev,
                  static_cast<int>(p.n_seqs), p.table_heads, p.pages_per_seq, p.page_size,
                  static_cast<int>(p.num_pages), p.queries};
}

// What every entry point over a paged relation needs of it.
inline int check_paged(const tgx_paged* p) {
  TGX_REQUIRE(p != nullptr, "null paged relation");
  TGX_REQUIRE(p->n_seqs >= 0 && p->table_heads >= 1 && p->pages_per_seq >= 0 &&
                  p->page_size >= 1 && p->num_pages >= 0 && p->queries >= 1,
              "paged relation with negative or zero sizes");
  TGX_REQUIRE(p->page_size < (1 << 30), "pages of fewer than 2^30 slots");
  TGX_REQUIRE(p->n_seqs < (int64_t{1} << 31) && p->num_pages < (int64_t{1} << 31) &&
                  static_cast<int64_t>(p->pages_per_seq) * p->page_size <
                      (int64_t{1} << 31) - 4096 &&   // (kernels look a few tiles ahead)
                  p->num_pages * p->page_size < (int64_t{1} << 31) &&
                  p->n_seqs * p->queries < (int64_t{1} << 31),
              "paged relation: sequences, rows, positions and slots must be fewer than 2^31");
  TGX_REQUIRE(p->n_seqs == 0 || p->lengths_dev, "paged relation without lengths");
  TGX_REQUIRE(p->n_seqs == 0 || p->pages_per_seq == 0 || p->page_table_dev,
              "paged relation without a page table");
  return TGX_OK;
}

// Inclusive prefix sum over the wave's lanes: shifts inside rows of 16 lanes,
// then the rows' last lanes broadcast to the rows after them (no LDS).
__device__ __forceinline__ int wave_prefix(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);   // row_shr:1
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);   // row_shr:2
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);   // row_shr:4
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);   // row_shr:8
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);   // row_bcast:15
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);   // row_bcast:31
  return v;
}

// Largest value of the wave's lanes.
__device__ __forceinline__ uint32_t wave_largest(uint32_t u) {
  int v = static_cast<int>(u);
  auto step = [&](int o) { v = static_cast<int>(max(static_cast<uint32_t>(v), static_cast<uint32_t>(o))); };
  step(__builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false));
  step(__builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false));
  step(__builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false));
  step(__builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false));
  step(__builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false));
  step(__builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false));
  return static_cast<uint32_t>(read_lane(v, 63));
}

// Cached tokens of sequence b: what its page table can hold at most.
__device__ __forceinline__ int paged_length(const PagedRel& r, int b) {
  return min(max(r.lengths[b], 0), r.pages_per_seq * r.page_size);
}

// Slot of position `pos` in a page table, -1 where the table names no page.
__device__ __forceinline__ int paged_slot(const PagedRel& r, const int32_t* table, int pos) {
  const int page = static_cast<unsigned>(pos) / static_cast<unsigned>(r.page_size);
  const int id = table[page];
  if (static_cast<unsigned>(id) >= static_cast<unsigned>(r.num_pages)) return -1;
  return id * r.page_size + (pos - page * r.page_size);
}

}  // namespace tgx
