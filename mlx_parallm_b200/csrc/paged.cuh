// What the kernels over a paged key-value cache share.
// Pages [P, G, page, D]: the slots of one page and key head are neighbours, so a page of a head is one run of page * D elements.
// Slot s of row r lies in page table[r * width + s / page] at s % page; page is a multiple of 16, so 16 slots never cross a page.
#pragma once
#include "common.cuh"

namespace b200p {

// The table of one call.  An id outside [0, P) names no page: nothing is read or written there.
struct PageTable {
  const int32_t* table;
  int64_t P;
  int rows, width, page;
};

__device__ __forceinline__ int64_t page_id(const PageTable& t, int row, int index) {
  const int id = t.table[(int64_t)row * t.width + index];
  return id >= 0 && id < t.P ? id : -1;
}
__device__ __forceinline__ int table_slots(const PageTable& t) { return t.width * t.page; }
// slots that lie at or before `slot` in the row's pages
__device__ __forceinline__ int slots_seen(const PageTable& t, int slot) {
  return slot < 0 ? 0 : (slot < table_slots(t) ? slot + 1 : table_slots(t));
}

// host: the checks every call makes of its pages and table
static inline int check_pages(const void* k, const void* v, const PageTable& t, int G, int D, int dtype) {
  B200P_REQUIRE(k && v && t.table, B200P_ERR_ARG, "null pointer");
  B200P_REQUIRE(dtype == B200P_F32 || dtype == B200P_F16 || dtype == B200P_BF16, B200P_ERR_ARG, "bad dtype %d", dtype);
  B200P_REQUIRE(t.page >= 16 && t.page % 16 == 0 && t.page <= 4096, B200P_ERR_ARG, "a page holds a multiple of 16 tokens, 4096 at most: got %d", t.page);
  B200P_REQUIRE(G > 0 && G < 65536, B200P_ERR_ARG, "bad number of key heads %d", G);
  B200P_REQUIRE(D >= 8 && D <= 256 && D % 8 == 0, B200P_ERR_ARG, "head_dim %d: a multiple of 8, 256 at most", D);
  B200P_REQUIRE(t.P > 0 && t.P < (1ll << 31) && t.rows > 0 && t.width > 0, B200P_ERR_ARG, "bad shape: %lld pages, table %d x %d", (long long)t.P, t.rows,
                t.width);
  B200P_REQUIRE((int64_t)t.width * t.page < (1ll << 30), B200P_ERR_ARG, "a row of %d pages of %d tokens: at most 2^30 tokens", t.width, t.page);
  B200P_REQUIRE(aligned(k, 16) && aligned(v, 16), B200P_ERR_ALIGN, "pages must be 16-byte aligned");
  return B200P_OK;
}

}  // namespace b200p
