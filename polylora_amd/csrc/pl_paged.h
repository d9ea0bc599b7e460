// What the paged cache's two kernels share: its element types and addressing.
#pragma once

#include "pl_common.h"

// Element type of a cache: the model's, or e4m3 with a scale per key head.
template <int CT>
struct pl_cache_elem {
  typedef typename pl_traits<CT>::T T;
};
template <>
struct pl_cache_elem<PL_F8E4M3> {
  typedef uint8_t T;
};

// A key or value cache: element (page, head, slot, d) lies at
// page * s_page + head * s_head + slot * s_slot + d.  Offsets are 64-bit: one
// layer's cache alone passes 4 G elements well within 288 GB.
struct pl_cache_view {
  void* p;
  int64_t s_page, s_head, s_slot;
};

struct pl_page_table {
  const int32_t* p;   // [rows][ld], a row's pages in order
  int64_t ld;
  int32_t max_pages;  // columns
  int32_t num_pages;  // pages in the pool: ids outside [0, num_pages) hold nothing
  int32_t page_shift; // log2 of the tokens per page
};

// The largest finite e4m3 value.
constexpr float kE4M3Max = 448.f;

// Smallest and largest tokens per page (powers of two) and the head sizes.
constexpr int kPageMin = 16, kPageMax = 1 << 16;
constexpr int kHeadDimMax = 256, kHeadDimStep = 16;

static inline int pl_cache_elem_size(int ct) { return ct == PL_F8E4M3 ? 1 : pl_elem_size(ct); }

static inline int pl_log2_exact(int32_t v) {
  int s = 0;
  while ((1 << s) < v) ++s;
  return (1 << s) == v ? s : -1;
}

// The checks both entry points make of their cache arguments; PL_OK or a
// status with the message set.
int pl_check_paged(const char* what, int32_t dtype, int32_t cache_dtype, const void* key_cache,
                   const int64_t* key_strides, const void* value_cache,
                   const int64_t* value_strides, int32_t num_pages, int32_t page_size,
                   const int32_t* page_table, int64_t table_ld, int32_t max_pages, int32_t rows,
                   int32_t heads, int32_t kv_heads, int32_t dim, const float* k_scale,
                   const float* v_scale);

// Whether no two elements of a cache share a place: from the smallest stride up,
// each dimension steps past all that those before it reach.
bool pl_elements_apart(const int64_t* strides, int32_t pages, int32_t kv_heads, int32_t page_size,
                       int32_t dim);
