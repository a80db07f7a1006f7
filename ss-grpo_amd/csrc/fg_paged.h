// K and V in pages. Token t of a cache row lies in page table[row][t / P], slot t % P (P a power of two). A page holds, for one
// layer, [kv heads][P][d] rows of K and of V: bf16, or MX e4m3 (fg_mx.h): codes of 8 bits and a scale byte per 32 elements
// of a row, [kv heads][P][d / 32]. Pages lie `page_bytes` apart (their scales `scale_bytes`), so that a pool may hold all
// layers of a page side by side.
#pragma once

#include "fg_common.h"
#include "fg_mx.h"

#include "../../include/flashgrpo_amd.h"

namespace fg {

enum PageFormat : int { kPageE4M3 = 0, kPageBF16 = 1 };

struct Pages {
  uint8_t* k;
  uint8_t* v;
  uint8_t* ks;  // scales (e4m3)
  uint8_t* vs;
  const int32_t* table;
  uint32_t page_bytes, scale_bytes;  // from page to page
  int64_t table_stride;
  int pages, table_rows, table_width, log2_page, kv_heads;

  FG_DEVICE int capacity() const { return table_width << log2_page; }
  // The page of token t (0 <= t < capacity) of the table row that begins at `row`; -1: none.
  FG_DEVICE int page(const int32_t* row, int t) const {
    const int p = row[t >> log2_page];
    return (unsigned)p < (unsigned)pages ? p : -1;
  }
  // Bytes from page 0 to page p (p >= 0), and from its scales.
  FG_DEVICE uint64_t at(int p) const { return (uint64_t)(uint32_t)p * page_bytes; }
  FG_DEVICE uint64_t scales_at(int p) const { return (uint64_t)(uint32_t)p * scale_bytes; }
  // The row of kv head h and token t within its page.
  FG_DEVICE int row_in_page(int h, int t) const { return (h << log2_page) + (t & ((1 << log2_page) - 1)); }
};

template <int FMT>
constexpr int page_elem_bytes = FMT == kPageBF16 ? 2 : 1;

// Checks the host's description and takes it over; an error code and its message otherwise.
inline int pages_of(const fg_kv_pages* p, const char* what, Pages& out) {
  const std::string w(what);
  FG_REQUIRE(p, w + ": null pointer (pages)");
  FG_REQUIRE(p->format == kPageE4M3 || p->format == kPageBF16, w + ": format must be 0 (MX e4m3) or 1 (bf16)");
  FG_REQUIRE(p->k && p->v && p->table && (p->format == kPageBF16 || (p->k_scales && p->v_scales)),
             w + ": null pointer (pages)");
  FG_REQUIRE(p->head_dim == 64 || p->head_dim == 128, w + ": head_dim must be 64 or 128");
  FG_REQUIRE(p->page_size >= 16 && p->page_size <= (1 << 20) && (p->page_size & (p->page_size - 1)) == 0,
             w + ": page_size must be a power of two in [16, 2^20]");
  FG_REQUIRE(p->pages > 0 && p->kv_heads > 0 && p->table_rows > 0 && p->table_width > 0, w + ": bad sizes");
  FG_REQUIRE((int64_t)p->table_width * p->page_size < (1ll << 31) - 65536, w + ": a row must hold less than 2^31 tokens");
  FG_REQUIRE((int64_t)p->kv_heads * p->page_size * p->head_dim < (1ll << 30) && p->page_stride < (1ll << 31) &&
                 p->scale_stride < (1ll << 32),
             w + ": a page must have less than 2^30 elements, pages lie less than 2^31 elements (scales 4 GiB) apart");
  const int es = p->format == kPageBF16 ? 2 : 1;
  FG_REQUIRE(p->page_stride >= (int64_t)p->kv_heads * p->page_size * p->head_dim && p->table_stride >= p->table_width,
             w + ": pages and table rows must not overlap");
  FG_REQUIRE(((uintptr_t)p->k & 15) == 0 && ((uintptr_t)p->v & 15) == 0 && (p->page_stride * es) % 16 == 0,
             w + ": pages must start 16-byte aligned");
  FG_REQUIRE(p->format == kPageBF16 ||
                 (((uintptr_t)p->k_scales & 3) == 0 && ((uintptr_t)p->v_scales & 3) == 0 && p->scale_stride % 4 == 0 &&
                  p->scale_stride >= (int64_t)p->kv_heads * p->page_size * (p->head_dim / kMxBlock)),
             w + ": scales must start 4-byte aligned and not overlap");
  out.k = (uint8_t*)p->k;
  out.v = (uint8_t*)p->v;
  out.ks = (uint8_t*)p->k_scales;
  out.vs = (uint8_t*)p->v_scales;
  out.table = p->table;
  out.page_bytes = (uint32_t)(p->page_stride * es);
  out.scale_bytes = (uint32_t)p->scale_stride;
  out.table_stride = p->table_stride;
  out.pages = p->pages;
  out.table_rows = p->table_rows;
  out.table_width = p->table_width;
  out.log2_page = __builtin_ctz(p->page_size);
  out.kv_heads = p->kv_heads;
  return 0;
}

}  // namespace fg
