// What the paged-cache kernels share: the device view of a cache with block tables, the argument checks, and the
// rules by which a query block's key rows are cut into tiles.
#pragma once

#include "common.cuh"
#include "tc5.cuh"

// A cache as the kernels see it (mb_paged_kv).
struct PagedView {
  const int32_t* table;
  const int32_t* lens;
  const int32_t* prefix;      // [batch] or null
  uint32_t batch, pages, page_size, kv_heads, table_width;
  size_t table_stride;
  mb_fastdiv page_div;
  uint32_t rows_max;          // table_width * page_size
  uint32_t window;            // 0 = none
  int* plan_flag;
};

// Rows of one sequence that a block of queries at positions [q_first, q_last] can see, as tiles of `tile` rows:
// tiles [lo, end) around the band, and tiles [0, pre) of the always-visible prefix where those lie below it.
struct PagedSpan {
  int len, prefix;            // live rows, always-visible rows (clamped to len)
  int k_lo, k_hi;             // the band's rows
  uint32_t lo, end, pre;      // tiles
  __device__ __forceinline__ uint32_t count() const { return end - lo + pre; }
  // i-th tile, first the band's from the last one down, then the prefix's from the last one down
  __device__ __forceinline__ uint32_t tile_down(uint32_t i) const {
    return i < end - lo ? end - 1 - i : pre - 1 - (i - (end - lo));
  }
  // whether rows [r, r + n) hold a row that may be seen
  __device__ __forceinline__ bool needed(int r, int n) const {
    return (r < k_hi && r + n > k_lo) || r < prefix;
  }
};

__device__ __forceinline__ int paged_len(const PagedView& c, uint32_t b) {
  const int len = __ldg(c.lens + b);
  return len < 0 ? 0 : min(len, int(c.rows_max));
}
// True when the length or the table is unusable as given; the caller raises the flag once.
__device__ __forceinline__ bool paged_len_bad(const PagedView& c, uint32_t b) {
  const int len = __ldg(c.lens + b);
  return len < 0 || len > int(c.rows_max);
}
__device__ __forceinline__ void paged_raise(const PagedView& c, uint32_t b) {
  if (c.plan_flag) atomicCAS(c.plan_flag, 0, int(b) + 1);
}

__device__ __forceinline__ PagedSpan paged_span(const PagedView& c, uint32_t b, int len, int q_first, int q_last, uint32_t tile) {
  PagedSpan s;
  s.len = len;
  s.prefix = c.prefix ? max(0, min(__ldg(c.prefix + b), len)) : 0;
  s.k_hi = max(0, min(len, q_last + 1));
  s.k_lo = c.window ? max(0, q_first + 1 - int(min(c.window, 0x7fffffffu))) : 0;
  s.k_lo = min(s.k_lo, s.k_hi);
  s.lo = uint32_t(s.k_lo) / tile;
  s.end = s.k_hi > s.k_lo ? (uint32_t(s.k_hi) + tile - 1) / tile : s.lo;
  s.pre = (uint32_t(s.prefix) + tile - 1) / tile;
  if (s.end > s.lo && s.pre >= s.lo) {            // prefix and band touch: one run of tiles
    s.end = max(s.end, s.pre);
    s.lo = 0;
    s.pre = 0;
  }
  return s;
}

// Page of table entry `e` of sequence b, or `pages` (one past the pool: a TMA box there is filled with zeros) with the
// flag raised when the entry is not a page.
__device__ __forceinline__ uint32_t paged_page(const PagedView& c, uint32_t b, uint32_t e) {
  const uint32_t page = e < c.table_width ? uint32_t(__ldg(c.table + size_t(b) * c.table_stride + e)) : c.pages;
  if (page < c.pages) return page;
  paged_raise(c, b);
  return c.pages;
}

// Checks an mb_paged_kv and fills the view. `terms` may be null (the append has none).
int paged_view(mb_ctx* ctx, const char* what, const mb_paged_kv* kv, const mb_score_terms* terms, size_t heads, PagedView* out);
// Rows of one TMA box: the largest power of two that divides the page and does not exceed `most` (page_size is a
// multiple of 16, so at least 16; a box never crosses a page).
inline uint32_t paged_box_rows(size_t page_size, uint32_t most) {
  uint32_t r = 16;
  while (r < most && page_size % (2 * r) == 0) r *= 2;
  return r;
}
// Tensor map over a bf16 pool [pages, page_size, kv_heads, d], box 64 x 1 x box_rows x 1 under the 128-byte swizzle.
int paged_pool_map(mb_ctx* ctx, CUtensorMap* tm, const void* pool, const mb_paged_kv* kv, uint32_t box_rows);
// bf16 tensor map of up to five dimensions, innermost first, 128-byte swizzle, zeros out of bounds.
int paged_encode_map(mb_ctx* ctx, CUtensorMap* tm, uint32_t rank, const void* base, const uint64_t* dims,
                     const uint64_t* strides_bytes, const uint32_t* box);

// 2^x on the special-function unit; its error (2 ulp) is far below the 2^-9 of the bf16 probabilities it becomes.
__device__ __forceinline__ float paged_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// tanh(x) of a score over its cap: 1 - 2 / (e^2x + 1), saturating at +-1 through e^2x = inf or 0, with an absolute error of a
// few 2^-24. The cap multiplies that error into an exponent of two: up to cap * log2(e) = 512 it stays below 2e-4, an eighth
// of the rounding of a bf16 probability. A larger cap may be any number of times the score, so there values below 1/2 are
// x + x^3 q(x^2), q of degree two (a weighted least-squares fit, reweighted towards the smallest maximum; off by 1.9e-7
// and by 1.0e-6 of its value at most). The one-instruction tanh is off by 2^-11 of its value, 0.02 in a score near a cap of
// 50. The decode kernels choose by the cap (83.5 us against 86.1 with the second form always, two tokens of 32 sequences over
// four-bit rows); the general form of the prompt kernel always takes both (263 us against 270 by the cap, 2 x 515 tokens
// over 12000 rows).
constexpr float PAGED_LARGE_CAP = 512.0f;
__device__ __forceinline__ float paged_tanh(float x, bool large_cap) {
  const float e = paged_ex2(x * 2.8853900817779268f);    // 2 log2(e)
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(e + 1.0f));
  r = fmaf(-2.0f, r, 1.0f);
  if (large_cap) {
    const float y = x * x;
    const float q = fmaf(fmaf(-4.422929382e-02f, y, 1.318586219e-01f), y, -3.332646081e-01f);
    r = fabsf(x) < 0.5f ? fmaf(x * y, q, x) : r;
  }
  return r;
}
