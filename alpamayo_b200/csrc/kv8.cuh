// kv8.cuh — the paged int8 key/value cache as the kernels see it.
//
// A page holds `page` tokens of one sequence for every KV head:
//   codes  int8  [num_pages][kv_heads][page][head_dim]   (K and V apart)
//   scales float [num_pages][kv_heads]                   (K and V apart)
// and stands for code * scale.  The page table is int32 [B][table_width];
// token t of sequence b lies in page table[b][t / page] at t % page.
#pragma once

#include "tc_ptx.cuh"

namespace paro {

constexpr float kKv8Max = 127.0f;   // largest code: symmetric, -128 is not used

struct Kv8View {
  int8_t* k_codes;
  int8_t* v_codes;
  float* k_scale;
  float* v_scale;
  int64_t num_pages;
  const int32_t* table;
  int table_width;
  int kv_heads;
  int page_shift;   // log2 of the page size (16, 32, 64, 128)
  int dim;          // 64 or 128
};

// Tokens of a sequence that its row of the page table can hold; a longer
// length is reported and cut (nothing outside the table is read).
__device__ __forceinline__ int kv8_len(const Kv8View& c, int len) {
  const int64_t cap = (int64_t)c.table_width << c.page_shift;
  if (len < 0 || len > cap) {
    report_error(kErrBadPage);
    return len < 0 ? 0 : (int)cap;
  }
  return len;
}

// Page of token block `blk` (< table_width) of sequence b, or -1 (reported)
// where the entry is not a page of the pool.
__device__ __forceinline__ int kv8_page(const Kv8View& c, int b, int blk) {
  const int id = c.table[(int64_t)b * c.table_width + blk];
  if (id < 0 || id >= c.num_pages) {
    report_error(kErrBadPage);
    return -1;
  }
  return id;
}

// First element of (page, head)'s token 0 in a code array.
__device__ __forceinline__ int64_t kv8_base(const Kv8View& c, int page, int h) {
  return (((int64_t)page * c.kv_heads + h) << c.page_shift) * c.dim;
}

// Code of x under `scale` (= absmax / 127): the nearest integer, ties to
// even; a zero scale (all-zero page) gives zero codes, a scale that is not
// finite reads back as NaN whatever the code.
__device__ __forceinline__ int kv8_code(float x, float scale) {
  if (!(scale > 0.f)) return 0;
  return max(-127, min(127, __float2int_rn(__fdiv_rn(x, scale))));
}

// Sequence b of packed item `item` when sequence b owns count(b) consecutive
// items: all lanes of a warp call it and get b and the first item of b, or
// b = -1 past the last one.
template <typename Count>
__device__ __forceinline__ int warp_find_seq(int64_t item, int B, Count count, int64_t* first) {
  const int lane = threadIdx.x & 31;
  int64_t before = 0;
  for (int b0 = 0; b0 < B; b0 += 32) {
    const int64_t mine = b0 + lane < B ? count(b0 + lane) : 0;
    int64_t incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t up = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += up;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, before + incl > item);
    if (hit) {
      const int src = __ffs(hit) - 1;
      *first = before + __shfl_sync(0xffffffffu, incl - mine, src);
      return b0 + src;
    }
    before += __shfl_sync(0xffffffffu, incl, 31);
  }
  *first = before;
  return -1;
}

}  // namespace paro
