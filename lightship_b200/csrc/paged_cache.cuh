// paged_cache.cuh -- the paged key-value cache as its kernels see it: addresses, lengths and the
// visibility rule, shared by the append (paged_cache.cu) and the attention kernels.
#pragma once
#include <stdint.h>

#include "lsc_internal.h"
#include "sm100.cuh"

namespace lsc {

struct PagedView {
  uint16_t* k;  // 16-bit elements of either type
  uint16_t* v;
  const int32_t* table;
  const int32_t* lens;
  int64_t table_stride, num_pages;
  int64_t page_stride, token_stride, head_stride;  // elements
  int32_t max_pages, batch, kv_heads;
  int32_t page_shift;  // log2(page_size)
  uint32_t* err;
};

// Checks a cache description on the host and fills `view` (all but the error word).
lsc_status paged_view(const lsc_paged_kv* cache, const char* who, PagedView* view);
// The current device's state, which has to be an sm_100 one; sets the view's error word.
lsc_status paged_device(const char* who, DeviceState** ds, PagedView* view);

__device__ __forceinline__ void raise_bad_arg(uint32_t* err) { atomicOr(err, LSC_DEVERR_BAD_ARG); }

// Lengths, tables and offsets are read by plain loads: a kernel whose launch overlaps the one before
// may share an SM with the writer, which the read-only path does not follow.
// kv_lens[b], clamped to the table's reach; `flag` raises the error word for a length out of range.
__device__ __forceinline__ int32_t paged_len(const PagedView& c, int b, bool flag) {
  const int32_t n = c.lens[b];
  const int32_t most = c.max_pages << c.page_shift;
  if (n >= 0 && n <= most) return n;
  if (flag) raise_bad_arg(c.err);
  return n < 0 ? 0 : most;
}

// Rows [begin, end) of sequence b among `tokens`; empty where the offsets decrease or leave them.
__device__ __forceinline__ void query_rows(const int32_t* offsets, int b, int64_t tokens, uint32_t* err,
                                           bool flag, int32_t& begin, int32_t& end) {
  begin = offsets[b];
  end = offsets[b + 1];
  if (begin >= 0 && begin <= end && end <= tokens) return;
  if (flag) raise_bad_arg(err);
  end = begin = 0;
}

// Raises the error word for offsets and lengths out of range; called by the threads of one CTA.
__device__ __forceinline__ void check_rows(const PagedView& c, const int32_t* offsets, int64_t tokens) {
  int32_t begin, end;
  for (int b = threadIdx.x; b < c.batch; b += blockDim.x) {
    query_rows(offsets, b, tokens, c.err, true, begin, end);
    paged_len(c, b, true);
  }
}

// Key j as the query at position p sees it.  `low` = p - window + 1, or 0 without a window.
__device__ __forceinline__ bool key_visible(int32_t j, int32_t p, int32_t low, int32_t sinks) {
  return (j <= p) & ((j >= low) | (j < sinks));
}

// Bits 0 .. n - 1 (all for n >= 32, none for n <= 0).
__device__ __forceinline__ uint32_t low_bits(int32_t n) {
  return n >= 32 ? 0xFFFFFFFFu : (n <= 0 ? 0u : (1u << n) - 1u);
}

// key_visible of keys j .. j + 31, as bits.
__device__ __forceinline__ uint32_t visible_mask(int32_t j, int32_t p, int32_t low, int32_t sinks) {
  return low_bits(p - j + 1) & (~low_bits(low - j) | low_bits(sinks - j));
}

}  // namespace lsc
