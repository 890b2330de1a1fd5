// attention_paged.cuh -- what the two attention kernels over the paged cache share: arguments,
// 16-bit packing, and which key tiles a range of query positions meets.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "epilogue.cuh"
#include "paged_cache.cuh"

namespace lsc {

constexpr float kLog2e = 1.4426950408889634f;

struct AttnArgs {
  const uint16_t* q;
  int64_t tokens, q_token, q_head;
  const int32_t* offsets;  // null: row b is sequence b's one new token
  int32_t q_heads, group;
  float scale_log2;  // alpha * log2(e): scores are kept as powers of two
  int32_t window, sinks;
  uint16_t* out;
  int8_t* out_i8;
  float s_out, inv_s_out;
  int32_t rounding;
};

// The checks that both entry points share; fills `a` but for the offsets.
lsc_status attention_args(const lsc_paged_kv* cache, const char* who, const void* q, int64_t tokens, int32_t q_heads,
                          int64_t q_token, int64_t q_head, float alpha, int64_t window, int64_t sinks, void* out,
                          int8_t* out_i8, float s_out, int32_t rounding, AttnArgs* a);

// Tensor map of the keys or values {64, page_size, head_dim / 64, heads, pages}: boxes of box_rows
// places x box_blocks column blocks of 64 elements, the blocks one after another in shared memory.
lsc_status paged_tensor_map(CUtensorMap* map, const lsc_paged_kv* cache, const PagedView& view, const void* base,
                            uint32_t box_rows, uint32_t box_blocks);

__device__ __forceinline__ float ex2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// mbarrier.try_wait that may suspend the thread for up to a millisecond: a waiting warp that comes
// back sooner spends issue slots that the softmax needs.
__device__ __forceinline__ bool mbar_try_wait_long(uint32_t bar_addr, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n .reg .pred P;\n mbarrier.try_wait.parity.shared::cta.b64 P, [%1], %2, %3;\n"
      " selp.u32 %0, 1, 0, P;\n}\n"
      : "=r"(ok)
      : "r"(bar_addr), "r"(parity), "r"(1000000u)
      : "memory");
  return ok != 0;
}

// mbar_wait by all lanes of a warp with one outcome (false for all when it ran out).  The global
// timer takes longer to read than most waits here last, so it is read at every 64th try only; the
// loop is kept small because it stands in many places.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile uint32_t* abort_flag, uint32_t* err) {
  const uint32_t at = smem_u32(bar);
  unsigned long long until = 0;
#pragma unroll 1
  for (uint32_t n = 1; !__all_sync(0xffffffffu, mbar_try_wait_long(at, parity)); ++n) {
    if ((n & 63u) != 0) continue;
    const unsigned long long now = globaltimer_ns();
    if (until == 0) until = now + kWaitLimitNs;
    if (__any_sync(0xffffffffu, *abort_flag != 0 || now > until)) {
      *abort_flag = 1u;
      if (now > until) atomicOr(err, LSC_DEVERR_TIMEOUT);
      return false;
    }
  }
  return true;
}

// f16 ends at 2^16 above and rounds below 2^-14 in steps of 2^-24, so a probability taken relative to the
// largest one would be lost from 2^-25 on, while the sum l still counts it: very many faint keys behind a
// strong one would then shrink the output (131072 of them by 0.4 %).  So f16 probabilities, which reach
// 2^MOST, go into the product with V times 2^kRaise, which brings those to 2^15.  bf16 has the exponents
// of f32 and needs no factor.
template <bool BF16, int MOST>
constexpr int kRaise = BF16 ? 0 : 15 - MOST;

// {lo, hi} rounded to the cache's type and packed
template <bool BF16>
__device__ __forceinline__ uint32_t pack16(float lo, float hi) {
  uint32_t d;
  if constexpr (BF16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
  else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
  return d;
}

// What packing left of both: {lo, hi} minus the packed values, rounded and packed
template <bool BF16>
__device__ __forceinline__ uint32_t pack16_rest(float lo, float hi, uint32_t packed) {
  float2 v;
  if constexpr (BF16) v = make_float2(__uint_as_float(packed << 16), __uint_as_float(packed & 0xFFFF0000u));
  else v = __half22float2(*reinterpret_cast<const __half2*>(&packed));
  return pack16<BF16>(lo - v.x, hi - v.y);
}

// The key tiles (of TILE places) that queries at positions first .. last meet, sinks apart from
// the window: tile i of n is key tile i < sink_tiles ? i : start + i - sink_tiles, counted from `skip`
// on where the list is a part of another.
template <int TILE>
struct TileList {
  int32_t n, sink_tiles, start, skip = 0;
  __device__ __forceinline__ TileList(int32_t first, int32_t last, int32_t window, int32_t sinks) {
    const int32_t low = window > 0 && first >= window ? first - window + 1 : 0;
    const int32_t kept = sinks < low ? sinks : low;
    sink_tiles = (kept + TILE - 1) / TILE;
    start = low / TILE;
    if (start <= sink_tiles) sink_tiles = start = 0;
    n = last < 0 ? 0 : sink_tiles + last / TILE + 1 - start;
  }
  __device__ __forceinline__ int32_t tile(int32_t i) const {
    i += skip;
    return i < sink_tiles ? i : start + i - sink_tiles;
  }
  // part x of `parts` equal ones (a few: a list of a sequence's 2^30 places has at most 2^24 tiles)
  __device__ __forceinline__ void take(uint32_t x, uint32_t parts) {
    const uint32_t all = static_cast<uint32_t>(n);
    skip = static_cast<int32_t>(all * x / parts);
    n = static_cast<int32_t>(all * (x + 1) / parts) - skip;
  }
};

}  // namespace lsc
