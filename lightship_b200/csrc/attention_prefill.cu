// attention_prefill.cu -- causal attention of a ragged batch of new tokens over the paged key-value
// cache, with a sliding window and sinks, on the 5th-generation tensor cores:
//   O[t, h, :] = sum_j p_j V[j, :] / l,  p_j = 2^(s_j - m),  s_j = alpha log2(e) Q[t, h, :] . K[j, :]
// over the visible places j of the row's sequence, in one pass over the keys with a running
// reference m and sum l.
//
// A unit of work is up to 256 rows, two tiles of 128: consecutive tokens of one sequence times the
// query heads that share a key-value head (hp of them), so a tile of K and V is read once for all
// of them and all heads of a token share one mask.  One persistent CTA per SM walks the units,
// those at the highest positions first (they meet the most keys) and turning at each end of the
// grid, which spreads the causal triangle evenly:
//   warps 0-3, 4-7  softmax of row tile 0 and 1: thread = row.  S (128 keys) comes from TMEM into
//                   registers, p goes back to TMEM, packed, in place of S;
//   warps 8, 9      issue the products of row tile 0 and 1: S = Q K^T (A and B in shared memory) and
//                   O += P V (A in TMEM, V MN-major), P part by part as the softmax writes it, so
//                   that one tile's softmax runs beside the other's products;
//   warp 11         brings the K and V tiles by TMA, page by page; boxes of pages without a visible
//                   place read out of the tensor's range: zeros, no traffic;
//   warp 10         finds the units, brings their Q, and zeroes the rows of V that no row of the unit
//                   sees (a product with p = 0 would keep a NaN) in the few tiles that have such
//                   rows, before they are released to the products.
// m moves only when a row's maximum passes it by more than 2^8: until then p stays below 2^8,
// which bf16 and the f32 sums hold as exactly as values below 1, and O needs no rescaling.  In f16 all of
// p, l and O carry a factor of 2^7 on top, so p stays below 2^15 and is not lost before 2^-32.  When it moves, the softmax thread rescales its row of O in TMEM; the products into O
// that it follows are complete, because S of this tile was issued behind them.
// What bounds it: 128 x 128 scores take 1024 clocks of the tensor cores with heads of 128 (both products) and
// the same of the special function units, and a row tile's softmax and products follow one another; two row tiles
// fill each other's gaps to 60 to 70 % of the tensor cores' measured rate.  Measured: 8192 tokens, 32 query
// heads on 8 of 128 (f16) in 555 to 565 us, 985 TFLOP/s, call after call (the power limit lowers the clock),
// and in 475 in bursts of a few calls at 1965 MHz, which is how the figures beside the rules below were
// taken; 16 on 4 of 64 with a window of 1024 in 95 us; 100 tokens of 12 heads of 64 in 7.7 us.  An int8
// output takes 1.3 times as long (475 and 617 us), for the second product with V.
// With few units (a chunk of a prompt on a long cache) a cluster of 2, 4 or 8 CTAs shares each long one:
// every CTA takes a part of the unit's key tiles, keeps its own m, l and O, and sends each CTA of the
// cluster a share of O's columns through distributed shared memory; the shares are joined there in
// the order of the parts.  No workspace, no second launch.
// Every wait is bounded (a timeout flags the device error word and ends the CTA's work).
#include <type_traits>

#include "attention_paged.cuh"
#include "device_count.h"

namespace lsc {
namespace {

constexpr int kTile = 128;       // rows of a row tile, places of a key tile
constexpr int kPrefillThreads = 384;
constexpr int kSchedSlots = 4;
constexpr int kParts = 2;        // parts of P that are passed on
// Keys of the first part.  The products of the last part are what the next scores wait for, so it is
// small; 64 keys took 477 us where 96 take 474 (8192 tokens, 32 query heads on 8 of 128).
constexpr int kFirstPart = 96;
// The quarter of the exponentials after which the other row tile may begin: 1, 2 and 3 took 476, 475 and
// 474 us there, no turns at all 490.
constexpr int kTurnAt = 3;
// Key tiles per CTA of a cluster that shares a unit, at least, and those of a unit from which on it is
// shared.  A cluster's exchange takes about 6 us, a tile 1.6.  Whole and shared, us, with 8 units: 512 places
// 13.0 and (2 parts) 13.5, 1024 places 19.5 and (4) 14.7, 4096 places 57 and (8) 22.6, 65536 places 810
// and 121.
constexpr int kPartTiles = 2, kSharedTiles = 8;
constexpr int kMoveBy = 8;  // log2 of how far a maximum may pass the reference

// max of three (NaN operands are ignored)
__device__ __forceinline__ float fmax3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

template <int D, bool FINE>
struct PrefillShape {
  static constexpr int kTileBytes = kTile * D * 2;    // Q, K or V of one tile
  static constexpr int kStages = D == 128 ? 5 : 10;   // K and V tiles in turn
  static constexpr int kBarBytes = 768;
  static constexpr int kSmem = (2 + kStages) * kTileBytes + kBarBytes + 1024;
  // TMEM columns of a row tile's S and P, then O of both.  Heads of 128 leave 128 columns for S, and P
  // takes its place: the next S waits for the products with P.  Heads of 64 leave 192 (kApart): tiles
  // take turns at S in the last or the first 128 and P in the last or the first 64 of them, so the next
  // S never meets the P in use and is there when the softmax comes for it.  FINE needs 64 more columns
  // for the low parts of P: there all heads do as heads of 128.
  static constexpr bool kApart = D == 64 && !FINE;
  static constexpr uint32_t kColsS = kApart ? 192 : 128, kColO = 2 * kColsS;
  static constexpr uint32_t s_at(uint32_t turn) { return kApart && turn == 0 ? 64 : 0; }
  static constexpr uint32_t p_at(uint32_t turn) { return kApart && turn == 0 ? 128 : 0; }
};
static_assert(PrefillShape<128, false>::kSmem <= 232448 && PrefillShape<64, false>::kSmem <= 232448, "shared memory budget");

struct PrefillArgs {
  AttnArgs a;
  int32_t hp;          // query heads of a tile
  int32_t tpt;         // tokens of a tile: 128 / hp
  int32_t unit_tokens; // tokens of a unit: tpt or 2 tpt
  int32_t pairs;       // key-value heads x (group / hp)
  int32_t parts;       // CTAs of a cluster that share a unit of one row tile; 1: no cluster
};

// A unit: tokens [row0, row0 + count) of the batch, the first at position pos0 of sequence b.
struct Unit {
  int32_t b, row0, count, pos0, kvh, head0;
};

// What the rows of tile w of a unit see.
struct TileRows {
  int32_t count, first, last, low;
  __device__ __forceinline__ TileRows(const PrefillArgs& p, const Unit& u, int w) {
    count = u.count - w * p.tpt;
    count = count < 0 ? 0 : (count > p.tpt ? p.tpt : count);
    first = u.pos0 + w * p.tpt;
    last = first + count - 1;
    low = p.a.window > 0 && first >= p.a.window ? first - p.a.window + 1 : 0;
  }
};

// The numbers (in a unit's tile list) of the tiles that a row tile meets: the first `kept` and
// [from, to).
struct TileSpan {
  int32_t kept, from, to, n;
  __device__ __forceinline__ TileSpan(const TileRows& r, const TileList<kTile>& tiles, int32_t sinks) {
    n = tiles.n;
    const int32_t shift = tiles.sink_tiles - tiles.start;  // key tile -> number, behind the sinks' tiles
    to = r.count > 0 && r.last >= 0 ? r.last / kTile + 1 + shift : 0;
    from = r.low / kTile + shift;
    from = from < tiles.sink_tiles ? tiles.sink_tiles : from;
    // with the sinks' tiles in front of the list, all tiles up to the one before the window's first
    // that hold a sink
    const int32_t sink_tiles = sinks > 0 ? (sinks - 1) / kTile + 1 : 0;
    kept = tiles.sink_tiles > 0 ? tiles.sink_tiles : sink_tiles;
    kept = kept < to ? kept : to;
    // numbers of the part that the list is
    auto clip = [&](int32_t i) { return i < tiles.skip ? 0 : (i - tiles.skip < n ? i - tiles.skip : n); };
    kept = clip(kept);
    from = clip(from);
    to = clip(to);
    if (kept >= from) kept = from = 0;
  }
  __device__ __forceinline__ bool has(int32_t i) const { return i < kept || (i >= from && i < to); }
  // the number after i (n: none)
  __device__ __forceinline__ int32_t next(int32_t i) const {
    ++i;
    if (i >= kept && i < from) i = from;
    return i < to ? i : n;
  }
};

// The units of this CTA, found by one warp.  Sequence b's units stand at levels
// base_b .. base_b + n_b - 1 (its position in units); F(t) counts those at level t or above.
struct Scheduler {
  const PagedView& c;
  const PrefillArgs& p;
  int lane;
  int64_t total;
  int32_t top;
  // What is known of sequence b: its rows, its length, its units and their first level.
  struct Seq {
    int32_t b, begin, count, len, n, base;
  };
  // Up to 32 sequences with new tokens are held by a lane each, and what follows never reads the batch again
  // (slots: 32); else the batch is read each time (slots: its size) and the first 32 are held.  Four
  // prompts that take 76 us alone take 87 in a batch of 1024 slots so, and took 167 to 195 without the list.
  Seq held;
  int slots;
  __device__ __forceinline__ Seq read(int b) const {
    Seq s{};
    s.b = b;
    if (b >= c.batch) return s;
    int32_t end;
    query_rows(p.a.offsets, b, p.a.tokens, c.err, false, s.begin, end);
    s.len = paged_len(c, b, false);
    s.count = end - s.begin;
    s.n = (s.count + p.unit_tokens - 1) / p.unit_tokens;
    s.base = s.len > s.count ? (s.len - s.count) / p.unit_tokens : 0;
    return s;
  }
  __device__ __forceinline__ Seq of(int i) const { return i == lane ? held : read(i); }
  __device__ __forceinline__ void hold() {
    held = read(lane);
    slots = c.batch;
    if (c.batch <= 32) return;
    Seq list{};
    int live = 0;
#pragma unroll 1
    for (int b = 0; b < c.batch; b += 32) {
      const Seq s = read(b + lane);
      for (uint32_t mask = __ballot_sync(0xffffffffu, s.n > 0); mask; mask &= mask - 1) {
        const int src = __ffs(mask) - 1;
        Seq t;
        t.b = b + src;
        t.begin = __shfl_sync(0xffffffffu, s.begin, src);
        t.count = __shfl_sync(0xffffffffu, s.count, src);
        t.len = __shfl_sync(0xffffffffu, s.len, src);
        t.n = __shfl_sync(0xffffffffu, s.n, src);
        t.base = __shfl_sync(0xffffffffu, s.base, src);
        if (live == 32) return;
        if (lane == live++) list = t;
      }
    }
    held = list;
    slots = 32;
  }
  __device__ __forceinline__ int64_t at_or_above(int32_t t) const {
    int64_t f = 0;
#pragma unroll 1
    for (int b = lane; b < slots; b += 32) {
      const Seq s = of(b);
      const int32_t x = s.base + s.n - t;
      f += x < 0 ? 0 : (x > s.n ? s.n : x);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) f += __shfl_xor_sync(0xffffffffu, f, o);
    return f;
  }
  __device__ __forceinline__ Scheduler(const PagedView& c_, const PrefillArgs& p_, int lane_)
      : c(c_), p(p_), lane(lane_), top(0) {
    hold();
#pragma unroll 1
    for (int b = lane; b < slots; b += 32) {
      const Seq s = of(b);
      top = s.n > 0 && s.base + s.n > top ? s.base + s.n : top;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const int32_t other = __shfl_xor_sync(0xffffffffu, top, o);
      top = other > top ? other : top;
    }
    total = at_or_above(0) * p.pairs;
    level = top;
    level_end = above = 0;
    scan_b = scan_k = 0;
  }
  // Unit number i (all lanes); calls come with growing i, so the level found and the place in the
  // batch are kept: a large batch is scanned once per level.
  int32_t level;               // of the unit before
  int64_t level_end, above;    // F(level), F(level + 1)
  int32_t scan_b, scan_k;      // first sequence of the block scanned last; units of the level before it
  __device__ __forceinline__ Unit find(int64_t i) {
    const int64_t u = i / p.pairs;
    const int32_t pair = static_cast<int32_t>(i - u * p.pairs);
    if (u >= level_end) {
      int32_t lo = 0, hi = level;  // F(lo) > u >= F(hi)
      above = level_end;
      level_end = total / p.pairs;
      while (hi - lo > 1) {
        const int32_t mid = lo + (hi - lo) / 2;
        const int64_t f = at_or_above(mid);
        if (f > u) {
          lo = mid;
          level_end = f;
        } else {
          hi = mid;
          above = f;
        }
      }
      level = lo;
      scan_b = scan_k = 0;
    }
    // the (u - above)-th sequence with a unit at this level
    const int32_t k = static_cast<int32_t>(u - above);
    Unit r{};
#pragma unroll 1
    for (; scan_b < slots; scan_b += 32) {
      const Seq s = of(scan_b + lane);
      const bool here = s.base <= level && level < s.base + s.n;
      const uint32_t mask = __ballot_sync(0xffffffffu, here);
      const int have = __popc(mask);
      if (k >= scan_k + have) {
        scan_k += have;
        continue;
      }
      uint32_t rest = mask;
      for (int x = scan_k; x < k; ++x) rest &= rest - 1;
      const int src = __ffs(rest) - 1;
      const int32_t first = (level - s.base) * p.unit_tokens;
      r.b = __shfl_sync(0xffffffffu, s.b, src);
      r.row0 = __shfl_sync(0xffffffffu, s.begin + first, src);
      r.count = __shfl_sync(0xffffffffu, s.count - first < p.unit_tokens ? s.count - first : p.unit_tokens, src);
      r.pos0 = __shfl_sync(0xffffffffu, s.len - s.count + first, src);
      break;
    }
    const int32_t per_head = p.pairs / c.kv_heads;
    r.kvh = pair / per_head;
    r.head0 = r.kvh * p.a.group + (pair - r.kvh * per_head) * p.hp;
    return r;
  }
};

// FINE, for an int8 output: each p goes into the products as two 16-bit numbers, its rounding and the
// rounding of what is left.  p rounded once moves a value by up to 2^-11 or 2^-8 of it, which is far
// below a step of the output but sends the values next to a border to the other code.
template <bool BF16, int D, bool FINE>
__global__ void __launch_bounds__(kPrefillThreads, 1)
    paged_prefill_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                         const __grid_constant__ CUtensorMap tm_v, const PagedView c, const PrefillArgs p) {
  using Shape = PrefillShape<D, FINE>;
  constexpr int kBlocks = D / 64;
  constexpr int kStages = Shape::kStages;
  constexpr int kBlockBytes = kTile * 128;  // 128 rows of one 128-byte column block
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t{1023});
  uint8_t* s_q = smem;
  uint8_t* s_kv = smem + 2 * Shape::kTileBytes;
  uint64_t* bars = reinterpret_cast<uint64_t*>(s_kv + kStages * Shape::kTileBytes);
  uint64_t* kv_full = bars;
  uint64_t* kv_empty = kv_full + kStages;
  uint64_t* landed = kv_empty + kStages;  // V tiles that the zeroing warp passes on
  uint64_t* q_full = landed + kStages;
  uint64_t* q_empty = q_full + 1;
  uint64_t* s_full = q_empty + 1;
  uint64_t* p_full = s_full + 2;  // [row tile][turn][part]
  uint64_t* o_last = p_full + 4 * kParts;  // (kApart) the product before a unit's last one is complete
  uint64_t* s_free = o_last + 2;           // (kApart) the softmax has S in registers
  uint64_t* o_full = s_free + 2;
  uint64_t* drain = o_full + 2;
  uint64_t* turn = drain + 2;  // [row tile]: the other one has done its exponentials
  uint64_t* sched_full = turn + 2;
  uint64_t* sched_empty = sched_full + kSchedSlots;
  Unit* sched = reinterpret_cast<Unit*>(sched_empty + kSchedSlots);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sched + kSchedSlots);
  volatile uint32_t* abort_flag = tmem_slot + 1;

  const AttnArgs& a = p.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(kv_full + s, 1);
      mbar_init(kv_empty + s, 2);
      mbar_init(landed + s, 1);
    }
    mbar_init(q_full, 1);
    mbar_init(q_empty, 2);
    for (int w = 0; w < 2; ++w) {
      mbar_init(s_full + w, 1);
      for (int x = 0; x < 2 * kParts; ++x) mbar_init(p_full + 2 * w * kParts + x, 4);
      mbar_init(o_last + w, 1);
      mbar_init(s_free + w, 4);
      mbar_init(o_full + w, 1);
    }
    for (int w = 0; w < 2; ++w) {
      mbar_init(drain + w, 1);
      mbar_init(turn + w, 4);
    }
    for (int s = 0; s < kSchedSlots; ++s) {
      mbar_init(sched_full + s, 1);
      mbar_init(sched_empty + s, 8 + 2 + 1);  // softmax, products, loads of K and V
    }
    *abort_flag = 0u;
    sched[0].b = -1;
    fence_barrier_init();
    tma_prefetch_desc(&tm_q);
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
  }
  if (warp == 8) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  griddep_wait();
  griddep_launch_dependents();

  // The next unit of this CTA for one warp; false when there is none (or after a timeout).
  uint32_t sched_at = 0, sched_phase = 0;
  auto next_unit = [&](Unit& u) -> bool {
    if (!warp_wait(sched_full + sched_at, sched_phase, abort_flag, c.err)) return false;
    u = sched[sched_at];
    __syncwarp();
    if (lane == 0) mbar_arrive(sched_empty + sched_at);
    if (++sched_at == kSchedSlots) {
      sched_at = 0;
      sched_phase ^= 1u;
    }
    return u.b >= 0;
  };
  auto tiles_of = [&](const Unit& u) {
    TileList<kTile> tiles(u.pos0, u.pos0 + u.count - 1, a.window, a.sinks);
    if (p.parts > 1) {
      const uint32_t most = static_cast<uint32_t>(p.parts), part = blockIdx.x % most;
      const uint32_t room = tiles.n < kSharedTiles ? 1 : static_cast<uint32_t>(tiles.n) / kPartTiles;
      if (part < room) tiles.take(part, room < most ? room : most);
      else tiles.n = 0;
    }
    return tiles;
  };
  // The host knows the table's width only: what a cluster does with its unit goes by the unit's own tiles.
  // Few of them belong to the first CTA alone, which writes the rows as a CTA without a cluster does.
  auto is_shared = [&](const Unit& u) {
    return TileList<kTile>(u.pos0, u.pos0 + u.count - 1, a.window, a.sinks).n >= kSharedTiles;
  };

  if (warp >= 8) {
    regs_shrink<88>();
    if (warp == 10) {
      // ------------------------------------------------------------------ units, zeroing of unseen V rows
      // the CTAs share the check of the batch
#pragma unroll 1
      for (int64_t b = blockIdx.x * 32 + lane; b < c.batch; b += gridDim.x * 32) {
        int32_t begin, end;
        query_rows(a.offsets, static_cast<int>(b), a.tokens, c.err, true, begin, end);
        paged_len(c, static_cast<int>(b), true);
      }
      Scheduler s(c, p, lane);
      int64_t round = 0;         // of the next unit to find: the grid walks them to and fro
      int found = 0, zeroed = 0; // units passed on; units whose V rows are done
      bool more = true, ok = true;
      uint32_t stage = 0, land_phase = 0;  // land_phase: one parity bit per stage
      uint32_t q_phase = 0;
      int q_loads = 0, q_units = 0;  // copies; units whose Q is on its way (or not needed)
      // Q of a unit, once the scores of the unit before are done (they need no more from this warp)
      auto bring_q = [&](const Unit& u) -> bool {
        ++q_units;
        if (tiles_of(u).n == 0) return true;
        if (!warp_wait(q_empty, q_phase ^ 1u, abort_flag, c.err)) return false;
        q_phase ^= 1u;
        if (lane == 0) {
          const int q_tiles = u.count > p.tpt ? 2 : 1;
          mbar_arrive_expect_tx(q_full, static_cast<uint32_t>(q_tiles * kBlocks * p.hp * p.tpt * 128));
          for (int w = 0; w < q_tiles; ++w)
            for (int x = 0; x < kBlocks; ++x)
              tma_load_3d(&tm_q, q_full, s_q + w * Shape::kTileBytes + x * kBlockBytes, x * 64, u.head0,
                          u.row0 + w * p.tpt);
        }
        __syncwarp();
        ++q_loads;
        return true;
      };
      while (ok && (more || zeroed < found)) {
        // Pass on the next unit as soon as its slot is free, but wait for a slot only when there is
        // nothing to zero: the others need no more from this warp to free one.
        // A slot is not used again before this warp has zeroed its unit.
        if (more && found - zeroed < kSchedSlots &&
            (zeroed == found ||
             __all_sync(0xffffffffu, mbar_test_wait(smem_u32(sched_empty + sched_at), sched_phase ^ 1u)))) {
          int64_t i = round * gridDim.x + ((round & 1) ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
          if (p.parts > 1) i = round == 0 ? blockIdx.x / p.parts : s.total;  // one unit per cluster
          ++round;
          Unit u{};
          u.b = -1;
          if (i < s.total) u = s.find(i);
          else if (p.parts == 1 && (round - 1) * gridDim.x < s.total) continue;  // the last round has none for this CTA
          more = u.b >= 0;
          if (!(ok = warp_wait(sched_empty + sched_at, sched_phase ^ 1u, abort_flag, c.err))) break;
          if (lane == 0) {
            sched[sched_at] = u;
            mbar_arrive(sched_full + sched_at);
          }
          __syncwarp();
          if (++sched_at == kSchedSlots) {
            sched_at = 0;
            sched_phase ^= 1u;
          }
          if (more) ++found;
          // the first unit's Q comes before the others are looked for
          if (more && q_units == 0 && !(ok = bring_q(u))) break;
          continue;
        }
        const Unit u = sched[zeroed % kSchedSlots];
        const TileList<kTile> tiles = tiles_of(u);
        if (q_units == zeroed && !(ok = bring_q(u))) break;
        ++zeroed;
        if (tiles.n == 0) continue;
        const int32_t last = u.pos0 + u.count - 1;
        const int32_t low = a.window > 0 && u.pos0 >= a.window ? u.pos0 - a.window + 1 : 0;
        for (int32_t i = 0; i < tiles.n; ++i) {
          const int32_t j0 = tiles.tile(i) * kTile;
          const bool whole = j0 + kTile <= last + 1 && (j0 >= low || j0 + kTile <= a.sinks);
          if (++stage >= kStages) stage -= kStages;  // past the K tile
          if (!whole) {
            if (!(ok = warp_wait(landed + stage, (land_phase >> stage) & 1u, abort_flag, c.err))) break;
            land_phase ^= 1u << stage;
            uint8_t* v = s_kv + stage * Shape::kTileBytes;
            // lanes 8 x .. 8 x + 7 write the eight 16-byte parts of row x (of four at a time)
            for (int r = lane >> 3; r < kTile; r += 4) {
              if (key_visible(j0 + r, last, low, a.sinks)) continue;
#pragma unroll
              for (int x = 0; x < kBlocks; ++x)
                *reinterpret_cast<uint4*>(v + x * kBlockBytes + r * 128 + (lane & 7) * 16) = make_uint4(0, 0, 0, 0);
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(kv_full + stage);
          }
          if (++stage >= kStages) stage -= kStages;
        }
      }
      if ((!ok || *abort_flag) && q_loads > 0) {
        // let the copies in flight land before the CTA exits
        volatile uint32_t no_abort = 0;
        mbar_wait(q_full, static_cast<uint32_t>((q_loads - 1) & 1), &no_abort, c.err);
      }
    } else if (warp == 11) {
      // ------------------------------------------------------------------ loads of K and V
      constexpr int32_t kUnseen = INT32_MIN;  // the page of a box without a visible place
      const int page_size = 1 << c.page_shift;
      const int box_rows = page_size < kTile ? page_size : kTile;
      const int per_tile = kTile / box_rows;
      // a box holds all column blocks where it has the whole tile's places, else one block
      const int boxes = per_tile == 1 ? 1 : per_tile * kBlocks;  // at most 32
      const int sub = lane % per_tile, block = lane / per_tile;
      uint32_t stage0 = 0, phase0 = 0;  // of the unit's first K tile
      uint32_t land_parity = 0;         // per stage: uses of `landed` mod 2
      uint32_t used = 0, by_land = 0, parity = 0;  // per stage: the last copy and its barrier
      bool ok = true;
      Unit u;
      while (ok && next_unit(u)) {
        const TileList<kTile> tiles = tiles_of(u);
        if (tiles.n == 0) continue;
        const int32_t last = u.pos0 + u.count - 1;
        const int32_t low = a.window > 0 && u.pos0 >= a.window ? u.pos0 - a.window + 1 : 0;
        auto page_of = [&](int32_t i) -> int32_t {
          const int32_t j0 = tiles.tile(i) * kTile + sub * box_rows;
          const bool seen = j0 <= last && (j0 + box_rows > low || j0 < a.sinks);
          return seen ? c.table[u.b * c.table_stride + (j0 >> c.page_shift)] : kUnseen;
        };
        const int32_t count = 2 * tiles.n;  // K tiles even, V tiles odd
        int32_t next = page_of(0);
        for (int32_t x = 0; x < count; ++x) {
          const uint32_t y = stage0 + static_cast<uint32_t>(x);
          const uint32_t stage = y % kStages, bit = 1u << stage, phase = phase0 ^ ((y / kStages) & 1u);
          int32_t page = next;
          if (x + 1 < count) next = page_of((x + 1) >> 1);
          if (page < 0 || page >= c.num_pages) {
            if (page != kUnseen) raise_bad_arg(c.err);
            page = static_cast<int32_t>(c.num_pages);
          }
          const int32_t t0 = tiles.tile(x >> 1) * kTile, j0 = t0 + sub * box_rows;
          const bool by_landed = (x & 1) != 0 && !(t0 + kTile <= last + 1 && (t0 >= low || t0 + kTile <= a.sinks));
          if (!(ok = warp_wait(kv_empty + stage, phase ^ 1u, abort_flag, c.err))) break;
          uint64_t* bar = (by_landed ? landed : kv_full) + stage;
          if (lane == 0) mbar_arrive_expect_tx(bar, Shape::kTileBytes);
          __syncwarp();
          if (lane < boxes)
            tma_load_5d((x & 1) != 0 ? &tm_v : &tm_k, bar,
                        s_kv + stage * Shape::kTileBytes + block * kBlockBytes + sub * box_rows * 128, 0,
                        j0 & (page_size - 1), block, u.kvh, page);
          __syncwarp();
          used |= bit;
          if (by_landed) {
            by_land |= bit;
            parity = (parity & ~bit) | (land_parity & bit);
            land_parity ^= bit;
          } else {
            by_land &= ~bit;
            parity = (parity & ~bit) | (phase ? bit : 0u);
          }
        }
        const uint32_t y = stage0 + static_cast<uint32_t>(count);
        phase0 ^= (y / kStages) & 1u;
        stage0 = y % kStages;
      }
      if (!ok || *abort_flag) {
        // let the copies in flight land before the CTA exits
        volatile uint32_t no_abort = 0;
        for (int s = 0; s < kStages; ++s)
          if ((used >> s) & 1u)
            mbar_wait(((by_land >> s) & 1u ? landed : kv_full) + s, (parity >> s) & 1u, &no_abort, c.err);
      }
    } else {
      // ------------------------------------------------------------------ products of one row tile
      // The whole warp walks the tiles and one elected lane issues: a lane that has left its warp
      // issues at half the rate.  One warp per row tile, because what a warp does between products
      // (waits, addresses, a commit that takes the time of three products) would leave the tensor
      // pipe idle; what describes the unit is made uniform, so that descriptors stay in uniform
      // registers.
      constexpr uint32_t idesc_s = BF16 ? idesc_bf16(128, kTile) : idesc_f16(128, kTile);
      constexpr uint32_t idesc_o = (BF16 ? idesc_bf16(128, D) : idesc_f16(128, D)) | (1u << 16);  // V MN-major
      constexpr uint32_t kDescTile = Shape::kTileBytes >> 4;
      auto uniform = [](int32_t x) { return __shfl_sync(0xffffffffu, x, 0); };
      const int w = uniform(warp == 8 ? 0 : 1);
      const uint64_t dq = smem_desc_sw128_kmajor(smem_u32(s_q + w * Shape::kTileBytes));
      const uint64_t dk = smem_desc_sw128_kmajor(smem_u32(s_kv));
      const uint64_t dv = smem_desc_sw128_mnmajor(smem_u32(s_kv), kBlockBytes);
      const uint32_t t_s = uniform(tmem) + w * Shape::kColsS, t_o = uniform(tmem) + Shape::kColO + w * D;
      uint32_t q_phase = 0, p_phase = 0, free_phase = 0;  // p_phase: a bit per turn
      uint32_t stage = 0, phase = 0;  // of the next K tile that has not been used
      bool ok = true, any = false;
      auto step = [](uint32_t& s, uint32_t& ph, uint32_t by) {
        s += by;
        if (s >= kStages) {
          s -= kStages;
          ph ^= 1u;
        }
      };
      // A commit holds up the issuing lane for about as long as three products, so there is one per key
      // tile, behind its scores.  The softmax warps, which wait for it, give back the stages that it
      // shows to be free.
      auto issue_scores = [&](uint32_t turn_of, uint64_t dka) {  // by the elected lane
        const uint32_t to = t_s + (turn_of == 0 ? Shape::s_at(0) : Shape::s_at(1));
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          constexpr int kStep = 32 >> 4, kBlock = kBlockBytes >> 4;
          mma_f16(to, dq + (k >> 2) * kBlock + (k & 3) * kStep, dka + (k >> 2) * kBlock + (k & 3) * kStep, idesc_s,
                  k != 0 ? 1u : 0u);
        }
        mma_commit(s_full + w);
      };
      Unit u;
      while (ok && next_unit(u)) {
        const TileList<kTile> tiles = tiles_of(u);
        const int32_t n = uniform(tiles.n);
        if (n == 0) continue;
        TileSpan span(TileRows(p, u, w), tiles, a.sinks);
        span.kept = uniform(span.kept);
        span.from = uniform(span.from);
        span.to = uniform(span.to);
        span.n = n;
        if (!(ok = warp_wait(q_full, q_phase, abort_flag, c.err))) break;
        q_phase ^= 1u;
        uint32_t more = 0;
        const int32_t first = span.next(-1);
        if (first < n) {
          uint32_t s = stage, ph = phase;
          for (int32_t i = 0; i < first; ++i) step(s, ph, 2);
          if (!(ok = warp_wait(kv_full + s, ph, abort_flag, c.err))) break;
          tc_fence_after();
          if (elect_one()) issue_scores(0, dk + s * kDescTile);
          __syncwarp();
          any = true;
        } else {
          if (lane == 0) mbar_arrive(q_empty);  // no softmax warp will
          __syncwarp();
        }
        uint32_t turn_of = 0;  // of the row tile's tiles, every other
        for (int32_t i = 0; i < n; ++i) {
          uint32_t vs = stage, vph = phase, ks = stage, kph = phase;
          step(vs, vph, 1);
          step(ks, kph, 2);
          const bool mine = span.has(i);
          if ((!Shape::kApart || !mine) && !(ok = warp_wait(kv_full + vs, vph, abort_flag, c.err))) break;
          if (!mine) {
            // Not this row tile's: give the stages back once they hold the tile (before, the arrival
            // would count for the tile that they held last).
            if (!(ok = warp_wait(kv_full + stage, phase, abort_flag, c.err))) break;
            if (lane == 0) {
              mbar_arrive(kv_empty + stage);
              mbar_arrive(kv_empty + vs);
            }
            __syncwarp();
            step(stage, phase, 2);
            continue;
          }
          const uint64_t dva = dv + vs * kDescTile;
          const int32_t j = span.next(i);
          for (int32_t x = i + 1; x < j; ++x) step(ks, kph, 2);
          const uint64_t dka = dk + ks * kDescTile;
          const uint32_t t_p = t_s + (turn_of == 0 ? Shape::p_at(0) : Shape::p_at(1));
          auto products = [&](auto part) {  // by the elected lane
            constexpr int x = decltype(part)::value, kCut = kFirstPart / 16;
#pragma unroll
            for (int k = x ? kCut : 0; k < (x ? kTile / 16 : kCut); ++k) {
              mma_f16_ts(t_o, t_p + k * 8, dva + k * (2048 >> 4), idesc_o, k != 0 ? 1u : more);
              if constexpr (FINE) mma_f16_ts(t_o, t_p + kTile / 2 + k * 8, dva + k * (2048 >> 4), idesc_o, 1u);
            }
          };
          if constexpr (Shape::kApart) {
            if (j < n) {
              if (!(ok = warp_wait(kv_full + ks, kph, abort_flag, c.err))) break;
              if (!(ok = warp_wait(s_free + w, free_phase, abort_flag, c.err))) break;
              free_phase ^= 1u;
              tc_fence_after();
              if (elect_one()) issue_scores(turn_of ^ 1u, dka);
              __syncwarp();
            }
            if (!(ok = warp_wait(kv_full + vs, vph, abort_flag, c.err))) break;
          }
          uint64_t* const p_ready = p_full + (2 * w + (Shape::kApart ? turn_of : 0)) * kParts;
          const uint32_t p_parity = (p_phase >> (Shape::kApart ? turn_of : 0)) & 1u;
          if (!(ok = warp_wait(p_ready, p_parity, abort_flag, c.err))) break;
          tc_fence_after();
          if (elect_one()) products(std::integral_constant<int, 0>{});
          __syncwarp();
          if (!Shape::kApart && j < n && !(ok = warp_wait(kv_full + ks, kph, abort_flag, c.err))) break;
          if (!(ok = warp_wait(p_ready + 1, p_parity, abort_flag, c.err))) break;
          tc_fence_after();
          if (elect_one()) {
            products(std::integral_constant<int, 1>{});
            // heads of 128: S of the row tile's next tile follows its products into O, which read P in S's
            // place; heads of 64: it was issued before
            if (j >= n) mma_commit(o_full + w);
            else if (!Shape::kApart) issue_scores(0, dka);
            else if (span.next(j) >= n) mma_commit(o_last + w);
          }
          __syncwarp();
          p_phase ^= Shape::kApart ? 1u << turn_of : 1u;
          turn_of ^= Shape::kApart ? 1u : 0u;
          more = 1;
          step(stage, phase, 2);
        }
      }
      if (any && (!ok || *abort_flag)) {
        volatile uint32_t no_abort = 0;
        if (elect_one()) {
          mma_commit(drain + w);
          mbar_wait(drain + w, 0u, &no_abort, c.err);
        }
        __syncwarp();
      }
    }
    if (p.parts > 1) {
      __syncwarp();
      cluster_sync();
      cluster_sync();
    }
  } else {
    // -------------------------------------------------------------------- softmax and output
    regs_grow<208>();
    const int w = warp >> 2, quarter = warp & 3;
    const int row = quarter * 32 + lane;
    const uint32_t lanes = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t t_s = tmem + lanes + w * Shape::kColsS;
    const uint32_t t_o = tmem + lanes + Shape::kColO + w * D;
    const int token = row / p.hp, head = row - token * p.hp;
    const float scale = a.scale_log2;
    uint32_t s_phase = 0, o_phase = 0, last_phase = 0;
    uint32_t stage0 = 0;  // of the unit's first K tile
    uint32_t turn_phase = w == 0 ? 1u : 0u;  // row tile 0 begins
    float ref = -INFINITY;  // the reference m, in units of the raw scores
    float l = 0.0f;
    int done = 0;
    Unit u;
    bool ok = true;
    while (ok && next_unit(u)) {
      const TileList<kTile> tiles = tiles_of(u);
      const TileRows rows(p, u, w);
      const uint32_t unit_stage = stage0;
      stage0 = (stage0 + 2u * static_cast<uint32_t>(tiles.n)) % kStages;
      if (rows.count == 0) continue;
      // gives K tile i (v = 0) or V tile i (v = 1) of the unit back to the loads
      auto release = [&](int32_t i, uint32_t v) {
        mbar_arrive(kv_empty + (unit_stage + 2u * static_cast<uint32_t>(i) + v) % kStages);
      };
      const TileSpan span(rows, tiles, a.sinks), other_span(TileRows(p, u, w ^ 1), tiles, a.sinks);
      const bool mine = token < rows.count;
      // positions of this row and of the warp's first and last one
      const int32_t pos = rows.first + (mine ? token : rows.count - 1);
      const int32_t low = a.window > 0 && pos >= a.window ? pos - a.window + 1 : 0;
      const int32_t pos_min = __shfl_sync(0xffffffffu, pos, 0), low_max = __shfl_sync(0xffffffffu, low, 31);
      ref = -INFINITY;
      l = 0.0f;
      done = 0;
      int32_t before = -1, before2 = -1;  // the tile before i, and the one before that
      for (int32_t i = span.next(-1); i < tiles.n;) {
        const int32_t j0 = tiles.tile(i) * kTile, after = span.next(i);
        const uint32_t turn_of = Shape::kApart ? done & 1u : 0u;
        const uint32_t s_here = t_s + (turn_of == 0 ? Shape::s_at(0) : Shape::s_at(1));
        const uint32_t p_here = t_s + (turn_of == 0 ? Shape::p_at(0) : Shape::p_at(1));
        if (!(ok = warp_wait(s_full + w, s_phase, abort_flag, c.err))) break;
        s_phase ^= 1u;
        tc_fence_after();
        // the unit's last scores are there: Q of the next one may come
        if (after >= tiles.n && quarter == 0 && lane == 0) mbar_arrive(q_empty);
        uint32_t s[4][32];
#pragma unroll
        for (int x = 0; x < 4; ++x) tmem_ld_32x32b_x32(s_here + 32 * x, s[x]);
        tmem_ld_wait();
        if constexpr (Shape::kApart) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0 && after < tiles.n) mbar_arrive(s_free + w);
        }
        if (j0 + kTile - 1 > pos_min || (j0 < low_max && j0 + kTile > a.sinks)) {
          // some row of the warp does not see the whole tile: -inf in the places it does not see
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const uint32_t see = visible_mask(j0 + 32 * x, pos, low, a.sinks);
#pragma unroll
            for (int e = 0; e < 32; ++e) s[x][e] = (see >> e) & 1u ? s[x][e] : 0xFF800000u;
          }
        }
        float top[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          top[x] = __uint_as_float(s[x][0]);
#pragma unroll
          for (int e = 1; e < 31; e += 2) top[x] = fmax3(top[x], __uint_as_float(s[x][e]), __uint_as_float(s[x][e + 1]));
          top[x] = fmaxf(top[x], __uint_as_float(s[x][31]));
        }
        const float m = fmax3(fmaxf(top[0], top[1]), top[2], top[3]);
        if (done == 0) {
          ref = m;
        } else {
          // also true where ref is -inf and m is not; false where both are
          const bool move = (m - ref) * scale > static_cast<float>(kMoveBy);
          if (__any_sync(0xffffffffu, move)) {
            if constexpr (Shape::kApart) {
              // The product of the tile before is complete when the next tile's scores, issued behind it,
              // are; where no scores follow it has a barrier of its own.
              if (after < tiles.n) ok = warp_wait(s_full + w, s_phase, abort_flag, c.err);
              else ok = warp_wait(o_last + w, last_phase, abort_flag, c.err);
              if (!ok) break;
              tc_fence_after();
            }
            const float f = move ? ex2_approx((ref - m) * scale) : 1.0f;
            if (move) ref = m;
            l *= f;
#pragma unroll 1
            for (int x = 0; x < D / 32; ++x) {
              uint32_t o[32];
              tmem_ld_32x32b_x32(t_o + 32 * x, o);
              tmem_ld_wait();
#pragma unroll
              for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
              tmem_st_32x32b_x32(t_o + 32 * x, o);
            }
          }
        }
        ++done;
        const float shift = ref == -INFINITY ? 0.0f : fmaf(-ref, scale, static_cast<float>(kRaise<BF16, kMoveBy>));
        const uint64_t scale2 = f2pack(scale, scale), shift2 = f2pack(shift, shift);
        uint64_t sum2[2] = {0ull, 0ull};
        // The two row tiles take turns at the special function units: in step with each other they would
        // wait for them together and for the products together.
        const bool shared = other_span.has(i);
        if (shared) {
          if (!(ok = warp_wait(turn + w, turn_phase, abort_flag, c.err))) break;
          turn_phase ^= 1u;
        }
        auto arrive = [&](int part) {
          tmem_st_wait();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(p_full + (2 * w + turn_of) * kParts + part);
        };
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          uint32_t packed[16], low[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            float y0, y1;
            f2unpack(f2fma(f2pack(__uint_as_float(s[x][2 * e]), __uint_as_float(s[x][2 * e + 1])), scale2, shift2), y0, y1);
            y0 = ex2_approx(y0);
            y1 = ex2_approx(y1);
            sum2[e & 1] = f2add(sum2[e & 1], f2pack(y0, y1));
            packed[e] = pack16<BF16>(y0, y1);
            if constexpr (FINE) low[e] = pack16_rest<BF16>(y0, y1, packed[e]);
          }
          if (shared && x == kTurnAt && lane == 0) mbar_arrive(turn + (w ^ 1));
          if (x == kFirstPart / 32) arrive(0);  // its stores have had the time of 32 keys to complete
          tmem_st_32x32b_x16(p_here + 16 * x, packed);
          if constexpr (FINE) tmem_st_32x32b_x16(p_here + kTile / 2 + 16 * x, low);
        }
        arrive(1);
        if (quarter == 0 && lane == 0) {
          // with the scores all products issued before them were complete
          release(i, 0);
          const int32_t past = Shape::kApart ? before2 : before;
          if (past >= 0) release(past, 1);
        }
        before2 = before;
        before = i;
        float s0, s1;
        f2unpack(f2add(sum2[0], sum2[1]), s0, s1);
        l += s0 + s1;
        i = after;
      }
      if (!ok) break;
      if (done) {
        if (!(ok = warp_wait(o_full + w, o_phase, abort_flag, c.err))) break;
        o_phase ^= 1u;
        tc_fence_after();
        if (quarter == 0 && lane == 0) {
          release(before, 1);
          if (Shape::kApart && before2 >= 0) release(before2, 1);
        }
        if (done >= 2) last_phase ^= 1u;
      }
      if (p.parts > 1 && (blockIdx.x % p.parts > 0 || is_shared(u))) break;
      const float inv = l == 0.0f ? 0.0f : __frcp_rn(l);
      const int64_t at = (static_cast<int64_t>(u.row0 + w * p.tpt + token) * a.q_heads + u.head0 + head) * D;
#pragma unroll 1
      for (int x = 0; x < D / 16; ++x) {
        uint32_t o[16];
        if (done) {
          tmem_ld_32x32b_x16(t_o + 16 * x, o);
          tmem_ld_wait();
        } else {
#pragma unroll
          for (int e = 0; e < 16; ++e) o[e] = 0u;
        }
        __syncwarp();
        if (mine) {
          float y[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) y[e] = __uint_as_float(o[e]) * inv;
          if (a.out) {
#pragma unroll
            for (int v = 0; v < 2; ++v)
              *reinterpret_cast<uint4*>(a.out + at + 16 * x + 8 * v) =
                  make_uint4(pack16<BF16>(y[8 * v], y[8 * v + 1]), pack16<BF16>(y[8 * v + 2], y[8 * v + 3]),
                             pack16<BF16>(y[8 * v + 4], y[8 * v + 5]), pack16<BF16>(y[8 * v + 6], y[8 * v + 7]));
          }
          if (a.out_i8) {
            uint32_t pk[4];
            requant_pack<16>(y, a.s_out, a.inv_s_out, false, a.rounding, pk);
            *reinterpret_cast<uint4*>(a.out_i8 + at + 16 * x) = make_uint4(pk[0], pk[1], pk[2], pk[3]);
          }
        }
        __syncwarp();
      }
      // the next unit's products into O follow p_full, which this warp signals behind these loads
      tc_fence_before();
    }
    if (p.parts > 1) {
      // CTA x of the cluster joins columns [x width, (x + 1) width) of O.  They arrive where the key
      // tiles were, [part][row][width], 16-byte pieces turned by the row against bank conflicts; m and
      // l of all parts where Q was.
      const uint32_t parts = static_cast<uint32_t>(p.parts), width = D / parts, pieces = width / 4;
      const uint32_t part = blockIdx.x % parts;
      float2* const s_ml = reinterpret_cast<float2*>(s_q);  // [part][row]
      __syncwarp();
      cluster_sync();  // every CTA's products and copies are complete
      u = sched[0];
      const bool here = u.b >= 0 && *abort_flag == 0u && is_shared(u);
      if (here && w == 0) {
        for (uint32_t x = 0; x < parts; ++x)
          asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(
                           mapa_shared(smem_u32(s_ml + part * kTile + row), x)),
                       "f"(ref), "f"(l)
                       : "memory");
        if (done) {
#pragma unroll 1
          for (uint32_t x = 0; x < D / 16; ++x) {
            uint32_t o[16];
            tmem_ld_32x32b_x16(t_o + 16 * x, o);
            tmem_ld_wait();
#pragma unroll
            for (uint32_t e = 0; e < 4; ++e) {
              const uint32_t column = 16 * x + 4 * e, to = column / width, piece = column % width / 4;
              const uint32_t at = ((part * kTile + row) * pieces + (piece ^ (row & (pieces - 1)))) * 16;
              asm volatile("st.shared::cluster.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(mapa_shared(smem_u32(s_kv) + at, to)),
                           "r"(o[4 * e]), "r"(o[4 * e + 1]), "r"(o[4 * e + 2]), "r"(o[4 * e + 3])
                           : "memory");
            }
          }
        }
      }
      __syncwarp();
      cluster_sync();
      if (here) {
        const uint32_t chunks = width / 8, rows = static_cast<uint32_t>(u.count * p.hp);
        for (uint32_t i = threadIdx.x; i < rows * chunks; i += 256) {
          const uint32_t r = i / chunks, piece = (i - r * chunks) * 2;
          // a part without a visible key has l = 0, and what it holds of O does not count
          float m = -INFINITY, sum = 0.0f, y[8] = {};
          for (uint32_t x = 0; x < parts; ++x) {
            const float2 ml = s_ml[x * kTile + r];
            if (ml.y != 0.0f) m = fmaxf(m, ml.x);
          }
          for (uint32_t x = 0; x < parts; ++x) {
            const float2 ml = s_ml[x * kTile + r];
            if (ml.y == 0.0f) continue;
            const float f = ex2_approx((ml.x - m) * scale);
            sum += ml.y * f;
#pragma unroll
            for (uint32_t e = 0; e < 2; ++e) {
              const float4 v = *reinterpret_cast<const float4*>(
                  s_kv + ((x * kTile + r) * pieces + ((piece + e) ^ (r & (pieces - 1)))) * 16);
              y[4 * e] += v.x * f;
              y[4 * e + 1] += v.y * f;
              y[4 * e + 2] += v.z * f;
              y[4 * e + 3] += v.w * f;
            }
          }
          const float inv = sum == 0.0f ? 0.0f : __frcp_rn(sum);
#pragma unroll
          for (int e = 0; e < 8; ++e) y[e] *= inv;
          const uint32_t t = r / p.hp;
          const int64_t at = (static_cast<int64_t>(u.row0 + t) * a.q_heads + u.head0 + (r - t * p.hp)) * D + part * width +
                             4 * piece;
          if (a.out)
            *reinterpret_cast<uint4*>(a.out + at) = make_uint4(pack16<BF16>(y[0], y[1]), pack16<BF16>(y[2], y[3]),
                                                               pack16<BF16>(y[4], y[5]), pack16<BF16>(y[6], y[7]));
          if (a.out_i8) {
            uint32_t pk[2];
            requant_pack<8>(y, a.s_out, a.inv_s_out, false, a.rounding, pk);
            *reinterpret_cast<uint2*>(a.out_i8 + at) = make_uint2(pk[0], pk[1]);
          }
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 8) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Whether the device runs `units` clusters of 2, 4 or 8 CTAs at the same time; no, where it does not say.
template <bool BF16, int D, bool FINE>
bool clusters_fit(const DeviceState* ds, int cluster, int64_t units) {
  static DeviceCount counts[3];
  const int at_once = counts[cluster / 4].get(ds->device, [&](int* n) {
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = static_cast<unsigned>(cluster);
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.gridDim = dim3(static_cast<unsigned>(cluster));
    cfg.blockDim = dim3(kPrefillThreads);
    cfg.dynamicSmemBytes = PrefillShape<D, FINE>::kSmem;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const bool known = cudaOccupancyMaxActiveClusters(n, paged_prefill_kernel<BF16, D, FINE>, &cfg) == cudaSuccess;
    if (!known) cudaGetLastError();  // the call goes on without clusters
    return known;
  });
  return units <= at_once;
}

template <bool BF16, int D, bool FINE>
lsc_status launch_prefill(const lsc_paged_kv* cache, const DeviceState* ds, const PagedView& c, PrefillArgs p,
                          cudaStream_t st) {
  using Shape = PrefillShape<D, FINE>;
  const AttnArgs& a = p.a;
  const uint32_t box = cache->page_size < kTile ? cache->page_size : kTile;
  CUtensorMap tq, tk, tv;
  const uint32_t blocks = box == kTile ? D / 64 : 1;
  lsc_status s = paged_tensor_map(&tk, cache, c, cache->k, box, blocks);
  if (s == LSC_SUCCESS) s = paged_tensor_map(&tv, cache, c, cache->v, box, blocks);
  if (s) return s;
  const uint64_t dims[3] = {D, static_cast<uint64_t>(a.q_heads), static_cast<uint64_t>(a.tokens)};
  const uint64_t strides[2] = {static_cast<uint64_t>(a.q_head) * 2, static_cast<uint64_t>(a.q_token) * 2};
  const uint32_t qbox[3] = {64, static_cast<uint32_t>(p.hp), static_cast<uint32_t>(p.tpt)};
  const uint32_t ones[3] = {1, 1, 1};
  s = encode_tmap_3d(&tq, BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, a.q, dims, strides,
                     qbox, ones, CU_TENSOR_MAP_SWIZZLE_128B);
  if (s) return s;
  // units: a sequence's last one may be short
  auto units = [&](int64_t tokens) {
    return (a.tokens + (a.tokens < c.batch ? a.tokens : c.batch) * (tokens - 1)) / tokens * p.pairs;
  };
  LSC_CUDA_TRY(cudaFuncSetAttribute(paged_prefill_kernel<BF16, D, FINE>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                    Shape::kSmem));
  // Two row tiles per unit hide one's softmax behind the other's products; with fewer units than SMs
  // one row tile each spreads the work over more of them.  One and two, us: 256 tokens of 12 heads of 64
  // 9.1 and 10.1; 32 query heads on 8 of 128, 512 tokens 15.2 and 16.5, 1024 tokens (136 units) 25.8 and
  // 25.5, 2048 tokens 68.4 and 44.9.
  p.unit_tokens = units(2 * p.tpt) < ds->sm_count ? p.tpt : 2 * p.tpt;
  const int64_t most = units(p.unit_tokens);
  int grid = static_cast<int>(most < ds->sm_count ? most : ds->sm_count);
  p.parts = 1;
  int64_t places = static_cast<int64_t>(c.max_pages) << c.page_shift;
  const int64_t seen = static_cast<int64_t>(a.window) + a.sinks + p.tpt;
  if (a.window > 0 && places > seen) places = seen;
  // As many CTAs as the longest sequence that the table has room for could use; more clusters than run at
  // once would take twice the time.
  if (p.unit_tokens == p.tpt && places >= kSharedTiles * kTile) {
    while (p.parts < 8 && 2 * p.parts * kPartTiles * kTile <= places &&
           clusters_fit<BF16, D, FINE>(ds, 2 * p.parts, most))
      p.parts *= 2;
  }
  if (p.parts > 1) grid = static_cast<int>(most) * p.parts;  // units of one row tile: there are few
  LSC_CUDA_TRY(launch_clusters(ds->overlap_launches, paged_prefill_kernel<BF16, D, FINE>, dim3(grid),
                               dim3(kPrefillThreads), Shape::kSmem, st, p.parts, tq, tk, tv, c, p));
  return LSC_SUCCESS;
}

}  // namespace

lsc_status attention_args(const lsc_paged_kv* cache, const char* who, const void* q, int64_t tokens, int32_t q_heads,
                          int64_t q_token, int64_t q_head, float alpha, int64_t window, int64_t sinks, void* out,
                          int8_t* out_i8, float s_out, int32_t rounding, AttnArgs* a) {
  if (tokens < 0 || tokens > (1 << 30))
    return set_error(LSC_ERROR_INVALID_ARGUMENT, "%s: bad token count (at most 2^30)", who);
  if (q_heads < 1 || q_heads > 65535 || q_heads % cache->kv_heads)
    return set_error(LSC_ERROR_INVALID_ARGUMENT, "%s: %d query heads are not a multiple of %d key-value heads", who,
                     q_heads, cache->kv_heads);
  if (!(alpha > 0.0f) || !(alpha <= 1.0e38f))
    return set_error(LSC_ERROR_INVALID_ARGUMENT, "%s: alpha must be positive and finite", who);
  if (window < 0 || sinks < 0) return set_error(LSC_ERROR_INVALID_ARGUMENT, "%s: negative window or sinks", who);
  if (rounding != LSC_ROUND_HALF_AWAY && rounding != LSC_ROUND_HALF_EVEN)
    return set_error(LSC_ERROR_INVALID_ARGUMENT, "%s: bad rounding %d", who, rounding);
  // the stride of an axis of one entry is never used: any value will do there
  if (q_heads == 1) q_head = cache->head_dim;
  if (tokens <= 1) q_token = static_cast<int64_t>(q_heads) * cache->head_dim;
  if (q_token < 0 || q_head < 0 || q_token % 8 || q_head % 8 || q_token >= (int64_t{1} << 39) ||
      q_head >= (int64_t{1} << 39))
    return set_error(LSC_ERROR_INVALID_ARGUMENT, "%s: query strides must be multiples of 8 elements", who);
  if (tokens > 0 && cache->batch > 0) {
    if (!q || (!out && !out_i8)) return set_error(LSC_ERROR_INVALID_ARGUMENT, "%s: null pointer", who);
    if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(out_i8)) & 15)
      return set_error(LSC_ERROR_INVALID_ARGUMENT, "%s: buffers must be 16-byte aligned", who);
    if (out_i8 && !(s_out > 0.0f))
      return set_error(LSC_ERROR_INVALID_ARGUMENT, "%s: int8 output needs a scale > 0", who);
  }
  a->q = static_cast<const uint16_t*>(q);
  a->tokens = tokens;
  a->q_token = q_token;
  a->q_head = q_head;
  a->q_heads = q_heads;
  a->group = q_heads / cache->kv_heads;
  a->scale_log2 = alpha * kLog2e;
  // positions stay below 2^30: a longer window is no window, more sinks see no more
  a->window = static_cast<int32_t>(window > (1 << 30) ? 0 : window);
  a->sinks = static_cast<int32_t>(window == 0 ? 0 : (sinks > (1 << 30) ? (1 << 30) : sinks));
  a->out = static_cast<uint16_t*>(out);
  a->out_i8 = out_i8;
  a->s_out = s_out;
  a->inv_s_out = out_i8 ? reciprocal_or_zero(s_out) : 0.0f;
  a->rounding = rounding;
  a->offsets = nullptr;
  return LSC_SUCCESS;
}

lsc_status paged_tensor_map(CUtensorMap* map, const lsc_paged_kv* cache, const PagedView& view, const void* base,
                            uint32_t box_rows, uint32_t box_blocks) {
  const uint64_t dims[5] = {64, static_cast<uint64_t>(cache->page_size), static_cast<uint64_t>(cache->head_dim / 64),
                            static_cast<uint64_t>(cache->kv_heads), static_cast<uint64_t>(cache->num_pages)};
  const uint64_t strides[4] = {static_cast<uint64_t>(view.token_stride) * 2, 128,
                               static_cast<uint64_t>(view.head_stride) * 2, static_cast<uint64_t>(view.page_stride) * 2};
  const uint32_t box[5] = {64, box_rows, box_blocks, 1, 1};
  const uint32_t ones[5] = {1, 1, 1, 1, 1};
  return encode_tmap_5d(map, cache->dtype == LSC_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                            : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                        base, dims, strides, box, ones, CU_TENSOR_MAP_SWIZZLE_128B);
}

}  // namespace lsc

using namespace lsc;

extern "C" lsc_status lsc_paged_attention_prefill(const lsc_paged_kv* cache, const void* q, int64_t tokens,
                                                  int32_t q_heads, int64_t q_token_stride, int64_t q_head_stride,
                                                  const int32_t* q_offsets, float alpha, int64_t window, int64_t sinks,
                                                  void* out, int8_t* out_i8, float s_out, int32_t rounding,
                                                  lsc_stream stream) {
  const char* who = "paged_attention_prefill";
  PagedView c;
  PrefillArgs p{};
  lsc_status st = paged_view(cache, who, &c);
  if (st) return st;
  st = attention_args(cache, who, q, tokens, q_heads, q_token_stride, q_head_stride, alpha, window, sinks, out, out_i8,
                      s_out, rounding, &p.a);
  if (st) return st;
  if (tokens == 0 || c.batch == 0) return LSC_SUCCESS;
  if (!q_offsets || (reinterpret_cast<uintptr_t>(q_offsets) & 3))
    return set_error(LSC_ERROR_INVALID_ARGUMENT, "%s: null or misaligned offsets", who);
  p.a.offsets = q_offsets;
  DeviceState* ds = nullptr;
  if ((st = paged_device(who, &ds, &c))) return st;
  // heads of a row tile: the group, or its largest divisor up to 32
  p.hp = p.a.group;
  if (p.hp > 32)
    for (p.hp = 32; p.a.group % p.hp; --p.hp) {
    }
  p.tpt = kTile / p.hp;
  p.pairs = c.kv_heads * (p.a.group / p.hp);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool bf16 = cache->dtype == LSC_DTYPE_BF16;
  const bool wide = cache->head_dim == 128;
  if (out_i8) {
    if (bf16) return wide ? launch_prefill<true, 128, true>(cache, ds, c, p, s) : launch_prefill<true, 64, true>(cache, ds, c, p, s);
    return wide ? launch_prefill<false, 128, true>(cache, ds, c, p, s) : launch_prefill<false, 64, true>(cache, ds, c, p, s);
  }
  if (bf16) return wide ? launch_prefill<true, 128, false>(cache, ds, c, p, s) : launch_prefill<true, 64, false>(cache, ds, c, p, s);
  return wide ? launch_prefill<false, 128, false>(cache, ds, c, p, s) : launch_prefill<false, 64, false>(cache, ds, c, p, s);
}
