// attention_decode.cu -- attention of one new token per sequence over the paged key-value cache,
// split over the cache's length and joined:
//   O[b, h, :] = sum_j p_j V[j, :] / l,  p_j = 2^(s_j - m),  s_j = alpha log2(e) Q[b, h, :] . K[j, :]
// with m the running maximum and l the sum of p over the visible places j.
//
// Every byte of K and V is read once (once per 64 heads of a larger group) and used for at most 4 flops per
// query head of its group, so the cache's bandwidth bounds it.  The work is cut by bytes, not by sequences: the key tiles (64
// places) of all (sequence, key-value head) pairs form one list, and CTA c of G takes tiles
// [c T / G, (c + 1) T / G) of it, so a ragged batch and a single long sequence load the GPU alike.
// A CTA meets whole pairs, which it writes out itself, and at most two cut ones (its first and its
// last), whose (m, l, O) go to the workspace; a second kernel joins the parts of each cut pair in
// the order of the CTAs, so results do not depend on timing.
//
// One warp per CTA brings tiles by TMA into a ring of 128-byte-swizzled stages, page by page (the
// boxes of pages without a visible place read out of the tensor's range: zeros, no traffic).
// Four warps multiply: the up to 16 query heads of a group are the rows of m16n8k16 products (the
// instruction needs one eighth of the rows that tcgen05 does, and at 4 flops a byte the legacy
// tensor path is far from its limit).  Measured: 131072 places of 8 bf16 heads of 128, 32 query heads, in
// 92 to 94 us (5.7 to 5.8 TB/s of keys and values); 64 sequences of up to 8192 places in 182 to 195 us
// (5.6 to 6.0 TB/s).  Groups of more than 16 heads give the warps heads instead of keys: MT row tiles x
// (4 / MT) key slices.  Each warp keeps its own m, l and O.  With heads of 128 that takes more registers
// than there are: two row tiles spill about 90 bytes a thread and four about 290 (350 for an int8
// output), and every warp reads the keys of its slice for itself (16 sequences of 4096 places, 64 heads on
// one, 31 us; its bytes alone would take 5).
#include "attention_paged.cuh"

namespace lsc {
namespace {

constexpr int kTile = 64;         // places per key tile
constexpr int kConsumers = 4;     // multiplying warps
constexpr int kDecodeThreads = 32 * (kConsumers + 1);
constexpr int kMaxCtas = 320;     // bound of the grid, and so of the workspace

template <int D>
struct DecodeShape {
  static constexpr int kTileBytes = kTile * D * 2;               // K or V of one tile
  static constexpr int kStages = D == 128 ? 3 : 6;               // 96 KB of tiles: two CTAs per SM
  static constexpr int kSwapBytes = 3 * 16 * 64 * 4;             // O of three warps, 64 columns at a time
  static constexpr int kSmem = kStages * 2 * kTileBytes + kSwapBytes + 2 * 64 * 4 + 256 + 1024;
};

struct DecodeArgs {
  AttnArgs a;
  int32_t head_tiles;  // row tiles of 16 * MT heads per key-value head
  int32_t split;       // 0: CTAs take whole pairs
  int32_t* desc;       // [grid][4]: sequence, pair, parts (0: none), unused
  float* part_m;       // [2 * grid][16 * MT]
  float* part_l;
  float* part_o;       // [2 * grid][16 * MT][D]
};

__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
template <bool BF16>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (BF16)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// A walk over (sequence, pair of the sequence, tile of the pair).
struct Cursor {
  int32_t b, pair, i;
  int32_t len;
  TileList<kTile> tiles;
  __device__ __forceinline__ Cursor() : tiles(-1, -1, 0, 0) {}
  __device__ __forceinline__ void load(const PagedView& c, const AttnArgs& a) {
    len = paged_len(c, b, false);
    tiles = TileList<kTile>(len - 1, len - 1, a.window, a.sinks);
  }
  // To the first tile of the next pair; called while there is one.  Empty sequences are passed eight at a time
  // (one after another, 8188 empty slots behind four live sequences took 880 us where this takes 30).
  __device__ __forceinline__ void next_pair(const PagedView& c, const AttnArgs& a, int32_t pairs) {
    i = 0;
    if (++pair < pairs) return;
    pair = 0;
    while (true) {
      if (++b >= c.batch) return;
      load(c, a);
      if (tiles.n > 0) return;
#pragma unroll 1
      while (b + 8 < c.batch) {
        int32_t most = 0;
#pragma unroll
        for (int x = 1; x <= 8; ++x) most = max(most, c.lens[b + x]);
        if (most > 0) break;
        b += 8;
      }
    }
  }
};

// Tiles of sequence b's pairs
__device__ __forceinline__ int64_t tiles_of(const PagedView& c, const AttnArgs& a, int b, int32_t pairs, bool flag) {
  const int32_t len = paged_len(c, b, flag);
  return static_cast<int64_t>(TileList<kTile>(len - 1, len - 1, a.window, a.sinks).n) * pairs;
}

// One output row of two columns
template <bool BF16>
__device__ __forceinline__ void write_pair(const AttnArgs& a, int64_t at, float x, float y) {
  if (a.out) *reinterpret_cast<uint32_t*>(a.out + at) = pack16<BF16>(x, y);
  if (a.out_i8) {
    int32_t u, v;
    if (a.rounding == LSC_ROUND_HALF_EVEN) {
      u = requant_one<LSC_ROUND_HALF_EVEN>(x, a.s_out, a.inv_s_out);
      v = requant_one<LSC_ROUND_HALF_EVEN>(y, a.s_out, a.inv_s_out);
    } else {
      u = requant_one<LSC_ROUND_HALF_AWAY>(x, a.s_out, a.inv_s_out);
      v = requant_one<LSC_ROUND_HALF_AWAY>(y, a.s_out, a.inv_s_out);
    }
    *reinterpret_cast<uint16_t*>(a.out_i8 + at) = static_cast<uint16_t>((u & 0xFF) | ((v & 0xFF) << 8));
  }
}

// FINE, for an int8 output: each p goes into the product as its rounding and the rounding of what is
// left (p rounded once sends values next to a border of the output's codes to the other side).
template <bool BF16, int D, int MT, bool FINE>
__global__ void __launch_bounds__(kDecodeThreads, 2)
    paged_decode_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                        const PagedView c, const DecodeArgs p) {
  using Shape = DecodeShape<D>;
  constexpr int kSlices = kConsumers / MT;  // key slices of a tile
  constexpr int kKeys = kTile / kSlices;    // places of a warp's slice
  constexpr int kRows = 16 * MT;
  constexpr int kBlocks = D / 64;           // 128-byte column blocks of a row
  constexpr int kStages = Shape::kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t{1023});
  float* swap = reinterpret_cast<float*>(smem + kStages * 2 * Shape::kTileBytes);
  float* swap_m = swap + Shape::kSwapBytes / 4;  // [4 warps][16 rows]
  float* swap_l = swap_m + 64;
  uint64_t* full = reinterpret_cast<uint64_t*>(swap_l + 64);
  uint64_t* empty = full + kStages;
  uint64_t* swap_bar = empty + kStages;
  int64_t* plan = reinterpret_cast<int64_t*>(swap_bar + 1);  // tiles before the first sequence, its index
  int64_t* warp_sum = plan + 2;                              // [5]
  volatile uint32_t* abort_flag = reinterpret_cast<volatile uint32_t*>(warp_sum + 5);

  const AttnArgs& a = p.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int32_t pairs = c.kv_heads * p.head_tiles;
  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(full + s, 1);
      mbar_init(empty + s, kConsumers);
    }
    mbar_init(swap_bar, kConsumers);
    *abort_flag = 0u;
    fence_barrier_init();
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
  }
  griddep_wait();

  // ---- which tiles: the total, and where this CTA's first tile lies.  Sequences are scanned 160 at a
  // time; one block of them is enough for most batches, and then lengths are read once.
  const bool once = c.batch <= kDecodeThreads;
  int64_t mine = 0, upto = 0, sum = 0;  // of this thread's sequence; tiles up to it; of all its sequences
  auto scan = [&](int b, bool flag) {
    mine = b < c.batch ? tiles_of(c, a, b, pairs, flag) : 0;
    upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t other = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += other;
    }
    if (lane == 31) warp_sum[warp] = upto;
    __syncthreads();
    int64_t all = 0;
    for (int w = 0; w <= kConsumers; ++w) {
      if (w == warp) upto += all;
      all += warp_sum[w];
    }
    return all;
  };
  int64_t total;
  if (once) {
    total = scan(threadIdx.x, blockIdx.x == 0);
  } else {
    for (int b = threadIdx.x; b < c.batch; b += kDecodeThreads) sum += tiles_of(c, a, b, pairs, blockIdx.x == 0);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) warp_sum[warp] = sum;
    __syncthreads();
    total = 0;
    for (int w = 0; w <= kConsumers; ++w) total += warp_sum[w];
  }
  const int64_t ctas = total < gridDim.x ? total : gridDim.x;
  int64_t begin = 0, end = 0;
  if (blockIdx.x < ctas) {
    begin = blockIdx.x * total / ctas;
    end = (blockIdx.x + 1) * total / ctas;
  }
  if (begin < end) {
    int64_t before = 0;  // tiles of the sequences before this block of 160
    for (int b0 = 0; b0 < c.batch; b0 += kDecodeThreads) {
      int64_t all = 0;
      if (!once) {
        __syncthreads();  // warp_sum has been read
        all = scan(b0 + threadIdx.x, false);
      }
      if (begin >= before + upto - mine && begin < before + upto) {
        plan[0] = before + upto - mine;
        plan[1] = b0 + threadIdx.x;
      }
      before += all;
      if (before > begin) break;
    }
  }
  __syncthreads();
  griddep_launch_dependents();

  // rows of empty sequences
  for (int b = blockIdx.x; b < c.batch; b += gridDim.x) {
    if (paged_len(c, b, false) > 0) continue;
    const int64_t row = static_cast<int64_t>(b) * a.q_heads * D;
    for (int e = threadIdx.x * 8; e < a.q_heads * D; e += kDecodeThreads * 8) {
      if (a.out) *reinterpret_cast<uint4*>(a.out + row + e) = make_uint4(0, 0, 0, 0);
      if (a.out_i8) *reinterpret_cast<uint2*>(a.out_i8 + row + e) = make_uint2(0, 0);
    }
  }
  if (p.desc && threadIdx.x == 0) p.desc[4 * blockIdx.x + 2] = 0;
  if (begin >= end) return;

  Cursor cur;
  cur.b = static_cast<int32_t>(plan[1]);
  cur.load(c, a);
  int64_t rem = begin - plan[0];
  cur.pair = static_cast<int32_t>(rem / cur.tiles.n);
  cur.i = static_cast<int32_t>(rem - static_cast<int64_t>(cur.pair) * cur.tiles.n);
  int64_t left = end - begin;
  if (!p.split) {
    // whole pairs: this CTA owns the pairs whose first tile lies in its range
    if (cur.i > 0) {
      left -= cur.tiles.n - cur.i;
      if (left > 0) cur.next_pair(c, a, pairs);
    }
  }

  if (warp == kConsumers) {
    // ------------------------------------------------------------------ TMA producer (whole warp)
    const int page_size = 1 << c.page_shift;
    const int box_rows = page_size < kTile ? page_size : kTile;
    const int per_tile = kTile / box_rows;  // boxes of K, and of V: at most 8
    const int sub = lane % per_tile;
    const bool is_v = lane / per_tile == 1;
    uint32_t stage = 0, phase = 0;
    int issued = 0;
    bool ok = true;
    while (left > 0 && ok) {
      int64_t count = cur.tiles.n - cur.i;
      if (p.split && count > left) count = left;
      const int kvh = cur.pair / p.head_tiles;
      const int32_t low = a.window > 0 && cur.len > a.window ? cur.len - a.window : 0;
      // this lane's page of tile i: out of the tensor's range when it holds no visible place
      auto page_of = [&](int32_t i) -> int32_t {
        const int32_t j0 = cur.tiles.tile(i) * kTile + sub * box_rows;
        const bool seen = j0 < cur.len && (j0 + box_rows > low || j0 < a.sinks);
        if (!seen) return static_cast<int32_t>(c.num_pages);
        const int32_t id = *(c.table + cur.b * c.table_stride + (j0 >> c.page_shift));
        if (id >= 0 && id < c.num_pages) return id;
        raise_bad_arg(c.err);
        return static_cast<int32_t>(c.num_pages);
      };
      int32_t page = page_of(cur.i);
      for (int32_t i = cur.i; i < cur.i + count; ++i) {
        const int32_t next = i + 1 < cur.i + count ? page_of(i + 1) : 0;
        if (!(ok = warp_wait(empty + stage, phase ^ 1u, abort_flag, c.err))) break;
        if (lane == 0) mbar_arrive_expect_tx(full + stage, 2 * Shape::kTileBytes);
        __syncwarp();
        if (lane < 2 * per_tile) {
          const int32_t j0 = cur.tiles.tile(i) * kTile + sub * box_rows;
          uint8_t* dst = smem + (2 * stage + (is_v ? 1 : 0)) * Shape::kTileBytes + sub * box_rows * (2 * D);
          tma_load_5d(is_v ? &tm_v : &tm_k, full + stage, dst, 0, j0 & (page_size - 1), 0, kvh, page);
        }
        ++issued;
        if (++stage == kStages) {
          stage = 0;
          phase ^= 1u;
        }
        page = next;
      }
      left -= count;
      if (left > 0) cur.next_pair(c, a, pairs);
    }
    if (!ok) {
      // let the copies in flight land before the CTA exits
      volatile uint32_t no_abort = 0;
      for (int s = 0; s < kStages && s < issued; ++s) {
        const int uses = (issued - s + kStages - 1) / kStages;
        mbar_wait(full + s, static_cast<uint32_t>((uses - 1) & 1), &no_abort, c.err);
      }
    }
    return;
  }

  // -------------------------------------------------------------------- multiplying warps
  const int slice = warp % kSlices, mt = warp / kSlices;
  const int r0 = lane >> 2, cpair = (lane & 3) * 2;
  // A tile lies box by box (box_rows places), each box column block by column block: the bytes
  // before place `key`, and between its column blocks
  const int row_shift = c.page_shift < 6 ? c.page_shift : 6;
  const uint32_t block_bytes = 128u << row_shift;
  auto place = [&](int key) -> uint32_t {
    return (static_cast<uint32_t>(key) >> row_shift) * (kBlocks * block_bytes) +
           ((static_cast<uint32_t>(key) & ((1u << row_shift) - 1u)) << 7);
  };
  uint32_t stage = 0, phase = 0, swap_phase = 0;
  int64_t at_tile = begin;
  if (!p.split && left < end - begin) at_tile = end - left;
  while (left > 0) {
    int64_t count = cur.tiles.n - cur.i;
    if (p.split && count > left) count = left;
    const int kvh = cur.pair / p.head_tiles;
    const int head0 = (cur.pair - kvh * p.head_tiles) * kRows;           // of the group
    const int heads = a.group - head0 < kRows ? a.group - head0 : kRows;  // rows that are heads
    const int32_t low = a.window > 0 && cur.len > a.window ? cur.len - a.window : 0;

    // Q of this warp's 16 rows as the A operand
    uint32_t q[D / 16][4];
    {
      const int ra = mt * 16 + r0, rb = ra + 8;
      const uint16_t* base = a.q + cur.b * a.q_token + (static_cast<int64_t>(kvh) * a.group + head0) * a.q_head + cpair;
      const uint16_t* qa = base + ra * a.q_head;
      const uint16_t* qb = base + rb * a.q_head;
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
        q[k][0] = ra < heads ? *reinterpret_cast<const uint32_t*>(qa + 16 * k) : 0u;
        q[k][1] = rb < heads ? *reinterpret_cast<const uint32_t*>(qb + 16 * k) : 0u;
        q[k][2] = ra < heads ? *reinterpret_cast<const uint32_t*>(qa + 16 * k + 8) : 0u;
        q[k][3] = rb < heads ? *reinterpret_cast<const uint32_t*>(qb + 16 * k + 8) : 0u;
      }
    }
    float o[D / 8][4];
#pragma unroll
    for (int n = 0; n < D / 8; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.0f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};

    for (int32_t i = cur.i; i < cur.i + count; ++i) {
      if (!warp_wait(full + stage, phase, abort_flag, c.err)) return;
      const uint32_t sk = smem_u32(smem + 2 * stage * Shape::kTileBytes);
      const uint32_t sv = sk + Shape::kTileBytes;
      const int32_t t0 = cur.tiles.tile(i) * kTile + slice * kKeys;  // this warp's first place
      const bool edge = !(t0 + kKeys <= cur.len && (t0 >= low || t0 + kKeys <= a.sinks));
      // s = Q K^T
      float s[kKeys / 8][4];
#pragma unroll
      for (int n = 0; n < kKeys / 8; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.0f;
#pragma unroll
      for (int n = 0; n < kKeys / 16; ++n) {
        const int key = slice * kKeys + n * 16 + ((lane >> 4) << 3) + (lane & 7);
        const int half = (lane >> 3) & 1;
        const uint32_t at = sk + place(key);
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          const int chunk = 2 * (k & 3) + half;
          uint32_t b[4];
          ldsm4(at + (k >> 2) * block_bytes + ((chunk ^ (key & 7)) << 4), b);
          mma16816<BF16>(s[2 * n], q[k], b[0], b[1]);
          mma16816<BF16>(s[2 * n + 1], q[k], b[2], b[3]);
        }
      }
      float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int n = 0; n < kKeys / 8; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float x = s[n][e] * a.scale_log2;
          if (edge) {
            const int32_t j = t0 + n * 8 + cpair + (e & 1);
            x = key_visible(j, cur.len - 1, low, a.sinks) ? x : -INFINITY;
          }
          s[n][e] = x;
          top[e >> 1] = fmaxf(top[e >> 1], x);
        }
      float f[2], ref[2];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 1));
        top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 2));
        const float now = fmaxf(m[r], top[r]);
        ref[r] = now == -INFINITY ? 0.0f : now;
        f[r] = ex2_approx(m[r] - ref[r]);
        m[r] = now;
        ref[r] -= kRaise<BF16, 0>;
      }
      if (__any_sync(0xffffffffu, f[0] != 1.0f || f[1] != 1.0f)) {
        l[0] *= f[0];
        l[1] *= f[1];
#pragma unroll
        for (int n = 0; n < D / 8; ++n) {
          o[n][0] *= f[0];
          o[n][1] *= f[0];
          o[n][2] *= f[1];
          o[n][3] *= f[1];
        }
      }
      // p = 2^(s - m), rounded to the cache's type for the product with V (the sums take it unrounded).  In
      // f16 all of p, l and O carry a factor of 2^15, here and where parts are joined.
#pragma unroll
      for (int n = 0; n < kKeys / 16; ++n) {
        float e[8];
#pragma unroll
        for (int x = 0; x < 8; ++x) {
          const int r = (x >> 1) & 1;
          e[x] = ex2_approx(s[2 * n + (x >> 2)][x & 3] - ref[r]);
          l[r] += e[x];
        }
        const uint32_t pa[4] = {pack16<BF16>(e[0], e[1]), pack16<BF16>(e[2], e[3]), pack16<BF16>(e[4], e[5]),
                                pack16<BF16>(e[6], e[7])};
        uint32_t pl[4];  // (FINE) what the rounding left
        if constexpr (FINE) {
#pragma unroll
          for (int x = 0; x < 4; ++x) pl[x] = pack16_rest<BF16>(e[2 * x], e[2 * x + 1], pa[x]);
        }
        // values of places that are not seen count as zero, whatever the cache holds there
        uint32_t keep0 = 0xFFFFFFFFu, keep1 = 0xFFFFFFFFu;
        if (edge) {
          const int32_t j = t0 + n * 16 + cpair;
          auto keep = [&](int32_t x) { return key_visible(x, cur.len - 1, low, a.sinks); };
          keep0 = (keep(j) ? 0xFFFFu : 0u) | (keep(j + 1) ? 0xFFFF0000u : 0u);
          keep1 = (keep(j + 8) ? 0xFFFFu : 0u) | (keep(j + 9) ? 0xFFFF0000u : 0u);
        }
        const int key = slice * kKeys + n * 16 + (((lane >> 3) & 1) << 3) + (lane & 7);
        const uint32_t at = sv + place(key);
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          const int chunk = 2 * (k & 3) + (lane >> 4);
          uint32_t b[4];
          ldsm4_t(at + (k >> 2) * block_bytes + ((chunk ^ (key & 7)) << 4), b);
          mma16816<BF16>(o[2 * k], pa, b[0] & keep0, b[1] & keep1);
          mma16816<BF16>(o[2 * k + 1], pa, b[2] & keep0, b[3] & keep1);
          if constexpr (FINE) {
            mma16816<BF16>(o[2 * k], pl, b[0] & keep0, b[1] & keep1);
            mma16816<BF16>(o[2 * k + 1], pl, b[2] & keep0, b[3] & keep1);
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(empty + stage);
      if (++stage == kStages) {
        stage = 0;
        phase ^= 1u;
      }
    }

    // ---- the warps' parts of this pair
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
    }
    auto swap_sync = [&]() -> bool {
      __syncwarp();
      if (lane == 0) mbar_arrive(swap_bar);
      const bool ok = warp_wait(swap_bar, swap_phase, abort_flag, c.err);
      swap_phase ^= 1u;
      return ok;
    };
    float top[2] = {m[0], m[1]};
    if constexpr (kSlices > 1) {
      if ((lane & 3) == 0) {
        swap_m[warp * 16 + r0] = m[0];
        swap_m[warp * 16 + r0 + 8] = m[1];
        swap_l[warp * 16 + r0] = l[0];
        swap_l[warp * 16 + r0 + 8] = l[1];
      }
      if (!swap_sync()) return;
      float f[2];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int row = r0 + 8 * r;
        for (int w = 0; w < kSlices; ++w) top[r] = fmaxf(top[r], swap_m[(mt * kSlices + w) * 16 + row]);
        const float ref = top[r] == -INFINITY ? 0.0f : top[r];
        f[r] = ex2_approx(m[r] - ref);
        l[r] = 0.0f;
        for (int w = 0; w < kSlices; ++w)
          l[r] += swap_l[(mt * kSlices + w) * 16 + row] * ex2_approx(swap_m[(mt * kSlices + w) * 16 + row] - ref);
      }
#pragma unroll
      for (int n = 0; n < D / 8; ++n) {
        o[n][0] *= f[0];
        o[n][1] *= f[0];
        o[n][2] *= f[1];
        o[n][3] *= f[1];
      }
#pragma unroll
      for (int h = 0; h < kBlocks; ++h) {
        if (slice > 0) {
          float* mine = swap + (mt * (kSlices - 1) + slice - 1) * 1024;
#pragma unroll
          for (int n = 0; n < 8; ++n) {
            *reinterpret_cast<float2*>(mine + r0 * 64 + n * 8 + cpair) = make_float2(o[8 * h + n][0], o[8 * h + n][1]);
            *reinterpret_cast<float2*>(mine + (r0 + 8) * 64 + n * 8 + cpair) =
                make_float2(o[8 * h + n][2], o[8 * h + n][3]);
          }
        }
        if (!swap_sync()) return;
        if (slice == 0) {
          for (int w = 0; w < kSlices - 1; ++w) {
            const float* other = swap + (mt * (kSlices - 1) + w) * 1024;
#pragma unroll
            for (int n = 0; n < 8; ++n) {
              const float2 x = *reinterpret_cast<const float2*>(other + r0 * 64 + n * 8 + cpair);
              const float2 y = *reinterpret_cast<const float2*>(other + (r0 + 8) * 64 + n * 8 + cpair);
              o[8 * h + n][0] += x.x;
              o[8 * h + n][1] += x.y;
              o[8 * h + n][2] += y.x;
              o[8 * h + n][3] += y.y;
            }
          }
        }
        if (!swap_sync()) return;
      }
    }
    if (slice == 0) {
      const bool opens = cur.i == 0, closes = cur.i + count == cur.tiles.n;
      if (opens && closes) {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const int row = mt * 16 + r0 + 8 * r;
          if (row < heads) {
            const float inv = l[r] == 0.0f ? 0.0f : __frcp_rn(l[r]);
            const int64_t at = (static_cast<int64_t>(cur.b) * a.q_heads + kvh * a.group + head0 + row) * D + cpair;
#pragma unroll
            for (int n = 0; n < D / 8; ++n) write_pair<BF16>(a, at + 8 * n, o[n][2 * r] * inv, o[n][2 * r + 1] * inv);
          }
        }
      } else {
        const int64_t slot = opens ? gridDim.x + blockIdx.x : blockIdx.x;
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const int row = mt * 16 + r0 + 8 * r;
          if (row < heads) {
            float* to = p.part_o + (slot * kRows + row) * D + cpair;
#pragma unroll
            for (int n = 0; n < D / 8; ++n)
              *reinterpret_cast<float2*>(to + 8 * n) = make_float2(o[n][2 * r], o[n][2 * r + 1]);
            if ((lane & 3) == 0) {
              p.part_m[slot * kRows + row] = top[r];
              p.part_l[slot * kRows + row] = l[r];
            }
          }
        }
        if (opens && warp == 0 && lane == 0) {
          const int64_t last = ((at_tile + cur.tiles.n) * ctas - 1) / total;  // the CTA of the pair's last tile
          p.desc[4 * blockIdx.x] = cur.b;
          p.desc[4 * blockIdx.x + 1] = cur.pair;
          p.desc[4 * blockIdx.x + 2] = static_cast<int32_t>(last - blockIdx.x + 1);
        }
      }
    }
    left -= count;
    at_tile += count;
    if (left > 0) cur.next_pair(c, a, pairs);
  }
}

// Joins the parts of the pair that CTA blockIdx.x opened and did not close, for rows blockIdx.y,
// blockIdx.y + gridDim.y, ...: eight warps take every eighth part, in the order of the CTAs.
template <bool BF16, int D, int MT>
__global__ void __launch_bounds__(256) paged_join_kernel(const PagedView c, const DecodeArgs p, int grid) {
  constexpr int kRows = 16 * MT, kVec = D / 32;
  __shared__ float acc[8][D];
  __shared__ float acc_l[8];
  griddep_wait();
  griddep_launch_dependents();
  const int cta = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int32_t parts = p.desc[4 * cta + 2];
  if (parts == 0) return;
  const int32_t b = p.desc[4 * cta], pair = p.desc[4 * cta + 1];
  const int kvh = pair / p.head_tiles, head0 = (pair - kvh * p.head_tiles) * kRows;
  for (int row = blockIdx.y; row < kRows && head0 + row < p.a.group; row += gridDim.y) {
    const int head = head0 + row;
    // part x lies in the opening slot (x = 0) or in the first-segment slot of CTA cta + x
    auto slot = [&](int x) { return static_cast<int64_t>(x == 0 ? grid + cta : cta + x) * kRows + row; };
    float top = -INFINITY;
    for (int x = lane; x < parts; x += 32) top = fmaxf(top, p.part_m[slot(x)]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const float ref = top == -INFINITY ? 0.0f : top;
    float v[kVec] = {}, l = 0.0f;
#pragma unroll 4
    for (int x = warp; x < parts; x += 8) {
      const int64_t s = slot(x);
      const float f = ex2_approx(p.part_m[s] - ref);
      l += f * p.part_l[s];
      const float* from = p.part_o + s * D + lane * kVec;
#pragma unroll
      for (int e = 0; e < kVec; ++e) v[e] += f * from[e];
    }
#pragma unroll
    for (int e = 0; e < kVec; ++e) acc[warp][lane * kVec + e] = v[e];
    if (lane == 0) acc_l[warp] = l;
    __syncthreads();
    const int d = threadIdx.x * 2;
    if (d < D) {
      float x = 0.0f, y = 0.0f;
      l = 0.0f;
#pragma unroll
      for (int w = 0; w < 8; ++w) {
        x += acc[w][d];
        y += acc[w][d + 1];
        l += acc_l[w];
      }
      const float inv = l == 0.0f ? 0.0f : __frcp_rn(l);
      write_pair<BF16>(p.a, (static_cast<int64_t>(b) * p.a.q_heads + kvh * p.a.group + head) * D + d, x * inv, y * inv);
    }
    __syncthreads();
  }
}

// Row tiles of a group: 16 heads while they suffice, then 32, then 64 (and several of those).
int row_tiles(int group) { return group <= 16 ? 1 : (group <= 32 ? 2 : 4); }

// Caches of short sequences are not cut: the join (2 us, and the parts' way through memory) would cost
// more than the tiles it spreads.  A CTA takes 0.9 us per tile of heads of 128, half of that for heads of
// 64, and with many pairs the GPU is full without a cut.  Cut and whole, us: 8 pairs of 128, 192 places
// 10.2 and 9.7, 320 places 10.6 and 11.8, 512 places 10.8 and 14.4; 32 pairs of 64, 512 places 9.7 and
// 9.5; 64 pairs of 128, 384 places 14.0 and 13.1, 512 places 14.5 and 14.9; 128 pairs of 128, 512 places
// 17.2 and 15.2, 768 places 18.2 and 18.7.
bool is_cut(const lsc_paged_kv* cache) {
  const int64_t pairs = static_cast<int64_t>(cache->batch) * cache->kv_heads;
  const int64_t whole = cache->head_dim == 128 && pairs < 64 ? 256 : 512;  // places
  return static_cast<int64_t>(cache->max_pages) * cache->page_size > whole;
}

uint64_t workspace_bytes_for(int group, int head_dim) {
  const uint64_t rows = 16 * row_tiles(group);
  return kMaxCtas * 16 + 2 * kMaxCtas * rows * (head_dim + 2) * 4;
}

template <bool BF16, int D, int MT, bool FINE>
lsc_status launch_decode(const lsc_paged_kv* cache, const DeviceState* ds, const PagedView& c, DecodeArgs p,
                         cudaStream_t st) {
  using Shape = DecodeShape<D>;
  const uint32_t box = cache->page_size < kTile ? cache->page_size : kTile;
  CUtensorMap tk, tv;
  lsc_status s = paged_tensor_map(&tk, cache, c, cache->k, box, D / 64);
  if (s == LSC_SUCCESS) s = paged_tensor_map(&tv, cache, c, cache->v, box, D / 64);
  if (s) return s;
  int grid = 2 * ds->sm_count;
  if (grid > kMaxCtas) grid = kMaxCtas;
  LSC_CUDA_TRY(cudaFuncSetAttribute(paged_decode_kernel<BF16, D, MT, FINE>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                    Shape::kSmem));
  LSC_CUDA_TRY(launch_dependent(ds->overlap_launches, paged_decode_kernel<BF16, D, MT, FINE>, dim3(grid),
                                dim3(kDecodeThreads), Shape::kSmem, st, tk, tv, c, p));
  if (p.split) {
    const int rows = p.a.group < 16 ? p.a.group : 16;
    LSC_CUDA_TRY(launch_dependent(ds->overlap_launches, paged_join_kernel<BF16, D, MT>, dim3(grid, rows), dim3(256), 0,
                                  st, c, p, grid));
  }
  return LSC_SUCCESS;
}

template <bool BF16, int D, bool FINE>
lsc_status launch_decode_rows(const lsc_paged_kv* cache, const DeviceState* ds, const PagedView& c, const DecodeArgs& p,
                              cudaStream_t st) {
  switch (row_tiles(p.a.group)) {
    case 1: return launch_decode<BF16, D, 1, FINE>(cache, ds, c, p, st);
    case 2: return launch_decode<BF16, D, 2, FINE>(cache, ds, c, p, st);
    default: return launch_decode<BF16, D, 4, FINE>(cache, ds, c, p, st);
  }
}

}  // namespace
}  // namespace lsc

using namespace lsc;

extern "C" {

uint64_t lsc_paged_attention_decode_workspace_size(const lsc_paged_kv* cache, int32_t q_heads) {
  if (!cache || cache->kv_heads < 1 || q_heads < 1 || !is_cut(cache)) return 0;
  return workspace_bytes_for(q_heads / cache->kv_heads, cache->head_dim);
}

lsc_status lsc_paged_attention_decode(const lsc_paged_kv* cache, const void* q, int32_t q_heads,
                                      int64_t q_token_stride, int64_t q_head_stride, float alpha, int64_t window,
                                      int64_t sinks, void* out, int8_t* out_i8, float s_out, int32_t rounding,
                                      void* workspace, uint64_t workspace_bytes, lsc_stream stream) {
  const char* who = "paged_attention_decode";
  PagedView c;
  DecodeArgs p{};
  lsc_status st = paged_view(cache, who, &c);
  if (st) return st;
  st = attention_args(cache, who, q, c.batch, q_heads, q_token_stride, q_head_stride, alpha, window, sinks, out, out_i8,
                      s_out, rounding, &p.a);
  if (st) return st;
  if (c.batch == 0) return LSC_SUCCESS;
  p.split = is_cut(cache);
  if (p.split && (!workspace || workspace_bytes < lsc_paged_attention_decode_workspace_size(cache, q_heads) ||
                  (reinterpret_cast<uintptr_t>(workspace) & 15)))
    return set_error(LSC_ERROR_INVALID_ARGUMENT, "%s: the workspace is missing, too small or not 16-byte aligned", who);
  DeviceState* ds = nullptr;
  if ((st = paged_device(who, &ds, &c))) return st;
  const int rows = 16 * row_tiles(p.a.group);
  p.head_tiles = (p.a.group + rows - 1) / rows;
  if (p.split) {
    p.desc = static_cast<int32_t*>(workspace);
    p.part_m = reinterpret_cast<float*>(p.desc + 4 * kMaxCtas);
    p.part_l = p.part_m + 2 * kMaxCtas * rows;
    p.part_o = p.part_l + 2 * kMaxCtas * rows;
  }
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool bf16 = cache->dtype == LSC_DTYPE_BF16;
  const bool wide = cache->head_dim == 128;
  if (out_i8) {
    if (bf16) return wide ? launch_decode_rows<true, 128, true>(cache, ds, c, p, s) : launch_decode_rows<true, 64, true>(cache, ds, c, p, s);
    return wide ? launch_decode_rows<false, 128, true>(cache, ds, c, p, s) : launch_decode_rows<false, 64, true>(cache, ds, c, p, s);
  }
  if (bf16) return wide ? launch_decode_rows<true, 128, false>(cache, ds, c, p, s) : launch_decode_rows<true, 64, false>(cache, ds, c, p, s);
  return wide ? launch_decode_rows<false, 128, false>(cache, ds, c, p, s) : launch_decode_rows<false, 64, false>(cache, ds, c, p, s);
}

}  // extern "C"
