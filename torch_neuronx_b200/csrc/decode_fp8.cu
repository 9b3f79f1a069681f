// Flash decoding against an 8-bit paged cache (cache_rows.cu has the format), products on tensor cores.
//
// The cache is read once for all query heads of a kv head.  Its blocks of 128 keys, over all sequences and kv heads, are one
// list that is cut into equal ranges, one for each CTA the GPU holds at a time: the lengths are read on the device, so ragged
// batches leave no SM without work and no CTA starts twice.  A CTA leaves fp32 partials (o, m, l), one of each computing warp, for
// each (sequence, kv head) that its range touches, in slot `CTA + number of the pair` (both only ever grow along the list, so no slot is used twice),
// and whoever has a pair's first or last block notes the slot; a second launch merges (cache_decode.cu).
// With a prefix that all sequences share (FrontKeys) and that is not worth launches of its own, every sequence is two in the list:
// the prefix's keys, then its own.
// What the format changes:
//   * e4m3 is exact in 16 bits, so both products are 16-bit m16n8k16 MMAs with the bytes expanded in registers (8-bit MMAs would
//     need P and Q in 8 bits).  Both are taken transposed, S^T = K Q^T and O^T = V^T P^T: the keys, then the columns of V,
//     fill the sixteen rows of an MMA and the query heads its eight columns, so that no row is empty and O of 8 heads
//     needs D / 4 registers.  A fragment word of K holds four consecutive elements of one key, and the order inside a
//     k-step is free as long as the query fragments use it too; a transposed fragment word of V holds two keys x two
//     columns, which one byte permutation makes rows 2 i and 2 i + 1 of V^T.  movmatrix turns the probabilities round.
//   * scores: s = (q . k8) * 2^e_k, the row's power of two applied to the finished fp32 score.  A bf16 query row is brought to a
//     maximum in [2^14, 2^15) by a power of two first (fp16 keeps its own scale unless it has room above); should fp16 not hold it
//     exactly even so -- elements below 2^-31 of the largest --, the pair's first product is a bf16 one, a byte shifted into
//     bf16's place being the value times 2^-120 (for all bf16 queries: 64 x 512..8192 keys 134 us, not 123).  That power goes back out with
//     the softmax's scale: maxima are kept in log2 units, which no ordinary score leaves.  Keys from 2^95 on are multiplied in another order.
//   * values: o += (p 2^(e_v - r + 9)) v8 with r the largest e_v the warp has met (o is rescaled when it grows), so the
//     probability stays inside fp16; it enters as hi + lo, two fp16 operands: 22 bits, and never coarser than 2^-34 of
//     the largest value row the warp has met.  That row may have no weight at all, so a warp's keys with a row 2^10 below it are
//     multiplied in bf16, hi + lo: 16 bits at any size.  (Either bf16 product in every block: 64 x 512..8192 keys 240 us, not 120.)
// One warp brings the rows into a ring of blocks by tensor copies, one for each page and operand, and another the scales; four
// warps compute, 32 keys of a block each, and wait for nothing but their block.  (With plain copies and one barrier a block of 64
// keys, as decode_mma.cu has them, the address arithmetic and the latency of table and scales stood in the way: 64 x 512..8192
// keys, 32/8 heads of 128, 194 us.)
// Softmax in the exp2 domain, statistics fp32, the running maximum raised lazily (2^6).
// Bound by HBM once the ring is full (2450 cycles for 128 keys in each of the two CTAs of an SM).  With the merge: 64 x 512..8192 keys,
// 32/8 heads of 128: 119 us, 4.9 TB/s; 16 x 128..4000 keys, 12 heads of 64: 24 us; one sequence of 2001 keys: 11 us.
#include "debug.cuh"
#include "fp8.cuh"
#include "tc_common.cuh"

namespace b200 {

namespace {

using namespace ptx;
using namespace tc;

constexpr int kWarps = kFp8Parts;                         // that compute; one more brings the rows, one the scales
constexpr int kThreads = (kWarps + 2) * 32;
constexpr int kBlockKeys = 128;
constexpr int kWarpKeys = kBlockKeys / kWarps;
constexpr float kRescaleThreshold = 6.0f;
constexpr float kProbShift = 9.0f;   // p <= 2^6, p 2^9 <= 2^15 in fp16
constexpr float kDeep = 10.0f;       // a row this many binades below the largest has its block multiplied in bf16 ...
constexpr float kDeepShift = 110.0f; // ... with probabilities of up to 2^125

// A block of the ring: its rows of K, then of V, swizzled in 16-byte pieces as a tensor copy leaves them (128-byte pattern for
// D = 128, 64-byte for D = 64), so that ldmatrix meets no bank twice.
template <int D, int HEADS> struct Geo {
  static constexpr int kTileBytes = kBlockKeys * D;
  static constexpr int kStageBytes = 2 * kTileBytes;
  static constexpr int kStages = D == 128 && HEADS == 16 ? 2 : 3;
  static constexpr int kRingBytes = kStages * kStageBytes;
  static constexpr int kChunksPerRow = D / 16;
  static constexpr int kCtas = D == 128 || HEADS == 16 ? 2 : 3;             // of an SM
  static __device__ __forceinline__ int swizzle(int row) { return D == 128 ? row & 7 : (row >> 1) & 3; }
};

// What the warps that compute have to know of a block, left beside it by the warp that brings the rows: they walk through the list
// without reading a length.
struct __align__(16) Block {
  int blk, n_keys, last, next_unit;   // last: of this CTA's blocks of the pair; the pair behind it (next_unit -1: none)
  int next_b, pad[3];
};

template <int D, int HEADS> struct Sync {
  static constexpr int kStages = Geo<D, HEADS>::kStages;
  uint64_t full[kStages];                  // the copies' arrivals and those of the warps that start them
  uint64_t empty[kStages];                 // the computing warps
  Block block[kStages];
  alignas(16) uint16_t query[kStages][HEADS][D + 16];   // with a pair's first block: its query rows (padded: fragments meet no bank twice)
  uint32_t scale[kStages][2][kBlockKeys];  // of the keys and of the values: the four bytes around a scale
  uint8_t shift[kStages][2][kBlockKeys];   // ... and the bit at which it starts
  int abort_flag;
  int issued[2];                           // (left by the warps of the rows and of the scales) blocks whose copies were started
};
// Arrivals of a block's barrier: of the warp that brings the rows (one with the bytes of its tensor copies, or its lanes' copies and the
// block's record), and of the warp that brings the scales (its lanes' copies, and what it stores itself).
template <bool TMA> constexpr int kRowArrivals = TMA ? 1 : 33;
constexpr int kScaleArrivals = 33;
template <int D, int HEADS> constexpr int smem_bytes() {
  return Geo<D, HEADS>::kRingBytes + 1024 + static_cast<int>(sizeof(Sync<D, HEADS>));
}

__device__ __forceinline__ void cp_async_16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }
// One of the barrier's counted arrivals, when this thread's copies so far have landed.
__device__ __forceinline__ void cp_async_arrive(uint32_t bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void ldsm_x4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void ldsm_x4_trans(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
template <bool BF16>
__device__ __forceinline__ void mma_16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if (BF16) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    return;
  }
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Four e4m3 values as two bf16 pairs, the even and the odd ones, times 2^-120: sign, exponent and mantissa in their places; subnormal
// numbers and NaN stay what they are.
__device__ __forceinline__ void unpack_e4m3_bf16(uint32_t w, uint32_t& even, uint32_t& odd) {
  const uint32_t x = w << 4 & 0x07f007f0u, y = w >> 4 & 0x07f007f0u;
  even = (w << 8 & 0x80008000u) | x | __vcmpeq2(x, 0x07f007f0u);
  odd = (w & 0x80008000u) | y | __vcmpeq2(y, 0x07f007f0u);
}
// The power of two that brings a query row, whose largest element has the bits `top`, into [2^want, 2^(want + 1)), up to 2^126.
template <bool BF16> __device__ __forceinline__ int power_up(uint32_t top, int want) {
  int up = top == 0u || top >= 0x7f800000u ? 0 : 127 + want - static_cast<int>(top >> 23);   // zeros, infinities and NaN stay as they are
  if (!BF16 && up < 0) up = 0;
  return up > 126 ? 126 : up;   // (-113 and more)
}
// (lo, hi) as a 16-bit pair, and what the rounding left over as another.
template <bool BF16> __device__ __forceinline__ void split_16(float lo, float hi, uint32_t& head, uint32_t& rest) {
  head = pack16<BF16>(lo, hi);
  const float h0 = half_to_f32<BF16>(static_cast<uint16_t>(head)), h1 = half_to_f32<BF16>(static_cast<uint16_t>(head >> 16));
  rest = pack16<BF16>(lo - h0, hi - h1);
}
// The transpose of an 8 x 8 matrix of 16-bit elements: lane 4 i + j holds elements 2 j, 2 j + 1 of row i.
__device__ __forceinline__ uint32_t turn8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// The list of blocks: for each sequence and unit (a kv head and a block of its query heads) the blocks of its keys.
struct List {
  const Problem& p;
  const FrontKeys& front;
  const int units, twice;   // twice: 1 with a front, sequence b is entries 2 b (the front) and 2 b + 1
  __device__ __forceinline__ int count() const { return p.B << twice; }
  __device__ __forceinline__ int keys(int e) const { return twice && (e & 1) == 0 ? front.len : valid_keys(p, e >> twice); }
  __device__ __forceinline__ int blocks(int e) const { return (keys(e) + kBlockKeys - 1) / kBlockKeys; }
  __device__ __forceinline__ int sequence(int e) const { return twice && (e & 1) == 0 ? kSharedPrefix : e >> twice; }   // as it is reported
  __device__ __forceinline__ const int* table(int e) const {
    return twice && (e & 1) == 0 ? front.table : p.block_table + static_cast<int64_t>(e >> twice) * p.table_stride;
  }
};

// A place in the list and the number of blocks behind it that the CTA still has to do; every role walks on its own.
struct Cursor {
  int b, unit, blk;     // entry (a sequence, or one of its two parts), unit, block of the entry
  int n_keys, n_blk;    // of the entry
  int left;

  __device__ __forceinline__ void enter(const List& l) {
    n_keys = l.keys(b);
    n_blk = (n_keys + kBlockKeys - 1) / kBlockKeys;
  }
  // The next block; `left` reaches 0 at the end of the range.
  __device__ __forceinline__ void step(const List& l) {
    if (--left <= 0) return;
    if (++blk < n_blk) return;
    next_pair(l);
  }
  // The first block of the next pair that has one.
  __device__ __forceinline__ void next_pair(const List& l) {
    blk = 0;
    if (++unit < l.units) return;
    unit = 0;
    do {
      ++b;
      enter(l);
    } while (n_blk == 0 && b + 1 < l.count());
  }
};

// The first place of this CTA's range.  Whole warp; lens are read 32 at a time, twice.
__device__ __forceinline__ Cursor first_place(const List& l, int fixed_blocks, int lane) {
  int64_t sum = 0;
  for (int b0 = 0; b0 < l.count(); b0 += 32) sum += __reduce_add_sync(0xffffffffu, b0 + lane < l.count() ? l.blocks(b0 + lane) : 0);
  const int64_t total = sum * l.units;
  int64_t per = fixed_blocks;
  if (per == 0) per = (total + gridDim.x - 1) / gridDim.x;
  const int64_t start = blockIdx.x * per;
  Cursor c = {0, 0, 0, 0, 0, 0};
  if (start >= total) return c;
  c.left = static_cast<int>(total - start < per ? total - start : per);
  int64_t before = 0;
  for (int b0 = 0; b0 < l.count(); b0 += 32) {
    const int mine = b0 + lane < l.count() ? l.blocks(b0 + lane) : 0;
    int upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
      const int x = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += x;
    }
    const unsigned here = __ballot_sync(0xffffffffu, start < (before + upto) * l.units);
    if (here != 0u) {
      const int at = __ffs(here) - 1;
      c.b = b0 + at;
      const int64_t off = start - (before + __shfl_sync(0xffffffffu, upto - mine, at)) * l.units;
      c.enter(l);
      c.unit = static_cast<int>(off / c.n_blk);
      c.blk = static_cast<int>(off % c.n_blk);
      return c;
    }
    before += __shfl_sync(0xffffffffu, upto, 31);
  }
  return c;   // (not reached: start < total)
}

// Table entry of a key position; -1 behind the end.  Looked at where it is used: a look here would wait for the load.
__device__ __forceinline__ int entry_of(const List& l, const Cursor& c, int row) {
  int page = -1;
  if (c.left > 0 && row < c.n_keys) page = l.table(c.b)[row >> l.p.page_shift];
  return page;
}
// A number outside the pool is reported, and page 0 read in its place.
__device__ __forceinline__ int page_of(const List& l, const CacheScales& sc, const Cursor& c, int entry, int row) {
  if (row >= c.n_keys) return -1;
  if (static_cast<unsigned>(entry) < static_cast<unsigned>(sc.n_pages)) return entry;
  report_page(l.p.status, B200_SDPA_ERR_PAGE, l.sequence(c.b), row >> l.p.page_shift << l.p.page_shift, sc.n_pages);
  return 0;
}

// The n-th block's stage is free: the warps that compute have read the block before it there.
template <typename S>
__device__ __forceinline__ bool wait_read(const Problem& p, S* sync, int n, int role, int lane, long long wait_limit) {
  const int s = n % S::kStages, round = n / S::kStages;
  if (round == 0) return true;
  const bool ok = __all_sync(0xffffffffu, wait_clocked(smem_u32(&sync->empty[s]), (round - 1) & 1, &sync->abort_flag, wait_limit));
  if (!ok && lane == 0) report(p.status, role, n, s);
  return ok;
}

// The warp that brings the rows.  Lane l looks up the pages of keys l, l + 32, ... of a block, a block ahead.  TMA: pages of 8
// rows or more, one tensor copy for each page and operand.  Smaller pages: 16-byte copies of single rows.
template <int D, int HEADS, bool TMA>
__device__ __forceinline__ void bring_rows(const List& l, const CacheScales& sc, const CUtensorMap* tm_k, const CUtensorMap* tm_v,
                                           Sync<D, HEADS>* sync, uint32_t ring, Cursor c, int lane, long long wait_limit) {
  using G = Geo<D, HEADS>;
  constexpr int kStages = G::kStages, kLook = kBlockKeys / 32;
  const Problem& p = l.p;
  const int page_mask = (1 << p.page_shift) - 1;
  int entries[kLook], next[kLook];   // of this block and the next (a loop of one block: unrolled over the stages, the code came slower
                                     // from behind the instruction caches than the table's latency is)
  Cursor after = c;
  auto look_up = [&](int (&e)[kLook]) {
#pragma unroll
    for (int i = 0; i < kLook; ++i) e[i] = entry_of(l, after, after.blk * kBlockKeys + lane + 32 * i);
  };
  look_up(entries);
  bool alive = true;
  int n = 0;
#pragma unroll 1
  while (c.left > 0) {
    const int s = n % kStages;
    after.step(l);
    look_up(next);
    alive = wait_read(p, sync, n, 1, lane, wait_limit);
    if (!alive) break;
    const int hk = c.unit % p.Hkv;
    const uint32_t stage = ring + s * G::kStageBytes, bar = smem_u32(&sync->full[s]);
    const int key0 = c.blk * kBlockKeys;
    if (lane == 0) {
      const bool more = after.left > 0;
      Block& k = sync->block[s];
      k.blk = c.blk;
      k.n_keys = c.n_keys;
      k.last = !more || after.b != c.b || after.unit != c.unit;
      k.next_unit = more ? after.unit : -1;
      k.next_b = after.b;
    }
    if constexpr (TMA) {
      const int rows = page_mask + 1 < kBlockKeys ? page_mask + 1 : kBlockKeys;   // of one copy
      const int first = (lane >> 1) * rows;                  // lanes 2 i and 2 i + 1: keys and values of copy i
      int entry = 0;
#pragma unroll
      for (int i = 0; i < kLook; ++i) {
        const int e = __shfl_sync(0xffffffffu, entries[i], first & 31);
        entry = (first >> 5) == i ? e : entry;
      }
      const int page = first < kBlockKeys ? page_of(l, sc, c, entry, key0 + first) : -1;
      const bool mine = page >= 0;
      const unsigned copies = __popc(__ballot_sync(0xffffffffu, mine));
      if (lane == 0) mbar_arrive_expect_tx(bar, copies * rows * D);
      __syncwarp();
      if (mine)
        tma_load_4d(stage + (lane & 1) * G::kTileBytes + first * D, (lane & 1) ? tm_v : tm_k, bar, 0, (key0 + first) & page_mask, hk, page);
    } else {
      // where this lane's rows start, in pieces of 16 bytes; then lanes of a row share out its pieces
      const uint8_t* k_head = static_cast<const uint8_t*>(p.k) + hk * p.ks[1];
      const uint8_t* v_head = static_cast<const uint8_t*>(p.v) + hk * p.vs[1];
      constexpr int kRowsAtOnce = 32 / G::kChunksPerRow;
      const int ch = lane % G::kChunksPerRow;
#pragma unroll
      for (int i = 0; i < kLook; ++i) {
        const int row = 32 * i + lane;
        const int page = page_of(l, sc, c, entries[i], key0 + row);
        const uint32_t in_page = static_cast<uint32_t>((key0 + row) & page_mask), at = static_cast<uint32_t>(page);
        const uint32_t k_at = at * static_cast<uint32_t>(p.ks[0] >> 4) + in_page * static_cast<uint32_t>(p.ks[2] >> 4);
        const uint32_t v_at = at * static_cast<uint32_t>(p.vs[0] >> 4) + in_page * static_cast<uint32_t>(p.vs[2] >> 4);
#pragma unroll 4
        for (int r = lane / G::kChunksPerRow; r < 32; r += kRowsAtOnce) {
          const int there = __shfl_sync(0xffffffffu, page, r);
          const uint32_t k_from = __shfl_sync(0xffffffffu, k_at, r), v_from = __shfl_sync(0xffffffffu, v_at, r);
          if (there < 0) continue;
          const uint32_t dst = stage + (32 * i + r) * D + ((ch ^ G::swizzle(32 * i + r)) << 4);
          cp_async_16(dst, k_head + (static_cast<uint64_t>(k_from) << 4) + ch * 16);
          cp_async_16(dst + G::kTileBytes, v_head + (static_cast<uint64_t>(v_from) << 4) + ch * 16);
        }
      }
      cp_async_arrive(bar);   // (every lane's copies; the barrier counts the 32 lanes)
      __syncwarp();
      if (lane == 0) mbar_arrive(bar);   // (the block's record)
    }
    ++n;
    c = after;
#pragma unroll
    for (int i = 0; i < kLook; ++i) entries[i] = next[i];
  }
  if constexpr (!TMA) cp_async_wait_all();
  if (lane == 0) sync->issued[0] = n;
}

// The warp that brings the scales of a block's keys l, l + 32, ... and of their values, and with the first block of a pair its query
// rows.  All by asynchronous copies: a value that passes through a register would be waited for, and under load each takes as
// long as a block.  (Scales are single bytes at any stride, so the four bytes around one are copied.)  Pages are looked up a block ahead.
template <int D, int HEADS>
__device__ __forceinline__ void bring_scales(const List& l, const CacheScales& sc, Sync<D, HEADS>* sync, Cursor c, int lane,
                                             long long wait_limit) {
  constexpr int kStages = Geo<D, HEADS>::kStages, kLook = kBlockKeys / 32;
  const Problem& p = l.p;
  const int page_mask = (1 << p.page_shift) - 1;
  const uint32_t k_page = static_cast<uint32_t>(sc.ks[0]), v_page = static_cast<uint32_t>(sc.vs[0]);
  const uint32_t k_row = static_cast<uint32_t>(sc.ks[2]), v_row = static_cast<uint32_t>(sc.vs[2]);
  int e[kLook];
  Cursor ahead = c;
  const int blocks = c.left;
  int b = -1, unit = -1;   // whose queries were brought last
  const uint8_t *k_base = nullptr, *v_base = nullptr;
  auto look_up = [&]() {
    const int* table = l.table(ahead.b);
    const int key0 = ahead.blk * kBlockKeys + lane;
#pragma unroll
    for (int i = 0; i < kLook; ++i) {
      e[i] = 0;   // (behind the end: a page that is there; what it says is not used)
      if (ahead.left > 0 && key0 + 32 * i < ahead.n_keys) e[i] = table[(key0 + 32 * i) >> p.page_shift];
    }
    ahead.step(l);
  };
  look_up();
  int n = 0;
#pragma unroll 1
  for (; n < blocks; ++n) {
    if (!wait_read(p, sync, n, 3, lane, wait_limit)) break;
    const int s = n % kStages;
    if (c.unit != unit || c.b != b) {
      b = c.b;
      unit = c.unit;
      const int hk = unit % p.Hkv, h0 = unit / p.Hkv * HEADS, heads = p.group - h0 < HEADS ? p.group - h0 : HEADS;
      k_base = sc.k + hk * sc.ks[1];
      v_base = sc.v + hk * sc.vs[1];
      const uint16_t* q = reinterpret_cast<const uint16_t*>(p.q) + (b >> l.twice) * p.qs[0] + static_cast<int64_t>(hk * p.group + h0) * p.qs[1];
      if (p.qs[3] == 1 && ((reinterpret_cast<uintptr_t>(q) | static_cast<uint64_t>(p.qs[1] * 2)) & 15) == 0) {
        for (int i = lane; i < heads * (D / 8); i += 32)
          cp_async_16(smem_u32(&sync->query[s][i / (D / 8)][i % (D / 8) * 8]), q + i / (D / 8) * p.qs[1] + i % (D / 8) * 8);
      } else {
        for (int i = lane; i < heads * D; i += 32) sync->query[s][i / D][i % D] = q[i / D * p.qs[1] + i % D * p.qs[3]];
      }
    }
    unsigned worst = 0;
#pragma unroll
    for (int i = 0; i < kLook; ++i) worst = max(worst, static_cast<unsigned>(e[i]));
    if (__any_sync(0xffffffffu, worst >= static_cast<unsigned>(sc.n_pages))) {
#pragma unroll
      for (int i = 0; i < kLook; ++i)
        if (static_cast<unsigned>(e[i]) >= static_cast<unsigned>(sc.n_pages)) {
          report_page(p.status, B200_SDPA_ERR_PAGE, l.sequence(b), (c.blk * kBlockKeys + lane + 32 * i) & ~page_mask, sc.n_pages);
          e[i] = 0;
        }
    }
#pragma unroll
    for (int i = 0; i < kLook; ++i) {
      const uint32_t row = static_cast<uint32_t>((c.blk * kBlockKeys + lane + 32 * i) & page_mask);
      const uint64_t page = static_cast<uint32_t>(e[i]);
      const uintptr_t k = reinterpret_cast<uintptr_t>(k_base) + page * k_page + static_cast<uint64_t>(row) * k_row;
      const uintptr_t v = reinterpret_cast<uintptr_t>(v_base) + page * v_page + static_cast<uint64_t>(row) * v_row;
      cp_async_4(smem_u32(&sync->scale[s][0][lane + 32 * i]), reinterpret_cast<const void*>(k & ~static_cast<uintptr_t>(3)));
      cp_async_4(smem_u32(&sync->scale[s][1][lane + 32 * i]), reinterpret_cast<const void*>(v & ~static_cast<uintptr_t>(3)));
      sync->shift[s][0][lane + 32 * i] = static_cast<uint8_t>((k & 3) * 8);
      sync->shift[s][1][lane + 32 * i] = static_cast<uint8_t>((v & 3) * 8);
    }
    cp_async_arrive(smem_u32(&sync->full[s]));
    __syncwarp();
    if (lane == 0) mbar_arrive(smem_u32(&sync->full[s]));
    c.step(l);
    look_up();
  }
  cp_async_wait_all();   // (before the CTA lets go of its memory, should it give up)
  if (lane == 0) sync->issued[1] = n;
}

// The CTA gives up (every warp has left its loop): what was started has to land before it lets go of its memory.  A block that
// one of the two warps started and the other did not lacks the other's arrivals, which are made up, so that every stage's barrier
// completes when its copies have landed.  The two warps are never more than a round of the ring apart.
template <int D, int HEADS, bool TMA>
__device__ __forceinline__ void land(Sync<D, HEADS>* sync, int warp, int lane) {
  constexpr int kStages = Geo<D, HEADS>::kStages;
  if (warp < kWarps || lane != 0) return;
  const int rows = sync->issued[0], scales = sync->issued[1], most = rows > scales ? rows : scales;
  if (warp == kWarps + 1) {
    for (int n = scales; n < rows; ++n)
      for (int i = 0; i < kScaleArrivals; ++i) mbar_arrive(smem_u32(&sync->full[n % kStages]));
    return;
  }
  for (int n = rows; n < scales; ++n)
    for (int i = 0; i < kRowArrivals<TMA>; ++i) mbar_arrive(smem_u32(&sync->full[n % kStages]));
  for (int s = 0; s < kStages && s < most; ++s) wait_drain(smem_u32(&sync->full[s]), ((most - 1 - s) / kStages) & 1);
}

// What fp16 has no room for goes through functions of their own, which take their operands through memory, so that the usual path keeps
// its registers and its place in the instruction caches (inlined, 128 sequences under a prefix took 80 us instead of 76).
//
// Query rows that fp16 does not hold exactly, in bf16: factor[i] is what goes back out of head 8 i + g's scores.
template <int D, int NB> struct Wide {
  uint2 q[NB][D / 16];
  float factor[NB], score[2][NB][4];
};
template <int D, int NB> __device__ __noinline__ void wide_query(Wide<D, NB>& d, const uint16_t* query, int g, int tq) {
#pragma unroll 1
  for (int i = 0; i < NB; ++i) {
    const uint16_t* row = query + (8 * i + g) * (D + 16);
    uint32_t top = 0;
#pragma unroll 1
    for (int e = 0; e < D; ++e) top = max(top, row[e] & 0x7fffu);
    const int up = power_up<true>(top << 16, 126);
    const float f = __int_as_float((127 + up) << 23);
    d.factor[i] = __int_as_float((127 - up) << 23) * 0x1p120f;
#pragma unroll 1
    for (int s = 0; s < D / 16; ++s) {
      const uint2 v = *reinterpret_cast<const uint2*>(row + 16 * s + 4 * tq);
      const uint32_t x = pack16<true>(half_to_f32<true>(static_cast<uint16_t>(v.x)) * f, half_to_f32<true>(static_cast<uint16_t>(v.x >> 16)) * f);
      const uint32_t y = pack16<true>(half_to_f32<true>(static_cast<uint16_t>(v.y)) * f, half_to_f32<true>(static_cast<uint16_t>(v.y >> 16)) * f);
      d.q[i][s] = make_uint2(__byte_perm(x, y, 0x5410), __byte_perm(x, y, 0x7632));   // (as unpack_e4m3_bf16 has the key's)
    }
  }
}
// Their products with a warp's keys.
template <int D, int NB> __device__ __noinline__ void wide_scores(Wide<D, NB>& d, uint32_t k_row, int lane) {
  float score[2][NB][4] = {};
#pragma unroll 1
  for (int s = 0; s < D / 16; s += 2) {
    const uint32_t at = k_row + static_cast<uint32_t>(((s + (lane >> 4)) ^ Geo<D, 8>::swizzle(lane & 7)) << 4);
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      uint32_t kf[4];
      ldsm_x4(at + t * 16 * D, kf);
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        uint32_t a0, a1, a2, a3;
        unpack_e4m3_bf16(kf[2 * u], a0, a2);
        unpack_e4m3_bf16(kf[2 * u + 1], a1, a3);
#pragma unroll
        for (int i = 0; i < NB; ++i) mma_16<true>(score[t][i], a0, a1, a2, a3, d.q[i][s + u].x, d.q[i][s + u].y);
      }
    }
  }
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int i = 0; i < NB; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) d.score[t][i][r] = score[t][i][r];
}
// A warp's products with its values where a row lies far below the largest.
template <int D, int NB> struct Deep {
  float o[D / 16][NB][4], sv[2][NB][4], nm[NB][2], lsum[NB][2];
  float w[2][2];   // 2^(e_v - r + 119)
};
template <int D, int NB> __device__ __noinline__ void deep_products(Deep<D, NB>& d, uint32_t v_row, int lane) {
  uint32_t ph[2][NB][2], pl[2][NB][2];
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      float x[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        x[r] = ex2(d.sv[t][i][r] + d.nm[i][r & 1]);
        d.lsum[i][r & 1] += x[r];
      }
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        split_16<true>(x[2 * y] * d.w[t][y], x[2 * y + 1] * d.w[t][y], ph[t][i][y], pl[t][i][y]);
        ph[t][i][y] = turn8x8(ph[t][i][y]);
        pl[t][i][y] = turn8x8(pl[t][i][y]);
      }
    }
#pragma unroll 1
  for (int j = 0; j < D / 16; j += 2) {
    const uint32_t at = v_row + static_cast<uint32_t>(((j + (lane >> 4)) ^ Geo<D, 8>::swizzle(lane & 7)) << 4);
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      uint32_t vf[4];
      ldsm_x4_trans(at + t * 16 * D, vf);
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        uint32_t a0, a1, a2, a3;
        unpack_e4m3_bf16(vf[2 * u], a0, a1);
        unpack_e4m3_bf16(vf[2 * u + 1], a2, a3);
#pragma unroll
        for (int i = 0; i < NB; ++i) {
          float part[4] = {0.f, 0.f, 0.f, 0.f};
          mma_16<true>(part, a0, a1, a2, a3, pl[t][i][0], pl[t][i][1]);
          mma_16<true>(part, a0, a1, a2, a3, ph[t][i][0], ph[t][i][1]);
#pragma unroll
          for (int r = 0; r < 4; ++r) d.o[j + u][i][r] = fmaf(part[r], 0x1p10f, d.o[j + u][i][r]);   // (2^120 of the bytes less 2^110)
        }
      }
    }
  }
}

// HEADS: query heads of a CTA, 8 or 16.
template <int D, bool BF16, int HEADS, bool TMA>
__global__ void __launch_bounds__(kThreads, Geo<D, HEADS>::kCtas)
    decode_fp8_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v, const Problem p, const CacheScales sc,
                      const FrontKeys front, const OwnPartials part, const int fixed_blocks, const long long wait_limit) {
  using G = Geo<D, HEADS>;
  constexpr int KS = D / 16, NB = HEADS / 8;
  extern __shared__ __align__(16) uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw), ring = (raw + 1023u) & ~1023u;
  uint8_t* smem = smem_raw + (ring - raw);
  auto* sync = reinterpret_cast<Sync<D, HEADS>*>(smem + G::kRingBytes);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (int s = 0; s < G::kStages; ++s) {
      mbar_init(smem_u32(&sync->full[s]), kRowArrivals<TMA> + kScaleArrivals);
      mbar_init(smem_u32(&sync->empty[s]), kWarps);
    }
    sync->abort_flag = 0;
    mbar_fence_init();
  }
  __syncthreads();
  pdl_wait();
  pdl_launch_dependents();   // (a gathering of the shared prefix may run beside this)
  const List list = {p, front, p.Hkv * ((p.group + HEADS - 1) / HEADS), front.len > 0 ? 1 : 0};
  Cursor c = first_place(list, fixed_blocks, lane);

  if (warp == kWarps) {
    bring_rows<D, HEADS, TMA>(list, sc, &tm_k, &tm_v, sync, ring, c, lane, wait_limit);
  } else if (warp == kWarps + 1) {
    bring_scales<D, HEADS>(list, sc, sync, c, lane, wait_limit);
  } else {
    const int g = lane >> 2, tq = lane & 3;
    uint2 q[NB][KS];
    float o[D / 16][NB][4];     // O^T: rows 2 g, 2 g + 1 of sixteen columns of V; heads 2 tq, 2 tq + 1 of eight
    float m[NB][2], lsum[NB][2], sl2[NB][2];   // of heads 2 tq, 2 tq + 1: maximum in log2 units, this lane's share of the sum, product to log2 units
    float r_exp = -CUDART_INF_F;
    int b = c.b, unit = c.unit, first = 0;     // the pair, and its first block here
    const int blocks = c.left;
    bool fresh = true, ok = true, wide = false;   // wide: the pair's query rows are bf16 ones here
    for (int n = 0; n < blocks; ++n) {
      const int st = n % G::kStages;
      ok = __all_sync(0xffffffffu, wait_clocked(smem_u32(&sync->full[st]), (n / G::kStages) & 1, &sync->abort_flag, wait_limit));
      if (!ok) {   // the CTA gives up
        if (lane == 0) report(p.status, 2, n, warp);
        break;
      }
      const int blk = sync->block[st].blk, n_keys = sync->block[st].n_keys;
      if (fresh) {
        fresh = false;
        first = blk;
        r_exp = -CUDART_INF_F;
        float factor[NB];
#pragma unroll
        for (int i = 0; i < NB; ++i) {
          // fragments: k-step s holds elements 16 s + 4 tq .. + 3 of head g, as the bytes of a key's fragment word; a head's
          // quad has all of it
          uint32_t top2 = 0, low2 = 0;   // (magnitudes of either type order like their bits) low2: 2^15 less the smallest that is not 0
#pragma unroll
          for (int s = 0; s < KS; ++s) {
            q[i][s] = *reinterpret_cast<const uint2*>(&sync->query[st][8 * i + g][16 * s + 4 * tq]);
            const uint32_t x = q[i][s].x & 0x7fff7fffu, y = q[i][s].y & 0x7fff7fffu;
            top2 = __vmaxu2(top2, __vmaxu2(x, y));
            if (BF16) low2 = __vmaxu2(low2, __vmaxu2((0x80008000u - x) & 0x7fff7fffu, (0x80008000u - y) & 0x7fff7fffu));
          }
          uint32_t top = max(top2 & 0xffffu, top2 >> 16);
          top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
          top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
          const bool here = unit / p.Hkv * HEADS + 8 * i + g < p.group;   // (else the row is whatever was there)
          if (i == 0) wide = false;
          // (2^15 at the top, 8 bits of 2^-17: the last is fp16's last, 2^-24)
          if (BF16 && here) wide |= static_cast<int>((0x8000u - max(low2 & 0xffffu, low2 >> 16)) >> 7) < static_cast<int>(top >> 7) - 31;
          top = __float_as_uint(half_to_f32<BF16>(static_cast<uint16_t>(top)));
          const int up = power_up<BF16>(top, 14);
          const float f = __int_as_float((127 + up) << 23);
          factor[i] = here ? p.scale * kLog2e * __int_as_float((127 - up) << 23) : 0.f;
#pragma unroll
          for (int s = 0; s < KS; ++s) {
            const uint2 v = q[i][s];
            q[i][s].x = here ? pack16<false>(half_to_f32<BF16>(static_cast<uint16_t>(v.x)) * f, half_to_f32<BF16>(static_cast<uint16_t>(v.x >> 16)) * f) : 0u;
            q[i][s].y = here ? pack16<false>(half_to_f32<BF16>(static_cast<uint16_t>(v.y)) * f, half_to_f32<BF16>(static_cast<uint16_t>(v.y >> 16)) * f) : 0u;
          }
        }
        wide = BF16 && __any_sync(0xffffffffu, wide);
        if (wide) {
          Wide<D, NB> d;
          wide_query<D, NB>(d, &sync->query[st][0][0], g, tq);
#pragma unroll
          for (int i = 0; i < NB; ++i) {
            const bool here = unit / p.Hkv * HEADS + 8 * i + g < p.group;
            if (here) factor[i] = p.scale * kLog2e * d.factor[i];
#pragma unroll
            for (int s = 0; s < KS; ++s) q[i][s] = here ? d.q[i][s] : make_uint2(0u, 0u);
          }
        }
#pragma unroll
        for (int i = 0; i < NB; ++i) {
#pragma unroll
          for (int j = 0; j < D / 16; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) o[j][i][r] = 0.f;
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            sl2[i][e] = __shfl_sync(0xffffffffu, factor[i], (2 * tq + e) * 4);
            m[i][e] = -CUDART_INF_F;
            lsum[i][e] = 0.f;
          }
        }
      }
      const int key_w = blk * kBlockKeys + warp * kWarpKeys;   // first key of this warp's 32
      if (key_w < n_keys) {
        // the rows in matrices of 8 rows x 16 bytes: rows 0-7 and 8-15 of one piece, then of the next
        const int row = warp * kWarpKeys + ((lane >> 3) & 1) * 8 + (lane & 7);
        const uint32_t k_row = ring + st * G::kStageBytes + row * D, v_row = k_row + G::kTileBytes;
        auto piece = [&](int x) { return static_cast<uint32_t>(((x + (lane >> 4)) ^ G::swizzle(lane & 7)) << 4); };
        float kx[2][2], ev[2][2];
        int e_max = -1;
        bool far = false;
        uint32_t kf[2][KS / 2][4];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
#pragma unroll
          for (int s = 0; s < KS; s += 2) ldsm_x4(k_row + t * 16 * D + piece(s), kf[t][s / 2]);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int at = warp * kWarpKeys + 16 * t + g + 8 * i;
            const uint32_t k = (sync->scale[st][0][at] >> sync->shift[st][0][at]) & 255u, v = (sync->scale[st][1][at] >> sync->shift[st][1][at]) & 255u;
            // 2^e as bits (2^-127 is subnormal), and e as a number, by way of 2^23 + code
            kx[t][i] = __uint_as_float(k == 255u ? 0x7fffffffu : max(k << 23, 0x00400000u));
            ev[t][i] = v == 255u ? CUDART_NAN_F : __uint_as_float(0x4b000000u | v) - (8388608.f + 127.f);
            far |= k - 222u < 33u;   // (not the NaN)
            if (v < 255u && key_w + 16 * t + g + 8 * i < n_keys) e_max = max(e_max, static_cast<int>(v));
          }
        }
        e_max = __reduce_max_sync(0xffffffffu, e_max);
        far = __any_sync(0xffffffffu, far);
        const float e_top = e_max < 0 ? -CUDART_INF_F : static_cast<float>(e_max - 127);   // the largest e of a value here
        const bool tail = key_w + kWarpKeys > n_keys;
        if (tail) {
          // what lies behind the end is anything: its weight is 0, and 0 times a NaN is not
          for (int i = lane; i < kWarpKeys * G::kChunksPerRow; i += 32)
            if (key_w + i / G::kChunksPerRow >= n_keys)
              *reinterpret_cast<uint4*>(smem + st * G::kStageBytes + G::kTileBytes + warp * kWarpKeys * D + i * 16) = make_uint4(0, 0, 0, 0);
          fence_proxy_async_smem();   // (the stage's next block comes by tensor copies)
          __syncwarp();
#pragma unroll
          for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int i = 0; i < 2; ++i)
              if (key_w + 16 * t + g + 8 * i >= n_keys) ev[t][i] = -CUDART_INF_F;
        }
        // ---- S^T = K Q^T: keys 16 t + g, + 8 x heads 2 tq, 2 tq + 1
        constexpr int kChains = NB == 1 ? 2 : 1;   // even and odd k-steps apart
        float sv[2][NB][4], part_s[2][NB][kChains][4];
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int i = 0; i < NB; ++i)
#pragma unroll
            for (int x = 0; x < kChains; ++x)
#pragma unroll
              for (int r = 0; r < 4; ++r) part_s[t][i][x][r] = 0.f;
        if (BF16 && wide) {
          Wide<D, NB> d;
#pragma unroll
          for (int i = 0; i < NB; ++i)
#pragma unroll
            for (int s = 0; s < KS; ++s) d.q[i][s] = q[i][s];
          wide_scores<D, NB>(d, k_row, lane);
#pragma unroll
          for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int i = 0; i < NB; ++i)
#pragma unroll
              for (int r = 0; r < 4; ++r) part_s[t][i][0][r] = d.score[t][i][r];
        } else {
#pragma unroll
          for (int s = 0; s < KS; ++s)
#pragma unroll
            for (int t = 0; t < 2; ++t) {
              uint32_t a0, a1, a2, a3;
              unpack_e4m3_f16(kf[t][s / 2][2 * (s & 1)], a0, a2);
              unpack_e4m3_f16(kf[t][s / 2][2 * (s & 1) + 1], a1, a3);
#pragma unroll
              for (int i = 0; i < NB; ++i) mma_16<false>(part_s[t][i][s % kChains], a0, a1, a2, a3, q[i][s].x, q[i][s].y);
            }
        }
        float mn[NB][2];
        bool grow = e_top > r_exp;
#pragma unroll
        for (int i = 0; i < NB; ++i) {
#pragma unroll
          for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const float x = kChains == 2 ? part_s[t][i][0][r] + part_s[t][i][kChains - 1][r] : part_s[t][i][0][r];
              // |x| <= 2^32, so below code 222 (2^95) the first product is finite; beyond, one that is not is none in the end either
              sv[t][i][r] = far ? x * sl2[i][r & 1] * kx[t][r >> 1] : x * kx[t][r >> 1] * sl2[i][r & 1];
              if (tail && key_w + 16 * t + g + 8 * (r >> 1) >= n_keys) sv[t][i][r] = -CUDART_INF_F;
            }
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float x = fmaxf(fmaxf(sv[0][i][e], sv[0][i][2 + e]), fmaxf(sv[1][i][e], sv[1][i][2 + e]));
#pragma unroll
            for (int d = 4; d < 32; d *= 2) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, d));
            mn[i][e] = fmaxf(m[i][e], x);
            grow |= mn[i][e] - m[i][e] > kRescaleThreshold;   // false for NaN (-inf - -inf)
          }
        }
        // ---- o is rescaled when the largest value exponent or a row maximum grows
        if (__any_sync(0xffffffffu, grow)) {
          const float re = fmaxf(r_exp, e_top);
          const float down = re == r_exp ? 1.f : ex2(r_exp - re);   // -inf -> 0
          r_exp = re;
#pragma unroll
          for (int i = 0; i < NB; ++i) {
            float f[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              f[e] = mn[i][e] == m[i][e] ? 1.f : ex2(m[i][e] - mn[i][e]);
              m[i][e] = mn[i][e];
              lsum[i][e] *= f[e];
              f[e] *= down;
            }
#pragma unroll
            for (int j = 0; j < D / 16; ++j)
#pragma unroll
              for (int r = 0; r < 4; ++r) o[j][i][r] *= f[r & 1];
          }
        }
        // ---- probabilities; times the value scale relative to r, hi and lo, turned round: heads g x keys 2 tq, 2 tq + 1.  Then
        // O^T += V^T P^T, sixteen columns of V at a time.
        bool deep = false;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int i = 0; i < 2; ++i) deep |= ev[t][i] < r_exp - kDeep && ev[t][i] != -CUDART_INF_F;
        if (__any_sync(0xffffffffu, deep)) {
          Deep<D, NB> d;
#pragma unroll
          for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int i = 0; i < 2; ++i) d.w[t][i] = ev[t][i] == -CUDART_INF_F ? 0.f : ex2(ev[t][i] - r_exp + (kProbShift + kDeepShift));
#pragma unroll
          for (int i = 0; i < NB; ++i) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              d.nm[i][e] = (m[i][e] == -CUDART_INF_F) ? 0.f : -m[i][e];
              d.lsum[i][e] = lsum[i][e];
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              d.sv[0][i][r] = sv[0][i][r];
              d.sv[1][i][r] = sv[1][i][r];
#pragma unroll
              for (int j = 0; j < D / 16; ++j) d.o[j][i][r] = o[j][i][r];
            }
          }
          deep_products<D, NB>(d, v_row, lane);
#pragma unroll
          for (int i = 0; i < NB; ++i) {
#pragma unroll
            for (int e = 0; e < 2; ++e) lsum[i][e] = d.lsum[i][e];
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
              for (int j = 0; j < D / 16; ++j) o[j][i][r] = d.o[j][i][r];
          }
        } else {
          uint32_t ph[2][NB][2], pl[2][NB][2];
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            float w[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) w[i] = ev[t][i] == -CUDART_INF_F ? 0.f : ex2(ev[t][i] - r_exp + kProbShift);
#pragma unroll
            for (int i = 0; i < NB; ++i) {
              float x[4];
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const float nm = (m[i][e] == -CUDART_INF_F) ? 0.f : -m[i][e];
                x[e] = ex2(sv[t][i][e] + nm);
                x[2 + e] = ex2(sv[t][i][2 + e] + nm);
                lsum[i][e] += x[e] + x[2 + e];
              }
#pragma unroll
              for (int y = 0; y < 2; ++y) {
                split_16<false>(x[2 * y] * w[y], x[2 * y + 1] * w[y], ph[t][i][y], pl[t][i][y]);
                ph[t][i][y] = turn8x8(ph[t][i][y]);
                pl[t][i][y] = turn8x8(pl[t][i][y]);
              }
            }
          }
#pragma unroll
          for (int j = 0; j < D / 16; j += 2)
#pragma unroll
            for (int t = 0; t < 2; ++t) {
              uint32_t vf[4];
              ldsm_x4_trans(v_row + t * 16 * D + piece(j), vf);
#pragma unroll
              for (int u = 0; u < 2; ++u) {
                uint32_t a0, a1, a2, a3;   // even and odd columns of keys 0-7, then of keys 8-15
                unpack_e4m3_f16(__byte_perm(vf[2 * u], 0, 0x3120), a0, a1);
                unpack_e4m3_f16(__byte_perm(vf[2 * u + 1], 0, 0x3120), a2, a3);
#pragma unroll
                for (int i = 0; i < NB; ++i) {
                  mma_16<false>(o[j + u][i], a0, a1, a2, a3, ph[t][i][0], ph[t][i][1]);
                  mma_16<false>(o[j + u][i], a0, a1, a2, a3, pl[t][i][0], pl[t][i][1]);
                }
              }
            }
        }
      }
      const int last = sync->block[st].last, next_unit = sync->block[st].next_unit, next_b = sync->block[st].next_b;
      const bool ends = blk + 1 == (n_keys + kBlockKeys - 1) / kBlockKeys;
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&sync->empty[st]));
      if (last == 0) continue;

      // ---- the pair's last block here: every warp leaves its partial, the merge is the second launch's.  (A merge of the
      // four in shared memory took longer than the few bytes more.)
      const int64_t pair = static_cast<int64_t>(b) * list.units + unit;
      const int64_t slot = pair + blockIdx.x;
      if (tid == 0) {
        if (first == 0) part.range[pair].x = static_cast<int>(slot);
        if (ends) part.range[pair].y = static_cast<int>(slot);
      }
      const float back = r_exp == -CUDART_INF_F ? 0.f : ex2(0.5f * (r_exp - kProbShift));   // 2^(r - 9), in two factors
#pragma unroll
      for (int i = 0; i < NB; ++i)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float sum = lsum[i][e];
#pragma unroll
          for (int d = 4; d < 32; d *= 2) sum += __shfl_xor_sync(0xffffffffu, sum, d);
          const int head = 8 * i + 2 * tq + e;
          if (unit / p.Hkv * HEADS + head >= p.group || !dbg_range(p.status, DBG_DECODE_FP8 * 100 + 1, slot, 1, part.slots)) continue;
          const int64_t row = (slot * kWarps + warp) * HEADS + head;
#pragma unroll
          for (int j = 0; j < D / 16; ++j)
            *reinterpret_cast<float2*>(part.o + row * D + 16 * j + 2 * g) = make_float2(o[j][i][e] * back * back, o[j][i][2 + e] * back * back);
          if (g == 0)
            *reinterpret_cast<float2*>(part.ml + row * 2) = make_float2(m[i][e], sum);
        }
      b = next_b;
      unit = next_unit;
      fresh = true;
    }
  }
  __syncthreads();
  if (*static_cast<volatile int*>(&sync->abort_flag) != 0) {
    land<D, HEADS, TMA>(sync, warp, lane);
    __syncthreads();
  }
}

// Pages of the pool as (bytes of a row, rows, heads, pages); one copy takes up to a block's rows of a page.
bool make_page_map(CUtensorMap* map, const void* pool, int d, int page, int heads, int pages, const int64_t* stride) {
  EncodeTiledFn fn = encode_fn();
  if (fn == nullptr) return false;
  const cuuint64_t dims[4] = {static_cast<cuuint64_t>(d), static_cast<cuuint64_t>(page), static_cast<cuuint64_t>(heads), static_cast<cuuint64_t>(pages)};
  auto fix = [&](int64_t s, int n) -> cuuint64_t { return static_cast<cuuint64_t>(n == 1 ? d : s); };   // (never stepped)
  const cuuint64_t strides[3] = {fix(stride[2], page), fix(stride[1], heads), fix(stride[0], pages)};
  const cuuint32_t box[4] = {static_cast<cuuint32_t>(d), static_cast<cuuint32_t>(page < kBlockKeys ? page : kBlockKeys), 1, 1};
  const cuuint32_t elem[4] = {1, 1, 1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, const_cast<void*>(pool), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
            d == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
// A tensor copy wants positive strides below 2^40 (the rows are on 16 bytes already) and whole swizzle patterns: 8 rows.
bool tma_pages(const Problem& p, int pages) {
  const int page = 1 << p.page_shift, n[3] = {pages, p.Hkv, page};
  if (page < 8) return false;
  for (int i = 0; i < 3; ++i)
    if (n[i] > 1 && (p.ks[i] <= 0 || p.vs[i] <= 0 || p.ks[i] >= (1LL << 40) || p.vs[i] >= (1LL << 40))) return false;
  return true;
}

template <int D, bool BF16, int HEADS, bool TMA>
int launch_one(const Problem& p, const CacheScales& sc, const Fp8Geometry& g, const FrontKeys& front, const OwnPartials& part, cudaStream_t stream) {
  CUtensorMap tk = {}, tv = {};
  if (TMA && (!make_page_map(&tk, p.k, D, 1 << p.page_shift, p.Hkv, sc.n_pages, p.ks) ||
              !make_page_map(&tv, p.v, D, 1 << p.page_shift, p.Hkv, sc.n_pages, p.vs)))
    return B200_SDPA_ERR_CUDA;
  auto kern = decode_fp8_kernel<D, BF16, HEADS, TMA>;
  constexpr int smem = smem_bytes<D, HEADS>();
  static_assert(Geo<D, HEADS>::kCtas * (smem + 1024) <= 228 * 1024, "the CTAs of an SM share its memory");
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess) {
    cudaGetLastError();
    return B200_SDPA_ERR_CUDA;
  }
  if (!launch_pdl(kern, dim3(g.grid), kThreads, smem, stream, tk, tv, p, sc, front, part, g.fixed_blocks, wait_limit_cycles())) return B200_SDPA_ERR_CUDA;
  count_launch(KID_DECODE);
  return B200_SDPA_OK;
}

template <int D, bool BF16>
int launch_heads(const Problem& p, const CacheScales& sc, const Fp8Geometry& g, const FrontKeys& front, const OwnPartials& part, cudaStream_t stream) {
  const bool tma = tma_pages(p, sc.n_pages);
  if (g.heads == 8) return tma ? launch_one<D, BF16, 8, true>(p, sc, g, front, part, stream) : launch_one<D, BF16, 8, false>(p, sc, g, front, part, stream);
  return tma ? launch_one<D, BF16, 16, true>(p, sc, g, front, part, stream) : launch_one<D, BF16, 16, false>(p, sc, g, front, part, stream);
}

}  // namespace

// Pools whose offsets the copies of small pages can count: rows in 32 bits of 16 bytes.
bool decode_fp8_served(const Problem& p, int n_pages) {
  if (tma_pages(p, n_pages)) return true;
  const int64_t page = 1LL << p.page_shift, limit = 1LL << 36;
  return p.ks[0] * n_pages + p.ks[2] * page < limit && p.vs[0] * n_pages + p.vs[2] * page < limit;
}

bool decode_fp8_geometry(const Problem& p, int front_keys, int kv_chunk, Fp8Geometry* g) {
  constexpr int64_t kSms = 148;
  g->heads = p.group <= 8 ? 8 : 16;
  g->units = p.Hkv * ((p.group + g->heads - 1) / g->heads);
  const int64_t one = static_cast<int64_t>(p.B) * g->units, pairs = front_keys > 0 ? 2 * one : one;
  const int64_t most = one * ((static_cast<int64_t>(p.S) + kBlockKeys - 1) / kBlockKeys + (static_cast<int64_t>(front_keys) + kBlockKeys - 1) / kBlockKeys);
  int64_t grid = kSms * (p.E == 128 || g->heads == 16 ? 2 : 3);
  static_assert(Geo<128, 8>::kCtas == 2 && Geo<128, 16>::kCtas == 2 && Geo<64, 16>::kCtas == 2 && Geo<64, 8>::kCtas == 3, "as above");
  g->fixed_blocks = 0;
  if (kv_chunk > 0) {
    g->fixed_blocks = (kv_chunk + kBlockKeys - 1) / kBlockKeys;
    grid = (most + g->fixed_blocks - 1) / g->fixed_blocks;
  }
  if (grid > most) grid = most;
  if (grid < 1 || grid + pairs > 0x7fffffffLL) return false;
  g->grid = static_cast<int>(grid);
  g->slots = grid + pairs;
  g->bytes = static_cast<uint64_t>(g->slots) * kWarps * g->heads * (p.E + 2) * sizeof(float) + static_cast<uint64_t>(pairs) * sizeof(int2);
  return true;
}

int launch_decode_partial_fp8(const Problem& p, const CacheScales& sc, int dtype, const Fp8Geometry& g, const FrontKeys& front, const OwnPartials& part, cudaStream_t stream) {
  const bool bf16 = dtype == B200_SDPA_BF16;
  if (p.E == 128) return bf16 ? launch_heads<128, true>(p, sc, g, front, part, stream) : launch_heads<128, false>(p, sc, g, front, part, stream);
  return bf16 ? launch_heads<64, true>(p, sc, g, front, part, stream) : launch_heads<64, false>(p, sc, g, front, part, stream);
}

}  // namespace b200
