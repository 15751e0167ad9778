// Attention of many query rows over paged keys and values: prompts, the last chunk
// of one, and the shared prefix of a batch, whose sequences' rows all read the same
// tokens.
//
// A kv head's rows are its query tokens x its group of q heads, in tiles of 256. A
// CTA takes a tile of rows through tiles of 128 tokens: for each half of the rows two
// products of 128 x 64 scores on the tensor cores, a softmax with a running maximum
// and sum in 32 bits, one thread for each row, and a product of the probabilities with
// the values. Scores, probabilities and the output's sums (32 bits) stay in tensor
// memory. The probabilities are rounded to the input type (half a step, as the output
// is; the two together leave 1.3 to 1.4 times the output's own error, and a second product
// with what the rounding leaves would take 0.4 more of the products' time) and take the place of the first 64 tokens' scores; the other 64 tokens' place is
// free as soon as its scores are read, so the next tile's are computed there while this
// one's first 64 are weighed. A row's sums are scaled to a new reference only where its
// maximum has grown by more than 2^8 (fp16: where a tile's leaves what the type holds),
// which the 32-bit sums carry exactly as well.
//
// Roles: warps 0-3 and 4-7 the halves' softmax, warps 8 and 10 issue the halves'
// products, warp 9 loads keys and values with TMA into a ring (a box for each run of
// rows in a page).
//
// Work: the visible (row tile, kv head, token tile) units laid end to end and cut
// into equal ranges, one CTA on every SM, whatever the prompts' lengths and masks
// are; row tiles cut by a border leave parts in the scratch, which are added up in the
// ranges' order by tile_join_kernel, or where a prefix has few rows in all by the CTA
// that comes last. tile_plan_kernel lays prompts' units out from the device's lengths; over a
// prefix all row tiles have the same ones.
//
// Bound by the softmax: a unit's products take 2560 cycles, its exponentials 1536 on
// the exponential units (a fourth of them runs on the FMA units), and the two warps of
// a scheduler take about 3700 for all of it (loads from tensor memory, waits and the
// exponentials of both at once); a piece of a row tile costs some 10000 more for its
// first scores, its masked tile and its output. Measured on B200: 2048 queries at the end
// of 40011 tokens, 32 / 8 heads of 128, 1.25 ms in five calls after a rest (1050 TFLOP/s,
// 0.62 of the measured burst rate), 1.43 to 1.51 ms back to back under the power cap (0.62
// to 0.65 of the sustained rate); six prompts of 107-2699 tokens behind a window of 1024
// 228 us.
#include <algorithm>
#include <type_traits>

#include "kv_attention.cuh"

namespace tcx {
namespace {

constexpr int kTokens = 128;
constexpr int kHalfRows = 128;
constexpr int kRows = 2 * kHalfRows;
constexpr int kThreads = 384;
constexpr int kPlanThreads = 1024;
constexpr int kPlanCache = 2048;
// What a piece of a row tile costs beside its token tiles (its queries, its first
// scores, its output), in token tiles: counted when the work is cut into ranges.
constexpr uint32_t kPieceCost = 3;

// Over a prefix: up to so many rows the CTA that comes last adds their parts up, one warp to a row
// at a time: 256 rows took it 115 us over 18 ranges, a launch of its own takes 18.
constexpr uint32_t kJoinHere = 32;

// A tile of rows: row r is query token q_first + (row0 + r) / group.
struct Item {
  uint32_t q_first, row0, rows;
  int pos0;                      // position of query token q_first, from the first token of `table`
  uint32_t tiles;                // token tiles: [0, sink_tiles) and from first_tile on
  int sink_tiles, first_tile;
  int limit, low, sinks;         // tokens seen lie below limit, and below sinks or from low on
  uint64_t table;                // first entry in the page table
};

struct RangeBegin {
  uint32_t item, head, tile;
  uint64_t unit;  // token tiles before it
};

struct RangeEnd {
  uint32_t item, head;  // of the last piece
  uint32_t starts, goes_on, slot;
};

struct TileArgs {
  AttnArgs a;
  uint32_t prefix;  // rows of all sequences over the shared prefix
  uint32_t join_here;  // few rows over a prefix: the CTA that comes last adds their parts up
  uint32_t max_q, max_ranges;
  uint32_t* item_first;  // [n_seq + 1]
  Item* items;
  uint64_t* unit_first;  // [items]: token tiles of all heads before it
  RangeBegin* begin;     // [max_ranges + 1]
  RangeEnd* end;         // [max_ranges]
  uint32_t* counts;      // items, ranges
  float* part_o;         // [max_ranges][2][kRows][D], sums of 2^(z - m) v
  float2* part_ml;       // the same rows' m and sum of 2^(z - m)
};

__device__ __forceinline__ uint32_t items_of(const TileArgs& d, uint32_t s) {
  const uint64_t rows = static_cast<uint64_t>(d.a.q_offsets[s + 1] - d.a.q_offsets[s]) * d.a.group;
  return static_cast<uint32_t>((rows + kRows - 1) / kRows);
}

__device__ Item make_item(const TileArgs& d, uint32_t s, uint32_t index, int prefix) {
  const AttnArgs& a = d.a;
  Item it;
  const uint32_t first = d.prefix ? 0 : a.q_offsets[s], last = d.prefix ? a.q_tokens : a.q_offsets[s + 1];
  it.q_first = first;
  it.row0 = index * kRows;
  it.rows = min(static_cast<uint32_t>(kRows), (last - first) * a.group - it.row0);
  int from, to;  // positions of the first and last row
  if (d.prefix) {
    it.table = 0;
    it.pos0 = 0;
    it.sinks = static_cast<int>(a.sinks);
    to = prefix - 1;
    from = prefix - static_cast<int>(d.max_q);  // at most: a row's own position decides
  } else {
    it.table = a.page_offsets[s];
    it.pos0 = static_cast<int>(seq_length(a, s)) - static_cast<int>(last - first);
    it.sinks = static_cast<int>(max(int64_t{0}, a.sinks - prefix));
    from = it.pos0 + static_cast<int>(it.row0 / a.group);
    to = it.pos0 + static_cast<int>((it.row0 + it.rows - 1) / a.group);
  }
  it.limit = max(to + 1, 0);
  it.low = a.window ? static_cast<int>(max(int64_t{0}, from - a.window + 1)) : 0;
  it.sink_tiles = it.low > 0 ? (min(it.sinks, it.limit) + kTokens - 1) / kTokens : 0;
  it.first_tile = max(it.low / kTokens, it.sink_tiles);
  // one tile at least, so that the rows are written
  it.tiles = max(it.sink_tiles + max((it.limit + kTokens - 1) / kTokens - it.first_tile, 0), 1);
  return it;
}

// Every range must hold more than a piece's cost to hold a tile.
__device__ __forceinline__ uint64_t piece_cost(uint64_t units, uint64_t pieces, uint32_t ranges) {
  return scaled(units + kPieceCost * pieces, 1, ranges) > kPieceCost ? kPieceCost : 0;
}

// Exclusive sum over the CTA; *total gets the sum.
__device__ uint64_t plan_scan(uint64_t v, uint64_t* sums, uint64_t* total) {
  const uint32_t lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  uint64_t inc = v;
  for (int x = 1; x < 32; x *= 2) {
    const uint64_t up = __shfl_up_sync(~0u, inc, x);
    if (lane >= x) inc += up;
  }
  __syncthreads();
  if (lane == 31) sums[warp] = inc;
  __syncthreads();
  uint64_t before = 0, all = 0;
  for (uint32_t w = 0; w < kPlanThreads / 32; ++w) {
    if (w < warp) before += sums[w];
    all += sums[w];
  }
  *total = all;
  return before + inc - v;
}

__global__ void __launch_bounds__(kPlanThreads) tile_plan_kernel(TileArgs d) {
  __shared__ uint64_t s_sums[kPlanThreads / 32], s_units[kPlanCache];
  __shared__ uint32_t s_first[kPlanCache];
  const AttnArgs& a = d.a;
  next_may_start();
  wait_for_previous();
  const int prefix = static_cast<int>(prefix_length(a));
  uint64_t total;
  uint32_t items;
  {
    const uint32_t share = (a.n_seq + kPlanThreads - 1) / kPlanThreads, s0 = min(threadIdx.x * share, a.n_seq),
                   s1 = min(s0 + share, a.n_seq);
    uint32_t mine = 0;
    for (uint32_t s = s0; s < s1; ++s) mine += items_of(d, s);
    uint32_t at = static_cast<uint32_t>(plan_scan(mine, s_sums, &total));
    items = static_cast<uint32_t>(total);
    for (uint32_t s = s0; s < s1; ++s) {
      if (s < kPlanCache) s_first[s] = at; else d.item_first[s] = at;
      at += items_of(d, s);
    }
    __syncthreads();
  }
  uint64_t units = 0;
  for (uint32_t i0 = 0; i0 < items; i0 += kPlanThreads) {
    const uint32_t i = i0 + threadIdx.x;
    uint64_t mine = 0;
    if (i < items) {
      uint32_t s = 0, hi = a.n_seq;  // the last sequence whose items begin at i or before
      while (hi - s > 1) {
        const uint32_t mid = (s + hi) / 2;
        if ((mid < kPlanCache ? s_first[mid] : d.item_first[mid]) <= i) s = mid; else hi = mid;
      }
      const uint32_t first = s < kPlanCache ? s_first[s] : d.item_first[s];
      const Item it = make_item(d, s, i - first, prefix);
      d.items[i] = it;
      mine = static_cast<uint64_t>(it.tiles) * a.kv_heads;
    }
    const uint64_t before = units + plan_scan(mine, s_sums, &total);
    units += total;
    if (i < items) {
      d.unit_first[i] = before;
      if (i < kPlanCache) s_units[i] = before;
    }
  }
  __syncthreads();
  const uint32_t ranges = static_cast<uint32_t>(min(static_cast<uint64_t>(d.max_ranges), units));
  const uint64_t pieces = static_cast<uint64_t>(items) * a.kv_heads, cost = piece_cost(units, pieces, ranges);
  if (threadIdx.x == 0) {
    d.counts[0] = items;
    d.counts[1] = ranges;
    d.begin[ranges] = RangeBegin{items, 0, 0, units};
  }
  for (uint32_t r = threadIdx.x; r < ranges; r += kPlanThreads) {
    const uint64_t at = (units + cost * pieces) * r / ranges;
    auto first_of = [&](uint32_t i) {
      return (i < kPlanCache ? s_units[i] : d.unit_first[i]) + cost * a.kv_heads * i;
    };
    uint32_t lo = 0, hi = items;
    while (hi - lo > 1) {
      const uint32_t mid = (lo + hi) / 2;
      if (first_of(mid) <= at) lo = mid; else hi = mid;
    }
    const uint64_t in = at - first_of(lo), tiles = d.items[lo].tiles, head = in / (tiles + cost);
    const uint64_t tile = max(in % (tiles + cost), cost) - cost;
    d.begin[r] = RangeBegin{lo, static_cast<uint32_t>(head), static_cast<uint32_t>(tile),
                            first_of(lo) - cost * a.kv_heads * lo + head * tiles + tile};
  }
}

template <int D>
struct TileLayout {
  static constexpr int kBlock = kTokens * 128;          // 64 values of 128 rows, swizzled
  static constexpr int kOperand = kBlock * (D / 64);    // 128 rows
  static constexpr int kStages = D == 128 ? 4 : 8;
  static constexpr int kOut = 8 * 32 * 128;              // 128 bytes of each row, on their way out
  static constexpr int kBytes = (2 + kStages) * kOperand + kOut + 1024;
  static constexpr uint32_t kScores = 0, kSums = 256, kColumns = 512;
};

__device__ __forceinline__ int first_token(const Item& it, uint32_t tile) {
  return (tile < static_cast<uint32_t>(it.sink_tiles) ? static_cast<int>(tile)
                                                     : it.first_tile + static_cast<int>(tile) - it.sink_tiles) * kTokens;
}

// The finite ones of two 16-bit values; 0 in place of the others.
template <typename T>
__device__ __forceinline__ uint32_t finite_only(uint32_t pair) {
  constexpr uint32_t kExponent = std::is_same<T, __half>::value ? 0x7c00 : 0x7f80;
  if ((pair & kExponent) == kExponent) pair &= 0xffff0000u;
  if ((pair >> 16 & kExponent) == kExponent) pair &= 0xffffu;
  return pair;
}

// Row r of an item and head, of which the ranges [from, to] hold parts: a warp adds them
// up in the ranges' order. The first of them is in place `first_slot` of its range.
template <typename T, int D>
__device__ __forceinline__ void join_row(const TileArgs& d, const Item& it, uint32_t head, uint32_t from, uint32_t to,
                                         uint32_t first_slot, uint32_t r, uint32_t lane) {
  constexpr int E = D / 32;
  const AttnArgs& a = d.a;
  auto row_of = [&](uint32_t k) { return static_cast<uint64_t>(k * 2 + (k == from ? first_slot : 0)) * kRows + r; };
  float top = -INFINITY, sum = 0.f, x[E] = {};
  for (uint32_t k = from + lane; k <= to; k += 32) top = fmaxf(top, __ldcg(&d.part_ml[row_of(k)].x));
  for (int i = 16; i; i /= 2) top = fmaxf(top, __shfl_xor_sync(~0u, top, i));
  const float ref = top == -INFINITY ? 0.f : top;
#pragma unroll 4
  for (uint32_t k = from; k <= to; ++k) {
    const uint64_t row = row_of(k);
    const float2 ml = __ldcg(&d.part_ml[row]);
    const float f = exp2_approx(ml.x - ref);
    sum += f * ml.y;
    if constexpr (E == 4) {
      const float4 v = __ldcg(reinterpret_cast<const float4*>(d.part_o + row * D) + lane);
      x[0] += f * v.x;
      x[1] += f * v.y;
      x[2] += f * v.z;
      x[3] += f * v.w;
    } else {
      const float2 v = __ldcg(reinterpret_cast<const float2*>(d.part_o + row * D) + lane);
      x[0] += f * v.x;
      x[1] += f * v.y;
    }
  }
  const uint32_t row = it.row0 + r, t = it.q_first + row / a.group, h = head * a.group + row % a.group;
  const Finish f = finish_row(a, static_cast<uint64_t>(t) * a.kv_heads * a.group + h, top, sum);
  if constexpr (E == 4) {
    store_row<T, D>(a, t, h, lane * 4, f, x);
  } else {  // two lanes' values in one
    const float y[4] = {x[0], x[1], __shfl_down_sync(~0u, x[0], 1), __shfl_down_sync(~0u, x[1], 1)};
    if (lane % 2 == 0) store_row<T, D>(a, t, h, lane * 2, f, y);
  }
  if (lane == 0) store_lse(a, t, h, f);
  __syncwarp();
}

// kPrefix: the rows of all sequences over the shared prefix.
template <typename T, int D, bool kPrefix>
__global__ void __launch_bounds__(kThreads, 1) tile_kernel(const __grid_constant__ CUtensorMap map, TileArgs d) {
  using L = TileLayout<D>;
  constexpr uint32_t kStages = L::kStages;
  extern __shared__ uint8_t raw[];
  __shared__ uint64_t s_bar[2 * kStages + 12];
  __shared__ uint32_t s_tmem, s_gave_up, s_drained, s_last;
  __shared__ uint32_t s_left_out[2];  // piece + 1 where values were kept from its products
  __shared__ __align__(16) int s_seen[2][8][4];
  const AttnArgs& a = d.a;
  const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32, range = blockIdx.x;
  const uint32_t base = (smem_addr(raw) + 1023) & ~1023u, ring = base + 2 * L::kOperand;
  // Ring place 2 i holds tile i's keys, 2 i + 1 its values. A tile's values and the
  // next one's keys are waited for together (pair p: places 2 p - 1 and 2 p); each is
  // given back by itself.
  // As many pairs' barriers as places: the first lap's copies wait for no place, and
  // must not arrive at a pair whose phase is still open.
  constexpr uint32_t kPairs = kStages;
  auto full = [&](uint32_t pair) { return smem_addr(&s_bar[pair % kPairs]); };
  auto full_phase = [&](uint32_t pair) { return pair / kPairs & 1; };
  auto empty = [&](uint32_t i) { return smem_addr(&s_bar[kPairs + i]); };
  auto bar = [&](uint32_t kind, uint32_t half) { return smem_addr(&s_bar[kPairs + kStages + kind * 2 + half]); };
  enum : uint32_t { kQueries, kScoredLow, kScoredHigh, kHighRead, kWeighed, kSummed };
  if (threadIdx.x == 0) {
    for (uint32_t i = 0; i < kPairs; ++i) mbar_init(full(i), 2);
    for (uint32_t i = 0; i < kStages; ++i) mbar_init(empty(i), 2);  // one arrival for each half
    for (uint32_t h = 0; h < 2; ++h) {
      mbar_init(bar(kQueries, h), 4);  // a warp's lane for all of them
      mbar_init(bar(kScoredLow, h), 1);
      mbar_init(bar(kScoredHigh, h), 1);
      mbar_init(bar(kHighRead, h), 4);
      mbar_init(bar(kWeighed, h), 4);
      mbar_init(bar(kSummed, h), 1);
    }
    s_gave_up = s_drained = s_left_out[0] = s_left_out[1] = 0;
    mbar_init_fence();
  }
  next_may_start();
  wait_for_previous();
  // The work: its row tiles, where the ranges begin, and this one.
  const int prefix = static_cast<int>(prefix_length(a));
  uint32_t items, ranges;
  uint64_t same_tiles = 0, cost = 0;  // over a prefix: every row tile's token tiles
  if (kPrefix) {
    items = static_cast<uint32_t>((static_cast<uint64_t>(a.q_tokens) * a.group + kRows - 1) / kRows);
    same_tiles = make_item(d, 0, 0, prefix).tiles;
    const uint64_t pieces = static_cast<uint64_t>(items) * a.kv_heads;
    ranges = static_cast<uint32_t>(min(static_cast<uint64_t>(d.max_ranges), pieces * same_tiles));
    cost = piece_cost(pieces * same_tiles, pieces, ranges);
  } else {
    items = d.counts[0];
    ranges = d.counts[1];
  }
  if (range >= ranges) {
    if (threadIdx.x == 0) d.end[range] = RangeEnd{0, 0, 0, 0, 0};
    return;
  }
  auto begin_of = [&](uint32_t r) {
    if (!kPrefix) return d.begin[r];
    const uint64_t pieces = static_cast<uint64_t>(items) * a.kv_heads, each = same_tiles + cost;
    const uint64_t at = scaled(pieces * each, r, ranges), piece = scaled(at, 1, each);
    const uint64_t tile = max(at - piece * each, cost) - cost, first = scaled(piece, 1, a.kv_heads);
    return RangeBegin{static_cast<uint32_t>(first), static_cast<uint32_t>(piece - first * a.kv_heads),
                      static_cast<uint32_t>(tile), piece * same_tiles + tile};
  };
  auto item_of = [&](uint32_t i) { return kPrefix ? make_item(d, 0, i, prefix) : d.items[i]; };
  if (warp == 8) tmem_alloc(smem_addr(&s_tmem), L::kColumns);
  tmem_fence_before();
  __syncthreads();
  tmem_fence_after();
  const uint32_t tmem = s_tmem;
  const RangeBegin begin = begin_of(range);
  const uint32_t count = static_cast<uint32_t>(begin_of(range + 1).unit - begin.unit);

  // Every role walks the range's pieces: the token tiles [at, at + n) of one item and head.
  uint32_t item = begin.item, head = begin.head, at = begin.tile;
  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    if (warp == 9) {  // ---- keys and values
      const uint32_t boxes = kTokens / a.box_rows;
      const uint32_t box = lane % boxes, half = lane / boxes;
      uint32_t slot_at = 0;  // ring position
      Item it = item_of(item);
      if (lane == 0) mbar_arrive(full(0));  // no values before the first keys
      bool alive = true;
      for (uint32_t left = count; left > 0 && alive;) {
        const uint32_t n = min(it.tiles - at, left);
        const uint32_t* table = (kPrefix ? a.prefix_table : a.page_table) + it.table;
        for (uint32_t j = 0; j < n && alive; ++j) {
          const int from = first_token(it, at + j) + static_cast<int>(box * a.box_rows),
                    to = from + static_cast<int>(a.box_rows);
          const bool wanted = half < D / 64 && from < it.limit && (to > it.low || from < it.sinks);
          const uint32_t bytes = __popc(__ballot_sync(~0u, wanted)) * a.box_rows * 128;
          uint64_t row = 0;
          if (wanted) row = checked_slot(a, table, from / a.page_tokens) * a.page_tokens + from % a.page_tokens;
#pragma unroll
          for (int plane = 0; plane < 2; ++plane, ++slot_at) {
            const uint32_t stage = slot_at % kStages;
            alive = alive && mbar_wait_warp(empty(stage), (slot_at / kStages & 1) ^ 1, &s_gave_up, a.status);
            if (!alive) break;
            const uint32_t arrived = full((slot_at + 1) / 2);
            if (lane == 0) {
              if (bytes) mbar_arrive_expect(arrived, bytes); else mbar_arrive(arrived);
            }
            __syncwarp();
            if (wanted)
              tma_load_3d(ring + stage * L::kOperand + half * L::kBlock + box * a.box_rows * 128, &map, half * 64,
                          head, static_cast<int>(row + (plane ? a.v_row0 : a.k_row0)), arrived);
          }
        }
        left -= n;
        at = 0;
        if (++head == a.kv_heads && left > 0) {
          head = 0;
          it = item_of(++item);
        }
      }
      const uint32_t last = slot_at / 2;
      if (lane == 0 && alive) mbar_arrive(full(last));  // no keys behind the last values
      // No copy may be in flight when the CTA ends.
      for (uint32_t p = last > kStages / 2 ? last - kStages / 2 : 0; p <= last; ++p)
        mbar_wait_warp(full(p), full_phase(p), &s_drained, a.status);
    } else if (warp == 8 || warp == 10) {  // ---- the products of half `h`
      // The tensor cores queue about two products, and a wait costs as long as two even
      // where the barrier is there: two warps issue, one for each half.
      constexpr uint32_t kScoreShape = mma_shape<T>(kTokens / 2, false), kValueShape = mma_shape<T>(D, true);
      const uint32_t h = warp == 10, tm = __shfl_sync(~0u, tmem, 0);
      const uint64_t q_operand = smem_operand(base + h * L::kOperand, 16, 1024),
                     k_operand = smem_operand(ring, 16, 1024), v_operand = smem_operand(ring, L::kBlock, 1024);
      const uint32_t scores = tm + L::kScores + h * kTokens, sums = tm + L::kSums + h * D;
      uint32_t slot_at = 0, pieces = 0, done = 0;
      auto wait = [&](uint32_t b, uint32_t phase) {
        const bool there = mbar_wait_warp(b, phase & 1, &s_gave_up, a.status);
        tmem_fence_after();
        return there;
      };
      // Scores: the half's queries x the first (high 0) or last 64 keys at `slot`, which
      // the first ones' give back. An operand's place is its descriptor's low bits, in
      // 16-byte units.
      auto score = [&](uint32_t slot, uint32_t high) {
        const uint64_t k = k_operand + slot % kStages * (L::kOperand / 16) + high * (64 * 128 / 16);
        if (elect_one()) {
#pragma unroll
          for (int e = 0; e < D / 16; ++e) {
            const uint32_t off = e / 4 * (L::kBlock / 16) + e % 4 * 2;
            mma_ss(scores + high * 64, q_operand + off, k + off, kScoreShape, e > 0);
          }
          mma_commit(bar(high ? kScoredHigh : kScoredLow, h));
          if (!high) mma_commit(empty(slot % kStages));
        }
        __syncwarp();
      };
      auto uniform = [&](uint32_t x) { return __shfl_sync(~0u, x, 0); };
      Item next = item_of(item);
      uint32_t tiles = uniform(next.tiles), rows = uniform(next.rows), next_item = min(item + 1, items - 1);
      next = item_of(next_item);
      at = uniform(at);
      head = uniform(head);
      bool alive = true;
      for (uint32_t left = uniform(count); left > 0 && alive;) {
        const uint32_t n = min(tiles - at, left);
        if (rows > h * kHalfRows) {
          alive = wait(bar(kQueries, h), pieces++) && wait(full(slot_at / 2), full_phase(slot_at / 2));
          if (!alive) break;
          score(slot_at, 1);
          score(slot_at, 0);
          for (uint32_t j = 0; j < n; ++j, ++done, slot_at += 2) {
            const uint32_t slot = slot_at + 1, k = slot_at + 2;
            const bool more = j + 1 < n;
            // The next scores of the last 64 tokens follow once these are read, those of
            // the first 64, whose place the probabilities take, behind the sums.
            alive = wait(full(k / 2), full_phase(k / 2));  // both places are there
            if (alive && more) {
              alive = wait(bar(kHighRead, h), done);
              if (alive) score(k, 1);
            }
            alive = alive && wait(bar(kWeighed, h), done);
            if (!alive) break;
            const uint64_t v = v_operand + slot % kStages * (L::kOperand / 16);
            if (elect_one()) {
#pragma unroll
              for (int i = 0; i < kTokens / 16; ++i)
                mma_ts(sums, scores + i * 8, v + i * 128, kValueShape, j > 0 || i > 0);
              mma_commit(empty(slot % kStages));
              if (!more) mma_commit(bar(kSummed, h));
            }
            __syncwarp();
            if (more) score(k, 0);
          }
        } else {  // no rows here: the tiles pass by
          for (uint32_t i = 0; i < 2 * n && alive; ++i, ++slot_at) {
            alive = wait(full((slot_at + 1) / 2), full_phase((slot_at + 1) / 2));
            mbar_arrive_warp(empty(slot_at % kStages), lane, alive);
          }
        }
        left -= n;
        at = 0;
        if (++head == a.kv_heads) {
          head = 0;
          tiles = uniform(next.tiles);
          rows = uniform(next.rows);
          next_item = min(next_item + 1, items - 1);
          next = item_of(next_item);
        }
      }
    }
    __syncwarp();
  } else {  // ---- the softmax of half `h`, one thread for each row
    asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    const uint32_t h = warp / 4, r = threadIdx.x, quarter = warp % 4 * 32 << 16;
    const uint32_t scores = tmem + quarter + L::kScores + h * kTokens, sums = tmem + quarter + L::kSums + h * D;
    const uint32_t staged = base + (2 + kStages) * L::kOperand + warp * 4096;
    uint32_t pieces = 0, done = 0, summed = 0, tiles_done = 0;
    bool alive = true;
    auto wait = [&](uint32_t b, uint32_t phase) { alive = alive && mbar_wait_warp(b, phase & 1, &s_gave_up, a.status); };
    // Starts the copies of this warp's 32 queries of a piece, D / 8 lanes to a row,
    // swizzled as the products read them.
    auto fetch = [&](uint32_t q_first, uint32_t row0, uint32_t rows, uint32_t kv_head) {
      constexpr uint32_t kLanes = D / 8;
      const uint32_t row = row0 + r, first = r & ~31u;
      const uint64_t from = (q_first + row / a.group) * a.q_token_stride +
                            (kv_head * a.group + row % a.group) * a.q_head_stride;
#pragma unroll
      for (uint32_t i = 0; i < kLanes; ++i) {
        const uint32_t src = i * (32 / kLanes) + lane / kLanes, c = lane % kLanes, mine = first + src;
        const bool valid = mine < rows;
        const uint64_t at_row = __shfl_sync(~0u, from, src);
        async_copy16(base + h * L::kOperand + c / 8 * L::kBlock + mine % kHalfRows * 128 + ((c % 8 ^ (mine & 7)) << 4),
                     a.q + (valid ? at_row + c * 16 : 0), valid ? 16 : 0);
      }
    };
    Item it = item_of(item);
    if (h * kHalfRows < it.rows) fetch(it.q_first, it.row0, it.rows, head);
    for (uint32_t left = count; left > 0; ++pieces) {
      const uint32_t n = min(it.tiles - at, left);
      const uint32_t row = it.row0 + r;
      const bool active = h * kHalfRows < it.rows;
      if (active) {
        async_copies_done();
        proxy_fence_smem();
        mbar_arrive_warp(bar(kQueries, h), lane, alive);
      }
      // The next piece's queries follow once this one's last scores are there.
      auto fetch_next = [&] {
        if (left == n) return;
        if (head + 1 < a.kv_heads) {
          if (active) fetch(it.q_first, it.row0, it.rows, head + 1);
        } else {
          const Item next = item_of(item + 1);
          if (h * kHalfRows < next.rows) fetch(next.q_first, next.row0, next.rows, 0);
        }
      };
      if (!active) fetch_next();
      // What this row sees: [0, hi] from lo on, and the sinks. What all rows of this
      // half see (all_*), and what any row of the item sees (any_*). Over a prefix, where
      // the rows are those of several sequences: what all rows of the item see (every_*).
      int hi = -1, lo = 0, all_hi, all_lo, any_hi, any_lo, every_hi, every_lo;
      auto low_of = [&](int pos) {
        return a.window ? static_cast<int>(max(int64_t{0}, pos - a.window + 1)) : 0;
      };
      if (kPrefix && d.max_q == 1 && a.window == 0) {
        // one query each stands behind the whole prefix, and sees it
        hi = r < it.rows ? prefix - 1 : -1;
        all_hi = any_hi = every_hi = prefix - 1;
        all_lo = any_lo = every_lo = 0;
      } else if (kPrefix) {
        if (r < it.rows) {
          const uint32_t t = it.q_first + row / a.group, s = seq_of(a, t);
          const int nq = static_cast<int>(a.q_offsets[s + 1] - a.q_offsets[s]);
          const int pos = prefix + static_cast<int>(seq_length(a, s)) - nq + static_cast<int>(t - a.q_offsets[s]);
          hi = min(pos, prefix - 1);
          lo = low_of(pos);
        }
        const bool valid = r < it.rows;
        all_hi = __reduce_min_sync(~0u, valid ? hi : 0x7fffffff);
        all_lo = __reduce_max_sync(~0u, valid ? lo : 0);
        any_hi = __reduce_max_sync(~0u, hi);
        any_lo = __reduce_min_sync(~0u, valid ? lo : 0x7fffffff);
        if (lane == 0) *reinterpret_cast<int4*>(s_seen[pieces & 1][warp]) = make_int4(all_hi, all_lo, any_hi, any_lo);
        asm volatile("bar.sync 1, 256;" ::: "memory");
        every_hi = 0x7fffffff;
        every_lo = 0;
#pragma unroll
        for (int w = 0; w < 8; ++w) {
          const int* v = s_seen[pieces & 1][w];
          every_hi = min(every_hi, v[0]);
          every_lo = max(every_lo, v[1]);
          if (static_cast<uint32_t>(w) / 4 == h) {
            all_hi = min(all_hi, v[0]);
            all_lo = max(all_lo, v[1]);
          }
          any_hi = max(any_hi, v[2]);
          any_lo = min(any_lo, v[3]);
        }
      } else {
        hi = r < it.rows ? it.pos0 + static_cast<int>(row / a.group) : -1;
        lo = low_of(hi);
        all_hi = it.pos0 + static_cast<int>((it.row0 + h * kHalfRows) / a.group);
        all_lo = low_of(it.pos0 + static_cast<int>((it.row0 + it.rows - 1) / a.group));
        any_hi = every_hi = it.limit - 1;
        any_lo = every_lo = it.low;
      }
      const bool mixed = kPrefix && (every_hi != any_hi || every_lo != any_lo);
      // Does the tile hold tokens that not every row of the item sees?
      auto partly_seen = [&](int token) {
        return token + kTokens - 1 > every_hi || (token < every_lo && token + kTokens > it.sinks);
      };
      constexpr bool kIsHalf = std::is_same<T, __half>::value;
      constexpr float kTop = kIsHalf ? kHalfTop : 8.f;  // the largest exponent before m rises
      float m = -INFINITY, l = 0.f, peak = -INFINITY;
      if (active) {
        for (uint32_t j = 0; j < n; ++j, ++done) {
          const int token = first_token(it, at + j);
          const bool masked = token + kTokens - 1 > all_hi || (token < all_lo && token + kTokens > it.sinks);
          // Scores that this row does not see become -inf: tokens from `from` on.
          auto hide = [&](uint32_t (&z)[kTokens / 2], int from) {
            auto below = [&](int x, int word) {  // bits of the word's tokens below x
              const int n_bits = min(max(x - from - word * 32, 0), 32);
              return n_bits == 32 ? ~0u : (1u << n_bits) - 1;
            };
#pragma unroll
            for (int w = 0; w < 2; ++w) {
              const uint32_t see = below(hi + 1, w) & (~below(lo, w) | below(it.sinks, w));
#pragma unroll
              for (int i = 0; i < 32; ++i)
                if (!(see >> i & 1)) z[w * 32 + i] = 0xff800000u;
            }
          };
          auto largest = [&](const uint32_t (&z)[kTokens / 2]) {
            float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int i = 0; i < kTokens / 2; i += 2)
              top[i / 2 % 4] = max3_nan(top[i / 2 % 4], __uint_as_float(z[i]), __uint_as_float(z[i + 1]));
            return max3_nan(max3_nan(top[0], top[1], top[2]), top[3], top[3]) * a.scale_log2;
          };
          const float2 c2 = make_float2(a.scale_log2, a.scale_log2);
          // 2^(z - m) of a pair, on the exponential units or (mixed: every fourth pair)
          // the FMA units, since the exponential units alone need nearly as long as
          // the products do.
          auto weigh = [&](uint32_t z0, uint32_t z1, int i, float ref, auto mixed) {
            float2 x = fma2(make_float2(__uint_as_float(z0), __uint_as_float(z1)), c2, make_float2(-ref, -ref));
            if (decltype(mixed)::value && i % 4 == 3) return exp2_fma(x);
            return make_float2(exp2_approx(x.x), exp2_approx(x.y));
          };
          auto reference = [&] { return m == -INFINITY ? 0.f : m; };
          float f = 1.f;  // what the sums so far are scaled by
          auto move = [&](float top, bool down) {
            const float old = m;
            if constexpr (kIsHalf) {
              m = half_reference(old, top, peak, down);
              peak = fmaxf(peak, m);
            } else if (top > m + kTop) {
              m = top;
            }
            const float by = m == old ? 1.f : exp2_approx(old - m);
            f *= by;
            return by;
          };

          // The last 64 tokens, whose scores were there early.
          float2 e[kTokens / 4], sum_e = make_float2(0.f, 0.f), sum_z = make_float2(0.f, 0.f);
          bool odd;  // a score that only the exponential units take: masked, infinite or NaN
          {
            wait(bar(kScoredHigh, h), done);
            tmem_fence_after();
            uint32_t z[kTokens / 2];
            tmem_load64(z, scores + kTokens / 2);
            tmem_fence_before();
            mbar_arrive_warp(bar(kHighRead, h), lane, alive);
            if (masked) hide(z, token + kTokens / 2);
            const float top = largest(z);
            move(top, true);
            odd = masked || __any_sync(~0u, !(fabsf(top) < INFINITY));
            const float ref = reference();
            auto all = [&](auto mixed) {
#pragma unroll
              for (int i = 0; i < kTokens / 4; ++i) {
                e[i] = weigh(z[2 * i], z[2 * i + 1], i, ref, mixed);
                sum_e = add2(sum_e, e[i]);
              }
            };
            if (odd) all(std::false_type{}); else all(std::true_type{});
          }
          auto store_high = [&] {
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              uint32_t p[16];
#pragma unroll
              for (int i = 0; i < 16; ++i) p[i] = pack2<T>(e[c * 16 + i].x, e[c * 16 + i].y);
              tmem_store16(scores + kTokens / 4 + c * 16, p);
            }
          };

          // The first 64 tokens. All probabilities take the place of their scores.
          {
            wait(bar(kScoredLow, h), done);
            tmem_fence_after();
            if (j + 1 == n) fetch_next();
            uint32_t z[kTokens / 2];
            tmem_load64(z, scores);
            if (masked) hide(z, token);
            // Values that no row sees are cleared (0 x NaN is not 0), half of them by each
            // half of the rows; both come here, and neither goes on alone. One that some
            // sequences' rows see must not reach the others': where it is not finite it is
            // kept from the product, and added to its rows' sums behind the last one.
            if ((masked || mixed) && partly_seen(token)) {
              const uint32_t v = 2 * (tiles_done + j) + 1, of = r % kHalfRows, halves = it.rows > kHalfRows ? 2 : 1;
              wait(full((v + 1) / 2), full_phase((v + 1) / 2));
              const int mine = token + static_cast<int>(of);
              const uint32_t to = ring + v % kStages * L::kOperand + of * 128;
              auto place_of = [&](uint32_t c) { return to + c / 8 * L::kBlock + ((c % 8 ^ (of & 7)) << 4); };
              auto put = [](uint32_t at, const uint32_t (&x)[4]) {
                asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(x[0]), "r"(x[1]), "r"(x[2]), "r"(x[3])
                             : "memory");
              };
              if (mine > any_hi || (mine < any_lo && mine >= it.sinks)) {
                for (uint32_t c = h; c < D / 8; c += halves) put(place_of(c), {0, 0, 0, 0});
              } else if (mixed && (mine > every_hi || (mine < every_lo && mine >= it.sinks))) {
#pragma unroll 1
                for (uint32_t c = h; c < D / 8; c += halves) {
                  uint32_t x[4], y[4];
                  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                               : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3])
                               : "r"(place_of(c))
                               : "memory");
#pragma unroll
                  for (int i = 0; i < 4; ++i) y[i] = finite_only<T>(x[i]);
                  if (((x[0] ^ y[0]) | (x[1] ^ y[1]) | (x[2] ^ y[2]) | (x[3] ^ y[3])) == 0) continue;
                  *static_cast<volatile uint32_t*>(&s_left_out[pieces & 1]) = pieces + 1;
                  put(place_of(c), y);
                }
              }
              proxy_fence_smem();
              if (halves == 2)
                asm volatile("bar.sync 2, 256;" ::: "memory");
              else if (kPrefix)  // half 1 is here no more: rows of half 0 alone are the last item's
                asm volatile("bar.sync 2, 128;" ::: "memory");
              else
                __syncwarp();
            }
            store_high();
            auto all = [&](auto mixed) {
              const float ref = reference();
              sum_z = make_float2(0.f, 0.f);
#pragma unroll
              for (int c = 0; c < 2; ++c) {
                uint32_t p[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                  const int k = c * 32 + 2 * i;
                  const float2 x = weigh(z[k], z[k + 1], i, ref, mixed);
                  sum_z = add2(sum_z, x);
                  p[i] = pack2<T>(x.x, x.y);
                }
                tmem_store16(scores + c * 16, p);
              }
            };
            // Where all rows see them whole they are weighed by the maximum so far at
            // once, while their own is found, and again where that has grown too far.
            bool again = true;
            float top;
            if (!odd) {
              all(std::true_type{});
              top = largest(z);
              again = __any_sync(~0u, !(top <= m + kTop));
            } else {
              top = largest(z);
            }
            if (again) {
              const float by = move(top, false);
              if (__any_sync(~0u, by != 1.f)) {
#pragma unroll
                for (int i = 0; i < kTokens / 4; ++i) e[i] = make_float2(e[i].x * by, e[i].y * by);
                sum_e = make_float2(sum_e.x * by, sum_e.y * by);
                store_high();
              }
              all(std::false_type{});
            }
          }
          if (__any_sync(~0u, f != 1.f) && j > 0) {  // these scores are there, so the sums before them are done
            for (int c = 0; c < D; c += 32) {
              uint32_t o[32];
              tmem_load32(o, sums + c);
#pragma unroll
              for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
              tmem_store32(sums + c, o);
            }
          }
          tmem_wait_store();
          tmem_fence_before();
          mbar_arrive_warp(bar(kWeighed, h), lane, alive);
          sum_e = add2(sum_e, sum_z);
          l = l * f + (sum_e.x + sum_e.y);
        }
        wait(bar(kSummed, h), summed++);
        tmem_fence_after();
        if (mixed && *static_cast<volatile uint32_t*>(&s_left_out[pieces & 1]) == pieces + 1) {
          // The values that were kept from this piece's products, read again: an infinity
          // or NaN is one whatever its weight.
#pragma unroll 1
          for (int c = 0; c < D; c += 32) {
            uint32_t o[32];
            tmem_load32(o, sums + c);
#pragma unroll 1
            for (uint32_t j = 0; j < n; ++j) {
              const int token = first_token(it, at + j);
              if (!partly_seen(token)) continue;
#pragma unroll 1
              for (int k = token; k < token + kTokens; ++k) {
                const bool every = k <= every_hi && (k >= every_lo || k < it.sinks);
                if (every || k > hi || (k < lo && k >= it.sinks)) continue;
                const uint64_t row = checked_slot(a, a.prefix_table, k / a.page_tokens) * a.page_tokens + k % a.page_tokens;
                const uint4* values = reinterpret_cast<const uint4*>(a.pool + (a.v_row0 + row) * a.token_bytes +
                                                                     head * a.row_bytes + c * 2);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                  const uint4 v = values[i];
                  const uint32_t x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                  for (int w = 0; w < 4; ++w) {
                    const float2 y = unpack2<T>(x[w] ^ finite_only<T>(x[w]));
                    uint32_t* to = o + i * 8 + w * 2;
                    to[0] = __float_as_uint(__uint_as_float(to[0]) + y.x);
                    to[1] = __float_as_uint(__uint_as_float(to[1]) + y.y);
                  }
                }
              }
            }
            __syncwarp();
            tmem_store32(sums + c, o);
          }
          tmem_wait_store();
        }
        const bool whole = at == 0 && n == it.tiles, final = whole && a.part_o == nullptr;
        const bool write = r < it.rows && alive;
        const uint32_t t = it.q_first + row / a.group, q_head = head * a.group + row % a.group;
        const uint64_t q_row = static_cast<uint64_t>(t) * a.kv_heads * a.group + q_head;
        const uint64_t part = static_cast<uint64_t>(range * 2 + (pieces > 0)) * kRows + r;
        Finish f{};
        if (write && whole) {
          f = finish_row(a, q_row, m, l);
          if (final) a.lse[q_row] = kLn2 * f.lse; else a.part_lse[q_row] = f.lse;
        } else if (write) {
          d.part_ml[part] = make_float2(m, l);
        }
        __syncwarp();
        const uint64_t to = !write ? 0
                            : final ? reinterpret_cast<uint64_t>(a.out + t * a.out_token_stride + q_head * a.out_head_stride)
                            : whole ? reinterpret_cast<uint64_t>(a.part_o + q_row * D)
                                    : reinterpret_cast<uint64_t>(d.part_o + part * D);
        // 32 values of the row, a finished one's with its factors
        auto values = [&](float (&x)[32], int c) {
          uint32_t o[32];
          tmem_load32(o, sums + c);
#pragma unroll
          for (int i = 0; i < 32; ++i) x[i] = __uint_as_float(o[i]);
          if (!whole) return;
#pragma unroll
          for (int i = 0; i < 32; ++i) x[i] = f.sees_own ? x[i] * f.own : 0.f;
          if (f.sees_prior) {
            const float4* y = reinterpret_cast<const float4*>(a.prior_o + q_row * D + c);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const float4 v = y[i];
              x[4 * i] += f.prior * v.x;
              x[4 * i + 1] += f.prior * v.y;
              x[4 * i + 2] += f.prior * v.z;
              x[4 * i + 3] += f.prior * v.w;
            }
          }
          __syncwarp();
        };
        // 128 bytes of each of the warp's rows go through shared memory, so that 8
        // lanes write one row's.
        auto place = [&](uint32_t of, uint32_t c) { return staged + of * 128 + ((c ^ (of & 7)) << 4); };
        auto leave = [&](uint32_t byte) {
          __syncwarp();
#pragma unroll
          for (uint32_t i = 0; i < 8; ++i) {
            const uint32_t src = i * 4 + lane / 8;
            const uint64_t at_row = __shfl_sync(~0u, to, src);
            uint4 v;
            asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                         : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                         : "r"(place(src, lane % 8))
                         : "memory");
            if (at_row) *reinterpret_cast<uint4*>(at_row + byte + lane % 8 * 16) = v;
          }
          __syncwarp();
        };
#pragma unroll 1
        for (int c = 0; c < D; c += 32) {
          float x[32];
          values(x, c);
          if (final) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
              asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(place(lane, c % 64 / 8 + i)),
                           "r"(pack2<T>(x[8 * i], x[8 * i + 1])), "r"(pack2<T>(x[8 * i + 2], x[8 * i + 3])),
                           "r"(pack2<T>(x[8 * i + 4], x[8 * i + 5])), "r"(pack2<T>(x[8 * i + 6], x[8 * i + 7]))
                           : "memory");
            if (c % 64 == 32) leave((c - 32) * 2);
          } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
              asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(place(lane, i)), "f"(x[4 * i]),
                           "f"(x[4 * i + 1]), "f"(x[4 * i + 2]), "f"(x[4 * i + 3])
                           : "memory");
            leave(c * 4);
          }
        }
        tmem_fence_before();
      }
      if (kPrefix && d.join_here && (at != 0 || n != it.tiles)) {
        // Another range has parts of these rows too: whoever comes last adds them up.
        const uint64_t first = begin.unit + tiles_done - at, last = first + it.tiles - 1;
        uint32_t from = 0, to = 0;  // the last ranges that begin at the first and last tile, or before
        for (uint32_t r0 = 0; r0 < ranges; r0 += 32) {
          const uint32_t r = r0 + lane;
          const uint64_t unit = r < ranges ? begin_of(r).unit : ~uint64_t{0};
          from += __popc(__ballot_sync(~0u, unit <= first));
          to += __popc(__ballot_sync(~0u, unit <= last));
        }
        --from;
        --to;
        asm volatile("bar.sync 1, 256;" ::: "memory");
        if (threadIdx.x == 0) s_last = alive && last_to_arrive(a.counters + TCX_KV_COUNTERS / 2 + from, to - from + 1);
        asm volatile("bar.sync 1, 256;" ::: "memory");
        if (s_last) {
          const uint32_t first_slot = begin_of(from).unit != first;
          for (uint32_t r = warp; r < it.rows; r += 8) join_row<T, D>(d, it, head, from, to, first_slot, r, lane);
        }
      }
      left -= n;
      tiles_done += n;
      if (left == 0 && threadIdx.x == 0)
        d.end[range] = RangeEnd{item, head, at == 0, at + n < it.tiles, pieces > 0};
      at = 0;
      if (++head == a.kv_heads && left > 0) {
        head = 0;
        it = item_of(++item);
      }
    }
  }
  tmem_fence_before();
  __syncthreads();
  tmem_fence_after();
  if (warp == 8) tmem_free(tmem, L::kColumns);
}

// Adds up the parts of the row tile that begins in a range and goes on in the next
// ones, in the ranges' order: one warp for each row.
template <typename T, int D>
__global__ void __launch_bounds__(256) tile_join_kernel(TileArgs d) {
  const AttnArgs& a = d.a;
  const uint32_t range = blockIdx.x, r = blockIdx.y * 8 + threadIdx.x / 32, lane = threadIdx.x % 32;
  next_may_start();
  wait_for_previous();
  const RangeEnd own = d.end[range];
  if (!own.goes_on || !own.starts) return;
  const Item it = d.prefix ? make_item(d, 0, own.item, static_cast<int>(prefix_length(a))) : d.items[own.item];
  if (r >= it.rows) return;
  uint32_t end = range + 1;  // the last range of these rows: the next one holds others, or they end here
  for (;; end += 32) {
    const RangeEnd next = d.end[min(end + lane, d.max_ranges - 1)];
    const uint32_t ends = __ballot_sync(~0u, next.item != own.item || next.head != own.head || !next.goes_on);
    if (ends == 0) continue;
    end += __ffs(ends) - 1;
    break;
  }
  join_row<T, D>(d, it, own.head, range, end, own.slot, r, lane);
}

uint64_t max_items(const tcx_kv_attention_args& x, bool prefix) {
  return x.q_tokens * (x.q_heads / x.kv_heads) / kRows + (prefix ? 1 : x.n_seq);
}

// One CTA on every SM; a range holds one unit at least.
uint32_t max_ranges(const tcx_kv_attention_args& x, bool prefix) {
  const uint64_t pages = prefix ? x.prefix_pages : x.max_pages;
  const uint64_t units = max_items(x, prefix) * x.kv_heads * (pages * x.page_tokens / kTokens + 2);
  return static_cast<uint32_t>(std::min<uint64_t>({static_cast<uint64_t>(sm_count()), units, TCX_KV_COUNTERS / 2}));
}

struct Parts {
  uint64_t item_first, items, unit_first, begin, end, counts, ml, o, total;
};

Parts parts(const tcx_kv_attention_args& x, bool prefix) {
  const uint64_t items = max_items(x, prefix), ranges = max_ranges(x, prefix);
  Parts p;
  uint64_t at = 0;
  auto take = [&](uint64_t bytes) {
    const uint64_t here = at;
    at += align256(bytes);
    return here;
  };
  p.item_first = take((x.n_seq + 1) * 4);
  p.items = take(items * sizeof(Item));
  p.unit_first = take(items * 8);
  p.begin = take((ranges + 1) * sizeof(RangeBegin));
  p.end = take(ranges * sizeof(RangeEnd));
  p.counts = take(8);
  p.ml = take(ranges * 2 * kRows * sizeof(float2));
  p.o = take(ranges * 2 * kRows * x.head_dim * sizeof(float));
  p.total = at;
  return p;
}

template <typename T, int D, bool kPrefix>
tcx_status launch(const TileArgs& d, const CUtensorMap& map, cudaStream_t stream) {
  using L = TileLayout<D>;
  static std::atomic<uint64_t> allowed{0};
  if (const tcx_status st = allow_shared(reinterpret_cast<const void*>(tile_kernel<T, D, kPrefix>), L::kBytes, &allowed);
      st != TCX_OK)
    return st;
  // The first kernel of the call follows the stream's earlier work whole.
  if (kPrefix) {
    tile_kernel<T, D, kPrefix><<<d.max_ranges, kThreads, L::kBytes, stream>>>(map, d);
    note_launches(1);
    TCX_CUDA_TRY(cudaGetLastError());
  } else {
    if (d.a.prior_o != nullptr) {
      if (const tcx_status st = launch_after(tile_plan_kernel, dim3(1), dim3(kPlanThreads), 0, stream, d); st != TCX_OK)
        return st;
    } else {
      tile_plan_kernel<<<1, kPlanThreads, 0, stream>>>(d);
      note_launches(1);
      TCX_CUDA_TRY(cudaGetLastError());
    }
    if (const tcx_status st = launch_after(tile_kernel<T, D, kPrefix>, dim3(d.max_ranges), dim3(kThreads), L::kBytes, stream, map, d);
        st != TCX_OK)
      return st;
  }
  if (d.max_ranges == 1 || d.join_here) return TCX_OK;
  return launch_after(tile_join_kernel<T, D>, dim3(d.max_ranges - 1, kRows / 8), dim3(256), 0, stream, d);
}

template <typename T, int D>
tcx_status launch(const TileArgs& d, const CUtensorMap& map, cudaStream_t stream) {
  return d.prefix ? launch<T, D, true>(d, map, stream) : launch<T, D, false>(d, map, stream);
}

}  // namespace

uint64_t tile_scratch_bytes(const tcx_kv_attention_args& x, bool prefix) { return parts(x, prefix).total; }

tcx_status launch_tile(const tcx_kv_attention_args& x, const AttnArgs& a, const CUtensorMap& map, bool prefix,
                       void* scratch, cudaStream_t stream) {
  const Parts p = parts(x, prefix);
  uint8_t* at = static_cast<uint8_t*>(scratch);
  TileArgs d{};
  d.a = a;
  d.prefix = prefix;
  d.max_q = static_cast<uint32_t>(x.max_q);
  d.join_here = prefix && x.q_tokens * a.group <= kJoinHere;
  d.max_ranges = max_ranges(x, prefix);
  d.item_first = reinterpret_cast<uint32_t*>(at + p.item_first);
  d.items = reinterpret_cast<Item*>(at + p.items);
  d.unit_first = reinterpret_cast<uint64_t*>(at + p.unit_first);
  d.begin = reinterpret_cast<RangeBegin*>(at + p.begin);
  d.end = reinterpret_cast<RangeEnd*>(at + p.end);
  d.counts = reinterpret_cast<uint32_t*>(at + p.counts);
  d.part_ml = reinterpret_cast<float2*>(at + p.ml);
  d.part_o = reinterpret_cast<float*>(at + p.o);
  if (x.dtype == TCX_KV_BF16)
    return x.head_dim == 128 ? launch<__nv_bfloat16, 128>(d, map, stream) : launch<__nv_bfloat16, 64>(d, map, stream);
  return x.head_dim == 128 ? launch<__half, 128>(d, map, stream) : launch<__half, 64>(d, map, stream);
}

}  // namespace tcx
