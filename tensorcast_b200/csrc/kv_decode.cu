// Attention of few query rows over long paged sequences (decode).
//
// A kv head's rows (query tokens x the head's group of q heads, up to 32) share
// the keys and values, so the call is bound by reading every visible key and value
// once from HBM. The visible tokens of all sequences are laid end to end in tiles
// of 64, and that axis is cut into equal ranges, one CTA for each range and kv
// head: every CTA reads the same number of bytes whatever the lengths are. CTAs of
// one range and neighbouring heads run side by side, so the 256-byte rows of a
// token's heads are fetched at about the same time.
//
// In a CTA one warp fills a ring of tiles with TMA (a box for each run of rows
// within a page). Of four warps (of each four, with more than 16 rows) each takes 16
// tokens of a tile: scores by mma, a running maximum and sum in 32 bits, probabilities
// rounded to the input type (half a step, as the output is: the two roundings together
// leave 1.1 to 1.2 times the output's own error) for the second product, sums in 32
// bits. Where a sequence ends inside a range the warps' parts are joined and written;
// a sequence cut by a range's border leaves parts in the scratch, and the CTA that
// comes last adds them up in the ranges' order. Where weights are accumulated, the
// scores go to the scratch as well (rows x 4 bytes for a token, against its 4 D), and
// decode_weights_kernel takes them up once the rows' sums are known.
//
// Measured on B200: 96 sequences of 64-4096 tokens, 32 / 8 heads of 128, 452 MB in
// 82 us (5.5 TB/s, 0.85 of the measured copy rate; about 10 us of it are the first
// loads' and the last joins' latencies); one sequence of 777 tokens 12.5 us.
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "kv_attention.cuh"
#include "kv_pieces.h"

namespace tcx {
namespace {

constexpr int kTile = 64;
constexpr int kWarps = 4;       // for each 16 rows: 16 tokens of a tile each
constexpr int kWarpRows = 16;

enum : uint32_t { kFirst = 1, kLast = 2, kMask = 4, kWhole = 8, kSecondSlot = 16 };

// What the consumers need to know of a tile.
struct TileInfo {
  uint32_t flags, seq, q_first, queries;
  int token, len, low, sinks;  // low: first token inside the first query's window
  uint32_t first_range, parts, first_slot;  // of a sequence that more than one range holds
};

struct DecodeArgs {
  AttnArgs a;
  uint32_t ranges, rows;  // at most
  uint32_t part_rows;     // 16 or 32
  float* part_o;    // [ranges][2][kv_heads][part_rows][D], sums of 2^(z - m) v
  float2* part_ml;  // the same rows' m and sum of 2^(z - m)
  float* scores;    // [kv_heads][rows][columns], in powers of two, where weights are added up
  uint32_t score_rows;
  uint64_t columns;
};

template <int D, int G>
struct Layout {
  static constexpr int kRows = kWarpRows * G;
  static constexpr int kHalf = kTile * 128;              // 64 values of each token: 128-byte rows, swizzled
  static constexpr int kKeys = kHalf * (D / 64);
  static constexpr int kQueryPitch = D * 2 + 16;          // 16 bytes more: rows in different banks
  static constexpr int kQueries = kRows * kQueryPitch;
  static constexpr int kStage = 2 * kKeys + (kQueries + 1023) / 1024 * 1024;
  // two CTAs fit an SM with 16 rows, one with 32
  static constexpr int kStages = (D == 128 ? 3 : 5) + (G == 1 ? 0 : D == 128 ? 2 : 3);
  static constexpr int kBytes = kStages * kStage + 1024;  // the first tile starts on a 1 KiB border
};

struct SeqInfo {
  int len, low, sinks, sink_tiles, first_tile;  // tiles: [0, sink_tiles) and from first_tile on
  uint32_t tiles, q_first, queries;
  uint64_t table;  // first entry in the page table

  __device__ __forceinline__ int token(uint32_t t) const {  // first token of tile t
    return (t < static_cast<uint32_t>(sink_tiles) ? static_cast<int>(t) : first_tile + static_cast<int>(t) - sink_tiles) *
           kTile;
  }
};

__device__ __forceinline__ SeqInfo seq_info(const AttnArgs& a, uint32_t s, int prefix) {
  SeqInfo i;
  i.table = a.page_offsets[s];
  i.q_first = a.q_offsets[s];
  i.queries = a.q_offsets[s + 1] - i.q_first;
  i.len = static_cast<int>(seq_length(a, s));
  i.low = a.window ? static_cast<int>(max(int64_t{0}, i.len - static_cast<int64_t>(i.queries) - a.window + 1)) : 0;
  i.sinks = static_cast<int>(max(int64_t{0}, a.sinks - prefix));
  const int tiles = (i.len + kTile - 1) / kTile;
  i.sink_tiles = i.low > 0 ? (min(i.sinks, i.len) + kTile - 1) / kTile : 0;
  i.first_tile = max(i.low / kTile, i.sink_tiles);
  // a sequence without tokens has one empty tile, so that its rows are written
  i.tiles = i.queries == 0 ? 0 : max(i.sink_tiles + tiles - i.first_tile, 1);
  return i;
}

// The rows of a sequence that several ranges hold: D / 4 threads to a row, the parts
// in the ranges' order.
template <typename T, int D, int G>
__device__ __forceinline__ void join_parts(const DecodeArgs& d, const TileInfo& info, uint32_t head, uint32_t rows) {
  const AttnArgs& a = d.a;
  constexpr uint32_t kLanes = D / 4;
  const uint32_t lane = threadIdx.x % kLanes, e = lane * 4;
  for (uint32_t r0 = 0; r0 < rows; r0 += 128 * G / kLanes) {
    const uint32_t r = min(r0 + threadIdx.x / kLanes, rows - 1);  // all lanes take part in the shuffles
    auto row_of = [&](uint32_t k) {
      return (static_cast<uint64_t>((info.first_range + k) * 2 + (k == 0 ? info.first_slot : 0)) * a.kv_heads + head) *
                 (kWarpRows * G) + r;
    };
    float top = -INFINITY, sum = 0.f, x[4] = {};
    for (uint32_t k = lane; k < info.parts; k += kLanes) top = fmaxf(top, __ldcg(&d.part_ml[row_of(k)].x));
    for (uint32_t i = kLanes / 2; i; i /= 2) top = fmaxf(top, __shfl_xor_sync(~0u, top, i));
    const float ref = top == -INFINITY ? 0.f : top;
#pragma unroll 8
    for (uint32_t k = 0; k < info.parts; ++k) {
      const uint64_t row = row_of(k);
      const float2 ml = __ldcg(&d.part_ml[row]);
      const float4 v = __ldcg(reinterpret_cast<const float4*>(d.part_o + row * D + e));
      const float f = exp2_approx(ml.x - ref);
      sum += f * ml.y;
      x[0] += f * v.x;
      x[1] += f * v.y;
      x[2] += f * v.z;
      x[3] += f * v.w;
    }
    if (r0 + threadIdx.x / kLanes >= rows) continue;
    const uint32_t t = info.q_first + r / a.group, h = head * a.group + r % a.group;
    const Finish f = finish_row(a, static_cast<uint64_t>(t) * a.kv_heads * a.group + h, top, sum);
    store_row<T, D>(a, t, h, e, f, x);
    if (e == 0) store_lse(a, t, h, f);
  }
  __syncwarp();
}

template <typename T, int D, bool kScores, int G>
__global__ void __launch_bounds__(32 * (kWarps * G + 1), G == 1 ? 2 : 1)
    decode_kernel(const __grid_constant__ CUtensorMap map, DecodeArgs d) {
  using L = Layout<D, G>;
  constexpr int kThreads = 32 * (kWarps * G + 1), kRows = L::kRows;
  extern __shared__ uint8_t raw[];
  __shared__ TileInfo s_info[L::kStages];
  __shared__ uint64_t s_full[L::kStages], s_empty[L::kStages];
  __shared__ uint32_t s_scan[kThreads / 32], s_begin[2], s_gave_up, s_drained, s_last;
  __shared__ float2 s_ml[kWarps * G][kWarpRows];
  const AttnArgs& a = d.a;
  const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const uint32_t head = blockIdx.x % a.kv_heads, range = blockIdx.x / a.kv_heads;
  const uint32_t base = (smem_addr(raw) + 1023) & ~1023u;
  next_may_start();
  if (threadIdx.x == 0) {
    for (int i = 0; i < L::kStages; ++i) {
      mbar_init(smem_addr(&s_full[i]), 1);
      mbar_init(smem_addr(&s_empty[i]), kWarps * G);
    }
    s_gave_up = s_drained = 0;
    mbar_init_fence();
  }
  // Rows of the query area that no query fills must hold finite values.
  for (uint32_t i = threadIdx.x; i < L::kStages * (L::kQueries / 16); i += kThreads)
    asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(base + i / (L::kQueries / 16) * L::kStage +
                                                                   2 * L::kKeys + i % (L::kQueries / 16) * 16),
                 "r"(0)
                 : "memory");
  proxy_fence_smem();
  const int prefix = static_cast<int>(prefix_length(a));
  // Tiles of this thread's share of the sequences, and where this range begins.
  const uint32_t share = (a.n_seq + kThreads - 1) / kThreads, s0 = min(threadIdx.x * share, a.n_seq),
                 s1 = min(s0 + share, a.n_seq);
  uint32_t mine = 0;
  for (uint32_t s = s0; s < s1; ++s) mine += seq_info(a, s, prefix).tiles;
  uint32_t inc = mine;
  for (int x = 1; x < 32; x *= 2) {
    const uint32_t up = __shfl_up_sync(~0u, inc, x);
    if (lane >= x) inc += up;
  }
  if (lane == 31) s_scan[warp] = inc;
  __syncthreads();
  uint32_t total = 0, before = inc - mine;
  for (uint32_t w = 0; w < kThreads / 32; ++w) {
    if (w < warp) before += s_scan[w];
    total += s_scan[w];
  }
  // A tile more in a range costs about 1400 cycles (what one SM fetches of it), a range
  // more for a sequence 90 for every four rows when its parts are joined: few tiles are
  // cut where the two together are least.
  const uint32_t least = max(1u, static_cast<uint32_t>(sqrtf(static_cast<float>(total) * d.rows * (1.f / 64))));
  const uint32_t ranges = min(d.ranges, (total + least - 1) / least);
  if (range >= ranges) {
    wait_for_previous();
    return;
  }
  const uint32_t t0 = static_cast<uint32_t>(scaled(range, total, ranges));
  const uint32_t t1 = static_cast<uint32_t>(scaled(range + 1, total, ranges));
  if (before <= t0 && t0 < before + mine) {
    uint32_t s = s0, at = before;
    for (;; ++s) {
      const uint32_t n = seq_info(a, s, prefix).tiles;
      if (t0 < at + n) break;
      at += n;
    }
    s_begin[0] = s;
    s_begin[1] = t0 - at;
  }
  __syncthreads();
  const uint32_t count = t1 - t0;

  if (warp == kWarps * G) {  // ---- the producer
    const uint32_t boxes = kTile / a.box_rows, halves = D / 64;
    // lane: one box of the keys or values and one half of the head
    const uint32_t box = lane % boxes, half = lane / boxes % halves, plane = lane / boxes / halves;
    const uint64_t plane_row = plane ? a.v_row0 : a.k_row0;
    // Page slots are looked up for 32 boxes at once, and for the next 32, or the next
    // sequence's first, while the tiles before them are fetched.
    const uint32_t per = 32 / boxes;  // tiles
    auto wanted_box = [&](const SeqInfo& q, int from) {
      const int to = from + static_cast<int>(a.box_rows);
      return from < q.len && (to > q.low || from < q.sinks);
    };
    auto slots_of = [&](const SeqInfo& q, uint32_t t0) {
      const uint32_t t = t0 + lane / boxes;
      if (t >= q.tiles) return 0u;
      const int from = q.token(t) + static_cast<int>(box * a.box_rows);
      return wanted_box(q, from) ? static_cast<uint32_t>(checked_slot(a, a.page_table + q.table, from / a.page_tokens)) : 0u;
    };
    uint32_t s = s_begin[0], t = s_begin[1], next_s = s;
    SeqInfo q = seq_info(a, s, prefix), next = q;
    uint32_t slots_from = t, slots = slots_of(q, t), next_slots = 0;
    uint32_t slots_ahead = count > per ? slots_of(q, t + per) : 0;
    bool fresh = true;  // the next tile is the first of its piece
    uint32_t pieces = 0;
    uint32_t i = 0;
    for (; i < count; ++i) {
      const uint32_t stage = i % L::kStages;
      const int token = q.token(t);
      if (t == slots_from + per) {
        slots = slots_ahead;
        slots_from = t;
        slots_ahead = slots_of(q, t + per);
      }
      const uint32_t slot = __shfl_sync(~0u, slots, (t - slots_from) * boxes + box);
      if (!mbar_wait_warp(smem_addr(&s_empty[stage]), (i / L::kStages & 1) ^ 1, &s_gave_up, a.status)) break;
      const uint32_t full = smem_addr(&s_full[stage]), at = base + stage * L::kStage;
      const int from = token + static_cast<int>(box * a.box_rows);
      const bool wanted = lane < 2 * halves * boxes && wanted_box(q, from);
      const uint32_t rows = fresh ? min(q.queries * a.group, static_cast<uint32_t>(kRows)) : 0;
      const uint32_t bytes = __popc(__ballot_sync(~0u, wanted)) * a.box_rows * 128 + rows * D * 2;
      if (lane == 0) mbar_expect(full, bytes);
      __syncwarp();
      if (wanted)
        tma_load_3d(at + plane * L::kKeys + half * L::kHalf + box * a.box_rows * 128, &map, half * 64, head,
                    static_cast<int>(plane_row + static_cast<uint64_t>(slot) * a.page_tokens + from % a.page_tokens), full);
      if (lane < rows)
        bulk_load(at + 2 * L::kKeys + lane * L::kQueryPitch,
                  a.q + (q.q_first + lane / a.group) * a.q_token_stride +
                      (head * a.group + lane % a.group) * a.q_head_stride,
                  D * 2, full);
      // What the consumers need is worked out while the copies run; they wait for both.
      TileInfo info{fresh ? kFirst : 0u, s, q.q_first, q.queries, token, q.len, q.low, q.sinks, 0, 0, 0};
      const bool seq_done = t + 1 == q.tiles;
      if (seq_done || i + 1 == count) info.flags |= kLast;
      const bool starts = s != s_begin[0] || s_begin[1] == 0;
      if (seq_done && starts) info.flags |= kWhole;
      if ((info.flags & kLast) && !(info.flags & kWhole)) {
        // the ranges that hold tiles [first, first + q.tiles)
        const uint64_t first = t0 + i - t;
        // the last range that begins at a tile or before: ((tile + 1) ranges - 1) / total
        auto range_of = [&](uint64_t tile) { return static_cast<uint32_t>(scaled((tile + 1) * ranges - 1, 1, total)); };
        info.first_range = range_of(first);
        info.parts = range_of(first + q.tiles - 1) - info.first_range + 1;
        info.first_slot = first != scaled(info.first_range, total, ranges);
      }
      if (pieces > 0) info.flags |= kSecondSlot;
      const int last_low = a.window ? q.low + static_cast<int>(q.queries) - 1 : 0;  // at least the last query's
      if (token + kTile - 1 > q.len - static_cast<int>(q.queries) ||
          (token < last_low && token + kTile > q.sinks))
        info.flags |= kMask;
      if (lane == 0) {
        s_info[stage] = info;
        mbar_arrive(full);
      }
      if (fresh && i + (q.tiles - t) < count) {  // the next sequence is this range's too
        next_s = s;
        do next = seq_info(a, ++next_s, prefix); while (next.tiles == 0);
        next_slots = slots_of(next, 0);
      }
      fresh = false;
      ++t;
      if (seq_done && i + 1 < count) {
        s = next_s;
        q = next;
        t = slots_from = 0;
        slots = next_slots;
        slots_ahead = slots_of(q, per);
        fresh = true;
        ++pieces;
      }
    }
    // No copy may be in flight when the CTA ends.
    for (uint32_t k = i > L::kStages ? i - L::kStages : 0; k < i; ++k)
      mbar_wait_warp(smem_addr(&s_full[k % L::kStages]), k / L::kStages & 1, &s_drained, a.status);
    return;
  }

  // ---- the consumers: rows row0 + lane / 4 and 8 more, tokens 16 part .. 16 part + 15 of each tile
  const uint32_t part = warp % kWarps, row0 = warp / kWarps * kWarpRows;
  auto meet = [&] { asm volatile("bar.sync 1, %0;" ::"n"(128 * G) : "memory"); };
  constexpr int kMeets = 2 * G + 1;  // at the end of a piece, and one more where its parts are joined
  uint32_t qf[D / 16][4];
  constexpr bool kIsHalf = std::is_same<T, __half>::value;
  float o[D / 8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f}, peak[2] = {-INFINITY, -INFINITY};
  uint32_t i = 0;
  for (; i < count; ++i) {
    const uint32_t stage = i % L::kStages, at = base + stage * L::kStage;
    if (!mbar_wait_warp(smem_addr(&s_full[stage]), i / L::kStages & 1, &s_gave_up, a.status)) break;
    const TileInfo info = s_info[stage];
    if (info.flags & kFirst) {
#pragma unroll
      for (int k = 0; k < D / 16; ++k)
        ldmatrix4(qf[k], at + 2 * L::kKeys + (row0 + lane % 16) * L::kQueryPitch + k * 32 + lane / 16 * 16);
#pragma unroll
      for (int n = 0; n < D / 8; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[n][e] = 0.f;
      m[0] = m[1] = peak[0] = peak[1] = -INFINITY;
      l[0] = l[1] = 0.f;
    }
    // All of the warp's keys are loaded before the first product, and its values before
    // the softmax, so that their latencies do not add up.
    uint32_t kf[D / 16][4], vf[D / 16][4];
    {
      const uint32_t token = part * 16 + lane / 16 * 8 + lane % 8, chunk = lane / 8 % 2;
      const uint32_t row = at + token * 128;
#pragma unroll
      for (int k = 0; k < D / 16; ++k)
        ldmatrix4(kf[k], row + k / 4 * L::kHalf + (((k % 4 * 2 + chunk) ^ (token & 7)) << 4));
    }
    if (info.flags & kMask) {
      // values that no row sees are cleared: 0 x NaN is not 0
      const int hidden = info.token + static_cast<int>(part * 16 + lane % 16);
      const bool clear = hidden >= info.len || (hidden < info.low && hidden >= info.sinks);
      if (__any_sync(~0u, clear)) {
        if (clear) {
          const uint32_t row = at + L::kKeys + lane / 16 * (L::kHalf * (D / 128)) + (part * 16 + lane % 16) * 128;
          if (lane < 16 || D == 128)
            for (int c = 0; c < 8; ++c)
              asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(row + c * 16), "r"(0) : "memory");
        }
        proxy_fence_smem();
        __syncwarp();
      }
    }
    {
      const uint32_t token = part * 16 + lane % 16;
      const uint32_t row = at + L::kKeys + token * 128;
#pragma unroll
      for (int n = 0; n < D / 16; ++n)
        ldmatrix4_t(vf[n], row + n / 4 * L::kHalf + (((n % 4 * 2 + lane / 16) ^ (token & 7)) << 4));
    }
    // scores: tokens 0-7 (z[0]) and 8-15 (z[1]) of this warp's 16, in two sums each
    float z[2][4] = {}, z2[2][4] = {};
#pragma unroll
    for (int k = 0; k < D / 16; k += 2) {
      mma16816<T>(z[0], qf[k], kf[k][0], kf[k][1]);
      mma16816<T>(z[1], qf[k], kf[k][2], kf[k][3]);
      mma16816<T>(z2[0], qf[k + 1], kf[k + 1][0], kf[k + 1][1]);
      mma16816<T>(z2[1], qf[k + 1], kf[k + 1][2], kf[k + 1][3]);
    }
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) z[n][e] += z2[n][e];
    if (info.flags & kMask) {
      const int first = info.token + static_cast<int>(part) * 16;
      const uint32_t r = row0 + lane / 4;
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int j = first + n * 8 + static_cast<int>(lane % 4) * 2 + e % 2;
          const int i_q = static_cast<int>((r + e / 2 * 8) / a.group);
          const int pos = info.len - static_cast<int>(info.queries) + i_q;
          const bool see = j <= pos && (a.window == 0 || j > pos - a.window || j < info.sinks);
          if (!see) z[n][e] = -INFINITY;
        }
    }
    if constexpr (kScores) {
      const uint64_t column = a.page_offsets[info.seq] * a.page_tokens;
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const uint32_t row = row0 + lane / 4 + 8 * r;
        if (row < info.queries * a.group && row < d.score_rows) {
          float* to = d.scores + (static_cast<uint64_t>(head) * d.score_rows + row) * d.columns + column;
#pragma unroll
          for (int n = 0; n < 2; ++n) {
            const int j = info.token + static_cast<int>(part * 16 + n * 8 + lane % 4 * 2);
            if (j < info.len)  // an even place: the pair's second is within the page
              *reinterpret_cast<float2*>(to + j) = make_float2(z[n][2 * r] * a.scale_log2, z[n][2 * r + 1] * a.scale_log2);
          }
        }
      }
    }
    uint32_t p[4];
    float scale[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      float top = fmaxf(fmaxf(z[0][2 * r], z[0][2 * r + 1]), fmaxf(z[1][2 * r], z[1][2 * r + 1]));
      top = fmaxf(top, __shfl_xor_sync(~0u, top, 1));
      top = fmaxf(top, __shfl_xor_sync(~0u, top, 2)) * a.scale_log2;
      if constexpr (kIsHalf) {
        top = half_reference(m[r], top, peak[r], true);
        peak[r] = fmaxf(peak[r], top);
      } else {
        top = fmaxf(top, m[r]);
      }
      const float ref = top == -INFINITY ? 0.f : top;
      scale[r] = exp2_approx(m[r] - ref);
      m[r] = top;
      float sum = 0.f;
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float& x = z[n][2 * r + e];
          x = exp2_approx(fmaf(x, a.scale_log2, -ref));
          sum += x;
        }
      l[r] = l[r] * scale[r] + sum;  // of this lane's columns
    }
    p[0] = pack2<T>(z[0][0], z[0][1]);
    p[1] = pack2<T>(z[0][2], z[0][3]);
    p[2] = pack2<T>(z[1][0], z[1][1]);
    p[3] = pack2<T>(z[1][2], z[1][3]);
    if (__any_sync(~0u, scale[0] != 1.f || scale[1] != 1.f)) {
#pragma unroll
      for (int n = 0; n < D / 8; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[n][e] *= scale[e / 2];
    }
#pragma unroll
    for (int n = 0; n < D / 16; ++n) {
      mma16816<T>(o[2 * n], p, vf[n][0], vf[n][1]);
      mma16816<T>(o[2 * n + 1], p, vf[n][2], vf[n][3]);
    }
    if (info.flags & kLast) {
      wait_for_previous();  // the rows' parts over a shared prefix
      // The four warps' parts are joined in this tile's memory, which all have read.
      const uint32_t rows = min(info.queries * a.group, static_cast<uint32_t>(kRows));
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        l[r] += __shfl_xor_sync(~0u, l[r], 1);
        l[r] += __shfl_xor_sync(~0u, l[r], 2);
        if (lane % 4 == 0) s_ml[warp][lane / 4 + 8 * r] = make_float2(m[r], l[r]);
      }
      meet();
      float* join = reinterpret_cast<float*>(raw + (at - smem_addr(raw)));  // [part][row][D]
      constexpr uint32_t kLanes = D / 4;  // threads of a row: 4 values each
#pragma unroll
      for (uint32_t g = 0; g < G; ++g) {  // 16 rows at a time: that is what the tile's memory holds
        if (g > 0) meet();
        if (row0 == g * kWarpRows) {
#pragma unroll
          for (int r = 0; r < 2; ++r)
            if (row0 + lane / 4 + 8 * r < rows)
#pragma unroll
              for (int n = 0; n < D / 8; ++n)
                *reinterpret_cast<float2*>(join + (part * kWarpRows + lane / 4 + 8 * r) * D + n * 8 + lane % 4 * 2) =
                    make_float2(o[n][2 * r], o[n][2 * r + 1]);
        }
        meet();
        const uint32_t here = min(rows - min(rows, g * kWarpRows), static_cast<uint32_t>(kWarpRows));
        for (uint32_t in = threadIdx.x / kLanes; in < here; in += 128 * G / kLanes) {
          const uint32_t e = threadIdx.x % kLanes * 4, r = g * kWarpRows + in;
          const float2(*ml)[kWarpRows] = s_ml + g * kWarps;
          float top = -INFINITY, sum = 0.f;
          for (int w = 0; w < kWarps; ++w) top = fmaxf(top, ml[w][in].x);
          const float ref = top == -INFINITY ? 0.f : top;
          float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
          for (int w = 0; w < kWarps; ++w) {
            const float f = exp2_approx(ml[w][in].x - ref);
            sum += f * ml[w][in].y;
            const float4 x = *reinterpret_cast<const float4*>(join + (w * kWarpRows + in) * D + e);
            v.x += f * x.x;
            v.y += f * x.y;
            v.z += f * x.z;
            v.w += f * x.w;
          }
          if (info.flags & kWhole) {
            const uint32_t t = info.q_first + r / a.group, h = head * a.group + r % a.group;
            const Finish f = finish_row(a, static_cast<uint64_t>(t) * a.kv_heads * a.group + h, top, sum);
            store_row<T, D>(a, t, h, e, f, {v.x, v.y, v.z, v.w});
            if (e == 0) store_lse(a, t, h, f);
          } else {
            const uint64_t row =
                (static_cast<uint64_t>(range * 2 + (info.flags & kSecondSlot ? 1 : 0)) * a.kv_heads + head) * kRows + r;
            *reinterpret_cast<float4*>(d.part_o + row * D + e) = v;
            if (e == 0) d.part_ml[row] = make_float2(top, sum);
          }
        }
      }
      meet();  // all have read s_ml: the next sequence's come there
      if (!(info.flags & kWhole)) {  // whoever comes last adds the parts up, in the ranges' order
        if (threadIdx.x == 0)
          s_last = last_to_arrive(a.counters + info.first_range * a.kv_heads + head, info.parts);
        meet();
        if (s_last) join_parts<T, D, G>(d, info, head, rows);
      }
      proxy_fence_smem();  // these accesses come before the copies of the next tile here
    }
    mbar_arrive_warp(smem_addr(&s_empty[stage]), lane, true);
  }
  // A wait of this warp ran out. The copies may still arrive for the other warps, which
  // then meet it at the ends of their pieces: it comes there as often as they do, by the
  // lengths alone (the notes may be another lap's), and neither reads nor stores.
  if (i < count) wait_for_previous();
  for (; i < count; ++i) {
    const TileEnd end = tile_end(s_begin[0], s_begin[1], count, i, [&](uint32_t s) { return seq_info(a, s, prefix).tiles; });
    if (!end.last) continue;
    for (int k = 0; k < kMeets; ++k) meet();
    if (!end.whole) {
      if (threadIdx.x == 0) s_last = 0;
      meet();
    }
  }
}

// The tokens' softmax weights, of the scores that decode_kernel left: a thread for
// four tokens and a kv head, the rows in their order.
__global__ void __launch_bounds__(128) decode_weights_kernel(DecodeArgs d) {
  const AttnArgs& a = d.a;
  const uint32_t s = blockIdx.z, head = blockIdx.y, q_first = a.q_offsets[s], queries = a.q_offsets[s + 1] - q_first;
  __shared__ float s_lse[kDecodeRows];
  const uint32_t rows = min(queries * a.group, d.score_rows);
  const SeqInfo q = seq_info(a, s, 0);
  if (rows == 0 || static_cast<int>(blockIdx.x * 512) >= q.len) {
    wait_for_previous();  // also here: this kernel's end stands for the one's before
    return;
  }
  const uint64_t column = a.page_offsets[s] * a.page_tokens;
  const float* z = d.scores + static_cast<uint64_t>(head) * d.score_rows * d.columns + column;
  float* w = a.weights + head * a.weights_head_stride + column;
  wait_for_previous();
  if (threadIdx.x < rows)
    s_lse[threadIdx.x] = kLog2e * a.lse[(q_first + threadIdx.x / a.group) * static_cast<uint64_t>(a.kv_heads) * a.group +
                                        head * a.group + threadIdx.x % a.group];
  __syncthreads();
  for (int j = static_cast<int>(blockIdx.x * 128 + threadIdx.x) * 4; j < q.len; j += static_cast<int>(gridDim.x * 512)) {
    float sum[4] = {};
#pragma unroll 4
    for (uint32_t r = 0; r < rows; ++r) {
      const float lse = s_lse[r];
      const float4 x = *reinterpret_cast<const float4*>(z + r * d.columns + j);  // whole pages: within the scratch
      if (lse == -INFINITY) continue;
      sum[0] += exp2_approx(x.x - lse);
      sum[1] += exp2_approx(x.y - lse);
      sum[2] += exp2_approx(x.z - lse);
      sum[3] += exp2_approx(x.w - lse);
    }
    // Tokens between the sinks and the window are seen by no row, and no tile held them.
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (j + k < q.len && (j + k >= q.low || j + k < q.sinks)) w[j + k] += sum[k];
  }
}

uint32_t part_rows(const tcx_kv_attention_args& x) {
  return x.max_q * (x.q_heads / x.kv_heads) <= kWarpRows ? kWarpRows : 2 * kWarpRows;
}

// Two CTAs fit an SM (one with 32 rows). Each range and head needs a counter where
// there are ranges to join; the other half of the counters is the tile kernel's, which
// may still run.
uint32_t decode_ranges(const tcx_kv_attention_args& x) {
  const uint64_t tiles = x.total_pages * x.page_tokens / kTile + x.n_seq;
  const uint64_t most = std::min<uint64_t>((part_rows(x) == kWarpRows ? 2ull : 1ull) * sm_count(), TCX_KV_COUNTERS / 2) / x.kv_heads;
  return static_cast<uint32_t>(std::max<uint64_t>(1, std::min<uint64_t>(tiles, most)));
}

template <typename T, int D, bool kScores, int G>
tcx_status launch(const DecodeArgs& d, const CUtensorMap& map, uint64_t max_tokens, cudaStream_t stream) {
  using L = Layout<D, G>;
  constexpr int kThreads = 32 * (kWarps * G + 1);
  static std::atomic<uint64_t> allowed{0};
  if (const tcx_status st = allow_shared(reinterpret_cast<const void*>(decode_kernel<T, D, kScores, G>), L::kBytes, &allowed);
      st != TCX_OK)
    return st;
  const dim3 grid(d.ranges * d.a.kv_heads);
  if (d.a.prior_o != nullptr) {  // behind the shared prefix's kernels
    if (const tcx_status st = launch_after(decode_kernel<T, D, kScores, G>, grid, dim3(kThreads), L::kBytes, stream, map, d);
        st != TCX_OK)
      return st;
  } else {
    decode_kernel<T, D, kScores, G><<<grid, kThreads, L::kBytes, stream>>>(map, d);
    note_launches(1);
    TCX_CUDA_TRY(cudaGetLastError());
  }
  if (!kScores || max_tokens == 0) return TCX_OK;
  const uint64_t blocks = std::min<uint64_t>((max_tokens + 511) / 512, 64);
  return launch_after(decode_weights_kernel, dim3(static_cast<unsigned>(blocks), d.a.kv_heads, d.a.n_seq), dim3(128), 0,
                      stream, d);
}

template <typename T, int D>
tcx_status launch(const DecodeArgs& d, const CUtensorMap& map, uint64_t max_tokens, cudaStream_t stream) {
  if (d.part_rows == kWarpRows)
    return d.scores != nullptr ? launch<T, D, true, 1>(d, map, max_tokens, stream)
                               : launch<T, D, false, 1>(d, map, max_tokens, stream);
  return d.scores != nullptr ? launch<T, D, true, 2>(d, map, max_tokens, stream)
                             : launch<T, D, false, 2>(d, map, max_tokens, stream);
}

uint64_t score_bytes(const tcx_kv_attention_args& x) {
  if (x.d_weights == nullptr) return 0;
  return align256(x.max_q * x.q_heads * x.total_pages * x.page_tokens * sizeof(float));
}

}  // namespace

// Up to 16 rows fill one tile of the products, up to 32 two, in warps of their own and one
// CTA on an SM; from there on the tile kernel. At 20 rows of one 500-token sequence the
// two take 18.6 and 23.6 us, at 32 rows of 96 sequences of 64-4096 tokens 165 and 156.
bool decode_fits(const tcx_kv_attention_args& x) {
  return x.max_q * (x.q_heads / x.kv_heads) <= kDecodeRows;
}

uint64_t decode_scratch_bytes(const tcx_kv_attention_args& x) {
  const uint64_t parts = decode_ranges(x) * 2ull * x.kv_heads * part_rows(x);
  return align256(parts * sizeof(float2)) +
         align256(parts * x.head_dim * 4) + score_bytes(x);
}

tcx_status launch_decode(const tcx_kv_attention_args& x, const AttnArgs& a, const CUtensorMap& map, void* scratch,
                         cudaStream_t stream) {
  DecodeArgs d{};
  d.a = a;
  d.ranges = decode_ranges(x);
  d.rows = static_cast<uint32_t>(x.max_q) * a.group;
  d.part_rows = part_rows(x);
  const uint64_t parts = d.ranges * 2ull * x.kv_heads * part_rows(x);
  uint8_t* at = static_cast<uint8_t*>(scratch);
  d.part_ml = reinterpret_cast<float2*>(at);
  d.part_o = reinterpret_cast<float*>(at += align256(parts * sizeof(float2)));
  const uint32_t rows = static_cast<uint32_t>(x.max_q) * a.group;
  if (x.d_weights != nullptr) {
    d.scores = reinterpret_cast<float*>(at + align256(parts * x.head_dim * 4));
    d.score_rows = rows;
    d.columns = x.total_pages * x.page_tokens;
  }
  const uint64_t max_tokens = x.max_pages * x.page_tokens;
  if (x.dtype == TCX_KV_BF16)
    return x.head_dim == 128 ? launch<__nv_bfloat16, 128>(d, map, max_tokens, stream)
                             : launch<__nv_bfloat16, 64>(d, map, max_tokens, stream);
  return x.head_dim == 128 ? launch<__half, 128>(d, map, max_tokens, stream) : launch<__half, 64>(d, map, max_tokens, stream);
}

}  // namespace tcx
