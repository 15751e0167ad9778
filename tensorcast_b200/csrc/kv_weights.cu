// The softmax weights of many query rows, added up for every token of a paged
// sequence: weight[j] += sum over rows of exp(scale q.k_j - lse).
//
// A CTA holds a tile of 128 keys and takes all rows that see one of them through it,
// 128 at a time: scores with the keys as the product's rows, so that a thread owns
// one key and half of the rows, adds up its 64 scores without exchanging anything, in
// the rows' order, and the key's two halves meet once at the end. The scores are
// recomputed from the keys: beside a prompt's products that is a third more, where
// keeping them would take rows x tokens x 4 bytes. Two CTAs share an SM, so that one's
// fetches run beside the other's exponentials. The exponential units bound it, at 0.45
// of their rate while an SM has work (a fourth of the exponentials as polynomials
// changed less than 1 %); over the whole call 0.36, because 657 CTAs are 2.2 rounds.
// Measured on B200: 256 queries at the ends of two sequences of 5000-6100 tokens, 32 / 8
// heads of 128, 58 to 62 us beside 70 us for their attention (4 us more with one thread
// for all 128 rows of a key).
#include <algorithm>
#include <type_traits>

#include "kv_attention.cuh"

namespace tcx {
namespace {

constexpr int kKeys = 128;
constexpr int kRows = 128;
constexpr int kWorkers = 2 * kKeys;  // a thread for each key and half of the rows
constexpr int kWarpRows = kRows * 32 / kWorkers;  // that a warp fetches
constexpr int kThreads = kWorkers + 32;

template <int D>
struct WeightLayout {
  static constexpr int kBlock = 128 * 128;            // 64 values of 128 rows, swizzled
  static constexpr int kOperand = kBlock * (D / 64);
  static constexpr int kBytes = 3 * kOperand + 1024;  // the keys, and two tiles of queries
};

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 2) weights_kernel(const __grid_constant__ CUtensorMap map, AttnArgs a) {
  using L = WeightLayout<D>;
  extern __shared__ uint8_t raw[];
  // Of the tiles' rows: lse in powers of two, infinite where the row counts for nothing,
  // and the keys that it sees, up to hi and from lo on (and the sinks).
  __shared__ __align__(16) float s_lse[4][kRows];
  __shared__ int2 s_sees[4][kRows];
  __shared__ float s_other[kKeys];
  __shared__ uint64_t s_bar[7];
  __shared__ uint32_t s_tmem, s_gave_up, s_drained;
  const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32, head = blockIdx.y, s = blockIdx.z;
  const int len = static_cast<int>(seq_length(a, s)), key0 = static_cast<int>(blockIdx.x) * kKeys;
  const uint32_t q_first = a.q_offsets[s], queries = a.q_offsets[s + 1] - q_first, rows = queries * a.group;
  if (key0 >= len || queries == 0) {
    wait_for_previous();  // also here: this kernel's end stands for the one's before
    return;
  }
  const int pos0 = len - static_cast<int>(queries), key_end = min(key0 + kKeys, len);
  const int sinks = static_cast<int>(a.sinks);
  auto low_of = [&](int pos) { return a.window ? static_cast<int>(max(int64_t{0}, pos - a.window + 1)) : 0; };
  // Rows that see a key of this tile: the queries from the first key on, up to the
  // last one whose window reaches back to the last key (all where a sink is among them).
  const int q_begin = max(key0 - pos0, 0);
  const int64_t q_last = a.window && key0 >= sinks ? key_end - 1 + a.window - 1 - pos0 : static_cast<int64_t>(queries) - 1;
  const int q_end = static_cast<int>(min(q_last + 1, static_cast<int64_t>(queries)));
  if (q_begin >= q_end) {
    wait_for_previous();
    return;
  }
  const uint32_t tile0 = q_begin * a.group / kRows, tile_end = (q_end * a.group + kRows - 1) / kRows;
  const uint32_t n = tile_end - tile0;

  const uint32_t base = (smem_addr(raw) + 1023) & ~1023u;
  const uint32_t keys_there = smem_addr(&s_bar[0]);
  auto queries_there = [&](uint32_t i) { return smem_addr(&s_bar[1 + i % 2]); };
  auto scored = [&](uint32_t i) { return smem_addr(&s_bar[3 + i % 2]); };
  auto taken = [&](uint32_t i) { return smem_addr(&s_bar[5 + i % 2]); };
  if (threadIdx.x == 0) {
    mbar_init(keys_there, 1);
    for (uint32_t i = 0; i < 2; ++i) {
      mbar_init(queries_there(i), kWorkers / 32);
      mbar_init(scored(i), 1);
      mbar_init(taken(i), kWorkers / 32);
    }
    s_gave_up = s_drained = 0;
    mbar_init_fence();
  }
  // The kernel before may still hold tensor memory, but on no SM of this CTA's: its
  // registers and shared memory leave no room beside it.
  if (warp == kWorkers / 32) tmem_alloc(smem_addr(&s_tmem), 2 * kRows);
  tmem_fence_before();
  __syncthreads();
  tmem_fence_after();
  const uint32_t tmem = s_tmem;

  if (warp == kWorkers / 32) {  // ---- the keys, and the products
    const uint32_t boxes = kKeys / a.box_rows, box = lane % boxes, half = lane / boxes;
    const int from = key0 + static_cast<int>(box * a.box_rows);
    const bool wanted = half < D / 64 && from < key_end;
    const uint32_t bytes = __popc(__ballot_sync(~0u, wanted)) * a.box_rows * 128;
    uint64_t row = 0;
    if (wanted)
      row = checked_slot(a, a.page_table + a.page_offsets[s], from / a.page_tokens) * a.page_tokens + from % a.page_tokens;
    if (lane == 0) mbar_arrive_expect(keys_there, bytes);
    __syncwarp();
    if (wanted)
      tma_load_3d(base + half * L::kBlock + box * a.box_rows * 128, &map, half * 64, head,
                  static_cast<int>(row + a.k_row0), keys_there);
    constexpr uint32_t kShape = mma_shape<T>(kRows, false);
    const uint64_t k_operand = smem_operand(base, 16, 1024), q_operand = smem_operand(base + L::kOperand, 16, 1024);
    auto wait = [&](uint32_t b, uint32_t phase) {
      const bool there = mbar_wait_warp(b, phase & 1, &s_gave_up, a.status);
      tmem_fence_after();
      return there;
    };
    const uint32_t tiles = __shfl_sync(~0u, n, 0);
    bool alive = wait(keys_there, 0);
    for (uint32_t i = 0; i < tiles && alive; ++i) {
      alive = wait(queries_there(i), i / 2) && (i < 2 || wait(taken(i), i / 2 - 1));
      if (!alive) break;
      const uint64_t q = q_operand + i % 2 * (L::kOperand / 16);
      if (elect_one()) {
#pragma unroll
        for (int e = 0; e < D / 16; ++e) {
          const uint32_t off = e / 4 * (L::kBlock / 16) + e % 4 * 2;
          mma_ss(tmem + i % 2 * kRows, k_operand + off, q + off, kShape, e > 0);
        }
        mma_commit(scored(i));
      }
      __syncwarp();
    }
    if (!alive) mbar_wait_warp(keys_there, 0, &s_drained, a.status);  // no copy may be in flight at the end
  } else {  // ---- one key and half of a tile's rows for each thread; the queries' copies
    bool alive = true;
    const uint32_t part = threadIdx.x / kKeys, mine = warp * kWarpRows + lane % kWarpRows;  // the row that it looks up
    const int key = key0 + static_cast<int>(threadIdx.x % kKeys);
    // Starts the copies of a tile's queries (this warp: 16 of them, D / 8 lanes to a
    // row, swizzled) and notes what its rows see.
    float of_row;
    int2 sees;
    auto fetch = [&](uint32_t i) {
      if (i < n) {
        constexpr uint32_t kLanes = D / 8;
        const uint32_t row = (tile0 + i) * kRows + mine, t = q_first + row / a.group,
                       h = head * a.group + row % a.group;
        const uint64_t at = t * a.q_token_stride + h * a.q_head_stride;
        const uint32_t first = (tile0 + i) * kRows + warp * kWarpRows;
#pragma unroll
        for (uint32_t k = 0; k < kWarpRows * kLanes / 32; ++k) {
          const uint32_t src = k * (32 / kLanes) + lane / kLanes, c = lane % kLanes, of = warp * kWarpRows + src;
          const bool valid = first + src < rows;
          const uint64_t from = __shfl_sync(~0u, at, src);
          async_copy16(base + (1 + i % 2) * L::kOperand + c / 8 * L::kBlock + of * 128 + ((c % 8 ^ (of & 7)) << 4),
                       a.q + (valid ? from + c * 16 : 0), valid ? 16 : 0);
        }
        of_row = -INFINITY;
        sees = make_int2(-1, 0);
        if (row < rows) {
          sees.x = pos0 + static_cast<int>(row / a.group);
          sees.y = low_of(sees.x);
          of_row = a.lse[static_cast<uint64_t>(t) * a.kv_heads * a.group + h];
        }
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    auto note = [&](uint32_t i) {  // what fetch found, once it is there
      if (i >= n || lane >= kWarpRows) return;
      s_lse[i % 4][mine] = of_row == -INFINITY ? INFINITY : of_row * kLog2e;
      s_sees[i % 4][mine] = sees;
    };
    auto ready = [&](uint32_t i) {  // tile i's copies of this warp are there
      if (i >= n) return;
      proxy_fence_smem();
      mbar_arrive_warp(queries_there(i), lane, alive);
    };
    wait_for_previous();  // the rows' lse
    fetch(0);
    note(0);
    fetch(1);
    note(1);
    asm volatile("cp.async.wait_group 1;" ::: "memory");
    ready(0);
    float2 sum[2] = {};
    for (uint32_t i = 0; i < n; ++i) {
      asm volatile("cp.async.wait_group 0;" ::: "memory");
      ready(i + 1);
      asm volatile("bar.sync 1, 256;" ::: "memory");  // the rows' notes are there, and those of tile i - 2 are read
      alive = alive && mbar_wait_warp(scored(i), i / 2 & 1, &s_gave_up, a.status);
      tmem_fence_after();
      fetch(i + 2);  // in place of tile i, which the product has read
      const uint32_t first = (tile0 + i) * kRows, last = min(first + kRows, rows) - 1;
      const int all_hi = pos0 + static_cast<int>(first / a.group), all_lo = low_of(pos0 + static_cast<int>(last / a.group));
      const bool masked = key0 + kKeys - 1 > all_hi || (key0 < all_lo && key0 + kKeys > sinks) || last != first + kRows - 1;
      const float4* lse = reinterpret_cast<const float4*>(s_lse[i % 4]);
      const float2 c2 = make_float2(a.scale_log2, a.scale_log2);
      auto add_up = [&](auto some_hidden) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const int c = static_cast<int>(part) * (kRows / 2) + half * (kRows / 4);
          uint32_t z[kRows / 4];
          tmem_load32(z, tmem + (warp % 4 * 32 << 16) + i % 2 * kRows + c);
          if (half == 1) {
            tmem_fence_before();
            mbar_arrive_warp(taken(i), lane, alive);
          }
#pragma unroll
          for (int k = 0; k < kRows / 4; k += 4) {
            const float4 x = lse[(c + k) / 4];
            float2 p = fma2(make_float2(__uint_as_float(z[k]), __uint_as_float(z[k + 1])), c2, make_float2(-x.x, -x.y));
            float2 q = fma2(make_float2(__uint_as_float(z[k + 2]), __uint_as_float(z[k + 3])), c2,
                            make_float2(-x.z, -x.w));
            p = make_float2(exp2_approx(p.x), exp2_approx(p.y));
            q = make_float2(exp2_approx(q.x), exp2_approx(q.y));
            if constexpr (decltype(some_hidden)::value) {
              auto see = [&](int of, float v) {
                const int2 row = s_sees[i % 4][c + k + of];
                return key <= row.x && (key >= row.y || key < sinks) ? v : 0.f;
              };
              p = make_float2(see(0, p.x), see(1, p.y));
              q = make_float2(see(2, q.x), see(3, q.y));
            }
            sum[0] = add2(sum[0], p);
            sum[1] = add2(sum[1], q);
          }
        }
      };
      if (masked) add_up(std::true_type{}); else add_up(std::false_type{});
      note(i + 2);
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    const float total = (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
    if (part == 1) s_other[threadIdx.x % kKeys] = total;
    asm volatile("bar.sync 1, 256;" ::: "memory");
    if (part == 0 && key < len && *static_cast<volatile uint32_t*>(&s_gave_up) == 0)
      a.weights[head * a.weights_head_stride + a.page_offsets[s] * a.page_tokens + key] += total + s_other[threadIdx.x];
  }
  tmem_fence_before();
  __syncthreads();
  tmem_fence_after();
  if (warp == kWorkers / 32) tmem_free(tmem, 2 * kRows);
}

template <typename T, int D>
tcx_status launch(const AttnArgs& a, const CUtensorMap& map, uint64_t max_tokens, cudaStream_t stream) {
  using L = WeightLayout<D>;
  static std::atomic<uint64_t> allowed{0};
  if (const tcx_status st = allow_shared(reinterpret_cast<const void*>(weights_kernel<T, D>), L::kBytes, &allowed);
      st != TCX_OK)
    return st;
  const dim3 grid(static_cast<unsigned>((max_tokens + kKeys - 1) / kKeys), a.kv_heads, a.n_seq);
  return launch_after(weights_kernel<T, D>, grid, dim3(kThreads), L::kBytes, stream, map, a);
}

}  // namespace

tcx_status launch_weights(const tcx_kv_attention_args& x, const AttnArgs& a, const CUtensorMap& map,
                          cudaStream_t stream) {
  const uint64_t max_tokens = x.max_pages * x.page_tokens;
  if (max_tokens == 0) return TCX_OK;
  if (x.dtype == TCX_KV_BF16)
    return x.head_dim == 128 ? launch<__nv_bfloat16, 128>(a, map, max_tokens, stream)
                             : launch<__nv_bfloat16, 64>(a, map, max_tokens, stream);
  return x.head_dim == 128 ? launch<__half, 128>(a, map, max_tokens, stream)
                           : launch<__half, 64>(a, map, max_tokens, stream);
}

}  // namespace tcx
