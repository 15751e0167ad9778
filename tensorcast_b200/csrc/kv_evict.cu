// Eviction from the paged KV pool: the tokens with the highest accumulated
// attention weight of every (sequence, layer, kv head) stay, and their rows are
// copied in their old order to the sequence's destination pages.
//
// One launch, one CTA per (layer, kv head, sequence), or some where those are few: it
// finds the budget's weight by radix selection over the weights' order-preserving
// integer images (11, 11 and 10 bits at a time, the images kept in shared memory),
// writes its share of the kept indices and moves those rows of its head in both planes,
// so that one list's selection runs beside others' copies.
// Bound by HBM: each kept row is read and written once; the places of 512 rows are
// looked up first, so that a thread has eight 16-byte loads under way. The destination
// pages are not the source's: a page may be shared with other sequences, and the copy
// needs no order between its CTAs. Measured on B200: 24 sequences of 500-8192 tokens, 4
// layers, budget 2048, 1.28 GB in 242 us (5.3 TB/s, 0.82 of the measured copy rate;
// 256 us with the copy as a second launch, 329 us with 256 threads in a CTA).
#include <cuda_runtime.h>

#include <algorithm>

#include "tcx_internal.h"

namespace tcx {
namespace {

constexpr int kThreads = 512;
constexpr int kBins = 2048;
constexpr int kBatch = 8;                 // tokens of a thread in a round of the last pass
constexpr uint32_t kHeldTokens = 14336;   // images that shared memory holds: 56 KiB (registers leave two CTAs on an SM)
constexpr int kSelectShared = kHeldTokens * 4;

struct EvictArgs {
  uint8_t* pool;
  uint64_t pool_pages, page_bytes, token_bytes, head_bytes;
  uint32_t page_tokens, kv_heads, n_seq;
  const uint32_t* page_table;
  const uint64_t* page_offsets;
  const uint32_t* seq_tokens;
  const uint32_t* dst_page_table;
  const uint64_t* dst_page_offsets;
  const uint32_t* budgets;
  uint64_t dst_capacity, sinks, recent;
  const float* weights;
  uint64_t weights_layer_stride, weights_head_stride;
  int32_t* keep;
  float* dst_weights;
  uint32_t* dst_tokens;
  uint32_t* status;
};

// Tokens of sequence s and how many of them it keeps, both cut at their pages.
__device__ __forceinline__ void lengths(const EvictArgs& a, uint32_t s, uint32_t* n, uint32_t* kept) {
  const uint64_t cap = (a.page_offsets[s + 1] - a.page_offsets[s]) * a.page_tokens;
  const uint64_t dst_cap = (a.dst_page_offsets[s + 1] - a.dst_page_offsets[s]) * a.page_tokens;
  uint64_t have = a.seq_tokens[s], budget = a.budgets[s];
  if (have > cap) {
    atomicCAS(a.status, 0u, 2u);
    have = cap;
  }
  if (budget > dst_cap) {
    atomicCAS(a.status, 0u, 3u);
    budget = dst_cap;
  }
  *n = static_cast<uint32_t>(have);
  *kept = static_cast<uint32_t>(min(have, budget));
}

// Larger weights have larger images; -0 and 0 have the same, NaN the lowest.
__device__ __forceinline__ uint32_t image(float w) {
  if (w != w) return 0;
  const uint32_t b = __float_as_uint(w + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// Exclusive sum over the CTA of one value per thread; *total gets the sum.
__device__ __forceinline__ uint32_t block_scan(uint32_t v, uint32_t* warp_sums, uint32_t* total) {
  const uint32_t lane = threadIdx.x % 32, warp = threadIdx.x / 32, warps = blockDim.x / 32;
  uint32_t inc = v;
  for (int d = 1; d < 32; d *= 2) {
    const uint32_t up = __shfl_up_sync(~0u, inc, d);
    if (lane >= d) inc += up;
  }
  __syncthreads();
  if (lane == 31) warp_sums[warp] = inc;
  __syncthreads();
  uint32_t before = 0, all = 0;
  for (uint32_t w = 0; w < warps; ++w) {
    if (w < warp) before += warp_sums[w];
    all += warp_sums[w];
  }
  *total = all;
  return before + inc - v;
}

// The indices (in order) and weights of the `kept` of n tokens that stay.
// Those from index r_begin to r_end are written.
__device__ void select_tokens(const EvictArgs& a, const float* w, uint32_t n, uint32_t kept, uint32_t r_begin,
                              uint32_t r_end, int32_t* keep, float* left, uint32_t* held) {
  __shared__ uint32_t bins[kBins], warp_sums[kThreads / 32], s_pick[2];
  // The first `first` and the tokens from `last` on stay; `want` more of those between.
  const uint32_t first = static_cast<uint32_t>(min(a.sinks, static_cast<uint64_t>(kept)));
  const uint32_t newest = static_cast<uint32_t>(min(a.recent, static_cast<uint64_t>(kept - first)));
  const uint32_t last = n - newest;
  uint32_t want = kept - first - newest;
  const bool any = want > 0, hold = n <= kHeldTokens;
  uint32_t prefix = 0;  // the wanted image's upper bits
  for (int pass = 0; any && pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11;
    const uint32_t known = pass == 0 ? 0 : ~0u << (shift + bits);
    for (uint32_t b = threadIdx.x; b < kBins; b += kThreads) bins[b] = 0;
    __syncthreads();
#pragma unroll 4
    for (uint32_t j = first + threadIdx.x; j < last; j += kThreads) {
      const uint32_t x = hold && pass > 0 ? held[j] : image(w[j]);
      if (hold && pass == 0) held[j] = x;
      if ((x & known) == prefix) atomicAdd(&bins[x >> shift & ((1u << bits) - 1)], 1u);
    }
    __syncthreads();
    // thread t: bins 2047 - 4 t down to 2044 - 4 t; how many lie above them
    uint32_t mine[4], all = 0, total;
    for (int k = 0; k < 4; ++k) all += mine[k] = bins[kBins - 1 - 4 * threadIdx.x - k];
    uint32_t above = block_scan(all, warp_sums, &total);
    if (above < want && above + all >= want) {
      int k = 0;
      while (above + mine[k] < want) above += mine[k++];
      s_pick[0] = kBins - 1 - 4 * threadIdx.x - k;
      s_pick[1] = above;
    }
    __syncthreads();
    prefix |= s_pick[0] << shift;
    want -= s_pick[1];
    __syncthreads();
  }
  // `want` of the tokens with exactly this image stay, the lowest indices first. A
  // thread takes consecutive tokens, so that one scan numbers a round of them.
  uint32_t done = 0, equal_done = 0;
  for (uint32_t j0 = 0; j0 < n; j0 += kThreads * kBatch) {
    const uint32_t from = j0 + threadIdx.x * kBatch;
    float v[kBatch];
    uint32_t equal = 0, stays = 0, total;  // bits of the thread's tokens
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const uint32_t j = from + k;
      v[k] = j < n ? w[j] : 0.f;
      const bool middle = j >= first && j < last;
      const uint32_t x = image(v[k]);
      if (any && middle && x == prefix) equal |= 1u << k;
      if ((j < n && !middle) || (any && middle && x > prefix)) stays |= 1u << k;
    }
    // both counts in one sum: at most 512 x 8 each
    const uint32_t before = block_scan(static_cast<uint32_t>(__popc(equal)) << 16 | __popc(stays), warp_sums, &total);
    uint32_t equals = equal_done + (before >> 16);
    uint32_t r = done + (before & 0xffff) + min(equals, want) - min(equal_done, want);
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const bool stay = (stays >> k & 1) || ((equal >> k & 1) && equals < want);
      equals += equal >> k & 1;
      if (stay && r >= r_begin && r < r_end) {
        keep[r] = static_cast<int32_t>(from + k);
        left[r] = v[k];
      }
      r += stay;
    }
    done += (total & 0xffff) + min(equal_done + (total >> 16), want) - min(equal_done, want);
    equal_done += total >> 16;
  }
}

__global__ void __launch_bounds__(kThreads, 2) evict_kernel(EvictArgs a) {
  extern __shared__ uint32_t held[];
  __shared__ uint64_t s_from[kThreads], s_to[kThreads];
  const uint32_t shares = gridDim.x / a.kv_heads, share = blockIdx.x % shares;
  const uint32_t head = blockIdx.x / shares, layer = blockIdx.y, s = blockIdx.z;
  uint32_t n, kept;
  lengths(a, s, &n, &kept);
  const uint64_t base = a.page_offsets[s] * a.page_tokens, dst_base = a.dst_page_offsets[s] * a.page_tokens;
  const uint64_t dst_cap = a.dst_page_offsets[s + 1] * a.page_tokens - dst_base;
  const float* w = a.weights + layer * a.weights_layer_stride + head * a.weights_head_stride + base;
  const uint64_t plane = (static_cast<uint64_t>(layer) * a.kv_heads + head) * a.dst_capacity + dst_base;
  int32_t* keep = a.keep + plane;
  float* left = a.dst_weights + plane;
  const uint32_t r_begin = static_cast<uint32_t>(static_cast<uint64_t>(kept) * share / shares);
  const uint32_t r_end = static_cast<uint32_t>(static_cast<uint64_t>(kept) * (share + 1) / shares);
  if (share == 0) {
    if (layer == 0 && head == 0 && threadIdx.x == 0) a.dst_tokens[s] = kept;
    for (uint64_t r = kept + threadIdx.x; r < dst_cap; r += blockDim.x) {
      keep[r] = -1;
      left[r] = 0.f;
    }
  }
  if (n == kept) {
    for (uint32_t j = r_begin + threadIdx.x; j < r_end; j += blockDim.x) {
      keep[j] = static_cast<int32_t>(j);
      left[j] = w[j];
    }
  } else {
    select_tokens(a, w, n, kept, r_begin, r_end, keep, left, held);
  }
  __syncthreads();
  // The kept rows of this head, 512 at a time.
  constexpr uint64_t kNone = ~uint64_t{0};
  const uint32_t* table = a.page_table + a.page_offsets[s];
  const uint32_t* dst_table = a.dst_page_table + a.dst_page_offsets[s];
  const uint32_t pieces = static_cast<uint32_t>(a.head_bytes / 16);
  for (uint32_t r0 = r_begin; r0 < r_end; r0 += kThreads) {
    const uint32_t r = r0 + threadIdx.x;
    if (r < r_end) {
      const uint32_t j = static_cast<uint32_t>(keep[r]);
      const uint32_t slot = table[j / a.page_tokens], dst_slot = dst_table[r / a.page_tokens];
      const bool good = slot < a.pool_pages && dst_slot < a.pool_pages;
      if (!good) atomicCAS(a.status, 0u, 1u);
      s_from[threadIdx.x] =
          good ? slot * a.page_bytes + j % a.page_tokens * a.token_bytes + head * a.head_bytes : kNone;
      s_to[threadIdx.x] = dst_slot * a.page_bytes + r % a.page_tokens * a.token_bytes + head * a.head_bytes;
    }
    __syncthreads();
    const uint32_t moves = min(r_end - r0, static_cast<uint32_t>(kThreads)) * pieces;
    for (uint32_t plane = 2 * layer; plane < 2 * layer + 2; ++plane) {
      uint8_t* rows = a.pool + plane * a.pool_pages * a.page_bytes;
      for (uint32_t i0 = threadIdx.x; i0 < moves; i0 += 8 * kThreads) {
        uint4 v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const uint32_t i = i0 + k * kThreads;
          if (i < moves && s_from[i / pieces] != kNone)
            v[k] = __ldcs(reinterpret_cast<const uint4*>(rows + s_from[i / pieces]) + i % pieces);
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const uint32_t i = i0 + k * kThreads;
          if (i < moves && s_from[i / pieces] != kNone)
            *(reinterpret_cast<uint4*>(rows + s_to[i / pieces]) + i % pieces) = v[k];
        }
      }
    }
    __syncthreads();
  }
}

}  // namespace
}  // namespace tcx

using namespace tcx;

extern "C" tcx_status tcx_kv_evict(const tcx_kv_evict_args* args, void* stream) {
  if (args == nullptr) return set_error(TCX_INVALID_ARGUMENT, "null arguments");
  const tcx_kv_evict_args& x = *args;
  if (x.n_seq == 0) return TCX_OK;
  if (x.d_pool == nullptr || x.d_page_offsets == nullptr || x.d_seq_tokens == nullptr ||
      x.d_dst_page_offsets == nullptr || x.d_budgets == nullptr || x.d_weights == nullptr ||
      x.d_dst_tokens == nullptr || x.d_status == nullptr)
    return set_error(TCX_INVALID_ARGUMENT, "null device pointer");
  if (x.dst_total_pages != 0 && (x.d_page_table == nullptr || x.d_dst_page_table == nullptr || x.d_keep == nullptr ||
                                 x.d_dst_weights == nullptr))
    return set_error(TCX_INVALID_ARGUMENT, "null device pointer");
  if (x.planes == 0 || x.planes % 2 != 0 || x.pool_pages == 0 || x.page_tokens == 0 || x.kv_heads == 0)
    return set_error(TCX_INVALID_ARGUMENT,
                     "planes must be even, and planes, pool_pages, page_tokens and kv_heads > 0");
  if (x.pool_pages > 0xffffffffull) return set_error(TCX_INVALID_ARGUMENT, "pool_pages exceeds 2^32");
  if (x.head_bytes == 0 || x.head_bytes % 16 != 0 || x.head_bytes > (1u << 20))
    return set_errorf(TCX_INVALID_ARGUMENT, "head_bytes must be a multiple of 16 up to 2^20, got %llu",
                      static_cast<unsigned long long>(x.head_bytes));
  if (x.planes > 65535 || x.kv_heads > 65535 || x.n_seq > 65535 || x.page_tokens > (1u << 20) ||
      x.page_tokens * x.kv_heads * (x.head_bytes / 16) > 0x7fffffffull)
    return set_error(TCX_INVALID_ARGUMENT, "planes, kv_heads, n_seq (65535) or page size out of range");
  if (x.dst_total_pages > 0x7fffffffull / x.page_tokens)
    return set_error(TCX_INVALID_ARGUMENT, "destination pages hold 2^31 tokens or more");
  if (reinterpret_cast<uintptr_t>(x.d_pool) & 15u) return set_error(TCX_INVALID_ARGUMENT, "pool must be 16-byte aligned");
  EvictArgs a{};
  a.pool = static_cast<uint8_t*>(x.d_pool);
  a.pool_pages = x.pool_pages;
  a.head_bytes = x.head_bytes;
  a.token_bytes = x.kv_heads * x.head_bytes;
  a.page_bytes = x.page_tokens * a.token_bytes;
  a.page_tokens = static_cast<uint32_t>(x.page_tokens);
  a.kv_heads = static_cast<uint32_t>(x.kv_heads);
  a.n_seq = static_cast<uint32_t>(x.n_seq);
  a.page_table = x.d_page_table;
  a.page_offsets = x.d_page_offsets;
  a.seq_tokens = x.d_seq_tokens;
  a.dst_page_table = x.d_dst_page_table;
  a.dst_page_offsets = x.d_dst_page_offsets;
  a.budgets = x.d_budgets;
  a.dst_capacity = x.dst_total_pages * x.page_tokens;
  a.sinks = x.sinks;
  a.recent = x.recent;
  a.weights = x.d_weights;
  a.weights_layer_stride = x.weights_layer_stride;
  a.weights_head_stride = x.weights_head_stride;
  a.keep = x.d_keep;
  a.dst_weights = x.d_dst_weights;
  a.dst_tokens = x.d_dst_tokens;
  a.status = x.d_status;
  static std::atomic<uint64_t> allowed{0};
  if (const tcx_status st = allow_shared(reinterpret_cast<const void*>(evict_kernel), kSelectShared, &allowed); st != TCX_OK)
    return st;
  // Few lists: several CTAs select the same one, and each moves a share of its rows.
  const uint64_t lists = static_cast<uint64_t>(a.kv_heads) * (x.planes / 2) * a.n_seq;
  const uint64_t shares = std::max<uint64_t>(1, std::min<uint64_t>(16, 2ull * sm_count() / lists));
  const dim3 grid(static_cast<unsigned>(a.kv_heads * shares), static_cast<unsigned>(x.planes / 2), a.n_seq);
  evict_kernel<<<grid, kThreads, kSelectShared, static_cast<cudaStream_t>(stream)>>>(a);
  note_launches(1);
  TCX_CUDA_TRY(cudaGetLastError());
  return TCX_OK;
}
