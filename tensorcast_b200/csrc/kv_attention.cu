// Attention of each sequence's newest tokens over its pages of the KV pool.
//
// Query i of a sequence stands at position p and sees the tokens of
//   [0, min(sinks, p + 1))  and  (p - window, p]        (all of [0, p] without a window),
// counted from the start of the shared prefix where there is one. A row of the
// computation is one query token of one q head.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cmath>

#include "kv_attention.cuh"

namespace tcx {
namespace {

tcx_status check_sizes(const tcx_kv_attention_args& a) {
  if (a.planes == 0 || a.pool_pages == 0 || a.page_tokens == 0 || a.kv_heads == 0 || a.q_heads == 0)
    return set_error(TCX_INVALID_ARGUMENT, "planes, pool_pages, page_tokens, kv_heads and q_heads must be > 0");
  if (a.page_tokens % 8 != 0 || a.page_tokens > (1u << 20))
    return set_errorf(TCX_INVALID_ARGUMENT, "page_tokens must be a multiple of 8 up to 2^20, got %llu",
                      static_cast<unsigned long long>(a.page_tokens));
  if (a.head_dim != 64 && a.head_dim != 128)
    return set_errorf(TCX_INVALID_ARGUMENT, "head_dim must be 64 or 128, got %llu",
                      static_cast<unsigned long long>(a.head_dim));
  if (a.dtype != TCX_KV_BF16 && a.dtype != TCX_KV_FP16) return set_error(TCX_INVALID_ARGUMENT, "unknown dtype");
  if (a.kv_heads > 1024 || a.q_heads > 65536 || a.q_heads % a.kv_heads != 0)
    return set_errorf(TCX_INVALID_ARGUMENT, "q_heads (%llu) must be a multiple of kv_heads (%llu, at most 1024)",
                      static_cast<unsigned long long>(a.q_heads), static_cast<unsigned long long>(a.kv_heads));
  if (a.k_plane >= a.planes || a.v_plane >= a.planes)
    return set_error(TCX_INVALID_ARGUMENT, "k_plane and v_plane must be planes of the pool");
  if (a.pool_pages > 0x7fffffffull || a.planes > 0x7fffffffull ||
      a.pool_pages * a.page_tokens > 0x7fffffffull / a.planes)
    return set_error(TCX_INVALID_ARGUMENT, "the pool's planes hold 2^31 token rows or more");
  if (a.n_seq > 65535) return set_error(TCX_INVALID_ARGUMENT, "more than 65535 sequences");
  if (a.q_tokens > 0x7fffffffull / a.q_heads) return set_error(TCX_INVALID_ARGUMENT, "2^31 query rows or more");
  if (a.max_q > a.q_tokens || a.total_pages > 0x7fffffffull || a.max_pages > a.total_pages ||
      a.max_pages > 0x3fffffffull / a.page_tokens || a.prefix_pages > 0x3fffffffull / a.page_tokens)
    return set_error(TCX_INVALID_ARGUMENT, "inconsistent size bounds");
  if (a.window > 0x3fffffffull || a.sinks > 0x3fffffffull)
    return set_error(TCX_INVALID_ARGUMENT, "window and sinks must be below 2^30");
  if (!(a.scale > 0) || !(a.scale * 1.4426950408889634 <= 3e38) || !(static_cast<float>(a.scale * kLog2e) > 0))
    return set_error(TCX_INVALID_ARGUMENT, "scale must be > 0 and finite");
  return TCX_OK;
}

tcx_status check(const tcx_kv_attention_args& a) {
  if (a.d_pool == nullptr || a.d_page_offsets == nullptr || a.d_seq_tokens == nullptr ||
      a.d_q_offsets == nullptr || a.d_q == nullptr || a.d_out == nullptr || a.d_lse == nullptr || a.d_status == nullptr ||
      a.d_counters == nullptr)
    return set_error(TCX_INVALID_ARGUMENT, "null device pointer");
  if (a.d_page_table == nullptr && a.total_pages != 0) return set_error(TCX_INVALID_ARGUMENT, "null device pointer");
  if (const tcx_status st = check_sizes(a); st != TCX_OK) return st;
  if ((reinterpret_cast<uintptr_t>(a.d_pool) | reinterpret_cast<uintptr_t>(a.d_q) |
       reinterpret_cast<uintptr_t>(a.d_out)) & 15u)
    return set_error(TCX_INVALID_ARGUMENT, "pool, q and out must be 16-byte aligned");
  if ((a.q_token_stride | a.q_head_stride | a.out_token_stride | a.out_head_stride) % 8 != 0)
    return set_error(TCX_INVALID_ARGUMENT, "strides of q and out must be multiples of 8 elements");
  if (a.d_prefix_table != nullptr) {
    if (a.d_prefix_tokens == nullptr) return set_error(TCX_INVALID_ARGUMENT, "null device pointer");
    if (a.d_weights != nullptr)
      return set_error(TCX_INVALID_ARGUMENT, "weights are not accumulated with a shared prefix");
  }
  return TCX_OK;
}

// The rows' parts over a shared prefix.
uint64_t prior_bytes(const tcx_kv_attention_args& x) {
  return align256(x.q_tokens * x.q_heads * (x.head_dim + 1) * sizeof(float));
}

AttnArgs device_args(const tcx_kv_attention_args& x) {
  AttnArgs a{};
  a.pool = static_cast<const uint8_t*>(x.d_pool);
  a.pool_pages = x.pool_pages;
  a.row_bytes = x.head_dim * 2;
  a.token_bytes = x.kv_heads * a.row_bytes;
  a.page_tokens = static_cast<uint32_t>(x.page_tokens);
  a.kv_heads = static_cast<uint32_t>(x.kv_heads);
  a.group = static_cast<uint32_t>(x.q_heads / x.kv_heads);
  a.page_table = x.d_page_table;
  a.page_offsets = x.d_page_offsets;
  a.seq_tokens = x.d_seq_tokens;
  a.q_offsets = x.d_q_offsets;
  a.n_seq = static_cast<uint32_t>(x.n_seq);
  a.q_tokens = static_cast<uint32_t>(x.q_tokens);
  a.prefix_table = x.d_prefix_table;
  a.prefix_tokens = x.d_prefix_tokens;
  a.prefix_pages = x.prefix_pages;
  a.window = static_cast<int64_t>(x.window);
  a.sinks = static_cast<int64_t>(x.sinks);
  a.scale_log2 = static_cast<float>(x.scale * 1.4426950408889634);
  a.q = static_cast<const uint8_t*>(x.d_q);
  a.out = static_cast<uint8_t*>(x.d_out);
  a.q_token_stride = x.q_token_stride * 2;
  a.q_head_stride = x.q_head_stride * 2;
  a.out_token_stride = x.out_token_stride * 2;
  a.out_head_stride = x.out_head_stride * 2;
  a.lse = x.d_lse;
  a.weights = x.d_weights;
  a.weights_head_stride = x.weights_head_stride;
  a.status = x.d_status;
  a.counters = x.d_counters;
  a.box_rows = std::min<uint32_t>(64, a.page_tokens & -a.page_tokens);
  a.k_row0 = x.k_plane * x.pool_pages * x.page_tokens;
  a.v_row0 = x.v_plane * x.pool_pages * x.page_tokens;
  return a;
}

}  // namespace

tcx_status encode_pool_map(const tcx_kv_attention_args& x, uint32_t box_rows, CUtensorMap* map) {
  using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                              const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                              CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
  static std::atomic<void*> entry{nullptr};
  void* f = entry.load(std::memory_order_relaxed);
  if (f == nullptr) {
    cudaDriverEntryPointQueryResult found;
    TCX_CUDA_TRY(cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &found));
    if (found != cudaDriverEntryPointSuccess || f == nullptr)
      return set_error(TCX_INTERNAL, "the driver has no cuTensorMapEncodeTiled");
    entry.store(f, std::memory_order_relaxed);
  }
  const cuuint64_t dims[3] = {x.head_dim, x.kv_heads, x.planes * x.pool_pages * x.page_tokens};
  const cuuint64_t strides[2] = {x.head_dim * 2, x.head_dim * 2 * x.kv_heads};
  const cuuint32_t box[3] = {64, 1, box_rows}, ones[3] = {1, 1, 1};
  const CUresult rc = reinterpret_cast<Encode>(f)(
      map, CU_TENSOR_MAP_DATA_TYPE_UINT16, 3, const_cast<void*>(x.d_pool), dims, strides, box, ones,
      CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
      CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (rc != CUDA_SUCCESS) return set_errorf(TCX_INTERNAL, "cuTensorMapEncodeTiled failed: %d", static_cast<int>(rc));
  return TCX_OK;
}

}  // namespace tcx

using namespace tcx;

extern "C" uint64_t tcx_kv_attention_scratch_bytes(const tcx_kv_attention_args* args) {
  if (args == nullptr || args->n_seq == 0 || args->q_tokens == 0 || check_sizes(*args) != TCX_OK) return 0;
  uint64_t own = decode_fits(*args) ? decode_scratch_bytes(*args) : tile_scratch_bytes(*args, false);
  if (args->d_prefix_table != nullptr) own += tile_scratch_bytes(*args, true) + prior_bytes(*args);
  return own;
}

extern "C" tcx_status tcx_kv_attention(const tcx_kv_attention_args* args, void* d_scratch, uint64_t scratch_bytes,
                                       void* stream) {
  if (args == nullptr) return set_error(TCX_INVALID_ARGUMENT, "null arguments");
  if (args->n_seq == 0 || args->q_tokens == 0) return TCX_OK;
  if (const tcx_status st = check(*args); st != TCX_OK) return st;
  const uint64_t need = tcx_kv_attention_scratch_bytes(args);
  if (scratch_bytes < need || d_scratch == nullptr || (reinterpret_cast<uintptr_t>(d_scratch) & 255u))
    return set_errorf(TCX_INVALID_ARGUMENT, "scratch of %llu bytes, 256-byte aligned, needed (got %llu)",
                      static_cast<unsigned long long>(need), static_cast<unsigned long long>(scratch_bytes));
  AttnArgs a = device_args(*args);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  CUtensorMap map;
  if (const tcx_status st = encode_pool_map(*args, a.box_rows, &map); st != TCX_OK) return st;
  uint8_t* scratch = static_cast<uint8_t*>(d_scratch);
  if (args->d_prefix_table != nullptr) {
    a.part_o = reinterpret_cast<float*>(scratch);
    a.part_lse = a.part_o + args->q_tokens * args->q_heads * args->head_dim;
    scratch += prior_bytes(*args);
    if (const tcx_status st = launch_tile(*args, a, map, true, scratch, s); st != TCX_OK) return st;
    scratch += tile_scratch_bytes(*args, true);
    a.prior_o = a.part_o;
    a.prior_lse = a.part_lse;
    a.part_o = a.part_lse = nullptr;
  }
  if (const tcx_status st = decode_fits(*args) ? launch_decode(*args, a, map, scratch, s)
                                               : launch_tile(*args, a, map, false, scratch, s);
      st != TCX_OK)
    return st;
  if (args->d_weights == nullptr || decode_fits(*args)) return TCX_OK;
  return launch_weights(*args, a, map, s);
}
