// Arguments and lookups shared by the attention kernels over the paged KV pool.
#pragma once

#include "sm100.cuh"
#include "tcx_internal.h"

namespace tcx {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr uint32_t kBadSlot = 1, kBadLength = 2;

struct AttnArgs {
  const uint8_t* pool;
  uint64_t pool_pages, page_bytes, token_bytes, row_bytes;  // row: one head of one token
  uint32_t page_tokens, kv_heads, group;
  uint64_t k_plane, v_plane;
  const uint32_t* page_table;
  const uint64_t* page_offsets;
  const uint32_t* seq_tokens;
  const uint32_t* q_offsets;
  uint32_t n_seq, q_tokens;
  const uint32_t* prefix_table;
  const uint32_t* prefix_tokens;
  uint64_t prefix_pages;
  int64_t window, sinks;
  float scale_log2;  // scale * log2(e): exponents are powers of two
  const uint8_t* q;
  uint8_t* out;
  uint64_t q_token_stride, q_head_stride, out_token_stride, out_head_stride;  // bytes
  float* lse;
  float* weights;
  uint64_t weights_head_stride;
  uint32_t* status;
  uint32_t box_rows;  // token rows of one TMA box: divides page_tokens and 64
  uint64_t k_row0, v_row0;  // first token row of the planes in the pool's map
};

// Tokens of sequence s, cut at its pages' capacity.
__device__ __forceinline__ uint32_t seq_length(const AttnArgs& a, uint32_t s) {
  const uint64_t cap = (a.page_offsets[s + 1] - a.page_offsets[s]) * a.page_tokens;
  const uint32_t n = a.seq_tokens[s];
  if (n > cap) {
    atomicCAS(a.status, 0u, kBadLength);
    return static_cast<uint32_t>(cap);
  }
  return n;
}

__device__ __forceinline__ uint32_t prefix_length(const AttnArgs& a) {
  if (a.prefix_table == nullptr) return 0;
  const uint64_t cap = a.prefix_pages * a.page_tokens;
  const uint32_t n = *a.prefix_tokens;
  if (n > cap) {
    atomicCAS(a.status, 0u, kBadLength);
    return static_cast<uint32_t>(cap);
  }
  return n;
}

// The sequence of query token t: q_offsets[s] <= t < q_offsets[s + 1].
__device__ __forceinline__ uint32_t seq_of(const AttnArgs& a, uint32_t t) {
  uint32_t lo = 0, hi = a.n_seq;
  while (hi - lo > 1) {
    const uint32_t mid = (lo + hi) / 2;
    if (a.q_offsets[mid] <= t) lo = mid; else hi = mid;
  }
  return lo;
}

__device__ __forceinline__ uint64_t checked_slot(const AttnArgs& a, const uint32_t* table, uint64_t page) {
  const uint32_t slot = table[page];
  if (slot < a.pool_pages) return slot;
  atomicCAS(a.status, 0u, kBadSlot);
  return 0;
}

// The pool as a tensor of [planes x slots x page tokens][kv heads][head_dim] 16-bit
// values, read in boxes of `box_rows` token rows of 64 values of one head.
tcx_status encode_pool_map(const tcx_kv_attention_args& x, uint32_t box_rows, CUtensorMap* map);

// Decode: few rows for each sequence and kv head (kv_decode.cu).
constexpr uint32_t kDecodeRows = 16;
bool decode_fits(const tcx_kv_attention_args& x);
uint64_t decode_scratch_bytes(const tcx_kv_attention_args& x);
tcx_status launch_decode(const tcx_kv_attention_args& x, const AttnArgs& a, const CUtensorMap& map, void* scratch,
                         cudaStream_t stream);

}  // namespace tcx
