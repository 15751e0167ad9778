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
  uint64_t pool_pages, token_bytes, row_bytes;  // row: one head of one token
  uint32_t page_tokens, kv_heads, group;
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
  uint32_t* counters;  // TCX_KV_COUNTERS, all 0 between launches
  // Where there is a shared prefix: the rows' parts over it (o normalised, lse in
  // powers of two, [q token][q head]) are written to `part` and then read as `prior`.
  float *part_o, *part_lse;
  const float *prior_o, *prior_lse;
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

// A finished row: o = sum of 2^(z - m) v and l = sum of 2^(z - m) become
//   o * own + prior_o * prior,  lse (in powers of two)
// A part that the row sees counts even where its weight has become 0, so that infinities
// and NaN show; one that it does not see is 0, whatever the sums hold.
struct Finish {
  float own, prior, lse;
  bool sees_own, sees_prior;
};

__device__ __forceinline__ Finish finish_row(const AttnArgs& a, uint64_t row, float m, float l) {
  Finish f;
  f.sees_own = l != 0.f;
  f.sees_prior = false;
  f.own = f.sees_own ? 1.f / l : 0.f;
  f.prior = 0.f;
  f.lse = m + log2f(l);  // l 0: m is -inf, and so is this
  if (a.prior_lse != nullptr) {
    const float p = a.prior_lse[row];
    const float top = fmaxf(f.lse, p), ref = top == -INFINITY ? 0.f : top;
    const float w = exp2f(f.lse - ref), wp = exp2f(p - ref), sum = w + wp;
    f.own = w == 0.f ? 0.f : f.own * w / sum;
    f.prior = wp == 0.f ? 0.f : wp / sum;
    f.sees_prior = p != -INFINITY;
    f.lse = top + log2f(sum);
  }
  return f;
}

// Four values of a finished row, from column e on.
template <typename T, int D>
__device__ __forceinline__ void store_row(const AttnArgs& a, uint32_t t, uint32_t h, uint32_t e, const Finish& f,
                                          const float (&v)[4]) {
  const uint64_t row = static_cast<uint64_t>(t) * a.kv_heads * a.group + h;
  float x[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = f.sees_own ? v[i] * f.own : 0.f;
  if (f.sees_prior) {
    const float4 y = *reinterpret_cast<const float4*>(a.prior_o + row * D + e);
    x[0] += f.prior * y.x;
    x[1] += f.prior * y.y;
    x[2] += f.prior * y.z;
    x[3] += f.prior * y.w;
  }
  if (a.part_o != nullptr) {
    *reinterpret_cast<float4*>(a.part_o + row * D + e) = make_float4(x[0], x[1], x[2], x[3]);
    return;
  }
  uint8_t* out = a.out + t * a.out_token_stride + h * a.out_head_stride + e * 2;
  *reinterpret_cast<uint2*>(out) = make_uint2(pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3]));
}

__device__ __forceinline__ void store_lse(const AttnArgs& a, uint32_t t, uint32_t h, const Finish& f) {
  const uint64_t row = static_cast<uint64_t>(t) * a.kv_heads * a.group + h;
  if (a.part_o != nullptr) a.part_lse[row] = f.lse; else a.lse[row] = kLn2 * f.lse;
}

// A row's probabilities are 2^(z - m), rounded to T for the product with the values,
// with a reference m that follows the largest score `top` of the tiles. bf16 has the
// range of 32 bits: m rises only. fp16 holds 2^-14 to 2^15 to the last bit (from 2^-25 on
// with fewer), and behind a strong first token all others can lie below that while
// they make up the output: there m leaves a tile's largest score between 2^-1 and 2^15,
// moves to where it is 2^11, and goes down as well, up to 40 below its highest, so that
// sums in 32 bits hold what came before. Measured against 64 bits, 40000 tokens 17 to
// 19 below the first in score, whose value is 0: off by 3e-4 of the largest output (its
// own rounding) at one query and at 40; with a reference that only rises by 1.2e-3 to
// 7.4e-3.
constexpr float kHalfTop = 15.f, kHalfSet = 11.f, kHalfLow = -1.f, kHalfDepth = 40.f;

// The reference after a tile whose largest score is `top`; `down`: it may go down.
__device__ __forceinline__ float half_reference(float m, float top, float peak, bool down) {
  if (top > m + kHalfTop) return top - kHalfSet;
  if (down && top < m + kHalfLow && top > -INFINITY) return fminf(m, fmaxf(top - kHalfSet, peak - kHalfDepth));
  return m;
}

// The last of `parts` CTAs to come here, all of whose writes the others' precede;
// it leaves the counter at 0 for the next call.
__device__ __forceinline__ bool last_to_arrive(uint32_t* counter, uint32_t parts) {
  __threadfence();
  const bool last = atomicAdd(counter, 1u) + 1 == parts;
  if (last) {
    *counter = 0;
    __threadfence();
  }
  return last;
}

inline uint64_t align256(uint64_t n) { return (n + 255) / 256 * 256; }

// The pool as a tensor of [planes x slots x page tokens][kv heads][head_dim] 16-bit
// values, read in boxes of `box_rows` token rows of 64 values of one head.
tcx_status encode_pool_map(const tcx_kv_attention_args& x, uint32_t box_rows, CUtensorMap* map);

// Decode: few rows for each sequence and kv head (kv_decode.cu).
constexpr uint32_t kDecodeRows = 32;
bool decode_fits(const tcx_kv_attention_args& x);
uint64_t decode_scratch_bytes(const tcx_kv_attention_args& x);
tcx_status launch_decode(const tcx_kv_attention_args& x, const AttnArgs& a, const CUtensorMap& map, void* scratch,
                         cudaStream_t stream);

// Many rows: prompts, and the shared prefix of a batch (kv_tile.cu). With
// `prefix` the rows of all sequences attend over the prefix.
uint64_t tile_scratch_bytes(const tcx_kv_attention_args& x, bool prefix);
tcx_status launch_tile(const tcx_kv_attention_args& x, const AttnArgs& a, const CUtensorMap& map, bool prefix,
                       void* scratch, cudaStream_t stream);

// Adds every token's softmax weights of many rows, whose lse is known (kv_weights.cu).
tcx_status launch_weights(const tcx_kv_attention_args& x, const AttnArgs& a, const CUtensorMap& map,
                          cudaStream_t stream);

}  // namespace tcx
