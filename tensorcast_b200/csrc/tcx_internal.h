// Internal helpers shared by the libtcx translation units: status/error plumbing
// and CUDA error checks. Not part of the C ABI.
#pragma once

#include <cuda_runtime.h>

#include <atomic>
#include <cstdarg>
#include <cstdint>
#include <cstdio>
#include <string>

#include "../../include/tcx.h"

namespace tcx {

// Records msg as this thread's last error and returns code (TCX_OK clears nothing).
tcx_status set_error(tcx_status code, const std::string& msg);
tcx_status set_errorf(tcx_status code, const char* fmt, ...) __attribute__((format(printf, 2, 3)));
void clear_error();

// Counts kernel launches of this library (tcx_kernel_launch_count).
void note_launches(uint64_t n);

// Kernel launchers shared between translation units (stream-ordered).
// max_ctas: cap on the persistent grid (0: 8 CTAs per SM), for copies that run
// beside other kernels.
tcx_status launch_copy_jobs(const void* d_src, void* d_dst, const tcx_copy_job* d_jobs, uint64_t n_jobs,
                            uint64_t* d_prefix, cudaStream_t stream, uint32_t max_ctas = 0);
int sm_count();
tcx_status launch_permute(const void* d_src, void* d_dst, const tcx_permute_job& pj, cudaStream_t stream);
tcx_status check_permute(const tcx_permute_job& pj);
tcx_status launch_leaf_pass(const void* d_src, uint64_t total, uint64_t leaf, uint32_t n, uint64_t seg_off,
                            uint64_t seg_len, uint32_t* states, void* d_digests, cudaStream_t stream);
// A pass over a slab buffer: bytes [seg_off, seg_off + seg_len) of leaf i (of
// the leaves [0, n) of a stream of `total` bytes cut at `leaf`) are at
// d_src + i * pitch.
tcx_status launch_leaf_pass_pitched(const void* d_src, uint64_t pitch, uint64_t total, uint64_t leaf, uint32_t n,
                                    uint64_t seg_off, uint64_t seg_len, uint32_t* states, void* d_digests,
                                    cudaStream_t stream);
tcx_status launch_merkle(const uint8_t* digests, uint64_t n, uint8_t* scratch, uint8_t* root, cudaStream_t stream);
uint64_t merkle_scratch_bytes(uint64_t n);
tcx_status preload_hash_kernels();
void encode_multihash(const uint8_t digest[32], char out[57]);

inline std::string cuda_msg(cudaError_t e) {
  return std::string(cudaGetErrorName(e)) + ": " + cudaGetErrorString(e);
}

}  // namespace tcx

// Returns TCX_INTERNAL with a message naming the failing call. The runtime's
// per-thread last error is reset (it is reported here), so that a later launch
// check on this thread does not pick up an error of this call, such as a failed
// allocation.
#define TCX_CUDA_TRY(call)                                                                         \
  do {                                                                                             \
    cudaError_t tcx_e_ = (call);                                                                   \
    if (tcx_e_ != cudaSuccess) {                                                                   \
      cudaGetLastError();                                                                          \
      return ::tcx::set_error(TCX_INTERNAL, std::string(#call " failed: ") + ::tcx::cuda_msg(tcx_e_)); \
    }                                                                                              \
  } while (0)

namespace tcx {

// Lets a kernel use `bytes` of dynamic shared memory, once for each device.
inline tcx_status allow_shared(const void* kernel, int bytes, std::atomic<uint64_t>* done) {
  int dev = 0;
  TCX_CUDA_TRY(cudaGetDevice(&dev));
  const uint64_t bit = 1ull << (dev & 63);
  if (dev < 64 && (done->load(std::memory_order_relaxed) & bit)) return TCX_OK;
  TCX_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
  if (dev < 64) done->fetch_or(bit, std::memory_order_relaxed);
  return TCX_OK;
}

// Launches a kernel that waits for the one before it in its own code
// (griddepcontrol.wait, in every thread that uses that one's memory or writes where it
// may still read, and in every CTA before it ends), so that its set-up runs beside that one's end. The first kernel of
// a call is launched without: it follows all earlier work of the stream.
template <typename... Params, typename... Args>
tcx_status launch_after(void (*kernel)(Params...), dim3 grid, dim3 block, size_t shared, cudaStream_t stream,
                        const Args&... args) {
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = shared;
  cfg.stream = stream;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  TCX_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, args...));
  note_launches(1);
  return TCX_OK;
}

}  // namespace tcx
