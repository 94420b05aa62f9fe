// Host-side pieces shared by the translation units of the paged-cache operators: this thread's error text, the launch
// count, the device check and the address of the per-device status word.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "b200_paged.h"

namespace txp {

// What kernels report through the status word (bits, so that several findings of one stretch of work are all kept).
enum PagedStatus : uint32_t {
  kBadPage = 1u,      // a page-table entry outside the cache where a used position needs a page
  kBadRow = 2u,       // a row index outside the table, a row listed twice, or a negative count
  kNoRoomInRow = 4u,  // a position past the width of the page table
  kNoFreePages = 8u,
  kBadLength = 16u,   // a negative length, or in an append more new tokens than cached tokens
  kTimeout = 32u,     // a bounded wait ran out
  kBadOffsets = 64u   // offsets of new tokens that fall or lie outside the tokens
};

int fail(int code, const char *fmt, ...);
void count_launches(int n);
// TXD_OK on an sm_100 device; *status receives the device address of its status word.
int device_ready(uint32_t **status);
// Checks a caller's view of a cache and copies it to *out in normal form.
int check_view(const tx_paged_view *c, tx_paged_view *out);
int shift_of(int page_size);  // log2

#define TXP_CUDA(expr)                                                                            \
  do {                                                                                            \
    cudaError_t e_ = (expr);                                                                      \
    if (e_ != cudaSuccess)                                                                        \
      return txp::fail(TXD_ERR_CUDA, "%s failed: %s", #expr, cudaGetErrorString(e_));             \
  } while (0)

// The programmatic attribute lets a kernel be scheduled while its predecessor drains; every kernel launched with it waits
// for its predecessor (griddepcontrol.wait) before it touches memory.
template <typename... P, typename... A>
cudaError_t launch(void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream, const A &...args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

}  // namespace txp
