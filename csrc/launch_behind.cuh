// Launches that overlap with the end of the kernel before them in the stream: blocks take their places on the GPU while that
// kernel runs out and wait there until all of it is done and visible. Saves about 2 us between two kernels, in a graph too:
// attention over 512 rows of 768 4-bit tokens in a row 30.9 -> 28.8 us, over one row of 333 8.3 -> 5.7. No kernel lets the next
// one's blocks come before its own have ended: they land where room is, not evenly (4 rows of 30000 tokens 35.7 -> 37.0 us when
// the attention kernel does so for the kernel that joins its parts, 33 rows of 700 7.5 -> 10.5 when it does for the next call).
#pragma once

#include "host_common.h"

namespace icb {

// First in such a kernel, by every thread of every block before it touches memory: what follows the kernel relies on the kernels
// before it having ended.
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

template <typename... P, typename... A>
inline int launch_behind(const char* name, void (*kernel)(P...), dim3 grid, int threads, size_t smem, cudaStream_t st,
                         const A&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args...);
  if (e != cudaSuccess) {
    cudaGetLastError();
    fprintf(stderr, "[ironcore_b200] %s: %s\n", name, cudaGetErrorString(e));
    return -(int)e;
  }
  return 0;
}

}  // namespace icb
