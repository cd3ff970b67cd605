// Launches of kernels that follow one another within a call.
#pragma once
#include "common.h"

// The kernels of one call follow one another closely: a block of the later one may start, and set itself up,
// while the last blocks of the earlier one end, and waits for its results before it touches them.  The earlier
// one's blocks say so at their start: the later one's blocks then come as room falls free.
// The later kernel's lifetime thus begins while the earlier one still writes, so it reads those results by plain
// loads: __ldg is for memory that nobody writes in the kernel's lifetime, and such a load may move above the wait.
// The inputs of the call were complete before its first kernel began: __ldg is right for them in all of them.
__device__ __forceinline__ void next_may_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
template <typename... P, typename... A>
int launch_behind(tx_ctx *ctx, const char *name, void (*kernel)(P...), dim3 grid, unsigned threads, int smem, A... args) {
  cudaLaunchAttribute close{};
  close.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  close.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = ctx->stream;
  cfg.attrs = &close;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, P(args)...);
  if (e == cudaSuccess) return TX_OK;
  cudaGetLastError();  // reported here, not by the next launch too
  return tx_cuda_fail(ctx, e, name);
}
