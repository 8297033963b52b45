// Host side of packed-sequence attention: the two kernels' launchers.
#pragma once
#include "host_common.cuh"
#include "packed_common.cuh"

namespace lbw {

// A launch that may start while the kernel before it in the stream is finishing (see pdl_wait).
template <typename... P, typename... A>
inline int launch_dependent(const char* what, void (*kernel)(P...), dim3 grid, int threads, int smem, cudaStream_t s,
                            A&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute at;
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  return cuda_check(cudaLaunchKernelEx(&cfg, kernel, P(args)...), what);
}

// packed_split.cu: the sequences with at most max_rows query rows per kv head. ws: split_workspace_floats(d) values.
// after: other kernels of the same call come before it.
long long split_workspace_floats(int d);
int launch_split(const void* k, long long k_tok, long long k_head, const void* v, long long v_tok, long long v_head,
                 const PackedArgs& a, int d, int dtype, const void* q, long long q_tok, long long q_head,
                 long long max_rows, bool after, float* ws, int* st, cudaStream_t s);

}  // namespace lbw
