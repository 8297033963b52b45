// Host side of packed-sequence attention: the two kernels' launchers.
#pragma once
#include "host_common.cuh"
#include "packed_common.cuh"

namespace lbw {

// packed_split.cu: the sequences with at most max_rows query rows per kv head. ws: split_workspace_floats(d) values.
long long split_workspace_floats(int d);
int launch_split(const void* k, long long k_tok, long long k_head, const void* v, long long v_tok, long long v_head,
                 const PackedArgs& a, int d, int dtype, const void* q, long long q_tok, long long q_head,
                 long long max_rows, float* ws, int* st, cudaStream_t s);

}  // namespace lbw
