// What the kernels of packed-sequence attention share: the description of a call, the lookup of a sequence in the
// device arrays of starts and lengths, and the rounding of probabilities and outputs to the tensors' type.
#pragma once
#include <cuda_fp16.h>
#include <math.h>

#include "lbw_common.cuh"

namespace lbw {

// Programmatic dependent launch between the kernels of one call: pdl_trigger lets the next kernel's blocks start as SMs
// become free, pdl_wait holds a block until the kernels before it have finished and their writes are visible. Every
// kernel that is launched this way waits before it ends, so what follows the call waits for all of them.
LBW_DEV void pdl_trigger() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
LBW_DEV void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// mbar_wait with the waiting itself in one function for all sites: inlined, the loops and their error paths are a third
// of the code of a kernel that has to stay in the instruction cache.
static __device__ __noinline__ bool mbar_wait_long(uint32_t bar, uint32_t parity, int* status, volatile int* flag, int site) {
  const long long t0 = clock64();
  while (!mbar_test(bar, parity)) {
    if (*flag) return false;
    if (clock64() - t0 > LBW_WAIT_CYCLES) {
      *flag = 1;
      if (status) atomicCAS(status, 0, LBW_DEV_TIMEOUT | site);
      return false;
    }
  }
  return true;
}
LBW_DEV bool mbar_wait_c(uint64_t* bar, uint32_t parity, const Abort& ab, int site) {
  const uint32_t a = smem_u32(bar);
  return mbar_test(a, parity) || mbar_wait_long(a, parity, ab.status, ab.flag, site);
}

struct PackedArgs {
  const int* cu_q;    // [n_seqs + 1] first query row of each sequence
  const int* cu_k;    // [n_seqs + 1] first key row
  const int* k_lens;  // [n_seqs] keys in use, or null: all of the sequence's rows
  int n_seqs;
  int tq, tk;         // rows of q and of k / v: every start and length is clamped to them
  int hq, hk, group;  // heads; group = hq / hk query heads share a kv head
  int causal;
  float scale_log2;
  void* out;
  long long os_tok, os_head;
};

struct PackedSeq {
  int q0, nq, k0, nk;
};

// Sequence b of the call. The arrays live on the device, so nothing on the host has checked them: a start or length
// that does not fit the tensors is cut to what does.
LBW_DEV PackedSeq packed_seq(const PackedArgs& a, int b) {
  PackedSeq s;
  s.q0 = min(max(a.cu_q[b], 0), a.tq);
  s.nq = min(max(a.cu_q[b + 1], s.q0), a.tq) - s.q0;
  s.k0 = min(max(a.cu_k[b], 0), a.tk);
  s.nk = min(max(a.cu_k[b + 1], s.k0), a.tk) - s.k0;
  if (a.k_lens) s.nk = min(max(a.k_lens[b], 0), s.nk);
  return s;
}

// Number of keys that query i of the sequence sees.
LBW_DEV int packed_visible(const PackedArgs& a, const PackedSeq& s, int i) {
  if (!a.causal) return s.nk;
  const int n = i + 1 + s.nk - s.nq;
  return n < 0 ? 0 : (n < s.nk ? n : s.nk);
}

// The whole block of NT threads: an item of a list in which sequence b has n.x items (SEARCH_Y: n.y) of (n.x, n.y) =
// count(b); which(sum of all n.y) says which item. Returns its sequence, its index in it, the sum of n.y before the
// sequence and that over all; seq = -1 past the end. Each thread counts a run of neighbouring sequences, and one thread's
// reading of the found sequence is what all get. `tmp`: NT / 32 entries of shared memory.
struct PackedAt {
  int seq;
  PackedSeq sq;
  long long local, before_y, total_y;
};

template <int NT, bool SEARCH_Y, typename F, typename W>
LBW_DEV PackedAt packed_locate(const PackedArgs& a, F count, W which, longlong2* tmp, PackedAt* at) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int per = (a.n_seqs + NT - 1) / NT;
  const int b0 = (int)min((long long)threadIdx.x * per, (long long)a.n_seqs), b1 = min(b0 + per, a.n_seqs);
  long long x = 0, y = 0;  // (x only for a search by n.x)
  for (int b = b0; b < b1; ++b) {
    const longlong2 n = count(b);
    if constexpr (!SEARCH_Y) x += n.x;
    y += n.y;
  }
  long long sx = x, sy = y;  // inclusive over the warp
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long vx = SEARCH_Y ? 0 : __shfl_up_sync(0xffffffffu, sx, o), vy = __shfl_up_sync(0xffffffffu, sy, o);
    if (lane >= o) {
      sx += vx;
      sy += vy;
    }
  }
  if (lane == 31) tmp[warp] = make_longlong2(sx, sy);
  if (threadIdx.x == 0) at->seq = -1;
  __syncthreads();
  long long ty = 0;
  sx -= x;
  sy -= y;
#pragma unroll
  for (int i = 0; i < NT / 32; ++i) {
    const longlong2 v = tmp[i];
    if (i < warp) {
      sx += v.x;
      sy += v.y;
    }
    ty += v.y;
  }
  const long long w = which(ty);
  long long from = SEARCH_Y ? sy : sx;
  if (w >= from && w < from + (SEARCH_Y ? y : x)) {
    for (int b = b0; b < b1; ++b) {
      const longlong2 n = count(b);
      const long long own = SEARCH_Y ? n.y : n.x;
      if (w < from + own) {
        at->seq = b;
        at->sq = packed_seq(a, b);
        at->local = w - from;
        at->before_y = sy;
        break;
      }
      from += own;
      sy += n.y;
    }
  }
  __syncthreads();
  PackedAt r = *at;
  r.total_y = ty;
  return r;
}

template <bool F16>
LBW_DEV uint32_t pack_16(float lo, float hi) {
  if constexpr (F16) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  } else {
    return pack_bf16(lo, hi);
  }
}

// The low 16 bits as a value.
template <bool F16>
LBW_DEV float unpack_16(uint32_t x) {
  if constexpr (F16)
    return __half2float(__ushort_as_half((unsigned short)x));
  else
    return __uint_as_float(x << 16);
}

}  // namespace lbw
