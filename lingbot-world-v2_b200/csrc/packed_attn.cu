// Attention over packed sequences on tcgen05: softmax(scale * Q K^T) V for every sequence of a batch, causal or not,
// with grouped heads, the sequences' starts and lengths read from device memory (lbw_packed_attention).
//
// Online softmax over 128-key tiles, fp32 scores, maxima, sums and accumulators; the probabilities are rounded once to
// the tensors' 16-bit type for the second product (off by 2^-8 or 2^-11 of themselves at most, in fp16 by 2^-25 where they are
// below 2^-14; the row's largest is 1 or more), while their sum takes them unrounded.
//
// A CTA has up to two tiles of 128 query rows of one kv head. A row is a (token, query head) pair: `pack` query heads of
// the kv head's group sit side by side in a tile (row = token * pack + head), so that a tile of a short sequence is
// filled by the group's heads. The two tiles are neighbours in the sequence; the "primary" is the later one, whose rows
// see at least as many keys, and the secondary stops at its own last visible key tile.
//   warps 0-7 / 8-15 softmax of the primary / secondary tile, two threads per row (= TMEM lane): warps 0-3 and 8-11 have
//                    the first 64 keys of a tile, 4-7 and 12-15 the others
//   warp 16          TMA producer: Q once, then K and V tiles through a 2-deep ring
//   warp 17          UMMA issuer, TMEM owner (S0 | S1 | O0 | O1)
//   warp 19          scheduler: the CTA stays for many windows; while it works on one, this warp takes the next from the
//                    blocks of the grid that have not started (cluster launch control) and works out its rows and keys,
//                    so that the next Q, K and S are under way before the last rows of the present window are written
//   warp 18          watches the K/V ring for the issuer (its arrival folds "V(j) and K(j + 1) landed" into the barrier that
//                    announces the primary's P) and clears the value rows past the sequence's last key: they belong to
//                    another sequence or to nobody, and 0 * NaN would reach the sum. On the diagonal it looks for values
//                    that are not finite, which rows may not see: they are taken out of the tile and noted, and the
//                    epilogue adds them to the rows that do see them
// P is written over S in TMEM, so a tile's chain is softmax, P V, next S; the two tiles take turns at the tensor pipe. The
// running maximum moves only when it grows by more than 2^8.
// What it measured (B200, D = 128, non-causal, cycles of one step = both tiles against 128 keys, 2,048 of them MMA at
// full rate): 3,600, with the exponentials left out 3,600, with one tile's chain shortened by a third 3,500, with S or P V
// left out 2,550, with all MMAs left out 1,470: the MMAs of a tile and the hand-overs around them (commit, softmax warps,
// arrival, issuer: ~600 cycles without any work in between) follow each other, and the exponentials hide behind the other
// tile. Tried and slower: exponentials on the FMA pipe (1/8 to 1/2 of them, +1 to +5%), an issuer per tile (+4 to +20%),
// one thread per row and two P releases (+10%), P beside S for D = 64 (-8% for long sequences, +10% for short ones), the
// maximum of the tile before as m (+5%), rolled MMA loops (+8%), waits of one lane (+17%) or with a suspend hint (+7%).
// Windows of one or two key tiles take ~9,000 cycles, softmax 2,500, P V 850, rows written 3,300: each role's code comes
// from beyond the instruction cache again in every window (390 misses, some 50 KB). Tried for them: a rolled loop over the
// two tiles in the issuer (-4 to -10%, but +3% for long sequences), the next window's first S behind the last P V (+1%), a
// run of the issuer's code without effect ahead of time (+5 to +10%), the softmax in halves (-1%, long +8%).
// Rows that see no key (causal with fewer keys than queries, no keys at all) get zeros.
#include <limits.h>

#include "host_common.cuh"
#include "overlap.cuh"
#include "packed_common.cuh"
#include "packed_host.cuh"

namespace lbw {

namespace pa {
constexpr int BM = 128, BN = 128, STAGES = 2;
constexpr int HALF = 128 * 64 * 2;  // 128 rows x 64 16-bit values: one 128-byte swizzled box
constexpr int SOFT_WARPS = 16;  // warps 0-15: (tile, key half) = (warp / 8, warp / 4 % 2), rows by warp % 4
constexpr int THREADS = (SOFT_WARPS + 4) * 32;
constexpr int STAGE_BYTES = SOFT_WARPS * 2048;  // output staging: 32 rows x 32 columns for each softmax warp
constexpr int smem_bytes(int d) { return (2 + 2 * STAGES) * (d / 64) * HALF + STAGE_BYTES + 1024; }
}  // namespace pa

struct TileArgs {
  int pack;        // query heads side by side in a tile
  int tile_toks;   // tokens of a tile: 128 / pack
  int head_tiles;  // hq / pack
  int short_rows;  // sequences with at most this many rows per kv head (nq * group) are packed_split_kernel's
  int n_split;     // key ranges per window (> 1: partial results, merged by packed_merge_kernel)
  float* part_o;   // [n_split][tq * hq][D]
  float* part_ml;  // [n_split][tq * hq][2]
};

// tcgen05 operations of a converged warp, issued by one of its lanes. Which: for D = 128 the elected one (always the same),
// elected in each operation's own asm; for D = 64 lane 0, by the predicate `lead`. A predicated MMA takes the issuer 79
// cycles, an elected one 65, and one runs for 64 (32 where D = 64 is its N). Measured (us, this rule / the other way round;
// bf16, replayed from a graph, the same inputs): D = 128 causal, 10,800 tokens of 40 / 8 heads 969 / 969, 64 x 300..900 of
// 16 / 2 heads 163 / 175; D = 64 without a mask, 16,000 tokens of 8 heads 834 / 857, 8 x 1,000 of 16 heads 68.1 / 68.6.
template <bool ELECT>
LBW_DEV void mma_f16_ss_one(uint32_t lead, uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t acc) {
  if constexpr (ELECT)
    asm volatile(
        "{\n\t.reg .pred p, e;\n\tsetp.ne.b32 p, %4, 0;\n\telect.sync _|e, 0xffffffff;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d_tmem),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(acc)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p, e;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 e, %5, 0;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d_tmem),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(acc), "r"(lead)
        : "memory");
}
template <bool ELECT>
LBW_DEV void mma_f16_ts_one(uint32_t lead, uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc, uint32_t acc) {
  if constexpr (ELECT)
    asm volatile(
        "{\n\t.reg .pred p, e;\n\tsetp.ne.b32 p, %4, 0;\n\telect.sync _|e, 0xffffffff;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d_tmem),
        "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(acc)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p, e;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 e, %5, 0;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d_tmem),
        "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(acc), "r"(lead)
        : "memory");
}
template <bool ELECT>
LBW_DEV void tc_commit_one(uint32_t lead, uint64_t* bar) {
  if constexpr (ELECT)
    asm volatile(
        "{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\t"
        "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}\n" ::"r"(smem_u32(bar))
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred e;\n\tsetp.ne.b32 e, %1, 0;\n\t"
        "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}\n" ::"r"(smem_u32(bar)),
        "r"(lead)
        : "memory");
}

// One window: the key range [g0, g0 + n_p) (in 128-key tiles) of a pair of query tiles.
struct PackedWin {
  PackedSeq sq;
  int tok[2];   // first token of the primary and of the secondary tile
  int n_p, n_s; // key tiles of the primary; the secondary takes the first n_s of them
  int g0, split, head0, two;
  int valid;
};

// Next window of the grid, for the block that calls it: takes the place of a block that has not been launched yet
// (cluster launch control). The answer arrives in `res` with 16 bytes on `bar`.
LBW_DEV void steal_request(void* res, uint64_t* bar) {
  asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(
                   smem_u32(res)),
               "r"(smem_u32(bar))
               : "memory");
}
LBW_DEV bool steal_answer(const void* res, unsigned& block) {
  uint32_t ok, x;
  asm volatile(
      "{\n\t.reg .b128 r;\n\t.reg .pred p;\n\t"
      "ld.shared.b128 r, [%2];\n\t"
      "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, r;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t"
      "mov.u32 %1, 0;\n\t"
      "@p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %1, r;\n\t}\n"
      : "=r"(ok), "=r"(x)
      : "r"(smem_u32(res))
      : "memory");
  block = x;
  return ok != 0;
}

// mbar_arrive of the lanes with lead != 0.
LBW_DEV void mbar_arrive_if(uint32_t lead, uint64_t* bar) {
  asm volatile("{\n\t.reg .pred e;\n\tsetp.ne.b32 e, %1, 0;\n\t@e mbarrier.arrive.shared::cta.b64 _, [%0];\n\t}\n" ::"r"(
                   smem_u32(bar)),
               "r"(lead)
               : "memory");
}

// The two warps of one group of rows meet (barrier `id`, 64 threads); pair_all: whether `ok` holds for all of them.
LBW_DEV void pair_sync(int id) { asm volatile("barrier.cta.sync %0, 64;" ::"r"(id) : "memory"); }
LBW_DEV bool pair_all(int id, bool ok) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %2, 0;\n\t"
      "barrier.cta.red.and.pred q, %1, 64, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}\n"
      : "=r"(r)
      : "r"(id), "r"((uint32_t)ok)
      : "memory");
  return r != 0;
}

// What a window keeps of the values that are not finite: for each column the first key with a NaN, with +inf and with
// -inf, 10 bits each, counted from `base` (the diagonal spans less than 640 keys); all ones: none.
constexpr uint32_t NO_KEY = 0x3ff, ALL_FINITE = 0x3fffffff;

// Whether rows [lo, hi) of a value tile (128 rows x D, swizzled) hold an infinity or a NaN: one answer for the warp. This
// look costs 2 to 7% of the time of short causal sequences (64 x 300..900 tokens 361 -> 375 us, 256 x 64..300 146 -> 156)
// and nothing that can be measured beyond 10,000 tokens or without a mask; unrolled by 4 or 1, or not inlined: 1% more.
template <int D, bool F16>
LBW_DEV bool v_not_finite(const uint8_t* tile, int lo, int hi) {
  uint32_t top = 0;
  auto take = [&](uint32_t x) {  // larger magnitude of either half, NaN above all
    if constexpr (F16) {
      const __half2 m = __hmax2_nan(*reinterpret_cast<__half2*>(&top), __habs2(*reinterpret_cast<__half2*>(&x)));
      top = *reinterpret_cast<const uint32_t*>(&m);
    } else {
      const __nv_bfloat162 m =
          __hmax2_nan(*reinterpret_cast<__nv_bfloat162*>(&top), __habs2(*reinterpret_cast<__nv_bfloat162*>(&x)));
      top = *reinterpret_cast<const uint32_t*>(&m);
    }
  };
#pragma unroll 2
  for (int r = lo * 8 + (threadIdx.x & 31); r < hi * 8; r += 32)
#pragma unroll
    for (int h = 0; h < D / 64; ++h) {
      const uint4 v = *reinterpret_cast<const uint4*>(tile + h * pa::HALF + r * 16);
      take(v.x);
      take(v.y);
      take(v.z);
      take(v.w);
    }
  constexpr uint32_t EXP = F16 ? 0x7c00u : 0x7f80u;
  return __any_sync(0xffffffffu, (top & EXP) == EXP || (top >> 16 & EXP) == EXP) != 0;
}

// Takes them out of rows [lo, hi) of a value tile whose first key is `key` (one column per lane); returns the new base.
// Not inlined, like all that is rare here: see mbar_wait_long.
template <int D, bool F16>
static __device__ __noinline__ int v_take_not_finite(uint8_t* tile, uint32_t* bad, int* s_base, int base, int key,
                                                      int lo, int hi) {
  const bool first = base < 0;
  if (first) base = key;
  constexpr uint32_t EXP = F16 ? 0x7c00u : 0x7f80u;
  for (int c = threadIdx.x & 31; c < D; c += 32) {
    uint32_t e = first ? ALL_FINITE : bad[c];
    for (int r = lo; r < hi; ++r) {
      uint16_t* p = reinterpret_cast<uint16_t*>(tile + (c >> 6) * pa::HALF + r * 128 + (((c >> 3 & 7) ^ (r & 7)) << 4)) + (c & 7);
      const uint32_t x = *p;
      if ((x & EXP) != EXP) continue;
      const int at = 10 * (x & (EXP ^ 0x7fff) ? 0 : x & 0x8000 ? 2 : 1);
      if ((e >> at & NO_KEY) == NO_KEY) e ^= (NO_KEY ^ (uint32_t)(key - base + r)) << at;
      *p = 0;
    }
    bad[c] = e;
  }
  *s_base = base;
  fence_async_shared();
  __syncwarp();
  return base;
}

// What they add to a column of a row that sees `seen` keys from `base` on.
LBW_DEV float not_finite_sum(uint32_t e, int seen) {
  const bool nan = (int)(e & NO_KEY) < seen, up = (int)(e >> 10 & NO_KEY) < seen, down = (int)(e >> 20) < seen;
  return nan || (up && down) ? __int_as_float(0x7fffffff) : up ? INFINITY : down ? -INFINITY : 0.f;
}

// Adds it to this thread's half of its row of the window, which the warp has just written.
template <int D, bool F16>
static __device__ __noinline__ void row_add_not_finite(const PackedArgs& a, const TileArgs& ta, const PackedWin& w,
                                                       const uint32_t* bad, int base) {
  const int warp = threadIdx.x >> 5, r0 = (warp & 3) * 32 + (threadIdx.x & 31), c0 = (warp >> 2 & 1) * (D / 2);
  const int tok = w.tok[warp >> 3] + r0 / ta.pack, head = w.head0 + r0 % ta.pack;
  __syncwarp();
  if (r0 < ta.pack * ta.tile_toks && tok < w.sq.nq) {
    const int seen = packed_visible(a, w.sq, tok) - base;
    const long long row = (long long)w.sq.q0 + tok;
    for (int c = c0; c < c0 + D / 2; ++c) {
      const float x = not_finite_sum(bad[c], seen);
      if (x == 0.f) continue;
      if (ta.n_split > 1) {
        ta.part_o[(((long long)w.split * a.tq + row) * a.hq + head) * D + c] += x;
      } else {
        uint16_t* p = reinterpret_cast<uint16_t*>(a.out) + row * a.os_tok + head * a.os_head + c;
        *p = (uint16_t)pack_16<F16>(unpack_16<F16>(*p) + x, 0.f);
      }
    }
  }
  __syncwarp();
}

template <int D, bool F16>
__global__ void __launch_bounds__(pa::THREADS, 1)
    packed_attn_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                       const __grid_constant__ CUtensorMap tmV, const __grid_constant__ PackedArgs a,
                       const __grid_constant__ TileArgs ta, int* status) {
  using namespace pa;
  constexpr int NH = D / 64;       // 64-wide boxes of a row
  constexpr int TILE = NH * HALF;  // 128 rows x D
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;
  uint8_t* sK = smem + 2 * TILE;
  uint8_t* sV = sK + STAGES * TILE;
  uint8_t* s_stage = sV + STAGES * TILE;
  __shared__ __align__(8) uint64_t q_full, q_empty, k_full[STAGES], k_empty[STAGES], v_full[STAGES], v_empty[STAGES],
      s_full[2], p_ready[2], o_done[2], win_full[2], win_empty[2], want_next, steal_bar, done_bar;
  __shared__ __align__(16) uint4 steal_res;
  __shared__ PackedWin s_win[2];
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag;
  __shared__ uint32_t s_bad[2][D];  // of window i in slot i & 1: values that are not finite
  __shared__ int s_bad_base[2];     // their first key, -1: there are none
  __shared__ int s_rank[32];        // the scheduler's

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    mbar_init(&q_full, 1);
    mbar_init(&q_empty, 1);
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&k_full[s], 1);
      mbar_init(&k_empty[s], 1);
      mbar_init(&v_full[s], 1);
      mbar_init(&v_empty[s], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_ready[i], 8 + (i == 0));  // P written by 8 warps (+ V(j) and K(j + 1) landed, for the primary)
      mbar_init(&o_done[i], 1);
      mbar_init(&win_full[i], 1);
      mbar_init(&win_empty[i], 3 + SOFT_WARPS);  // producer, issuer, watcher and the softmax warps have read the window
    }
    mbar_init(&want_next, 1);
    mbar_init(&steal_bar, 1);
    mbar_init(&done_bar, 1);
    abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 17) tmem_alloc(&tmem_slot, 512);
  // Rows that no token fills (pack does not divide 128): zeros, so that they never ask for a rescale.
  const int filled = ta.pack * ta.tile_toks;
  for (int e = filled * 8 + threadIdx.x; e < 128 * 8; e += THREADS)
    for (int t = 0; t < 2 * NH; ++t) *reinterpret_cast<uint4*>(sQ + t * HALF + e * 16) = make_uint4(0, 0, 0, 0);
  fence_async_shared();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_trigger();
  const uint32_t tmem = tmem_slot;
  const Abort ab{status, &abort_flag};

  if (warp == 19) {
    // ---------------- scheduler ----------------
    // Takes the next window when the producer loads the last key tile of the present one: about two tiles before its end,
    // enough to hide the answer and the search, and late enough that no CTA holds work which another could start.
    // The search for a window's sequence goes on where the last one ended, as windows mostly come in the grid's order. That
    // no later answer names an earlier block is promised nowhere: then the search starts again at the first sequence.
    bool have = true;
    unsigned block = blockIdx.x, asked = 0;  // (asked: lane 0's)
    int b_at = 0, loaded = -1;
    unsigned before = 0;  // windows of the sequences before b_at (all counts are below the grid's 2^31)
    PackedSeq s{0, 0, 0, 0};
    unsigned own = 0, upto = 0;
    for (int i = 0;; ++i) {
      const int slot = i & 1;
      bool ok = true;
      PackedWin w;
      w.valid = 0;
      if (i > 0 && lane == 0) ok = mbar_wait_c(&want_next, (i - 1) & 1, ab, 0x13);
      // The grid is an upper bound: a block past the last window is passed over (a later answer may name one with a window),
      // and none of them has to start. (3,000 single tokens beside a prompt of 700, whose bound is 6,000 blocks too high:
      // 262 us, 255 where the other warps left at the first such block.)
      for (bool ask = i > 0; have && !w.valid; ask = true) {
        if (ask) {
          if (lane == 0) {
            do {
              if (ok) {
                mbar_expect_tx(&steal_bar, 16);
                steal_request(&steal_res, &steal_bar);
                ok = mbar_wait_c(&steal_bar, asked++ & 1, ab, 0x11);
              }
              have = ok && steal_answer(&steal_res, block);
              fence_async_shared();  // (read before the next answer overwrites it)
            } while (have && b_at >= a.n_seqs && block / (ta.n_split * ta.head_tiles) >= before);  // (all counted: no window)
          }
          have = __shfl_sync(0xffffffffu, have, 0);
          block = __shfl_sync(0xffffffffu, block, 0);
          if (!have) break;
        }
        const unsigned rest = ta.n_split > 1 ? block / ta.n_split : block;
        w.split = (int)(block - rest * ta.n_split);
        const unsigned pair = rest / ta.head_tiles;
        w.head0 = (int)(rest - pair * ta.head_tiles) * ta.pack;
        if (pair < before) {
          b_at = 0;
          before = 0;
        }
        while (b_at < a.n_seqs) {
          if (loaded != b_at) {  // 32 sequences, one per lane, kept while windows come from them
            const int b = b_at + lane;
            s = b < a.n_seqs ? packed_seq(a, b) : PackedSeq{0, 0, 0, 0};
            if (a.n_seqs > 1) {
              // Those with most keys first: their windows are the longest, and a CTA that took one last would be alone.
              // Measured (us, so / in the batch's order, as above): 256 x 64..300 tokens of 16 / 2 heads 141.1 / 144.5, three
              // clips of 1,560 to 4,680 111.5 / 112.8, 48 x 1..509 of 32 / 8 90.0 / 90.8, 64 x 300..900 163.3 / 162.7.
              int rank = 0;
#pragma unroll
              for (int o = 0; o < 32; ++o) {
                const int nk = __shfl_sync(0xffffffffu, s.nk, o);
                rank += nk > s.nk || (nk == s.nk && o < lane);
              }
              s_rank[rank] = lane;
              __syncwarp();
              const int from = s_rank[lane];
              s.q0 = __shfl_sync(0xffffffffu, s.q0, from);
              s.nq = __shfl_sync(0xffffffffu, s.nq, from);
              s.k0 = __shfl_sync(0xffffffffu, s.k0, from);
              s.nk = __shfl_sync(0xffffffffu, s.nk, from);
              __syncwarp();
            }
            own = (long long)s.nq * a.group <= ta.short_rows ? 0 : (s.nq + 2 * ta.tile_toks - 1) / (2 * ta.tile_toks);
            upto = own;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
              const unsigned v = __shfl_up_sync(0xffffffffu, upto, o);
              if (lane >= o) upto += v;
            }
            loaded = b_at;
          }
          const unsigned hit = __ballot_sync(0xffffffffu, before + upto > pair);
          if (hit) {
            const int at = __ffs(hit) - 1;
            w.valid = 1;
            w.sq.q0 = __shfl_sync(0xffffffffu, s.q0, at);
            w.sq.nq = __shfl_sync(0xffffffffu, s.nq, at);
            w.sq.k0 = __shfl_sync(0xffffffffu, s.k0, at);
            w.sq.nk = __shfl_sync(0xffffffffu, s.nk, at);
            // Pairs of tiles are taken from the sequence's end, where causal rows see most keys. (The minimum is for starts
            // that overlap so often that the counts wrap.)
            const unsigned n_pairs = __shfl_sync(0xffffffffu, own, at);
            const unsigned l = min(pair - before - __shfl_sync(0xffffffffu, upto - own, at), n_pairs - 1);
            const int tok0 = (int)(n_pairs - 1 - l) * 2 * ta.tile_toks;
            w.two = tok0 + ta.tile_toks < w.sq.nq;
            w.tok[0] = w.two ? tok0 + ta.tile_toks : tok0;
            w.tok[1] = tok0;
            const int keys_p = packed_visible(a, w.sq, min(w.tok[0] + ta.tile_toks, w.sq.nq) - 1);
            const int keys_s = w.two ? packed_visible(a, w.sq, tok0 + ta.tile_toks - 1) : 0;
            const int all_p = (keys_p + BN - 1) / BN, all_s = (keys_s + BN - 1) / BN;
            w.g0 = 0;
            w.n_p = all_p;
            if (ta.n_split > 1) {  // (n_split <= 32 and all_p < 2^24: no overflow)
              w.g0 = w.split * all_p / ta.n_split;
              w.n_p = (w.split + 1) * all_p / ta.n_split - w.g0;
            }
            w.n_s = min(max(all_s - w.g0, 0), w.n_p);
            break;
          }
          before += __shfl_sync(0xffffffffu, upto, 31);
          b_at += 32;
        }
      }
      if (lane == 0) {
        ok = mbar_wait_c(&win_empty[slot], ((i >> 1) & 1) ^ 1, ab, 0x10) && ok;
        s_win[slot] = w;
        mbar_arrive(&win_full[slot]);
      }
      ok = __shfl_sync(0xffffffffu, ok, 0);
      if (!w.valid || !ok) break;
    }
  } else if (warp == 16) {
    // ---------------- producer ----------------
    if (lane == 0) {
      tma_prefetch_desc(&tmQ);
      tma_prefetch_desc(&tmK);
      tma_prefetch_desc(&tmV);
      int j = 0, nq_loads = 0;  // K/V tiles and Q pairs loaded so far
      bool ok = true;
      for (int i = 0; ok; ++i) {
        if (!mbar_wait_c(&win_full[i & 1], (i >> 1) & 1, ab, 0x20)) break;
        const PackedWin w = s_win[i & 1];
        mbar_arrive(&win_empty[i & 1]);
        if (!w.valid) break;
        const int kv_head = w.head0 / a.group;
        if (w.n_p == 0) mbar_arrive(&want_next);
        for (int t = 0; t < w.n_p; ++t, ++j) {
          if (t + 1 == w.n_p) mbar_arrive(&want_next);
          const int s = j & 1;
          const uint32_t ph = (j >> 1) & 1;
          const int row = w.sq.k0 + (w.g0 + t) * BN;
          if (!(ok = mbar_wait_c(&k_empty[s], ph ^ 1, ab, 0x21))) break;
          mbar_expect_tx(&k_full[s], TILE);
          for (int h = 0; h < NH; ++h) tma_load_3d(sK + s * TILE + h * HALF, &tmK, &k_full[s], h * 64, kv_head, row);
          if (t == 0) {  // the pair's Q goes where the last window's was, once its last S is computed
            if (!(ok = mbar_wait_c(&q_empty, (nq_loads & 1) ^ 1, ab, 0x23))) { mbar_wait_drain(&k_full[s], ph); break; }
            const int tiles = w.n_s > 0 ? 2 : 1;
            mbar_expect_tx(&q_full, tiles * NH * ta.pack * ta.tile_toks * 128);
            for (int q = 0; q < tiles; ++q)
              for (int h = 0; h < NH; ++h)
                tma_load_3d(sQ + q * TILE + h * HALF, &tmQ, &q_full, h * 64, w.head0, w.sq.q0 + w.tok[q]);
            ++nq_loads;
          }
          if (!(ok = mbar_wait_c(&v_empty[s], ph ^ 1, ab, 0x22))) { mbar_wait_drain(&k_full[s], ph); break; }
          mbar_expect_tx(&v_full[s], TILE);
          for (int h = 0; h < NH; ++h) tma_load_3d(sV + s * TILE + h * HALF, &tmV, &v_full[s], h * 64, kv_head, row);
        }
      }
      // Let the last loads of each ring slot land before the CTA can exit.
      if (nq_loads > 0) mbar_wait_drain(&q_full, (nq_loads - 1) & 1);
      for (int t = (j > STAGES ? j - STAGES : 0); t < j; ++t) {
        mbar_wait_drain(&k_full[t & 1], (t >> 1) & 1);
        mbar_wait_drain(&v_full[t & 1], (t >> 1) & 1);
      }
    }
  } else if (warp == 17) {
    // ---------------- MMA issuer ----------------
    // MMAs execute in issue order: S of a window's first tile may be issued right behind the last P V of the window
    // before, and its O is overwritten only by a P V that waits for a P written after that O was read.
    // The whole warp runs this code and one lane issues (by predicate): in a branch of one lane every descriptor would have
    // to be moved to the uniform registers that the MMA reads.
    constexpr bool ELECT = D == 128;
    const uint32_t lead = lane == 0;
    const uint32_t idesc_s = F16 ? idesc_f16(BM, BN, 0, 0) : idesc_bf16(BM, BN, 0, 0);  // S = Q K^T, both K-major
    const uint32_t idesc_o = F16 ? idesc_f16(BM, D, 0, 1) : idesc_bf16(BM, D, 0, 1);    // O += P V, V MN-major
    const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
    const uint64_t dQ = sdesc_kmajor_sw128(smem_u32(sQ));
    const uint64_t dK = sdesc_kmajor_sw128(smem_u32(sK));
    const uint64_t dV = sdesc_mnmajor_sw128(smem_u32(sV), HALF);
    auto issue_s = [&](int i, int stage) {
      const uint64_t q = dQ + (uint64_t)((i * TILE) >> 4), k = dK + (uint64_t)((stage * TILE) >> 4);
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        const uint64_t off = (uint64_t)(((kk >> 2) * HALF + (kk & 3) * 32) >> 4);
        mma_f16_ss_one<ELECT>(lead, tm + i * 128, q + off, k + off, idesc_s, kk > 0);
      }
    };
    auto issue_pv = [&](int i, int stage, bool first) {
      const uint64_t v = dV + (uint64_t)((stage * TILE) >> 4);
#pragma unroll
      for (int kk = 0; kk < 8; ++kk)  // P of keys 64.. lies over its own scores, 64 columns on
        mma_f16_ts_one<ELECT>(lead, tm + 256 + i * D, tm + i * 128 + (kk >> 2) * 64 + (kk & 3) * 8,
                      v + (uint64_t)((kk * 2048) >> 4), idesc_o, !(first && kk == 0));
    };
    auto wait = [&](uint64_t* bar, uint32_t parity, int site) {
      return __all_sync(0xffffffffu, mbar_wait_c(bar, parity, ab, site)) != 0;
    };
    int jp = 0, js = 0, nq_loads = 0;  // tiles of the primaries and secondaries, Q pairs, so far
    bool ok = true;
    for (int i = 0; ok; ++i) {
      if (!wait(&win_full[i & 1], (i >> 1) & 1, 0x30)) break;
      const int n_p = __shfl_sync(0xffffffffu, s_win[i & 1].n_p, 0), n_s = __shfl_sync(0xffffffffu, s_win[i & 1].n_s, 0);
      const int valid = __shfl_sync(0xffffffffu, s_win[i & 1].valid, 0);
      mbar_arrive_if(lead, &win_empty[i & 1]);
      if (!valid) break;
      if (n_p == 0) continue;
      if (!wait(&q_full, nq_loads & 1, 0x31) || !wait(&k_full[jp & 1], (jp >> 1) & 1, 0x32)) break;
      ++nq_loads;
      tc_fence_after();
      // Step j: P V of tile j, then S of tile j + 1 (step -1 has only the first S): the same code for all steps, so that
      // it is in the instruction cache when a window begins.
      for (int j = -1; ok && j < n_p; ++j) {
        const int s = jp & 1, s1 = j < 0 ? s : s ^ 1;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const int n = t ? n_s : n_p;
          if (t && j >= 0 && (j >= n || !ok)) tc_commit_one<ELECT>(lead, &v_empty[s]);
          if (j >= n || !ok) continue;
          if (j >= 0) {
            if (!(ok = wait(&p_ready[t], (t ? js : jp) & 1, 0x34 + t))) continue;
            tc_fence_after();
            issue_pv(t, s, j == 0);
            js += t;
            if (t) tc_commit_one<ELECT>(lead, &v_empty[s]);
          }
          if (j + 1 < n) {
            issue_s(t, s1);
            tc_commit_one<ELECT>(lead, &s_full[t]);
          } else if (n > 0) {
            tc_commit_one<ELECT>(lead, &o_done[t]);
          }
        }
        if (j + 1 < n_p) tc_commit_one<ELECT>(lead, &k_empty[s1]);
        if (j + 2 == n_p) tc_commit_one<ELECT>(lead, &q_empty);  // the window's last S has been issued
        jp += j >= 0;
      }
    }
    tc_commit_one<ELECT>(lead, &done_bar);
    mbar_wait_drain(&done_bar, 0);
  } else if (warp == 18) {
    // ---------------- K/V watcher ----------------
    // One phase of each P barrier at a time (see attn.cu). It must never wait for a phase that can be lapped: it does not
    // look at a window's first K, whose S and whose slot's next load (K two tiles on) do not depend on it, so that two
    // phases could pass before it looked. Every K and V that it waits for is followed by its own arrival before the
    // slot can be loaded again, and the phase before it is over: its S or P V was needed for the P seen before.
    int jp = 0;
    // All lanes wait: a wait of one lane of a converged warp costs ~500 cycles more (a round trip of two warps over mbarriers
    // takes 290 cycles when all lanes wait, 1,220 when lane 0 waits for the others), and these are on every tile's path.
    bool ok = true;
    for (int i = 0; ok; ++i) {
      if (!__all_sync(0xffffffffu, mbar_wait_c(&win_full[i & 1], (i >> 1) & 1, ab, 0x5f))) break;
      const int n_p = s_win[i & 1].n_p, g0 = s_win[i & 1].g0, valid = s_win[i & 1].valid;
      const int left = s_win[i & 1].sq.nk - g0 * BN;
      // Keys that all rows of the pair see, and all rows of the primary alone (it goes on when the secondary has ended).
      const int n_s = s_win[i & 1].n_s;
      const int see_p = packed_visible(a, s_win[i & 1].sq, s_win[i & 1].tok[0]) - g0 * BN;
      const int see_s = n_s > 0 ? packed_visible(a, s_win[i & 1].sq, s_win[i & 1].tok[1]) - g0 * BN : see_p;
      int base = -1;  // (the softmax warps have left the slot's last window: it is this one's now)
      if (lane == 0) s_bad_base[i & 1] = -1;
      __syncwarp();
      mbar_arrive_if(lane == 0, &win_empty[i & 1]);
      if (!valid) break;
      for (int j = 0; j < n_p; ++j, ++jp) {
        const int s = jp & 1;
        ok = __all_sync(0xffffffffu, mbar_wait_c(&v_full[s], (jp >> 1) & 1, ab, 0x61));
        if (!ok) break;
        const int rows = left - j * BN;  // value rows of this tile that are the sequence's
        if (rows < BN) {
          for (int r = rows * 8 + lane; r < BN * 8; r += 32)
#pragma unroll
            for (int h = 0; h < NH; ++h)
              *reinterpret_cast<uint4*>(sV + s * TILE + h * HALF + r * 16) = make_uint4(0, 0, 0, 0);
          fence_async_shared();
          __syncwarp();
        }
        // Keys that some row does not see (what all see goes the usual way).
        const int lo = max((j < n_s ? see_s : see_p) - j * BN, 0), hi = min(rows, BN);
        if (lo < hi && v_not_finite<D, F16>(sV + s * TILE, lo, hi))
          base = v_take_not_finite<D, F16>(sV + s * TILE, s_bad[i & 1], &s_bad_base[i & 1], base, (g0 + j) * BN, lo, hi);
        ok = j + 1 >= n_p || __all_sync(0xffffffffu, mbar_wait_c(&k_full[s ^ 1], ((jp + 1) >> 1) & 1, ab, 0x62));
        if (!ok) break;
        mbar_arrive_if(lane == 0, &p_ready[0]);
        ok = __all_sync(0xffffffffu, mbar_wait_c(&p_ready[0], jp & 1, ab, 0x63));
        if (!ok) break;
      }
    }
  } else {
    // ---------------- softmax / correction / epilogue ----------------
    // Two threads per row, one for each half of a tile's keys, in two warps that meet at a named barrier for the row's
    // maximum. They take every branch together: their row values are equal, and they agree on the waits (a warp that
    // left alone would leave the other at the barrier).
    const int wg = warp >> 3, half = (warp >> 2) & 1;
    const int r0 = (warp & 3) * 32 + lane;  // row of the tile
    const int pair_bar = 1 + wg * 4 + (warp & 3);
    uint8_t* stage = s_stage + warp * 2048;  // this warp's 2 KB: its rows' maxima and sums, and the output on its way
    float* my_row = reinterpret_cast<float*>(stage) + lane;
    const float* other_row = reinterpret_cast<const float*>(s_stage + (warp ^ 4) * 2048) + lane;
    const uint32_t lane_off = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t tS = tmem + lane_off + wg * 128 + half * 64;
    const uint32_t tO = tmem + lane_off + 256 + wg * D + half * (D / 2);  // this thread's columns of O
    uint32_t phases = 0;  // bit 0: parity of s_full (tiles so far), bit 1: of o_done (windows with a tile)
    for (int i = 0;; ++i) {
      const bool got = mbar_wait_c(&win_full[i & 1], (i >> 1) & 1, ab, 0x40);
      if (!pair_all(pair_bar, got && !abort_flag)) break;
      const volatile PackedWin& w = s_win[i & 1];  // read again at the end: registers are short in between
      if (!w.valid) break;
      if (wg == 1 && !w.two) {
        __syncwarp();
        if (lane == 0) mbar_arrive(&win_empty[i & 1]);
        continue;
      }
      // Keys this row sees, from this thread's first on; a row that is nobody's is never masked (nor written).
      int seen = 1 << 30;
      {
        const int nq = w.sq.nq, nk = w.sq.nk, tok = w.tok[wg] + r0 / ta.pack;
        if (r0 < ta.pack * ta.tile_toks && tok < nq)
          seen = packed_visible(a, PackedSeq{0, nq, 0, nk}, tok) - w.g0 * BN - half * 64;
      }
      const int n_tiles = wg == 0 ? w.n_p : w.n_s;
      float m = -INFINITY, l = 0.f;
      for (int left = n_tiles; left > 0; --left, seen -= BN, phases ^= 1) {
        mbar_wait_c(&s_full[wg], phases & 1, ab, 0x41 + wg);  // (after a timeout the window runs on, and ends the loop)
        tc_fence_after();
        uint32_t r[64];
        float* sv = reinterpret_cast<float*>(r);
        tmem_ld32(tS, *reinterpret_cast<uint32_t(*)[32]>(&r[0]));
        tmem_ld32(tS + 32, *reinterpret_cast<uint32_t(*)[32]>(&r[32]));
        tmem_ld_wait();
        if (!__all_sync(0xffffffffu, seen >= 64)) {  // the diagonal, or the sequence's last tile
#pragma unroll
          for (int cc = 0; cc < 2; ++cc) {
            const int n = min(max(seen - cc * 32, 0), 32);
            const uint32_t keep = n == 32 ? 0xffffffffu : (1u << n) - 1u;
#pragma unroll
            for (int e = 0; e < 32; ++e) sv[cc * 32 + e] = keep >> e & 1 ? sv[cc * 32 + e] : -INFINITY;
          }
        }
        float t8[8];
#pragma unroll
        for (int q = 0; q < 8; ++q) t8[q] = fmax3(sv[q], sv[8 + q], sv[16 + q]);
#pragma unroll
        for (int e = 24; e < 56; e += 16)
#pragma unroll
          for (int q = 0; q < 8; ++q) t8[q] = fmax3(t8[q], sv[e + q], sv[e + 8 + q]);
#pragma unroll
        for (int q = 0; q < 8; ++q) t8[q] = fmaxf(t8[q], sv[56 + q]);
        float mx = fmaxf(fmax3(t8[0], t8[1], t8[2]), fmax3(fmax3(t8[3], t8[4], t8[5]), t8[6], t8[7]));
        *my_row = mx;
        pair_sync(pair_bar);
        mx = fmaxf(mx, *other_row) * a.scale_log2;
        // The running maximum only moves when it grows by more than 2^8 (or from -inf). O and l are rescaled then, O by
        // both threads of the row; it stands still: S is behind every P V before it.
        const bool grow = mx > m + 8.f;
        const bool rescale = __any_sync(0xffffffffu, grow);
        const float alpha = !grow ? 1.f : m == -INFINITY ? 0.f : fast_exp2(m - mx);
        if (grow) m = mx;
        l *= alpha;
        // A row that has seen no key yet has m = -inf and scores of -inf: p = 2^(-inf - 0) = 0.
        const float m_use = m == -INFINITY ? 0.f : m;
        const uint64_t a2 = f2_pack(a.scale_log2, a.scale_log2), b2 = f2_pack(-m_use, -m_use);
        uint64_t lsum[2] = {0ull, 0ull};
#pragma unroll
        for (int cc = 0; cc < 4; ++cc) {
          uint32_t pk[8];
#pragma unroll
          for (int e = 0; e < 16; e += 2) {
            const int col = cc * 16 + e;
            float x0, x1, p0, p1;
            f2_unpack(f2_fma(f2_pack(sv[col], sv[col + 1]), a2, b2), x0, x1);
            p0 = fast_exp2(x0);
            p1 = fast_exp2(x1);
            lsum[(e >> 1) & 1] = f2_add(lsum[(e >> 1) & 1], f2_pack(p0, p1));
            pk[e >> 1] = pack_16<F16>(p0, p1);
          }
          tmem_st8(tS + cc * 8, pk);
        }
        if (rescale && left != n_tiles) {  // (the scores' registers are free now; before a window's first P V there is no O)
#pragma unroll 1
          for (int cc = 0; cc < D / 64; ++cc) {
            uint32_t o[32];
            tmem_ld32(tO + cc * 32, o);
            tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
            tmem_st32(tO + cc * 32, o);
          }
          tmem_st_wait();
          tc_fence_before();
          pair_sync(pair_bar);  // either thread's arrival may start a P V into all of O
        }
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        mbar_arrive_if(lane == 0, &p_ready[wg]);  // (one arrival per warp: 32 on one barrier take turns)
        float l0, l1;
        f2_unpack(f2_add(lsum[0], lsum[1]), l0, l1);
        l += l0 + l1;
      }
      if (n_tiles > 0) {
        mbar_wait_c(&o_done[wg], phases >> 1, ab, 0x48 + wg);
        phases ^= 2;
        tc_fence_after();
      }
      *my_row = l;  // for the row's sum over both halves (the last maxima have been read: O waited for both threads' P)
      pair_sync(pair_bar);
      l += *other_row;
      pair_sync(pair_bar);  // (read before the next window's maxima)
      const int tok = w.tok[wg] + r0 / ta.pack, head = w.head0 + r0 % ta.pack, split = w.split;
      const bool mine = r0 < ta.pack * ta.tile_toks && tok < w.sq.nq && !abort_flag;
      const long long row = (long long)w.sq.q0 + tok;
      // Values that are not finite and that this row sees (ordered by O's barrier behind the watcher's arrivals; what it
      // writes for later tiles of the primary is of keys that the secondary's rows do not see).
      const int base = n_tiles > 0 ? *(volatile int*)&s_bad_base[i & 1] : -1;
      __syncwarp();
      if (lane == 0 && base < 0) mbar_arrive(&win_empty[i & 1]);
      if (ta.n_split > 1) {
        // unnormalised fp32 row and its (m, l); a row without a key leaves only l = 0
        const long long pr = ((long long)split * a.tq + row) * a.hq + head;
        if (mine && half == 0) *reinterpret_cast<float2*>(ta.part_ml + pr * 2) = make_float2(m, l);
        float* dst = ta.part_o + pr * D + half * (D / 2);
        if (n_tiles > 0) {
#pragma unroll 1
          for (int cc = 0; cc < D / 64; ++cc) {
            uint32_t r[32];
            tmem_ld32(tO + cc * 32, r);
            tmem_ld_wait();
            if (mine) {
#pragma unroll
              for (int q = 0; q < 8; ++q)
                reinterpret_cast<float4*>(dst + cc * 32)[q] =
                    make_float4(__uint_as_float(r[4 * q]), __uint_as_float(r[4 * q + 1]), __uint_as_float(r[4 * q + 2]),
                                __uint_as_float(r[4 * q + 3]));
            }
          }
        }
      } else {
        const bool none = l == 0.f;  // no key seen: zeros (a NaN stays)
        const float inv = 1.f / l;
        // 32 columns at a time through shared memory (16-byte pieces, the piece's place turned by the row), so that 4
        // lanes store 64 contiguous bytes of a row: a row per thread would touch 32 lines with every store.
        const unsigned long long at = reinterpret_cast<unsigned long long>(reinterpret_cast<uint16_t*>(a.out) +
                                                                           row * a.os_tok + head * a.os_head + half * (D / 2));
        const uint32_t some = none ? 0u : 0xffffffffu;
#pragma unroll 1
        for (int cc = 0; cc < D / 64; ++cc) {
#pragma unroll 1
          for (int hh = 0; hh < 2; ++hh) {
            uint32_t r[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) r[e] = 0;
            if (n_tiles > 0) {
              tmem_ld16(tO + cc * 32 + hh * 16, r);
              tmem_ld_wait();
            }
#pragma unroll
            for (int q = 0; q < 2; ++q) {
              uint32_t pk[4];
#pragma unroll
              for (int e = 0; e < 4; ++e)
                pk[e] = some & pack_16<F16>(__uint_as_float(r[8 * q + 2 * e]) * inv, __uint_as_float(r[8 * q + 2 * e + 1]) * inv);
              *reinterpret_cast<uint4*>(stage + lane * 64 + (((hh * 2 + q) ^ ((lane >> 1) & 3)) << 4)) =
                  make_uint4(pk[0], pk[1], pk[2], pk[3]);
            }
          }
          __syncwarp();
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const int row_l = q * 8 + (lane >> 2);
            const uint4 v = *reinterpret_cast<const uint4*>(stage + row_l * 64 + (((lane & 3) ^ ((row_l >> 1) & 3)) << 4));
            const unsigned long long to = __shfl_sync(0xffffffffu, at, row_l);
            if (__shfl_sync(0xffffffffu, mine, row_l)) *reinterpret_cast<uint4*>(to + cc * 64 + (lane & 3) * 16) = v;
          }
          __syncwarp();
        }
      }
      if (base >= 0) {
        if (!abort_flag) row_add_not_finite<D, F16>(a, ta, s_win[i & 1], s_bad[i & 1], base);
        if (lane == 0) mbar_arrive(&win_empty[i & 1]);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 17) tmem_dealloc(tmem, 512);
}

// Joins the key ranges of split windows: out = sum_z 2^(m_z - M) O_z / sum_z 2^(m_z - M) l_z, M = max over the ranges
// with a key. One warp per (token, head); tokens of no sequence and of the other kernel's sequences are left alone.
template <int D, bool F16>
__global__ void __launch_bounds__(128) packed_merge_kernel(const __grid_constant__ PackedArgs a,
                                                           const __grid_constant__ TileArgs ta) {
  const int lane = threadIdx.x & 31;
  const long long wid = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (wid >= (long long)a.tq * a.hq) {
    pdl_wait();
    return;
  }
  pdl_trigger();
  const long long tok = wid / a.hq;
  const int head = (int)(wid % a.hq);
  bool ours = false;
  for (int b = lane; b < a.n_seqs; b += 32) {
    const PackedSeq s = packed_seq(a, b);
    ours |= tok >= s.q0 && tok < s.q0 + s.nq && (long long)s.nq * a.group > ta.short_rows;
  }
  pdl_wait();
  if (!__any_sync(0xffffffffu, ours)) return;
  // Lane z weighs range z (at most 32); then the rows, with the loads of 8 ranges in flight.
  const long long step = (long long)a.tq * a.hq;
  const float2 ml = lane < ta.n_split ? *reinterpret_cast<const float2*>(ta.part_ml + (lane * step + wid) * 2)
                                      : make_float2(-INFINITY, 0.f);
  float M = ml.x;
#pragma unroll
  for (int o = 16; o; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
  const bool some = ml.y != 0.f;  // (no key of the range visible: nothing was written. All scores NaN: so is the sum)
  const float w = !some ? 0.f : ml.x == -INFINITY ? ml.y : exp2f(ml.x - M);
  float L = some ? w * ml.y : 0.f;
#pragma unroll
  for (int o = 16; o; o >>= 1) L += __shfl_xor_sync(0xffffffffu, L, o);
  constexpr int PER = D / 32, UN = 8;
  const uint32_t there = __ballot_sync(0xffffffffu, some);
  float acc[PER] = {};
  for (int z = 0; z < ta.n_split; z += UN) {
    float f[UN][PER];
#pragma unroll
    for (int i = 0; i < UN; ++i) {
      const float* o = ta.part_o + ((z + i) * step + wid) * D + lane * PER;
#pragma unroll
      for (int e = 0; e < PER; e += 2) {
        const float2 v = there >> (z + i) & 1 ? *reinterpret_cast<const float2*>(o + e) : make_float2(0.f, 0.f);
        f[i][e] = v.x;
        f[i][e + 1] = v.y;
      }
    }
#pragma unroll
    for (int i = 0; i < UN; ++i) {
      const float wz = __shfl_sync(0xffffffffu, w, z + i);
#pragma unroll
      for (int e = 0; e < PER; ++e) acc[e] += wz * f[i][e];
    }
  }
  const float inv = L == 0.f ? 0.f : 1.f / L;
  uint32_t* dst = reinterpret_cast<uint32_t*>(reinterpret_cast<uint16_t*>(a.out) + tok * a.os_tok + head * a.os_head +
                                              lane * PER);
#pragma unroll
  for (int i = 0; i < PER; i += 2) dst[i / 2] = pack_16<F16>(acc[i] * inv, acc[i + 1] * inv);
}

}  // namespace lbw

using namespace lbw;

template <int D, bool F16>
static int launch_tiles(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const PackedArgs& a,
                        const TileArgs& ta, dim3 grid, int* st, cudaStream_t s) {
  static bool attr[64] = {};
  const int dix = device_index();
  if (dix < 0) return set_error(LBW_ERR_CUDA, "packed_attention: cudaGetDevice failed");
  int err;
  if (!attr[dix]) {
    err = cuda_check(cudaFuncSetAttribute(packed_attn_kernel<D, F16>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                          pa::smem_bytes(D)),
                     "packed_attention smem attribute");
    if (err) return err;
    attr[dix] = true;
  }
  packed_attn_kernel<D, F16><<<grid, pa::THREADS, pa::smem_bytes(D), s>>>(tq, tk, tv, a, ta, st);
  if ((err = cuda_check(cudaGetLastError(), "packed_attention launch"))) return err;
  if (ta.n_split > 1) {
    const long long rows = (long long)a.tq * a.hq;
    err = launch_dependent("packed_attention merge launch", packed_merge_kernel<D, F16>, dim3((unsigned)((rows + 3) / 4)),
                           128, 0, s, a, ta);
  }
  return err;
}

// Query heads side by side in a tile: the divisor d of the group that needs the fewest 128-row tiles for sequences of
// `avg` tokens, ceil(avg / floor(128 / d)) tiles for each of hq / d head tiles; the larger divisor where two are equal.
// (Group 4: always 4. Group 6: 6 below 21 tokens, where one tile takes all heads, 2 for long sequences, which it fills
// to 128 of 128 rows; 6 heads fill 126.) Measured (us, this rule / always one head, 32 heads over 8, 128 wide, causal):
// 256 x 20 tokens 63 / 214, 128 x 50 44 / 115, 32 x 300 69 / 102, 8 x 1,000 89 / 96, 2 x 4,000 264 / 281.
static int pick_pack(int group, long long avg) {
  int best = 1;
  double best_cost = 1e300;
  for (int d = 1; d <= group && d <= 128; ++d) {
    if (group % d) continue;
    const long long toks = 128 / d;
    const double cost = (double)((avg + toks - 1) / toks) / d;
    if (cost <= best_cost * (1 + 1e-9)) {
      best_cost = cost;
      best = d;
    }
  }
  return best;
}

// Rows per kv head (queries x group) up to which a sequence is packed_split_kernel's, which has 16 in a unit: it reads the
// keys and values once for each unit, the tile kernel once for 256 rows. Measured (us, split / tile kernel, 8 kv heads,
// 128 wide) at 1, 16 and 32 rows: 32 x 16,384 keys 329 / 422, 341 / 431, 655 / 430; 8 x 4,096 33 / 42, 35 / 39, 42 / 37;
// 1 x 30,000 28 / 34, 31 / 37, 48 / 37; 1 x 1,000 8 / 11, 10 / 11, 11 / 11; 128 x 500 50 / 67, 61 / 71, 108 / 68.
constexpr int SHORT_ROWS = 16;

// The call's launch plan, from the host's numbers alone. The sequences' own lengths are on the device: where they may be
// of both kinds, both kernels are launched and each takes its own.
struct PackedPlan {
  bool tiles, split;
  long long split_rows;   // packed_split_kernel's limit
  TileArgs tile;
  long long windows;      // upper bound of the tile kernel's windows
  long long tile_floats, split_floats;  // workspace, fp32 values
};

static PackedPlan make_plan(long long tq, long long tk, int hq, int hk, int d, int n_seqs, int max_q, bool same_lens) {
  PackedPlan p{};
  const int group = hq / hk;
  const long long most = max_q > 0 && max_q < tq ? max_q : tq;
  p.tiles = most * group > SHORT_ROWS;
  // Both kernels where there may be short sequences among the others: not where all have the promised number of rows, nor
  // where they have as many keys as queries (a short one is one tile).
  p.split = !p.tiles || (n_seqs > 1 && !same_lens && !(max_q > 0 && (long long)n_seqs * max_q == tq));
  p.split_rows = p.tiles ? SHORT_ROWS : LLONG_MAX;  // (a sequence longer than max_q promised is still computed)
  if (p.split) p.split_floats = split_workspace_floats(d);
  if (!p.tiles) return p;
  const long long avg = n_seqs > 0 ? (tq + n_seqs - 1) / n_seqs : tq;
  p.tile.pack = pick_pack(group, avg > 0 ? avg : 1);
  p.tile.tile_toks = 128 / p.tile.pack;
  p.tile.head_tiles = hq / p.tile.pack;
  p.tile.short_rows = p.split ? SHORT_ROWS : 0;
  long long pairs = tq / (2 * p.tile.tile_toks) + n_seqs;
  if (pairs > tq) pairs = tq;
  p.windows = pairs * p.tile.head_tiles;
  // Few windows: their keys are cut into ranges while the windows fill the SMs at most once, from 8 key tiles (of the mean
  // sequence) on, 16 for two ranges, each of 2 tiles or more, and of 8 or more beyond 16 ranges; 32 at most (a lane each in
  // the merge).
  // Measured (us, with / without, 8 heads): 200 queries of 30,000 keys 44 / 417, of 8,192 25 / 120, of 1,000 16 / 23; 1,000
  // of 8,192 48 / 121. Ranges of 4 tiles at least: 20 at 200 of 1,000, 18 for 15 at 128 of 4,096; ranges from 4 tiles on: 17
  // for 15 at 500 of 500, 24 for 18 at 3 x 96 of 550; 16 ranges at most: 68 for 44 at 64 of 60,000; 32 of any length: 26.6
  // for 24.9 at 40 of 16,000; as many as fill the SMs twice: 62 for 50 at 1,000 of 8,192. Two ranges / one, 32 heads over 8:
  // 26.8 / 24.5 at 3 x 96 of 1,000, 33.8 / 38.4 of 2,000; 35.8 / 30.3 at 1,500 of 1,500 (12 heads).
  const long long key_tiles = n_seqs > 0 ? (tk / n_seqs + 127) / 128 : 0;
  long long split = p.windows > 0 ? num_sms() / p.windows : 1;
  if (split > key_tiles / 2) split = key_tiles / 2;
  if (split > 16 && split > key_tiles / 8) split = key_tiles / 8 > 16 ? key_tiles / 8 : 16;
  if (split > 32) split = 32;
  if (key_tiles < (split == 2 ? 16 : 8)) split = 1;
  p.tile.n_split = split < 1 ? 1 : (int)split;
  if (p.tile.n_split > 1) p.tile_floats = (long long)p.tile.n_split * tq * hq * (d + 2);
  return p;
}

static int check_packed(long long tq, long long tk, int hq, int hk, int d, int n_seqs) {
  const char* who = "packed_attention";
  if (d != 64 && d != 128) return set_error(LBW_ERR_SHAPE, "%s: head_dim %d (64 or 128)", who, d);
  if (hk < 1 || hq < hk || hq % hk || hq > 65536)
    return set_error(LBW_ERR_SHAPE, "%s: %d query heads over %d kv heads", who, hq, hk);
  // (Below 2^31 with room for a tile: rows and their products with heads are 32-bit in the kernels.)
  if (tq < 0 || tq >= 1ll << 31 || tk < 0 || tq * hq >= (1ll << 31) - 1024 || tk >= (1ll << 31) - 1024)
    return set_error(LBW_ERR_SHAPE, "%s: %lld query rows of %d heads, %lld key rows", who, tq, hq, tk);
  if (n_seqs < 0 || n_seqs >= 1 << 30) return set_error(LBW_ERR_SHAPE, "%s: %d sequences", who, n_seqs);
  return LBW_OK;
}

extern "C" {

int lbw_packed_attention_workspace(long long tq, long long tk, int hq, int hk, int head_dim, int n_seqs, int max_q,
                                   int same_lens, long long* bytes, int* launches) {
  if (!bytes) return set_error(LBW_ERR_INVALID, "packed_attention_workspace: null pointer");
  const int err = check_packed(tq, tk, hq, hk, head_dim, n_seqs);
  if (err) return err;
  const PackedPlan p = make_plan(tq, tk, hq, hk, head_dim, n_seqs, max_q, same_lens != 0);
  const bool any = tq > 0 && n_seqs > 0;
  *bytes = any ? (p.tile_floats + p.split_floats) * 4 : 0;
  if (launches) *launches = any ? (p.tiles ? 1 + (p.tile.n_split > 1) : 0) + (p.split ? 2 : 0) : 0;
  return LBW_OK;
}

int lbw_packed_attention(const lbw_packed_batch* batch, void* workspace, long long ws_bytes, void* stream) {
  if (!batch) return set_error(LBW_ERR_INVALID, "packed_attention: null batch");
  const auto& [q, q_tok, q_head, k, k_tok, k_head, v, v_tok, v_head, out, out_tok, out_head, cu_q, cu_k, k_lens, tq, tk,
               n_seqs, hq, hk, head_dim, dtype, causal, max_q, softmax_scale] = *batch;
  const char* who = "packed_attention";
  int err = check_packed(tq, tk, hq, hk, head_dim, n_seqs);
  if (err) return err;
  if (dtype != LBW_BF16 && dtype != LBW_FP16) return set_error(LBW_ERR_INVALID, "%s: dtype %d (bf16 or fp16)", who, dtype);
  const float scale_log2 = softmax_scale * 1.4426950408889634f;  // (log2 e: the exponentials are powers of two)
  if (!(scale_log2 > 0.f) || isinf(scale_log2))
    return set_error(LBW_ERR_INVALID, "%s: softmax_scale %g (a positive number)", who, (double)softmax_scale);
  if (tq == 0 || n_seqs == 0) return LBW_OK;
  if (!q || !out || !cu_q || !cu_k || (tk > 0 && (!k || !v))) return set_error(LBW_ERR_INVALID, "%s: null pointer", who);
  if (!aligned(cu_q, 4) || !aligned(cu_k, 4) || !aligned(k_lens, 4) || !aligned(out, 16) || out_tok % 8 || out_head % 8)
    return set_error(LBW_ERR_ALIGN, "%s: the output needs a 16-byte aligned pointer and strides", who);
  const PackedPlan p = make_plan(tq, tk, hq, hk, head_dim, n_seqs, max_q, cu_q == cu_k && !k_lens);
  if (p.windows * 32 >= 1ll << 31) return set_error(LBW_ERR_SHAPE, "%s: %lld windows", who, p.windows);
  const long long need = (p.tile_floats + p.split_floats) * 4;
  if (need > 0 && (!workspace || !aligned(workspace, 16) || ws_bytes < need))
    return set_error(LBW_ERR_INVALID, "%s: %lld bytes of 16-byte aligned workspace needed (%lld given)", who, need,
                     ws_bytes);
  // Rows are written while others are still computed from q, k and v; a row of out in the place of its own q is not.
  const ByteGrid o = ByteGrid::of(out, tq, out_tok, hq, out_head, head_dim, 2);
  if (overlap(o, ByteGrid::of(k, tk, k_tok, hk, k_head, head_dim, 2)) ||
      overlap(o, ByteGrid::of(v, tk, v_tok, hk, v_head, head_dim, 2)))
    return set_error(LBW_ERR_INVALID, "%s: out is k or v, or overlaps them", who);
  if (out == q ? (tq > 1 && q_tok != out_tok) || (hq > 1 && q_head != out_head)
               : overlap(o, ByteGrid::of(q, tq, q_tok, hq, q_head, head_dim, 2)))
    return set_error(LBW_ERR_INVALID, "%s: out is q with other strides, or overlaps it", who);
  int* st = device_status(&err);
  if (!st) return err;
  const PackedArgs a{cu_q, cu_k, k_lens, n_seqs, (int)tq, (int)tk, hq, hk, hq / hk, causal != 0,
                     scale_log2, out, out_tok, out_head};
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  float* ws = reinterpret_cast<float*>(workspace);
  if (p.tiles) {
    const CUtensorMapDataType ty = dtype == LBW_FP16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    CUtensorMap tmQ, tmK, tmV;
    if ((err = make_tmap_3d(&tmQ, q, ty, head_dim, hq, tq, q_head, q_tok, p.tile.pack, p.tile.tile_toks))) return err;
    if (tk > 0) {
      if ((err = make_tmap_3d(&tmK, k, ty, head_dim, hk, tk, k_head, k_tok, 1, pa::BN))) return err;
      if ((err = make_tmap_3d(&tmV, v, ty, head_dim, hk, tk, v_head, v_tok, 1, pa::BN))) return err;
    } else {
      tmK = tmV = tmQ;  // no key tile is ever loaded
    }
    TileArgs ta = p.tile;
    ta.part_o = ws;
    ta.part_ml = ws ? ws + (long long)ta.n_split * tq * hq * head_dim : nullptr;
    const dim3 grid((unsigned)(p.windows * ta.n_split));
    if (head_dim == 128)
      err = dtype == LBW_FP16 ? launch_tiles<128, true>(tmQ, tmK, tmV, a, ta, grid, st, s)
                              : launch_tiles<128, false>(tmQ, tmK, tmV, a, ta, grid, st, s);
    else
      err = dtype == LBW_FP16 ? launch_tiles<64, true>(tmQ, tmK, tmV, a, ta, grid, st, s)
                              : launch_tiles<64, false>(tmQ, tmK, tmV, a, ta, grid, st, s);
    if (err) return err;
  }
  if (!p.split) return LBW_OK;
  if (!aligned(q, 16) || q_tok % 8 || q_head % 8)
    return set_error(LBW_ERR_ALIGN, "%s: q needs a 16-byte aligned pointer and strides", who);
  return launch_split(k, k_tok, k_head, v, v_tok, v_head, a, head_dim, dtype, q, q_tok, q_head, p.split_rows,
                      p.tiles, ws + p.tile_floats, st, s);
}

}  // extern "C"
