// Attention over packed sequences on tcgen05: softmax(scale * Q K^T) V for every sequence of a batch, causal or not,
// with grouped heads, the sequences' starts and lengths read from device memory (lbw_packed_attention).
//
// Online softmax over 128-key tiles, fp32 scores, maxima, sums and accumulators; the probabilities are rounded once to
// the tensors' 16-bit type for the second product (half a step of 2^-8 or 2^-11 each, averaged over the keys).
//
// A CTA has up to two tiles of 128 query rows of one kv head. A row is a (token, query head) pair: `pack` query heads of
// the kv head's group sit side by side in a tile (row = token * pack + head), so that a tile of a short sequence is
// filled by the group's heads. The two tiles are neighbours in the sequence; the "primary" is the later one, whose rows
// see at least as many keys, and the secondary stops at its own last visible key tile.
//   warps 0-3 / 4-7  softmax of the primary / secondary tile (thread = row = TMEM lane)
//   warp 8           TMA producer: Q once, then K and V tiles through a 2-deep ring
//   warp 9           UMMA issuer, TMEM owner (S0 | S1 | O0 | O1)
//   warp 10          watches the K/V ring for the issuer (its arrivals fold "V(j) landed" and "K(j + 1) landed" into the
//                    primary's two P barriers) and clears the value rows past the sequence's last key: they belong to
//                    another sequence or to nobody, and 0 * NaN would reach the sum
// The pipeline (P written over S in TMEM and released in two halves, a running maximum that moves only when it grows by
// more than 2^8, a quarter of the exponentials on the FMA pipe) is the chunk attention's, see attn.cu for its figures.
// Rows that see no key (causal with fewer keys than queries, no keys at all) get zeros.
#include <limits.h>

#include "host_common.cuh"
#include "packed_common.cuh"
#include "packed_host.cuh"

namespace lbw {

namespace pa {
constexpr int BM = 128, BN = 128, STAGES = 2;
constexpr int HALF = 128 * 64 * 2;  // 128 rows x 64 16-bit values: one 128-byte swizzled box
constexpr int THREADS = 352;
constexpr int smem_bytes(int d) { return (2 + 2 * STAGES) * (d / 64) * HALF + 1024; }
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

// Two 2^x on the FMA pipe (see exp2_poly2), NaN kept.
LBW_DEV void exp2_poly2_nan(float x0, float x1, float& y0, float& y1) {
  float a, b;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(a) : "f"(x0), "f"(-126.f));
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(b) : "f"(x1), "f"(-126.f));
  const uint64_t x = f2_pack(a, b);
  const uint64_t t = f2_add(x, f2_pack(12582912.f, 12582912.f));
  const uint64_t n = f2_add(t, f2_pack(-12582912.f, -12582912.f));
  const uint64_t f = f2_fma(n, f2_pack(-1.f, -1.f), x);
  uint64_t p = f2_fma(f2_pack(0.054602623f, 0.054602623f), f, f2_pack(0.24192412f, 0.24192412f));
  p = f2_fma(p, f, f2_pack(0.69331646f, 0.69331646f));
  p = f2_fma(p, f, f2_pack(1.f, 1.f));
  float p0, p1, t0, t1;
  f2_unpack(p, p0, p1);
  f2_unpack(t, t0, t1);
  y0 = __int_as_float(__float_as_int(p0) + ((__float_as_int(t0) - 0x4B400000) << 23));
  y1 = __int_as_float(__float_as_int(p1) + ((__float_as_int(t1) - 0x4B400000) << 23));
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
  __shared__ __align__(8) uint64_t q_full, k_full[STAGES], k_empty[STAGES], v_full[STAGES], v_empty[STAGES], s_full[2],
      p_ready[2][2], o_done[2], done_bar;
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag;
  __shared__ int found;
  __shared__ PackedSeq found_seq;
  __shared__ int found_item;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (warp == 0) {
    int b = -1;
    long long l = 0;
    const bool ok = packed_find(a.n_seqs, (long long)(blockIdx.x / ta.head_tiles), [&](int i) {
      const PackedSeq s = packed_seq(a, i);
      if ((long long)s.nq * a.group <= ta.short_rows) return 0;
      return (s.nq + 2 * ta.tile_toks - 1) / (2 * ta.tile_toks);
    }, b, l);
    if (lane == 0) {
      found = ok;
      found_item = (int)l;
      if (ok) found_seq = packed_seq(a, b);
    }
  }
  if (threadIdx.x == 0) {
    mbar_init(&q_full, 1);
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&k_full[s], 1);
      mbar_init(&k_empty[s], 1);
      mbar_init(&v_full[s], 1);
      mbar_init(&v_empty[s], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_ready[i][0], 128 + (i == 0));  // P of keys 0..63 written (+ V(j) landed, for the primary)
      mbar_init(&p_ready[i][1], 128 + (i == 0));  // P of keys 64..127 written (+ K(j + 1) landed, for the primary)
      mbar_init(&o_done[i], 1);
    }
    mbar_init(&done_bar, 1);
    abort_flag = 0;
    fence_mbar_init();
  }
  __syncthreads();
  pdl_trigger();
  if (!found) return;  // the grid is an upper bound made from the row counts alone
  if (warp == 9) tmem_alloc(&tmem_slot, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  const Abort ab{status, &abort_flag};

  // The window: pairs of tiles of a sequence are taken from its end, where causal rows see most keys.
  const PackedSeq sq = found_seq;
  const int n_pairs = (sq.nq + 2 * ta.tile_toks - 1) / (2 * ta.tile_toks);
  const int tok0 = (n_pairs - 1 - found_item) * 2 * ta.tile_toks;
  const bool two = tok0 + ta.tile_toks < sq.nq;
  const int head0 = (int)(blockIdx.x % ta.head_tiles) * ta.pack;
  const int kv_head = head0 / a.group;
  int tile_tok[2];  // first token of the primary and of the secondary tile
  tile_tok[0] = two ? tok0 + ta.tile_toks : tok0;
  tile_tok[1] = tok0;
  const int keys_p = packed_visible(a, sq, min(tile_tok[0] + ta.tile_toks, sq.nq) - 1);
  const int keys_s = two ? packed_visible(a, sq, tok0 + ta.tile_toks - 1) : 0;
  const int all_p = (keys_p + BN - 1) / BN, all_s = (keys_s + BN - 1) / BN;
  // This CTA's key tiles [g0, g0 + n_p); the secondary takes the first n_s of them.
  const int g0 = (int)((long long)blockIdx.y * all_p / ta.n_split);
  const int n_p = (int)((long long)(blockIdx.y + 1) * all_p / ta.n_split) - g0;
  const int n_s = min(max(all_s - g0, 0), n_p);

  if (warp == 8) {
    // ---------------- producer ----------------
    if (lane == 0 && n_p > 0) {
      tma_prefetch_desc(&tmK);
      tma_prefetch_desc(&tmV);
      mbar_expect_tx(&q_full, (n_s > 0 ? 2 : 1) * NH * ta.pack * ta.tile_toks * 128);
      for (int i = 0; i < (n_s > 0 ? 2 : 1); ++i)
        for (int h = 0; h < NH; ++h)
          tma_load_3d(sQ + i * TILE + h * HALF, &tmQ, &q_full, h * 64, head0, sq.q0 + tile_tok[i]);
      int j = 0;
      for (; j < n_p; ++j) {
        const int s = j & 1;
        const uint32_t ph = (j >> 1) & 1;
        const int row = sq.k0 + (g0 + j) * BN;
        if (!mbar_wait(&k_empty[s], ph ^ 1, ab, 0x21)) break;
        mbar_expect_tx(&k_full[s], TILE);
        for (int h = 0; h < NH; ++h) tma_load_3d(sK + s * TILE + h * HALF, &tmK, &k_full[s], h * 64, kv_head, row);
        if (!mbar_wait(&v_empty[s], ph ^ 1, ab, 0x22)) {
          mbar_wait_drain(&k_full[s], ph);
          break;
        }
        mbar_expect_tx(&v_full[s], TILE);
        for (int h = 0; h < NH; ++h) tma_load_3d(sV + s * TILE + h * HALF, &tmV, &v_full[s], h * 64, kv_head, row);
      }
      // Let the last loads of each ring slot land before the CTA can exit.
      mbar_wait_drain(&q_full, 0);
      for (int i = (j > STAGES ? j - STAGES : 0); i < j; ++i) {
        mbar_wait_drain(&k_full[i & 1], (i >> 1) & 1);
        mbar_wait_drain(&v_full[i & 1], (i >> 1) & 1);
      }
    }
  } else if (warp == 9) {
    // ---------------- MMA issuer ----------------
    if (lane == 0 && n_p > 0) {
      const uint32_t idesc_s = F16 ? idesc_f16(BM, BN, 0, 0) : idesc_bf16(BM, BN, 0, 0);  // S = Q K^T, both K-major
      const uint32_t idesc_o = F16 ? idesc_f16(BM, D, 0, 1) : idesc_bf16(BM, D, 0, 1);    // O += P V, V MN-major
      const uint64_t dQ = sdesc_kmajor_sw128(smem_u32(sQ));
      const uint64_t dK = sdesc_kmajor_sw128(smem_u32(sK));
      const uint64_t dV = sdesc_mnmajor_sw128(smem_u32(sV), HALF);
      auto issue_s = [&](int i, int stage) {
        const uint64_t q = dQ + (uint64_t)((i * TILE) >> 4), k = dK + (uint64_t)((stage * TILE) >> 4);
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          const uint64_t off = (uint64_t)(((kk >> 2) * HALF + (kk & 3) * 32) >> 4);
          mma_f16_ss(tmem + i * 128, q + off, k + off, idesc_s, kk > 0);
        }
      };
      auto issue_pv = [&](int i, int stage, bool first, int half) {  // keys 0..63 (half 0) or 64..127
        const uint64_t v = dV + (uint64_t)((stage * TILE) >> 4);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int kk = half * 4 + q;
          mma_f16_ts(tmem + 256 + i * D, tmem + i * 128 + kk * 8, v + (uint64_t)((kk * 2048) >> 4), idesc_o,
                     !(first && kk == 0));
        }
      };
      bool ok = mbar_wait(&q_full, 0, ab, 0x31) && mbar_wait(&k_full[0], 0, ab, 0x32);
      if (ok) {
        tc_fence_after();
        issue_s(0, 0);
        tc_commit(&s_full[0]);
        if (n_s > 0) {
          issue_s(1, 0);
          tc_commit(&s_full[1]);
        }
        tc_commit(&k_empty[0]);
        for (int j = 0; j < n_p; ++j) {
          const int s = j & 1, s1 = (j + 1) & 1;
          const bool more = j + 1 < n_p;
          if (!mbar_wait(&p_ready[0][0], j & 1, ab, 0x34)) break;
          tc_fence_after();
          issue_pv(0, s, j == 0, 0);
          if (!mbar_wait(&p_ready[0][1], j & 1, ab, 0x37)) break;
          tc_fence_after();
          issue_pv(0, s, j == 0, 1);
          if (more) {
            issue_s(0, s1);
            tc_commit(&s_full[0]);
          } else {
            tc_commit(&o_done[0]);
          }
          if (j < n_s) {
            if (!mbar_wait(&p_ready[1][0], j & 1, ab, 0x36)) break;
            tc_fence_after();
            issue_pv(1, s, j == 0, 0);
            if (!mbar_wait(&p_ready[1][1], j & 1, ab, 0x38)) break;
            tc_fence_after();
            issue_pv(1, s, j == 0, 1);
          }
          tc_commit(&v_empty[s]);
          if (j + 1 < n_s) {
            issue_s(1, s1);
            tc_commit(&s_full[1]);
          } else if (j + 1 == n_s) {
            tc_commit(&o_done[1]);
          }
          if (more) tc_commit(&k_empty[s1]);
        }
      }
      tc_commit(&done_bar);
      mbar_wait_drain(&done_bar, 0);
    }
  } else if (warp == 10) {
    // ---------------- K/V watcher ----------------
    // In landing order, one phase of each P barrier at a time (see attn.cu).
    bool ok = n_p > 0;
    if (ok && lane == 0) ok = mbar_wait(&k_full[0], 0, ab, 0x60);
    ok = __shfl_sync(0xffffffffu, ok, 0);
    for (int j = 0; j < n_p && ok; ++j) {
      const int s = j & 1;
      if (lane == 0) ok = mbar_wait(&v_full[s], (j >> 1) & 1, ab, 0x61);
      ok = __shfl_sync(0xffffffffu, ok, 0);
      if (!ok) break;
      const int rows = sq.nk - (g0 + j) * BN;  // value rows of this tile that are the sequence's
      if (rows < BN) {
        for (int i = rows * 8 + lane; i < BN * 8; i += 32)
#pragma unroll
          for (int h = 0; h < NH; ++h)
            *reinterpret_cast<uint4*>(sV + s * TILE + h * HALF + i * 16) = make_uint4(0, 0, 0, 0);
        fence_async_shared();
        __syncwarp();
      }
      if (lane == 0) {
        mbar_arrive(&p_ready[0][0]);
        ok = j + 1 >= n_p || mbar_wait(&k_full[s ^ 1], ((j + 1) >> 1) & 1, ab, 0x62);
        if (ok) {
          mbar_arrive(&p_ready[0][1]);
          ok = mbar_wait(&p_ready[0][0], j & 1, ab, 0x63) && mbar_wait(&p_ready[0][1], j & 1, ab, 0x64);
        }
      }
      ok = __shfl_sync(0xffffffffu, ok, 0);
    }
  } else {
    // ---------------- softmax / correction / epilogue ----------------
    const int wg = warp >> 2;
    const int r0 = (warp & 3) * 32 + lane;  // row of the tile
    const uint32_t lane_off = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t tS = tmem + lane_off + wg * 128;
    const uint32_t tO = tmem + lane_off + 256 + wg * D;
    const int tok = tile_tok[wg] + r0 / ta.pack;
    const bool mine = (wg == 0 || two) && r0 < ta.pack * ta.tile_toks && tok < sq.nq;
    const int seen = mine ? packed_visible(a, sq, tok) - g0 * BN : 0;  // keys this row sees, from this CTA's first on
    const int n_tiles = wg == 0 ? n_p : n_s;
    float m = -INFINITY, l = 0.f;
    bool ok = true;
    for (int j = 0; j < n_tiles; ++j) {
      const int valid = seen - j * BN;
      if (!mbar_wait(&s_full[wg], j & 1, ab, 0x40 + wg)) { ok = false; break; }
      tc_fence_after();
      uint32_t r[128];
      tmem_ld32(tS + 0, *reinterpret_cast<uint32_t(*)[32]>(&r[0]));
      tmem_ld32(tS + 32, *reinterpret_cast<uint32_t(*)[32]>(&r[32]));
      tmem_ld32(tS + 64, *reinterpret_cast<uint32_t(*)[32]>(&r[64]));
      tmem_ld32(tS + 96, *reinterpret_cast<uint32_t(*)[32]>(&r[96]));
      tmem_ld_wait();
      float* sv = reinterpret_cast<float*>(r);
      const bool whole = __all_sync(0xffffffffu, valid >= BN || !mine);
      if (!whole) {  // the diagonal, or the sequence's last tile
#pragma unroll
        for (int e = 0; e < BN; ++e)
          if (e >= valid) sv[e] = -INFINITY;
      }
      float t8[8];
#pragma unroll
      for (int q = 0; q < 8; ++q) t8[q] = sv[q];
#pragma unroll
      for (int e = 8; e < 120; e += 16)
#pragma unroll
        for (int q = 0; q < 8; ++q) t8[q] = fmax3(t8[q], sv[e + q], sv[e + 8 + q]);
#pragma unroll
      for (int q = 0; q < 8; ++q) t8[q] = fmaxf(t8[q], sv[120 + q]);
      const float mx =
          fmaxf(fmax3(t8[0], t8[1], t8[2]), fmax3(fmax3(t8[3], t8[4], t8[5]), t8[6], t8[7])) * a.scale_log2;
      const float m_new = fmaxf(m, mx);
      float alpha = 1.f;
      bool rescale = false;
      if (j == 0) {
        m = m_new;
      } else {
        const bool need = m_new > m + 8.f;
        rescale = __any_sync(0xffffffffu, need);
        if (need) {
          alpha = fast_exp2(m - m_new);
          l *= alpha;
          m = m_new;
        }
      }
      // A row that has seen no key yet has m = -inf: its scores are all -inf and p = 2^(-inf - 0) = 0.
      const float m_use = m == -INFINITY ? 0.f : m;
      const uint64_t a2 = f2_pack(a.scale_log2, a.scale_log2), b2 = f2_pack(-m_use, -m_use);
      uint64_t lsum[4] = {0ull, 0ull, 0ull, 0ull};
      if (whole) {
#pragma unroll
        for (int cc = 0; cc < 4; ++cc) {
          if (cc == 2 && !rescale) {  // keys 0..63 are in TMEM: let P V start on them (warp-uniform)
            tmem_st_wait();
            tc_fence_before();
            mbar_arrive(&p_ready[wg][0]);
          }
          uint32_t pk[16];
#pragma unroll
          for (int e = 0; e < 32; e += 2) {
            const int col = cc * 32 + e;
            float x0, x1, p0, p1;
            f2_unpack(f2_fma(f2_pack(sv[col], sv[col + 1]), a2, b2), x0, x1);
            if (((e >> 1) & 3) == 3) {
              exp2_poly2_nan(x0, x1, p0, p1);
            } else {
              p0 = fast_exp2(x0);
              p1 = fast_exp2(x1);
            }
            lsum[(e >> 1) & 3] = f2_add(lsum[(e >> 1) & 3], f2_pack(p0, p1));
            pk[e >> 1] = pack_16<F16>(p0, p1);
          }
          tmem_st16(tS + cc * 16, pk);
        }
      } else {
#pragma unroll
        for (int cc = 0; cc < 4; ++cc) {
          uint32_t pk[16];
#pragma unroll
          for (int e = 0; e < 32; e += 2) {
            const int col = cc * 32 + e;
            float x0, x1;
            f2_unpack(f2_fma(f2_pack(sv[col], sv[col + 1]), a2, b2), x0, x1);
            const float p0 = fast_exp2(x0), p1 = fast_exp2(x1);
            lsum[(e >> 1) & 3] = f2_add(lsum[(e >> 1) & 3], f2_pack(p0, p1));
            pk[e >> 1] = pack_16<F16>(p0, p1);
          }
          tmem_st16(tS + cc * 16, pk);
        }
      }
      float l0, l1, l2, l3;
      f2_unpack(f2_add(lsum[0], lsum[1]), l0, l1);
      f2_unpack(f2_add(lsum[2], lsum[3]), l2, l3);
      l += (l0 + l1) + (l2 + l3);
      if (rescale) {  // warp-uniform
#pragma unroll 1
        for (int cc = 0; cc < D / 32; ++cc) {
          uint32_t o[32];
          tmem_ld32(tO + cc * 32, o);
          tmem_ld_wait();
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
          tmem_st32(tO + cc * 32, o);
        }
      }
      tmem_st_wait();
      tc_fence_before();
      if (rescale || !whole) mbar_arrive(&p_ready[wg][0]);
      mbar_arrive(&p_ready[wg][1]);
    }
    if (n_tiles > 0 && ok) ok = mbar_wait(&o_done[wg], 0, ab, 0x48 + wg);
    if (ok && (wg == 0 || two)) {
      tc_fence_after();
      const long long row = (long long)(sq.q0 + tok);
      const int head = head0 + r0 % ta.pack;
      if (ta.n_split > 1) {
        // unnormalised fp32 row and its (m, l); a row without a key leaves only l = 0
        const long long pr = ((long long)blockIdx.y * a.tq + row) * a.hq + head;
        if (mine) *reinterpret_cast<float2*>(ta.part_ml + pr * 2) = make_float2(m, l);
        float* dst = ta.part_o + pr * D;
        if (n_tiles > 0) {
#pragma unroll 1
          for (int cc = 0; cc < D / 32; ++cc) {
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
        const bool none = l == 0.f;  // no key seen: zeros (NaN sums stay NaN)
        const float inv = 1.f / l;
        uint16_t* dst = reinterpret_cast<uint16_t*>(a.out) + row * a.os_tok + head * a.os_head;
#pragma unroll 1
        for (int cc = 0; cc < D / 32; ++cc) {
          uint32_t r[32];
          if (n_tiles > 0) {
            tmem_ld32(tO + cc * 32, r);
            tmem_ld_wait();
          }
          uint32_t pk[16];
#pragma unroll
          for (int e = 0; e < 32; e += 2)
            pk[e >> 1] = none ? 0u : pack_16<F16>(__uint_as_float(r[e]) * inv, __uint_as_float(r[e + 1]) * inv);
          if (mine) {
#pragma unroll
            for (int q = 0; q < 4; ++q)
              reinterpret_cast<uint4*>(dst + cc * 32)[q] = make_uint4(pk[4 * q], pk[4 * q + 1], pk[4 * q + 2], pk[4 * q + 3]);
          }
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 9) tmem_dealloc(tmem, 512);
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
  const long long step = (long long)a.tq * a.hq;
  float M = -INFINITY;
  for (int z = 0; z < ta.n_split; ++z) M = fmaxf(M, ta.part_ml[(z * step + wid) * 2]);
  constexpr int PER = D / 32;
  float L = 0.f, acc[PER] = {};
  for (int z = 0; z < ta.n_split; ++z) {
    const float2 ml = *reinterpret_cast<const float2*>(ta.part_ml + (z * step + wid) * 2);
    if (ml.y == 0.f) continue;  // no key of this range is visible: nothing was written
    const float w = exp2f(ml.x - M);
    L += w * ml.y;
    const float* o = ta.part_o + (z * step + wid) * D + lane * PER;
#pragma unroll
    for (int i = 0; i < PER; ++i) acc[i] += w * o[i];
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
// to 128 of 128 rows; 6 heads fill 126.)
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

// Rows per kv head (queries x group) up to which a sequence is packed_split_kernel's, which has 16 in a unit.
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
  p.split = !p.tiles || (n_seqs > 1 && !same_lens);  // (as many keys as queries: a short sequence is one tile)
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
  const long long key_tiles = (tk + 127) / 128;
  long long split = p.windows > 0 ? num_sms() / p.windows : 1;
  if (split > key_tiles / 4) split = key_tiles / 4;
  if (split > 16) split = 16;
  p.tile.n_split = split < 1 ? 1 : (int)split;
  if (p.tile.n_split > 1) p.tile_floats = (long long)p.tile.n_split * tq * hq * (d + 2);
  return p;
}

static int check_packed(long long tq, long long tk, int hq, int hk, int d, int n_seqs) {
  const char* who = "packed_attention";
  if (d != 64 && d != 128) return set_error(LBW_ERR_SHAPE, "%s: head_dim %d (64 or 128)", who, d);
  if (hk < 1 || hq < hk || hq % hk || hq > 65536)
    return set_error(LBW_ERR_SHAPE, "%s: %d query heads over %d kv heads", who, hq, hk);
  if (tq < 0 || tk < 0 || tq >= 1ll << 31 || tk >= 1ll << 31)
    return set_error(LBW_ERR_SHAPE, "%s: %lld query rows, %lld key rows", who, tq, tk);
  if (n_seqs < 0) return set_error(LBW_ERR_SHAPE, "%s: %d sequences", who, n_seqs);
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

int lbw_packed_attention(const void* q, long long q_tok, long long q_head, const void* k, long long k_tok,
                         long long k_head, const void* v, long long v_tok, long long v_head, void* out,
                         long long out_tok, long long out_head, const int* cu_q, const int* cu_k, const int* k_lens,
                         int n_seqs, long long tq, long long tk, int hq, int hk, int head_dim, int dtype, int causal,
                         float softmax_scale, int max_q, void* workspace, long long ws_bytes, void* stream) {
  const char* who = "packed_attention";
  int err = check_packed(tq, tk, hq, hk, head_dim, n_seqs);
  if (err) return err;
  if (dtype != LBW_BF16 && dtype != LBW_FP16) return set_error(LBW_ERR_INVALID, "%s: dtype %d (bf16 or fp16)", who, dtype);
  if (!(softmax_scale > 0.f) || isinf(softmax_scale))
    return set_error(LBW_ERR_INVALID, "%s: softmax_scale %g (a positive number)", who, (double)softmax_scale);
  if (tq == 0 || n_seqs == 0) return LBW_OK;
  if (!q || !out || !cu_q || !cu_k || (tk > 0 && (!k || !v))) return set_error(LBW_ERR_INVALID, "%s: null pointer", who);
  if (!aligned(cu_q, 4) || !aligned(cu_k, 4) || !aligned(k_lens, 4) || !aligned(out, 16) || out_tok % 8 || out_head % 8)
    return set_error(LBW_ERR_ALIGN, "%s: the output needs a 16-byte aligned pointer and strides", who);
  const PackedPlan p = make_plan(tq, tk, hq, hk, head_dim, n_seqs, max_q, cu_q == cu_k && !k_lens);
  if (p.windows >= 1ll << 31) return set_error(LBW_ERR_SHAPE, "%s: %lld windows", who, p.windows);
  const long long need = (p.tile_floats + p.split_floats) * 4;
  if (need > 0 && (!workspace || !aligned(workspace, 16) || ws_bytes < need))
    return set_error(LBW_ERR_INVALID, "%s: %lld bytes of 16-byte aligned workspace needed (%lld given)", who, need,
                     ws_bytes);
  int* st = device_status(&err);
  if (!st) return err;
  const PackedArgs a{cu_q, cu_k, k_lens, n_seqs, (int)tq, (int)tk, hq, hk, hq / hk, causal != 0,
                     softmax_scale * 1.4426950408889634f, out, out_tok, out_head};
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
    const dim3 grid((unsigned)p.windows, ta.n_split);
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
