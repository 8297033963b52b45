// Attention of few query rows over many keys: the sequences of a packed batch that have at most 16 rows per kv head
// (single tokens, a few drafted ones), whose time is the reading of their keys and values.
//
// A unit is the 16 rows (token, query head of the kv head's group) of one sequence and kv head against its keys, in
// tiles of 64. All tiles of all units form one list, and each CTA (one per SM) takes an equal run of it, so the bytes
// are spread evenly whatever the lengths are; a unit that crosses CTAs leaves fp32 partial rows with their maximum and
// sum, joined by packed_join_kernel. Every CTA finds its run from the device arrays by itself (packed_locate), so the
// host needs no lengths and a captured call follows new ones.
//   warp 8       producer: K and V tiles by TMA through a ring of 32 KB stages (head_dim 128)
//   warps 0-7    two groups of four take the stages in turn; each warp has 16 of a stage's 64 keys and its own running
//                maximum, sums and 16 x D accumulator (mma.sync m16n8k16), joined over the 8 warps at the unit's end
// mma.sync and not tcgen05: the rows of a unit fill an eighth of a 128-row tile, and 16 rows are enough to read at full
// rate (a warp spends ~150 instructions on 16 keys = 8 KB; the SM's share of the memory rate is 23 bytes a clock).
// Bound: the bytes of K and V. Measured (B200, bf16, 128-wide heads, 8 kv heads, both kernels, replayed from a graph):
// 32 sequences of 16,384 keys 326 us with 1 row per kv head, 336 with 16 (6.6 and 6.4 TB/s: a plain copy's rate);
// 128 x 500 keys 50 and 60 us (5.3 and 4.4 TB/s: 7 units a CTA, whose ends - the join of 8 warps, masks, the next Q - are
// not all hidden behind 8 tiles of loads); 1 x 30,000 keys 28 and 31 us (4.3 and 4.0 TB/s); 1 x 1,000 keys 8.2 and 10.4 us,
// which is two launches, the look-up of the sequences and one trip to memory.
#include "host_common.cuh"
#include "packed_common.cuh"
#include "packed_host.cuh"

namespace lbw {

namespace ps {
constexpr int KEYS = 64, ROWS = 16, WARPS = 8;
constexpr int THREADS = (WARPS + 1) * 32;
constexpr int HALF = KEYS * 128;  // 64 keys x 64 16-bit values
__host__ __device__ constexpr int stages(int d) { return d == 128 ? 6 : 8; }
__host__ __device__ constexpr int smem_bytes(int d) { return stages(d) * 2 * (d / 64) * HALF + WARPS * 8 * d * 4 + 1024; }
}  // namespace ps

LBW_DEV void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
LBW_DEV void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
template <bool F16>
LBW_DEV void mma_16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (F16)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// (units, tiles) of sequence b: row tiles x kv heads, and those times its key tiles. (0, 0) if it is not this kernel's.
LBW_DEV longlong2 split_count(const PackedArgs& a, long long max_rows, int b) {
  const PackedSeq s = packed_seq(a, b);
  const long long rows = (long long)s.nq * a.group;
  if (rows == 0 || rows > max_rows) return make_longlong2(0, 0);
  const long long units = (rows + ps::ROWS - 1) / ps::ROWS * a.hk;
  return make_longlong2(units, units * ((s.nk + ps::KEYS - 1) / ps::KEYS));
}

// Key tiles of each CTA: an equal share. (A minimum of 2 or 4 measures the same or slower: 1 x 1,000 keys 8.8 / 9.5 us
// against 8.5, 4 x 500 keys of 2 kv heads 8.7 / 9.3 against 8.2.)
LBW_DEV long long split_share(long long total, int ctas) {
  const long long w = (total + ctas - 1) / ctas;
  return w < 1 ? 1 : w;
}

// Where a CTA stands in the list: a unit of sequence b, from its key tile t0 on.
struct SplitUnit {
  PackedSeq sq;
  int b, n_tiles, units, unit, t0;
};

// The next unit, in the sequence or in the next one that has any; n_tiles = 0 past the last.
LBW_DEV void split_advance(const PackedArgs& a, long long max_rows, SplitUnit& u) {
  u.t0 = 0;
  if (++u.unit < u.units) return;
  u.unit = 0;
  while (++u.b < a.n_seqs) {
    const longlong2 n = split_count(a, max_rows, u.b);
    if (n.y == 0) continue;
    u.sq = packed_seq(a, u.b);
    u.n_tiles = (u.sq.nk + ps::KEYS - 1) / ps::KEYS;
    u.units = (int)n.x;
    return;
  }
  u.n_tiles = 0;
}

template <int D, bool F16>
__global__ void __launch_bounds__(ps::THREADS, 1)
    packed_split_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                        const __grid_constant__ PackedArgs a, const uint16_t* __restrict__ q, long long qs_tok,
                        long long qs_head, long long max_rows, float* __restrict__ part_o, float* __restrict__ part_ml,
                        int* status) {
  using namespace ps;
  constexpr int STAGES = stages(D), NH = D / 64, TILE = NH * HALF;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float* s_o = reinterpret_cast<float*>(smem + STAGES * 2 * TILE);  // [8 warps][8 rows][D]
  __shared__ float2 s_ml[WARPS][ROWS];
  __shared__ __align__(8) uint64_t full[STAGES], empty[STAGES];
  __shared__ int abort_flag;
  __shared__ longlong2 tmp[WARPS + 2];
  __shared__ PackedAt at_s;
  __shared__ SplitUnit next_s;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 4);
    }
    abort_flag = 0;
    fence_mbar_init();
  }
  const PackedAt at = packed_locate<THREADS, true>(
      a, [&](int b) { return split_count(a, max_rows, b); },
      [&](long long total) { return (long long)blockIdx.x * split_share(total, gridDim.x); }, tmp, &at_s);
  const long long share = split_share(at.total_y, gridDim.x);
  const long long first = blockIdx.x * share;
  pdl_trigger();
  if (at.seq < 0 || at.sq.nk == 0) {  // no tiles left for this CTA
    pdl_wait();
    return;
  }
  const long long last = min(first + share, at.total_y);
  const Abort ab{status, &abort_flag};
  SplitUnit u;
  u.b = at.seq;
  u.sq = at.sq;
  u.n_tiles = (u.sq.nk + KEYS - 1) / KEYS;
  u.units = (int)(((long long)u.sq.nq * a.group + ROWS - 1) / ROWS * a.hk);
  u.unit = (int)(at.local / u.n_tiles);
  u.t0 = (int)(at.local % u.n_tiles);

  if (warp == WARPS) {
    // ---------------- producer ----------------
    if (lane == 0) {
      tma_prefetch_desc(&tmK);
      tma_prefetch_desc(&tmV);
      int j = 0;
      bool ok = true;
      for (long long g = first; g < last && ok;) {
        const int n = (int)min((long long)(u.n_tiles - u.t0), last - g);
        if (n <= 0) break;  // only if the lengths were changed under the kernel
        const int head = u.unit % a.hk;
        for (int t = u.t0; t < u.t0 + n; ++t, ++j) {
          const int s = j % STAGES;
          if (!mbar_wait(&empty[s], ((j / STAGES) & 1) ^ 1, ab, 0x71)) { ok = false; break; }
          uint8_t* st = smem + s * 2 * TILE;
          mbar_expect_tx(&full[s], 2 * TILE);
          for (int h = 0; h < NH; ++h) tma_load_3d(st + h * HALF, &tmK, &full[s], h * 64, head, u.sq.k0 + t * KEYS);
          for (int h = 0; h < NH; ++h) tma_load_3d(st + TILE + h * HALF, &tmV, &full[s], h * 64, head, u.sq.k0 + t * KEYS);
        }
        g += n;
        if (g < last) split_advance(a, max_rows, u);
      }
      for (int i = (j > STAGES ? j - STAGES : 0); i < j; ++i) mbar_wait_drain(&full[i % STAGES], (i / STAGES) & 1);
    }
    pdl_wait();  // (it reads nothing of the kernels before it in the call: only its end comes after theirs)
    return;
  }

  // ---------------- consumers ----------------
  const int grp = warp >> 2, kb = (warp & 3) * 16;  // this warp's keys of a stage
  const int r_lo = lane >> 2, c0 = (lane & 3) * 2;
  uint8_t* smem_q = reinterpret_cast<uint8_t*>(s_o);
  const int q_row = threadIdx.x / (D / 8), q_chunk = threadIdx.x % (D / 8);
  auto load_q = [&](const SplitUnit& w) {
    const int row0 = w.unit / a.hk * ROWS, r = row0 + q_row;
    if (q_row >= ROWS || r >= w.sq.nq * a.group) return make_uint4(0, 0, 0, 0);
    const int tok = r / a.group, head = w.unit % a.hk * a.group + r - tok * a.group;
    return *reinterpret_cast<const uint4*>(q + (long long)(w.sq.q0 + tok) * qs_tok + (long long)head * qs_head + q_chunk * 8);
  };
  uint4 q_piece;
  bool have_q = false;
  int j = 0;
  for (long long g = first; g < last;) {
    const PackedSeq sq = u.sq;
    const int t0 = u.t0, n = (int)min((long long)(u.n_tiles - u.t0), last - g);
    if (n <= 0) break;  // as above; the same for all consumers, which follow one thread's reading
    const int head = u.unit % a.hk, row0 = u.unit / a.hk * ROWS;
    const int rows = min(sq.nq * a.group - row0, ROWS);
    int seen[2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
      seen[i] = r_lo + 8 * i < rows ? packed_visible(a, sq, (row0 + r_lo + 8 * i) / a.group) : 0;
    // The unit's Q, a 16-byte piece per thread, through shared memory into the fragments of all warps (4-byte loads of 8
    // rows at a time by every warp took 1 us of a unit's 9).
    if (!have_q) q_piece = load_q(u);
    if (q_row < ROWS) *reinterpret_cast<uint4*>(smem_q + q_row * D * 2 + ((q_chunk ^ (q_row & 7)) << 4)) = q_piece;
    asm volatile("bar.sync 1, 256;" ::: "memory");
    uint32_t qf[D / 16][4];
#pragma unroll
    for (int st = 0; st < D / 16; ++st) {
      const int r = lane & 15, ch = st * 2 + (lane >> 4);
      ldsm4(qf[st], smem_u32(smem_q) + r * D * 2 + ((ch ^ (r & 7)) << 4));
    }
    asm volatile("bar.sync 1, 256;" ::: "memory");  // (its place is the join's)
    const int all_see = packed_visible(a, sq, row0 / a.group);  // keys that every row of the unit sees
    float o[D / 8][4];
#pragma unroll
    for (int i = 0; i < D / 8; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[i][e] = 0.f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
    for (int t = t0; t < t0 + n; ++t, ++j) {
      if ((j & 1) != grp) continue;
      const int s = j % STAGES;
      mbar_wait(&full[s], (j / STAGES) & 1, ab, 0x72);  // (after a timeout the loop runs on: the block meets below)
      const uint32_t sk = smem_u32(smem + s * 2 * TILE), sv = sk + TILE;
      const int key0 = t * KEYS + kb;
      const int left = sq.nk - key0;  // keys of this warp that are the sequence's
      if (left < 16) {                // the value rows behind them may hold anything, NaN too
        for (int i = max(left, 0) * 8 + lane; i < 16 * 8; i += 32)
#pragma unroll
          for (int h = 0; h < NH; ++h)
            *reinterpret_cast<uint4*>(smem + s * 2 * TILE + TILE + h * HALF + kb * 128 + i * 16) = make_uint4(0, 0, 0, 0);
        fence_async_shared();
        __syncwarp();
      }
      float c[2][4];
#pragma unroll
      for (int nb = 0; nb < 2; ++nb) {
#pragma unroll
        for (int e = 0; e < 4; ++e) c[nb][e] = 0.f;
#pragma unroll
        for (int c4 = 0; c4 < D / 32; ++c4) {
          uint32_t f[4];
          const int key = kb + nb * 8 + (lane & 7), ch = c4 * 4 + (lane >> 3);
          ldsm4(f, sk + (ch >> 3) * HALF + key * 128 + (((ch & 7) ^ (key & 7)) << 4));
          mma_16816<F16>(c[nb], qf[c4 * 2], f[0], f[1]);
          mma_16816<F16>(c[nb], qf[c4 * 2 + 1], f[2], f[3]);
        }
      }
      if (key0 + 16 > all_see) {
#pragma unroll
        for (int nb = 0; nb < 2; ++nb)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (key0 + nb * 8 + c0 + (e & 1) >= seen[e >> 1]) c[nb][e] = -INFINITY;
      }
      uint32_t p[4];
      float alpha[2];
      bool moved = false;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float mx = fmaxf(fmaxf(c[0][2 * i], c[0][2 * i + 1]), fmaxf(c[1][2 * i], c[1][2 * i + 1]));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2)) * a.scale_log2;
        alpha[i] = 1.f;
        if (mx > m[i] + 8.f) {  // the running maximum moves only when it grows by more than 2^8
          alpha[i] = fast_exp2(m[i] - mx);
          m[i] = mx;
          l[i] *= alpha[i];
          moved = true;
        }
        const float mu = m[i] == -INFINITY ? 0.f : m[i];
        const float p0 = fast_exp2(fmaf(c[0][2 * i], a.scale_log2, -mu));
        const float p1 = fast_exp2(fmaf(c[0][2 * i + 1], a.scale_log2, -mu));
        const float p2 = fast_exp2(fmaf(c[1][2 * i], a.scale_log2, -mu));
        const float p3 = fast_exp2(fmaf(c[1][2 * i + 1], a.scale_log2, -mu));
        l[i] += (p0 + p1) + (p2 + p3);
        p[i] = pack_16<F16>(p0, p1);
        p[i + 2] = pack_16<F16>(p2, p3);
      }
      if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
        for (int i = 0; i < D / 8; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[i][e] *= alpha[e >> 1];
      }
      // Where rows do not see a key, its value must not reach them, and 0 * NaN would: such keys go by hand.
      bool by_hand = false;
      if (all_see < sq.nk && key0 + 16 > all_see) {
        constexpr uint32_t EXP = F16 ? 0x7c00u : 0x7f80u;
        for (int i = max(all_see - key0, 0) * 8 + lane; i < min(left, 16) * 8; i += 32)
#pragma unroll
          for (int h = 0; h < NH; ++h) {
            const uint4 x = *reinterpret_cast<const uint4*>(smem + s * 2 * TILE + TILE + h * HALF + kb * 128 + i * 16);
            const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) by_hand |= (w[e] & EXP) == EXP || (w[e] >> 16 & EXP) == EXP;
          }
        by_hand = __any_sync(0xffffffffu, by_hand);
      }
      if (by_hand) {
#pragma unroll 1
        for (int kk = 0; kk < 16; ++kk) {
          const int key = kb + kk, from = (lane & ~3) | (kk >> 1 & 3);
          const uint32_t w0 = __shfl_sync(0xffffffffu, kk < 8 ? p[0] : p[2], from) >> (kk & 1) * 16;
          const uint32_t w1 = __shfl_sync(0xffffffffu, kk < 8 ? p[1] : p[3], from) >> (kk & 1) * 16;
          const float p0 = unpack_16<F16>(w0), p1 = unpack_16<F16>(w1);
          const bool in0 = key0 + kk < seen[0], in1 = key0 + kk < seen[1];
#pragma unroll
          for (int ch = 0; ch < D / 8; ++ch) {
            const uint32_t x = *reinterpret_cast<const uint32_t*>(smem + s * 2 * TILE + TILE + (ch >> 3) * HALF + key * 128 +
                                                                  (((ch & 7) ^ (key & 7)) << 4) + c0 * 2);
            const float v0 = unpack_16<F16>(x), v1 = unpack_16<F16>(x >> 16);
            if (in0) o[ch][0] = fmaf(p0, v0, o[ch][0]), o[ch][1] = fmaf(p0, v1, o[ch][1]);
            if (in1) o[ch][2] = fmaf(p1, v0, o[ch][2]), o[ch][3] = fmaf(p1, v1, o[ch][3]);
          }
        }
      } else
#pragma unroll
      for (int ch = 0; ch < D / 8; ch += 2) {
        uint32_t f[4];
        const int key = kb + ((lane >> 3) & 1) * 8 + (lane & 7), cc = ch + (lane >> 4);
        ldsm4_t(f, sv + (cc >> 3) * HALF + key * 128 + (((cc & 7) ^ (key & 7)) << 4));
        mma_16816<F16>(o[ch], p, f[0], f[1]);
        mma_16816<F16>(o[ch + 1], p, f[2], f[3]);
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[s]);
    }

    // The next unit's Q is on its way during the join, if it is of the same sequence.
    have_q = g + n < last && u.unit + 1 < u.units;
    if (have_q) {
      SplitUnit w = u;
      ++w.unit;
      q_piece = load_q(w);
    }
    // The unit's end: join the 8 warps, 8 rows at a time.
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
      l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
      if ((lane & 3) == 0) s_ml[warp][r_lo + 8 * i] = make_float2(m[i], l[i]);
    }
    const bool begins = t0 == 0, ends = t0 + n == u.n_tiles;
    const long long slot = begins ? 2ll * blockIdx.x + 1 : 2ll * blockIdx.x;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (8 * i >= rows) break;
      if (8 * i + r_lo < rows) {  // (8 columns' place turned by the row: the 8 rows of a store would be in the same banks)
#pragma unroll
        for (int ch = 0; ch < D / 8; ++ch)
          *reinterpret_cast<float2*>(s_o + (warp * 8 + r_lo) * D + (ch ^ r_lo) * 8 + c0) =
              make_float2(o[ch][2 * i], o[ch][2 * i + 1]);
      }
      asm volatile("bar.sync 1, 256;" ::: "memory");
      const int r = threadIdx.x >> 5;  // a warp per row, D / 32 values per lane
      if (8 * i + r < rows) {
        float M = -INFINITY;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) M = fmaxf(M, s_ml[w][8 * i + r].x);
        constexpr int PER = D / 32;
        float L = 0.f, acc[PER] = {};
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
          const float2 ml = s_ml[w][8 * i + r];
          const float k = ml.x == -INFINITY ? 0.f : fast_exp2(ml.x - M);
          L += k * ml.y;
#pragma unroll
          for (int e = 0; e < PER; ++e) acc[e] += k * s_o[(w * 8 + r) * D + ((lane * PER) ^ (r * 8)) + e];
        }
        if (begins && ends) {
          const int tok = (row0 + 8 * i + r) / a.group, hh = head * a.group + (row0 + 8 * i + r) % a.group;
          uint32_t* dst = reinterpret_cast<uint32_t*>(reinterpret_cast<uint16_t*>(a.out) +
                                                      (long long)(sq.q0 + tok) * a.os_tok + hh * a.os_head + lane * PER);
          const float inv = L == 0.f ? 0.f : 1.f / L;
#pragma unroll
          for (int e = 0; e < PER; e += 2) dst[e / 2] = pack_16<F16>(acc[e] * inv, acc[e + 1] * inv);
        } else {
          float* dst = part_o + (slot * ROWS + 8 * i + r) * D + lane * PER;
#pragma unroll
          for (int e = 0; e < PER; ++e) dst[e] = acc[e];
          if (lane == 0) *reinterpret_cast<float2*>(part_ml + (slot * ROWS + 8 * i + r) * 2) = make_float2(M, L);
        }
      }
      if (threadIdx.x == 0 && (i == 1 || rows <= 8)) {
        SplitUnit w = u;
        if (g + n < last) split_advance(a, max_rows, w);
        next_s = w;
      }
      asm volatile("bar.sync 1, 256;" ::: "memory");
    }
    g += n;
    u = next_s;
  }
  pdl_wait();
}

// Joins the units that crossed CTAs and writes the rows of sequences without keys. Block (unit, y) has the y-th share of
// the unit's rows, a warp per row, or two or four warps where the share is fewer rows than warps (`W`: they take the
// row's parts in turn), with the loads of 8 parts in flight. Many blocks for few units: one sequence of 8 kv heads over
// 148 CTAs leaves 19 parts a row, and one block per unit reading 16 rows of them one by one took 20 us of 55.
template <int D, bool F16>
__global__ void __launch_bounds__(128) packed_join_kernel(const __grid_constant__ PackedArgs a, long long max_rows,
                                                          int ctas, const float* __restrict__ part_o,
                                                          const float* __restrict__ part_ml) {
  constexpr int PER = D / 32, UN = 8;
  __shared__ longlong2 tmp[5];
  __shared__ PackedAt at_s;
  __shared__ float s_acc[4][D], s_l[4];
  const PackedAt at = packed_locate<128, false>(
      a, [&](int b) { return split_count(a, max_rows, b); }, [&](long long) { return (long long)blockIdx.x; }, tmp,
      &at_s);
  pdl_wait();
  if (at.seq < 0) return;
  const PackedSeq sq = at.sq;
  const int n_tiles = (sq.nk + ps::KEYS - 1) / ps::KEYS;
  const long long share = split_share(at.total_y, ctas);
  const long long t_first = at.before_y + at.local * n_tiles;
  const int c0 = (int)min(t_first / share, ctas - 1ll);
  const int c1 = n_tiles ? (int)min((t_first + n_tiles - 1) / share, ctas - 1ll) : c0 - 1;
  if (c0 == c1) return;
  const int head = (int)(at.local % a.hk), row0 = (int)(at.local / a.hk) * ps::ROWS;
  const int rows = min(sq.nq * a.group - row0, ps::ROWS);
  const int rows_y = (rows + gridDim.y - 1) / gridDim.y;
  const int r0 = blockIdx.y * rows_y, r1 = min(rows, r0 + rows_y);
  const int W = rows_y >= 4 ? 1 : rows_y >= 2 ? 2 : 4;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int rb = r0; rb < r1; rb += 4 / W) {
    const int r = rb + warp / W, part = warp % W;
    float L = 0.f, acc[PER] = {};
    if (r < r1) {
      float M = -INFINITY;
      for (int c = c0 + lane; c <= c1; c += 32) M = fmaxf(M, part_ml[((2ll * c + (c == c0)) * ps::ROWS + r) * 2]);
#pragma unroll
      for (int o = 16; o; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
      for (int cb = c0 + part; cb <= c1; cb += W * UN) {
        float2 ml[UN];
        float f[UN][PER];
#pragma unroll
        for (int i = 0; i < UN; ++i) {
          const int c = cb + i * W;
          ml[i] = make_float2(-INFINITY, 0.f);
#pragma unroll
          for (int e = 0; e < PER; ++e) f[i][e] = 0.f;
          if (c > c1) continue;
          const long long at_row = (2ll * c + (c == c0)) * ps::ROWS + r;
          ml[i] = *reinterpret_cast<const float2*>(part_ml + at_row * 2);
#pragma unroll
          for (int e = 0; e < PER; e += 2) {
            const float2 v = *reinterpret_cast<const float2*>(part_o + at_row * D + lane * PER + e);
            f[i][e] = v.x;
            f[i][e + 1] = v.y;
          }
        }
#pragma unroll
        for (int i = 0; i < UN; ++i) {
          const float k = ml[i].x == -INFINITY ? 0.f : fast_exp2(ml[i].x - M);
          L += k * ml[i].y;
#pragma unroll
          for (int e = 0; e < PER; ++e) acc[e] += k * f[i][e];
        }
      }
    }
    if (W > 1) {  // (the same for the whole block)
#pragma unroll
      for (int e = 0; e < PER; ++e) s_acc[warp][lane * PER + e] = acc[e];
      if (lane == 0) s_l[warp] = L;
      __syncthreads();
      if (part == 0)
        for (int w = warp + 1; w < warp + W; ++w) {
          L += s_l[w];
#pragma unroll
          for (int e = 0; e < PER; ++e) acc[e] += s_acc[w][lane * PER + e];
        }
      __syncthreads();
    }
    if (part > 0 || r >= r1) continue;
    const float inv = L == 0.f ? 0.f : 1.f / L;
    const int tok = (row0 + r) / a.group, hh = head * a.group + (row0 + r) % a.group;
    uint32_t* dst = reinterpret_cast<uint32_t*>(reinterpret_cast<uint16_t*>(a.out) +
                                                (long long)(sq.q0 + tok) * a.os_tok + hh * a.os_head + lane * PER);
#pragma unroll
    for (int e = 0; e < PER; e += 2) dst[e / 2] = pack_16<F16>(acc[e] * inv, acc[e + 1] * inv);
  }
}

long long split_workspace_floats(int d) { return 2ll * num_sms() * ps::ROWS * (d + 2); }

template <int D, bool F16>
static int launch_split_t(const CUtensorMap& tmK, const CUtensorMap& tmV, const PackedArgs& a, const void* q,
                          long long q_tok, long long q_head, long long max_rows, bool after, float* ws, int* st, cudaStream_t s) {
  static bool attr[64] = {};
  const int dix = device_index();
  if (dix < 0) return set_error(LBW_ERR_CUDA, "packed_attention: cudaGetDevice failed");
  int err;
  if (!attr[dix]) {
    err = cuda_check(cudaFuncSetAttribute(packed_split_kernel<D, F16>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                          ps::smem_bytes(D)),
                     "packed_attention smem attribute");
    if (err) return err;
    attr[dix] = true;
  }
  // Row tiles: one per sequence of at most 16 rows; else at most one per sequence beyond tq * group / 16 full ones.
  const long long per_tok = (a.group + ps::ROWS - 1) / ps::ROWS;
  long long units = max_rows <= ps::ROWS ? a.n_seqs : (long long)a.tq * a.group / ps::ROWS + a.n_seqs;
  if (units > a.tq * per_tok) units = a.tq * per_tok;
  if (units * a.hk >= 1ll << 31) return set_error(LBW_ERR_SHAPE, "packed_attention: %lld units", units * a.hk);
  const int ctas = num_sms();
  float* part_ml = ws + 2ll * ctas * ps::ROWS * D;
  const uint16_t* q16 = reinterpret_cast<const uint16_t*>(q);
  if (after) {
    err = launch_dependent("packed_attention split launch", packed_split_kernel<D, F16>, dim3(ctas), ps::THREADS,
                           ps::smem_bytes(D), s, tmK, tmV, a, q16, q_tok, q_head, max_rows, ws, part_ml, st);
  } else {
    packed_split_kernel<D, F16><<<ctas, ps::THREADS, ps::smem_bytes(D), s>>>(tmK, tmV, a, q16, q_tok, q_head, max_rows,
                                                                            ws, part_ml, st);
    err = cuda_check(cudaGetLastError(), "packed_attention split launch");
  }
  if (err) return err;
  // A block per row of the unit (of the batch's mean) while that makes less than four blocks per SM.
  const long long mean = ((long long)a.tq * a.group + a.n_seqs - 1) / a.n_seqs;
  long long row_blocks = 4ll * ctas / (units * a.hk);
  if (row_blocks > mean) row_blocks = mean;
  if (row_blocks > ps::ROWS) row_blocks = ps::ROWS;
  const dim3 grid((unsigned)(units * a.hk), row_blocks < 1 ? 1u : (unsigned)row_blocks);
  return launch_dependent("packed_attention join launch", packed_join_kernel<D, F16>, grid, 128, 0, s, a, max_rows, ctas,
                          ws, part_ml);
}

int launch_split(const void* k, long long k_tok, long long k_head, const void* v, long long v_tok, long long v_head,
                 const PackedArgs& a, int d, int dtype, const void* q, long long q_tok, long long q_head,
                 long long max_rows, bool after, float* ws, int* st, cudaStream_t s) {
  CUtensorMap tmK{}, tmV{};
  const CUtensorMapDataType ty = dtype == LBW_FP16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  int err;
  if (a.tk > 0) {
    if ((err = make_tmap_3d(&tmK, k, ty, d, a.hk, a.tk, k_head, k_tok, 1, ps::KEYS))) return err;
    if ((err = make_tmap_3d(&tmV, v, ty, d, a.hk, a.tk, v_head, v_tok, 1, ps::KEYS))) return err;
  }
  if (d == 128)
    return dtype == LBW_FP16 ? launch_split_t<128, true>(tmK, tmV, a, q, q_tok, q_head, max_rows, after, ws, st, s)
                             : launch_split_t<128, false>(tmK, tmV, a, q, q_tok, q_head, max_rows, after, ws, st, s);
  return dtype == LBW_FP16 ? launch_split_t<64, true>(tmK, tmV, a, q, q_tok, q_head, max_rows, after, ws, st, s)
                           : launch_split_t<64, false>(tmK, tmV, a, q, q_tok, q_head, max_rows, after, ws, st, s);
}

}  // namespace lbw
