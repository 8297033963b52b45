// Row kernels over (token, head) vectors: the rotation by positions on several axes (lbw_axial_rope), and the RMSNorm
// of every q and k head with that rotation in the same pass (lbw_qk_headnorm_rope).
//
// For one head vector x of D values, R rotated pairs and the token's integer positions pos[axis]:
//   n_d  = x_d * rsqrt(mean_d(x_d^2) + eps) * gamma_d            (norm form; n = x otherwise)
//   t_i  = pos[axis(i)] * f_i                                    (angle of pair i)
//   y    = (a cos t - b sin t, a sin t + b cos t)                for the pair (a, b) of n; dims beyond 2R: y = n
// All in fp32 with one rounding to the output type. The angle is reduced in integers: with F_i = floor(f_i / 2pi * 2^64)
// the product pos * F_i mod 2^64 is the angle in 2^-64 turns, off by less than |pos| of them: below 2^-32 turns for every
// 32-bit position, where the 24 bits that sincospif takes are off by 2^-26 (an fp32 product pos * f_i is 6e-3 rad off at
// position 100,000). 64-bit positions take 64 more bits of f_i / 2pi, F' : the upper half of pos * (F_i 2^64 + F'_i) mod
// 2^128 is off by less than 2^-63 turns at any of them (F_i alone: 4e-7 rad at 2^40, 4e-4 at 2^50, nothing right at 2^63).
//
// Bound: bytes (each value read once and written once, ~7 flops each). A head is D / 8 "units" of 8 values, one per
// lane: unit u holds the pairs 4u .. 4u + 3, which are 8 neighbouring values (interleaved pairs: one 16-byte access)
// or two runs of 4 values R apart (half layout: two 8-byte accesses), so a pair never crosses lanes and the only exchange
// is the norm's sum over the head's 8, 16 or 32 lanes. The lanes of a head stay with one token: each computes its four
// angles once and uses them, with the gains multiplied in, for the same unit of all of the token's heads.
// Measured (B200, 10,800 tokens, 128-wide heads, bf16): norm of 40 + 40 heads out of the fused projection 78 us (442 MB,
// 5.7 TB/s, 87% of a plain copy's rate; 84 us in the half layout), rotation of 120 heads 109-114 us (5.8-6.1 TB/s).
#include <cuda_fp16.h>
#include <string.h>

#include <type_traits>

#include "host_common.cuh"
#include "lbw_common.cuh"
#include "overlap.cuh"

namespace lbw {

namespace hr {
constexpr int THREADS = 128;
constexpr int MINB = 6;  // blocks per SM: 80 registers; 8 blocks spill and are 5% slower, 4 have too few loads in flight
constexpr int UN = 4;    // heads loaded ahead by a lane group; 2 or 8 are 5-10% slower
}  // namespace hr

// One group of heads of every token: q, k or v. Strides in elements.
struct HeadSeg {
  const void* x;
  void* out;
  const void* gamma;  // null: no gain
  long long xs_tok, xs_head, os_tok, os_head;
  int heads;
  int gamma_f32;
};

struct HeadArgs {
  HeadSeg seg[3];
  long long tokens;
  int dim, units;     // units = dim / 8
  int chunk, chunks;  // heads per work item, items per token
  float eps;
  const void* pos;
  int pos_bits;
  long long ps_tok, ps_axis;
  const void* rows;
  int rows_bits;
  long long out_rows;
  struct {  // the part of lbw_rope_axes that every call needs
    int pairs, layout;
    unsigned char axis[128];
    unsigned long long step[128];
  } rope;
};

// A call with 64-bit positions and 128-bit steps has kernels of its own: with the lower halves in all, calls with 32-bit
// positions took 0.5 us more on the host (1 KB of arguments) and the kernel 0.7 to 1.2%.
struct HeadArgsWide : HeadArgs {
  unsigned long long step_low[128];
};

template <typename T>
struct Vec8;  // 8 values of T as raw registers
template <>
struct Vec8<float> {
  float4 a, b;
};
template <>
struct Vec8<__nv_bfloat16> {
  uint2 a, b;
};
template <>
struct Vec8<__half> {
  uint2 a, b;
};

template <typename T, bool HALF>
LBW_DEV void load8(Vec8<T>& r, const T* p, int o0, int o1) {
  if constexpr (sizeof(T) == 2 && !HALF) {
    const uint4 v = *reinterpret_cast<const uint4*>(p + o0);
    r.a = make_uint2(v.x, v.y);
    r.b = make_uint2(v.z, v.w);
  } else {
    r.a = *reinterpret_cast<const decltype(r.a)*>(p + o0);
    r.b = *reinterpret_cast<const decltype(r.b)*>(p + o1);
  }
}
template <typename T, bool HALF>
LBW_DEV void store8(const Vec8<T>& r, T* p, int o0, int o1) {
  if constexpr (sizeof(T) == 2 && !HALF) {
    *reinterpret_cast<uint4*>(p + o0) = make_uint4(r.a.x, r.a.y, r.b.x, r.b.y);
  } else {
    *reinterpret_cast<decltype(r.a)*>(p + o0) = r.a;
    *reinterpret_cast<decltype(r.b)*>(p + o1) = r.b;
  }
}

LBW_DEV void unpack8(const Vec8<float>& r, float (&f)[8]) {
  f[0] = r.a.x, f[1] = r.a.y, f[2] = r.a.z, f[3] = r.a.w;
  f[4] = r.b.x, f[5] = r.b.y, f[6] = r.b.z, f[7] = r.b.w;
}
LBW_DEV void pack8(Vec8<float>& r, const float (&f)[8]) {
  r.a = make_float4(f[0], f[1], f[2], f[3]);
  r.b = make_float4(f[4], f[5], f[6], f[7]);
}
LBW_DEV void unpack8(const Vec8<__nv_bfloat16>& r, float (&f)[8]) {
  const uint32_t w[4] = {r.a.x, r.a.y, r.b.x, r.b.y};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = __uint_as_float(w[i] << 16);
    f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}
LBW_DEV void pack8(Vec8<__nv_bfloat16>& r, const float (&f)[8]) {
  r.a = make_uint2(pack_bf16(f[0], f[1]), pack_bf16(f[2], f[3]));
  r.b = make_uint2(pack_bf16(f[4], f[5]), pack_bf16(f[6], f[7]));
}
LBW_DEV void unpack8(const Vec8<__half>& r, float (&f)[8]) {
  const uint32_t w[4] = {r.a.x, r.a.y, r.b.x, r.b.y};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    f[2 * i] = v.x;
    f[2 * i + 1] = v.y;
  }
}
LBW_DEV uint32_t pack_f16(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
LBW_DEV void pack8(Vec8<__half>& r, const float (&f)[8]) {
  r.a = make_uint2(pack_f16(f[0], f[1]), pack_f16(f[2], f[3]));
  r.b = make_uint2(pack_f16(f[4], f[5]), pack_f16(f[6], f[7]));
}

LBW_DEV float load_as_float(const float* p) { return *p; }
LBW_DEV float load_as_float(const __nv_bfloat16* p) { return __bfloat162float(*p); }
LBW_DEV float load_as_float(const __half* p) { return __half2float(*p); }

LBW_DEV long long load_index(const void* p, int bits, long long i) {
  return bits == 64 ? reinterpret_cast<const long long*>(p)[i] : (long long)reinterpret_cast<const int*>(p)[i];
}

// Gains of a unit (1 without any).
template <typename T, bool HALF>
LBW_DEV void load_gain(float (&gain)[8], const HeadSeg& g, bool on, int o0, int o1) {
#pragma unroll
  for (int e = 0; e < 8; ++e) gain[e] = 1.f;
  if (!g.gamma || !on) return;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int d = e < 4 ? o0 + e : o1 + e - 4;
    gain[e] = g.gamma_f32 ? reinterpret_cast<const float*>(g.gamma)[d]
                          : load_as_float(reinterpret_cast<const T*>(g.gamma) + d);
  }
}

// Heads [h0, h1) of one segment of the lane group's token, UN at a time: their loads all come before the first store
// (input and output may be the same tensor). The factors of the unit's pairs, (a, b) -> (a w0 - b w1, a w2 + b w3),
// hold the gains.
template <typename T, bool NORM, bool HALF, int G>
LBW_DEV void head_run(const HeadArgs& a, const HeadSeg& g, long long tok, long long row, bool on, int h0, int h1, int o0,
                      int o1, bool rotated, const float (&c)[4], const float (&s)[4]) {
  const T* px = reinterpret_cast<const T*>(g.x) + tok * g.xs_tok + h0 * g.xs_head;
  T* po = reinterpret_cast<T*>(g.out) + row * g.os_tok + h0 * g.os_head;
  float w[4][4];
  {
    float gain[8];
    if constexpr (NORM) load_gain<T, HALF>(gain, g, on, o0, o1);
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      const float g0 = NORM ? gain[HALF ? p : 2 * p] : 1.f, g1 = NORM ? gain[HALF ? p + 4 : 2 * p + 1] : 1.f;
      w[p][0] = g0 * c[p];
      w[p][1] = g1 * s[p];
      w[p][2] = g0 * s[p];
      w[p][3] = g1 * c[p];
    }
  }
  const float inv_d = 1.f / (float)a.dim;
  for (int h = h0; h < h1; h += hr::UN) {
    Vec8<T> r[hr::UN];
#pragma unroll
    for (int i = 0; i < hr::UN; ++i) {
      r[i] = Vec8<T>{};
      if (on && h + i < h1) load8<T, HALF>(r[i], px + i * g.xs_head, o0, o1);
    }
#pragma unroll
    for (int i = 0; i < hr::UN; ++i) {
      float f[8];
      unpack8(r[i], f);
      float k = 1.f;
      if constexpr (NORM) {
        float ss = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) ss = fmaf(f[e], f[e], ss);
#pragma unroll
        for (int o = G / 2; o; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        k = rsqrtf(fmaf(ss, inv_d, a.eps));
      }
#pragma unroll
      for (int p = 0; p < 4; ++p) {
        const int lo = HALF ? p : 2 * p, hi = HALF ? p + 4 : 2 * p + 1;
        const float x0 = f[lo], x1 = f[hi];
        f[lo] = x0 * w[p][0];
        f[hi] = x1 * w[p][3];
        if (rotated) {
          f[lo] = fmaf(-x1, w[p][1], f[lo]);
          f[hi] = fmaf(x0, w[p][2], f[hi]);
        }
        if constexpr (NORM) {
          f[lo] *= k;
          f[hi] *= k;
        }
      }
      if (NORM || rotated) pack8(r[i], f);  // (what is only copied keeps its bits, a NaN's too)
      if (on && h + i < h1) store8<T, HALF>(r[i], po + i * g.os_head, o0, o1);
    }
    px += hr::UN * g.xs_head;
    po += hr::UN * g.os_head;
  }
}

template <typename T, bool HALF>
LBW_DEV void head_copy(const HeadSeg& g, long long tok, long long row, bool on, int h0, int h1, int o0, int o1) {
  const T* px = reinterpret_cast<const T*>(g.x) + tok * g.xs_tok;
  T* po = reinterpret_cast<T*>(g.out) + row * g.os_tok;
  if (!on) return;
  for (int h = h0; h < h1; ++h) {
    Vec8<T> r;
    load8<T, HALF>(r, px + h * g.xs_head, o0, o1);
    store8<T, HALF>(r, po + h * g.os_head, o0, o1);
  }
}

// Work item = (32 / G neighbouring tokens, chunk of the q | k | v heads), one warp each, grid-stride; a group of G lanes
// has one token.
template <typename T, bool NORM, bool HALF, int G, typename A>
__global__ void __launch_bounds__(hr::THREADS, hr::MINB) head_rope_kernel(const __grid_constant__ A a) {
  constexpr bool WIDE = std::is_same_v<A, HeadArgsWide>;
  __shared__ __align__(16) unsigned long long step[128], step_low[WIDE ? 128 : 1];
  __shared__ __align__(4) unsigned char axis[128];
  for (int i = threadIdx.x; i < a.rope.pairs; i += hr::THREADS) {
    step[i] = a.rope.step[i];
    axis[i] = a.rope.axis[i];
    if constexpr (WIDE) step_low[i] = a.step_low[i];
  }
  __syncthreads();
  const int lane = threadIdx.x & 31;
  const int u = lane & (G - 1), sub = lane / G;
  const bool rotated = 4 * u < a.rope.pairs;
  const int o0 = HALF && rotated ? 4 * u : 8 * u;
  const int o1 = HALF && rotated ? a.rope.pairs + 4 * u : 8 * u + 4;
  const int hq = a.seg[0].heads, hk = a.seg[1].heads, hv = a.seg[2].heads;
  const long long items = (a.tokens + 32 / G - 1) / (32 / G) * a.chunks;
  const long long stride = (long long)gridDim.x * (hr::THREADS / 32);
  for (long long it = (long long)blockIdx.x * (hr::THREADS / 32) + (threadIdx.x >> 5); it < items; it += stride) {
    const long long block = it / a.chunks;
    const long long tok = block * (32 / G) + sub;
    const bool here = tok < a.tokens;
    const bool on = here && u < a.units;
    const int lo = (int)(it - block * a.chunks) * a.chunk;
    const int hi = min(lo + a.chunk, hq + hk + hv);
    float c[4] = {1.f, 1.f, 1.f, 1.f}, s[4] = {0.f, 0.f, 0.f, 0.f};
    if (rotated && here && lo < hq + hk) {
      const uchar4 ax = *reinterpret_cast<const uchar4*>(axis + 4 * u);
      const unsigned char axs[4] = {ax.x, ax.y, ax.z, ax.w};
#pragma unroll
      for (int p = 0; p < 4; ++p) {
        const long long ps = load_index(a.pos, a.pos_bits, tok * a.ps_tok + axs[p] * a.ps_axis);
        unsigned long long turns = (unsigned long long)ps * step[4 * u + p];
        if constexpr (WIDE) {  // the carry of the lower halves; a negative position is ps + 2^64 as an unsigned factor
          const unsigned long long low = step_low[4 * u + p];
          turns += __umul64hi((unsigned long long)ps, low) - (ps < 0 ? low : 0ull);
        }
        sincospif((float)(int)(turns >> 32) * 4.656612873077393e-10f, &s[p], &c[p]);  // 2^-31: half turns in [-1, 1]
      }
    }
    if (lo < hq) head_run<T, NORM, HALF, G>(a, a.seg[0], tok, tok, on, lo, min(hi, hq), o0, o1, rotated, c, s);
    if (hi <= hq) continue;
    long long row = tok;
    bool keep = on;
    if (a.rows && here) {
      row = load_index(a.rows, a.rows_bits, tok);
      keep = on && row >= 0 && row < a.out_rows;
    }
    if (lo < hq + hk)
      head_run<T, NORM, HALF, G>(a, a.seg[1], tok, row, keep, max(lo, hq) - hq, min(hi, hq + hk) - hq, o0, o1, rotated, c,
                                 s);
    if (hi > hq + hk) head_copy<T, HALF>(a.seg[2], tok, row, keep, max(lo, hq + hk) - hq - hk, hi - hq - hk, o0, o1);
  }
}

}  // namespace lbw

using namespace lbw;

// Checks one operand's pointers and strides.
static int check_seg(const char* who, const char* name, const lbw_head_rows& r, int dtype) {
  if (!r.x || !r.out) return set_error(LBW_ERR_INVALID, "%s: null %s", who, name);
  if (r.heads < 1 || r.heads > 1 << 20) return set_error(LBW_ERR_SHAPE, "%s: %d %s heads", who, r.heads, name);
  const long long per = dtype == LBW_FP32 ? 4 : 8;
  if (!aligned(r.x, 16) || !aligned(r.out, 16) || r.x_tok % per || r.x_head % per || r.out_row % per || r.out_head % per)
    return set_error(LBW_ERR_ALIGN, "%s: %s needs 16-byte aligned pointers and strides", who, name);
  return LBW_OK;
}

// Work items read and write in any order, so no output may share memory with an operand, but for its own in place, where every
// vector has to stay where it is. moved: rows of k and v go elsewhere, to a cache of out_rows.
static int check_in_place(const char* who, const HeadSeg (&seg)[3], const char* const (&names)[3], long long tokens, int dim,
                          int dtype, bool moved, long long out_rows) {
  const int size = dtype == LBW_FP32 ? 4 : 2;
  ByteGrid in[3], out[3];
  for (int i = 0; i < 3; ++i) {
    const HeadSeg& g = seg[i];
    if (!g.x) continue;
    const bool away = moved && i > 0;
    in[i] = ByteGrid::of(g.x, tokens, g.xs_tok, g.heads, g.xs_head, dim, size);
    out[i] = ByteGrid::of(g.out, away ? out_rows : tokens, g.os_tok, g.heads, g.os_head, dim, size);
    if (g.x == g.out && (away || (tokens > 1 && g.xs_tok != g.os_tok) || (g.heads > 1 && g.xs_head != g.os_head)))
      return set_error(LBW_ERR_INVALID, "%s: %s in place with other strides or rows", who, names[i]);
  }
  for (int i = 0; i < 3; ++i)
    for (int j = 0; j < 3; ++j) {
      if (!seg[i].x || !seg[j].x) continue;
      if (overlap(out[i], in[j]) && !(i == j && seg[i].x == seg[i].out))
        return set_error(LBW_ERR_INVALID, "%s: the output of %s overlaps %s and is not it in place", who, names[i], names[j]);
      if (i < j && overlap(out[i], out[j]))
        return set_error(LBW_ERR_INVALID, "%s: the outputs of %s and %s overlap", who, names[i], names[j]);
    }
  return LBW_OK;
}

static int check_common(const char* who, long long tokens, int head_dim, int dtype, const void* positions,
                        int pos_bits, const lbw_rope_axes* rope) {
  if (dtype != LBW_BF16 && dtype != LBW_FP16 && dtype != LBW_FP32)
    return set_error(LBW_ERR_INVALID, "%s: dtype %d", who, dtype);
  if (tokens < 0 || head_dim < 8 || head_dim % 8 || head_dim > 256)
    return set_error(LBW_ERR_SHAPE, "%s: head_dim %d (a multiple of 8, at most 256)", who, head_dim);
  if (!rope) return LBW_OK;
  if (rope->pairs < 4 || rope->pairs % 4 || rope->pairs > 128 || 2 * rope->pairs > head_dim)
    return set_error(LBW_ERR_SHAPE, "%s: %d rotated pairs of a %d-wide head (a multiple of 4, at most half of it)", who,
                     rope->pairs, head_dim);
  if (rope->axes < 1 || rope->axes > 8) return set_error(LBW_ERR_SHAPE, "%s: %d axes (1 to 8)", who, rope->axes);
  for (int i = 0; i < rope->pairs; ++i)
    if (rope->axis[i] >= rope->axes)
      return set_error(LBW_ERR_INVALID, "%s: pair %d turns by axis %d of %d", who, i, rope->axis[i], rope->axes);
  if (rope->layout != LBW_ROPE_INTERLEAVED && rope->layout != LBW_ROPE_HALF)
    return set_error(LBW_ERR_INVALID, "%s: rope layout %d", who, rope->layout);
  if (tokens > 0 && !positions) return set_error(LBW_ERR_INVALID, "%s: null positions", who);
  if (pos_bits != 32 && pos_bits != 64) return set_error(LBW_ERR_INVALID, "%s: %d-bit positions", who, pos_bits);
  return LBW_OK;
}

// The rotation of the call, turned the other way if `inverse`; of a description without the lower halves only what it has
// is read.
static void set_rope(HeadArgsWide& a, bool& wide, const lbw_rope_axes& rope, bool inverse) {
  wide = rope.wide && a.pos_bits == 64;
  a.rope.pairs = rope.pairs;
  a.rope.layout = rope.layout;
  memcpy(a.rope.axis, rope.axis, rope.pairs);
  memcpy(a.rope.step, rope.step, rope.pairs * 8);
  if (wide) memcpy(a.step_low, rope.step_low, rope.pairs * 8);
  for (int i = 0; inverse && i < rope.pairs; ++i) {  // minus the 64- or 128-bit number
    a.rope.step[i] = ~a.rope.step[i] + (!wide || a.step_low[i] == 0);
    if (wide) a.step_low[i] = 0ull - a.step_low[i];
  }
}

template <typename T, bool NORM, bool HALF, typename A>
static void launch_g(const A& a, int group, unsigned blocks, cudaStream_t s) {
  if (group == 8)
    head_rope_kernel<T, NORM, HALF, 8, A><<<blocks, hr::THREADS, 0, s>>>(a);
  else if (group == 16)
    head_rope_kernel<T, NORM, HALF, 16, A><<<blocks, hr::THREADS, 0, s>>>(a);
  else
    head_rope_kernel<T, NORM, HALF, 32, A><<<blocks, hr::THREADS, 0, s>>>(a);
}

template <typename T, bool NORM>
static void launch_t(const HeadArgsWide& a, bool wide, int group, unsigned blocks, cudaStream_t s) {
  const HeadArgs& narrow = a;
  if (a.rope.layout == LBW_ROPE_HALF)
    wide ? launch_g<T, NORM, true>(a, group, blocks, s) : launch_g<T, NORM, true>(narrow, group, blocks, s);
  else
    wide ? launch_g<T, NORM, false>(a, group, blocks, s) : launch_g<T, NORM, false>(narrow, group, blocks, s);
}

template <bool NORM>
static int launch_head_rope(HeadArgsWide& a, bool wide, int dtype, cudaStream_t s, const char* who) {
  a.units = a.dim / 8;
  const int group = a.units <= 8 ? 8 : a.units <= 16 ? 16 : 32;
  const int total = a.seg[0].heads + a.seg[1].heads + a.seg[2].heads;
  const long long most = (long long)num_sms() * hr::MINB;
  const long long blocks_tok = (a.tokens + 32 / group - 1) / (32 / group);
  // Heads per item: all of a token's, halved while the warps would have fewer than 8 items each (the last round is then
  // a small part of the time), but not below 12, where the four angles of a lane (~240 instructions, a head is ~60) would
  // weigh more than a third; below that only while there are fewer items than warps. Measured (us, this rule / all heads /
  // 12 / 4 at a time): norm of 10,800 tokens x 80 heads 75.5 / 79 / 76 / 101, of 40,000 x 32 106 / 109 / 122 / 150, of
  // 64 x 96 4.0 / 16 / 4.8 / 4.0; rotation of 10,800 x 120 112 / 119 / 110 / 118, of 64 x 48 3.0 / 7.6 / 4.0 / 3.3.
  const long long warps = most * (hr::THREADS / 32);
  a.chunk = total;
  while (a.chunk > hr::UN) {
    const long long items = blocks_tok * ((total + a.chunk - 1) / a.chunk);
    if (items >= (a.chunk > 12 ? 8 * warps : warps)) break;
    a.chunk = (a.chunk + 1) / 2;
  }
  a.chunk = (a.chunk + hr::UN - 1) / hr::UN * hr::UN;
  a.chunks = (total + a.chunk - 1) / a.chunk;
  const long long items = blocks_tok * a.chunks;
  const long long want = (items + hr::THREADS / 32 - 1) / (hr::THREADS / 32);
  const unsigned blocks = (unsigned)(want < most ? want : most);
  if (dtype == LBW_BF16)
    launch_t<__nv_bfloat16, NORM>(a, wide, group, blocks, s);
  else if (dtype == LBW_FP16)
    launch_t<__half, NORM>(a, wide, group, blocks, s);
  else
    launch_t<float, NORM>(a, wide, group, blocks, s);
  return cuda_check(cudaGetLastError(), who);
}

extern "C" {

int lbw_axial_rope(const lbw_head_rows* x, long long tokens, int head_dim, int dtype, const void* positions, int pos_bits,
                   long long pos_tok, long long pos_axis, const lbw_rope_axes* rope, int inverse, void* stream) {
  const char* who = "axial_rope";
  if (!x || !rope) return set_error(LBW_ERR_INVALID, "%s: null %s", who, x ? "rope" : "x");
  int err = check_common(who, tokens, head_dim, dtype, positions, pos_bits, rope);
  if (err) return err;
  if (tokens == 0) return LBW_OK;
  if ((err = check_seg(who, "x", *x, dtype))) return err;
  HeadArgsWide a;
  static_cast<HeadArgs&>(a) = HeadArgs{};
  a.seg[0] = HeadSeg{x->x, x->out, nullptr, x->x_tok, x->x_head, x->out_row, x->out_head, x->heads, 0};
  if ((err = check_in_place(who, a.seg, {"x", "", ""}, tokens, head_dim, dtype, false, 0))) return err;
  a.tokens = tokens;
  a.dim = head_dim;
  a.pos = positions;
  a.pos_bits = pos_bits;
  a.ps_tok = pos_tok;
  a.ps_axis = pos_axis;
  bool wide;
  set_rope(a, wide, *rope, inverse != 0);
  return launch_head_rope<false>(a, wide, dtype, reinterpret_cast<cudaStream_t>(stream), "axial_rope launch");
}

int lbw_qk_headnorm_rope(const lbw_head_rows* q, const lbw_head_rows* k, const lbw_head_rows* v, long long tokens,
                         int head_dim, int dtype, float eps, const void* positions, int pos_bits, long long pos_tok,
                         long long pos_axis, const lbw_rope_axes* rope, const void* k_rows, int k_rows_bits,
                         long long out_rows, void* stream) {
  const char* who = "qk_headnorm_rope";
  if (!q || !k) return set_error(LBW_ERR_INVALID, "%s: null q or k", who);
  int err = check_common(who, tokens, head_dim, dtype, positions, pos_bits, rope);
  if (err) return err;
  if (!(eps >= 0.f)) return set_error(LBW_ERR_INVALID, "%s: eps %g", who, (double)eps);
  if (k_rows && (k_rows_bits != 32 && k_rows_bits != 64))
    return set_error(LBW_ERR_INVALID, "%s: %d-bit cache rows", who, k_rows_bits);
  if (tokens == 0) return LBW_OK;
  if (k_rows && out_rows < 0) return set_error(LBW_ERR_SHAPE, "%s: %lld cache rows", who, out_rows);
  HeadArgsWide a;
  static_cast<HeadArgs&>(a) = HeadArgs{};
  const lbw_head_rows* in[3] = {q, k, v};
  const char* const names[3] = {"q", "k", "v"};
  for (int i = 0; i < 3; ++i) {
    if (!in[i]) continue;
    const lbw_head_rows& r = *in[i];
    if ((err = check_seg(who, names[i], r, dtype))) return err;
    if (r.gamma && !aligned(r.gamma, r.gamma_f32 ? 4 : 2))
      return set_error(LBW_ERR_ALIGN, "%s: gamma of %s is misaligned", who, names[i]);
    a.seg[i] = HeadSeg{r.x, r.out, r.gamma, r.x_tok, r.x_head, r.out_row, r.out_head, r.heads, r.gamma_f32};
  }
  if ((err = check_in_place(who, a.seg, names, tokens, head_dim, dtype, k_rows != nullptr, out_rows))) return err;
  a.tokens = tokens;
  a.dim = head_dim;
  a.eps = eps;
  a.pos = positions;
  a.pos_bits = pos_bits;
  a.ps_tok = pos_tok;
  a.ps_axis = pos_axis;
  a.rows = k_rows;
  a.rows_bits = k_rows_bits;
  a.out_rows = out_rows;
  bool wide = false;
  if (rope) set_rope(a, wide, *rope, false);
  return launch_head_rope<true>(a, wide, dtype, reinterpret_cast<cudaStream_t>(stream), "qk_headnorm_rope launch");
}

}  // extern "C"
