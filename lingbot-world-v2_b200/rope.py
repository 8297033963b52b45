"""3-D RoPE tables for the B200 kernels.

The reference rotates interleaved (re, im) pairs of each 128-wide head with angles split
22 / 21 / 21 pairs over (frame, height, width) (wan/modules/model_fast.py:878-931, :933-979;
freqs built at :3273-3278 from rope_params, wan/modules/model.py:47-53). Its grids are full
[L, 1, 64] cos/sin tensors; the rmsnorm_rope kernel instead takes the three small factor tables
(frames of this chunk x 22, grid_h x 21, grid_w x 21) and indexes them per token, so only
(f + h + w) x 21-22 values cross to the device. The angles are the same fp32 products and cos/sin
are taken on the CPU in fp32 exactly as the reference does, so the tables are bit-identical to the
reference grids' entries.
"""
import ctypes
import decimal
import math

import torch

HEAD_DIM = 128

# Arithmetic of the rotation, process-wide as in the reference (model_fast.py:985-1003): fp32 until a model forward
# sees a chunk of 4,096 or more tokens, bf16 from then on (cos / sin rounded to bf16 and every product and sum of the
# rotation rounded to bf16: lbw.h LBW_ROPE_BF16). The block reads it at each call.
ROPE_DTYPE = torch.float32


def mark_bf16_rope():
    """bf16 RoPE for the rest of this process (model_fast.py:1000-1003)."""
    global ROPE_DTYPE
    ROPE_DTYPE = torch.bfloat16


def set_bf16_rope_for_forward(seq_len):
    """Called once per model forward with its seq_len, as the reference does (model_fast.py:1144-1148, :3348)."""
    if seq_len >= 4096:
        mark_bf16_rope()


def rope_params(max_seq_len, dim, theta=10000):
    pos = torch.arange(max_seq_len).float()
    inv = 1.0 / torch.pow(theta, torch.arange(0, dim, 2).float().div(dim))
    return torch.outer(pos, inv)


def rope_freqs(head_dim=HEAD_DIM, max_frames=2880):
    """[max_frames, head_dim / 2] angle table (frame part | height part | width part)."""
    d = head_dim
    dt = d - 4 * (d // 6)
    return torch.cat([rope_params(max_frames, dt), rope_params(max_frames, 2 * (d // 6)),
                      rope_params(max_frames, 2 * (d // 6))], dim=1)


def split_sizes(freqs):
    c = freqs.shape[1]
    return c - 2 * (c // 3), c // 3


_CACHE = {}


def rope_tables(freqs, grid, start_frame, device):
    """(cos, sin) fp32 device tables [f*22 + h*21 + w*21] for a chunk of grid (f, h, w) whose first
    frame is `start_frame` (= current_start // frame_seqlen)."""
    f, h, w = (int(v) for v in grid)
    if torch.compiler.is_compiling():   # no host-side cache inside a traced graph
        return _tables(freqs, f, h, w, int(start_frame), device)
    key = (id(freqs), tuple(freqs.shape), f, h, w, int(start_frame), str(device))
    hit = _CACHE.get(key)
    if hit is not None and hit[0] is freqs:
        return hit[1]
    out = _tables(freqs, f, h, w, int(start_frame), device)
    _CACHE[key] = (freqs, out)
    return out


def _tables(freqs, f, h, w, start_frame, device):
    fc = freqs.detach().cpu().float()
    s0, s1 = split_sizes(fc)
    if (s0, s1) != (22, 21):
        raise ValueError(f"rope tables are laid out for head_dim 128 (22/21/21 pairs), got {s0}/{s1}/{s1}")
    ang = torch.cat([fc[start_frame:start_frame + f, :s0].reshape(-1), fc[:h, s0:s0 + s1].reshape(-1),
                     fc[:w, s0 + s1:].reshape(-1)])
    return torch.cos(ang).to(device), torch.sin(ang).to(device)


class RopeAxes(ctypes.Structure):
    """lbw_rope_axes (include/lbw.h)."""
    _fields_ = [("pairs", ctypes.c_int), ("axes", ctypes.c_int), ("layout", ctypes.c_int), ("wide", ctypes.c_int),
                ("axis", ctypes.c_ubyte * 128), ("step", ctypes.c_ulonglong * 128), ("step_low", ctypes.c_ulonglong * 128)]


def _pi(digits):
    """pi to `digits` decimal digits: 16 atan(1/5) - 4 atan(1/239) (Machin's formula) in integers."""
    one = 10 ** (digits + 10)

    def atan(n):
        total, term, k = 0, one // n, 1
        while term:
            total += term // k if k % 4 == 1 else -(term // k)
            term //= n * n
            k += 2
        return total

    return decimal.Decimal(16 * atan(5) - 4 * atan(239)) / one


def _frequency(theta, exponent, scale):
    """f = scale * theta^-exponent, exponent a pair (numerator, denominator), as a float, and the turns that it makes per
    position, round(f / (2 pi) * 2^128) mod 2^128. (From the float, with its 53 bits, an angle is 0.07 rad off at position
    2^50.)"""
    with decimal.localcontext() as c:
        size = abs(math.log10(theta)) + (abs(math.log10(abs(scale))) if scale else 0)
        c.prec = 60 + int(size)   # 2^128 has 39 digits
        c.rounding = decimal.ROUND_HALF_EVEN
        f = decimal.Decimal(scale) * decimal.Decimal(theta) ** (decimal.Decimal(-exponent[0]) / exponent[1])
        return float(f), int((f * 2 ** 127 / _pi(c.prec)).to_integral_value()) % (1 << 128)


class AxialRope:
    """Rotation of a head by integer positions on several axes, given per token (kernels.axial_rope,
    kernels.qk_headnorm_rope): packed clips and images, each on a grid of its own.

    sections   pairs turned by each axis, in order, e.g. (22, 21, 21) for (frame, height, width); their sum is a
               multiple of 4 and at most half of the head; the head's dims beyond twice the sum stay as they are
    theta      base of the angular frequencies
    layout     "interleaved": pair i is dims (2i, 2i + 1); "half": dims (i, i + pairs)
    spectrum   "axis": pair j of an axis with n pairs has theta^(-j / n), as rope_freqs does for each axis;
               "head": pair i of all has theta^(-i / pairs), whichever axis turns it
    scale      factor on an axis's positions (position interpolation), one number or one per axis

    A model makes it once and keeps it; it holds no device memory.
    """

    LAYOUTS = {"interleaved": 0, "half": 1}

    def __init__(self, sections, theta=10000.0, layout="interleaved", spectrum="axis", scale=1.0):
        self.sections = tuple(int(n) for n in sections)
        self.theta, self.layout, self.spectrum = float(theta), layout, spectrum
        self.axes, self.pairs = len(self.sections), sum(self.sections)
        self.scale = tuple(float(s) for s in scale) if isinstance(scale, (tuple, list)) else (float(scale),) * self.axes
        if not 1 <= self.axes <= 8 or min(self.sections) < 0:
            raise ValueError(f"AxialRope: sections {self.sections} (1 to 8 axes, no negative counts)")
        if self.pairs < 4 or self.pairs % 4 or self.pairs > 128:
            raise ValueError(f"AxialRope: {self.pairs} pairs (a multiple of 4, at most 128)")
        if layout not in self.LAYOUTS:
            raise ValueError(f"AxialRope: layout {layout!r} (one of {sorted(self.LAYOUTS)})")
        if spectrum not in ("axis", "head"):
            raise ValueError(f"AxialRope: spectrum {spectrum!r} ('axis' or 'head')")
        if len(self.scale) != self.axes or not all(math.isfinite(s) for s in self.scale):
            raise ValueError(f"AxialRope: scale {scale!r} needs one finite value per axis")
        if not (math.isfinite(self.theta) and self.theta > 0):
            raise ValueError(f"AxialRope: theta {theta!r}")
        self.axis_of_pair = [a for a, n in enumerate(self.sections) for _ in range(n)]
        self.inv_freq = []                                   # radians per position, as floats
        self.c = RopeAxes(self.pairs, self.axes, self.LAYOUTS[layout], 1)
        for a, n in enumerate(self.sections):
            for j in range(n):
                i = len(self.inv_freq)
                f, turns = _frequency(self.theta, (j, n) if spectrum == "axis" else (i, self.pairs), self.scale[a])
                self.inv_freq.append(f)
                self.c.axis[i] = a
                self.c.step[i], self.c.step_low[i] = turns >> 64, turns & (1 << 64) - 1
        self.ref = ctypes.byref(self.c)

    def __reduce__(self):
        return AxialRope, (self.sections, self.theta, self.layout, self.spectrum, self.scale)
