"""64-bit forms of the packed-sequence operators, with the error that a correct kernel may make beside each value.

The bounds count roundings. u = eps / 2 of the tensors' type is half a step (bf16 2^-8, fp16 2^-11, fp32 2^-24).
"""
import decimal
import functools
import math

import torch

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TINY = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -25, torch.float32: 0.0}   # half the spacing of fp16 subnormals


def attention(q, k, v, cu_q, cu_k, k_lens=None, causal=True, scale=None):
    """(out, bound) [tq, hq, d] fp64; rows of no sequence are NaN in both.

    out = sum_j p_j v_j / sum_j p_j. A probability is off by u where it is rounded for the second product, by 2^-21 where its
    exponential is (ex2.approx), and by the error s of its score, |q|.|k| scale times 2^-23 for each of the d products summed
    in fp32 (2^-23: sums may be cut, not rounded); the sum of probabilities has the same without u, and the second product's
    n additions cost 2^-23 each. A probability below the fp16 normals is off by 2^-25 at most where it is rounded, against a
    sum of 1 or more: the maximum that is subtracted is never above the row's largest score, whose probability is then 1 or
    more (with the keys in ranges this holds for the range of the largest maximum, and the others are scaled down to it)."""
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    group = q.shape[1] // k.shape[1]
    out = torch.full(q.shape, float("nan"), dtype=torch.float64, device=q.device)
    bound = out.clone()
    u, tiny = U[q.dtype], TINY[q.dtype]
    cq, ck = cu_q.tolist(), cu_k.tolist()
    for b in range(len(cq) - 1):
        n = ck[b + 1] - ck[b] if k_lens is None else int(k_lens[b])
        m = cq[b + 1] - cq[b]
        if m == 0:
            continue
        if n == 0:
            out[cq[b]:cq[b + 1]] = 0
            bound[cq[b]:cq[b + 1]] = 0
            continue
        qq = q[cq[b]:cq[b + 1]].double().transpose(0, 1)                                  # [hq, m, d]
        kk = k[ck[b]:ck[b] + n].double().transpose(0, 1).repeat_interleave(group, 0)     # [hq, n, d]
        vv = v[ck[b]:ck[b] + n].double().transpose(0, 1).repeat_interleave(group, 0)
        z = qq @ kk.transpose(1, 2) * scale
        mag = qq.abs() @ kk.abs().transpose(1, 2) * scale
        if causal:
            hide = torch.arange(n, device=q.device)[None] > torch.arange(m, device=q.device)[:, None] + (n - m)
            z = z.masked_fill(hide, -math.inf)
            mag = mag.masked_fill(hide, 0.0)
        top = z.amax(-1, keepdim=True)
        p = torch.exp(z - top.clamp(min=-1e300))
        total = p.sum(-1, keepdim=True).clamp(min=1e-300)
        o = (p @ vv) / total
        spread = (p @ vv.abs()) / total                                                  # sum p |v| / sum p
        s = mag.amax(-1, keepdim=True) * qq.shape[-1] * 2.0 ** -23
        rel = u + 2 * 2.0 ** -21 + 2.2 * s + n * 2.0 ** -23
        low = n * tiny * vv.abs().amax() if tiny else 0.0
        empty = torch.isinf(top) & (top < 0)
        out[cq[b]:cq[b + 1]] = torch.where(empty, torch.zeros((), dtype=torch.float64, device=q.device), o).transpose(0, 1)
        bound[cq[b]:cq[b + 1]] = torch.where(empty, torch.zeros((), dtype=torch.float64, device=q.device),
                                             spread * rel * 1.01 + u * o.abs() + low + tiny).transpose(0, 1)
    return out, bound


TURN = 192   # bits of a turn in `turns_per_position`


@functools.lru_cache(None)
def turns_per_position(sections, theta, spectrum, scale):
    """round(scale theta^-e / (2 pi) 2^192) of every pair, from the description alone: exp and ln with 150 digits, pi by the
    arithmetic-geometric mean."""
    D = decimal.Decimal
    with decimal.localcontext() as c:
        c.prec = 150
        a, b, t, p = D(1), 1 / D(2).sqrt(), D(1) / 4, D(1)
        for _ in range(9):
            a, b, t, p = (a + b) / 2, (a * b).sqrt(), t - p * ((a - b) / 2) ** 2, 2 * p
        pi = (a + b) ** 2 / (4 * t)
        out, pairs = [], sum(sections)
        for axis, n in enumerate(sections):
            for j in range(n):
                e = D(j) / n if spectrum == "axis" else D(len(out)) / pairs
                f = D(scale[axis]) * (-e * D(theta).ln()).exp()
                out.append(int((f / (2 * pi) * 2 ** TURN).to_integral_value()))
    return out


def rotate(x, positions, rope, inverse=False):
    """(y, size) fp64: x [tokens, heads, d] fp64 rotated by rope at integer positions, and |a| + |b| of each pair. The
    position times the turns per position is an integer, reduced exactly (fp64 loses digits beyond position 2^20)."""
    pos = positions.cpu()
    pos = pos[:, None] if pos.dim() == 1 else pos
    step = turns_per_position(rope.sections, rope.theta, rope.spectrum, rope.scale)
    axis = [a for a, n in enumerate(rope.sections) for _ in range(n)]
    ang = torch.empty(pos.shape[0], len(step), dtype=torch.float64)
    whole, half = 1 << TURN, 1 << TURN - 1
    for t, row in enumerate(pos.tolist()):
        for i, st in enumerate(step):
            ang[t, i] = math.ldexp((row[axis[i]] * st + half) % whole - half, -TURN) * 2 * math.pi
    ang = ang.to(x.device)
    c, s = ang.cos()[:, None], ang.sin()[:, None]
    if inverse:
        s = -s
    n = len(step)
    y, size = x.clone(), x.abs()
    i0 = slice(0, n) if rope.layout == "half" else slice(0, 2 * n, 2)
    i1 = slice(n, 2 * n) if rope.layout == "half" else slice(1, 2 * n, 2)
    a, b = x[..., i0], x[..., i1]
    y[..., i0], y[..., i1] = a * c - b * s, a * s + b * c
    both = a.abs() + b.abs()
    size[..., i0], size[..., i1] = both, both
    return y, size


def head_bound(y, size, dtype, dim, normed):
    """Error of a rotated (and normed) value: the rounding of the result, and in fp32 before it the squares' sum (dim / 2
    steps on the root), eps, the root (2), the gain and the scale (2), cos and sin (2 each and 1 for the rounded angle)
    and the two products and the sum (3), each half a step of the pair's size; 2^-24 turned by a full angle step (pi
    2^-25 absolute) is within the 16."""
    steps = 16 + (dim / 2 if normed else 0)
    return U[dtype] * y.abs() + steps * 2.0 ** -24 * size + TINY[dtype]


def norm(x, gamma, eps):
    x = x.double()
    y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    return y if gamma is None else y * gamma.double()


def within(got, want, bound):
    """Largest error over its bound (0 where both are equal)."""
    e = (got.double() - want).abs()
    assert not torch.isnan(e).any(), "NaN in the result"
    return float(torch.where(e == 0, torch.zeros_like(e), e / bound.clamp(min=1e-300)).max()) if e.numel() else 0.0
