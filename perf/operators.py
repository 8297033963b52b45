"""Measured cases of the packed-sequence operators: packed_attention, qk_headnorm_rope and axial_rope.

A case is one call as a serving program makes it. `run` computes it from elementary torch operations in 32 bits
(`own` false) or through the package's kernels (`own` true); `exact` restates the definitions in 64 bits.

The sequences of a case have lengths between `lo` and `hi` that follow from the case alone (`_lengths`), the data
from the seed. Attention: sequence b owns `q` rows cu_q[b]..cu_q[b+1] and its keys; `cached` sequences have their keys
in a slab of `cap` rows each, of which the first k_lens[b] are in use and the rest holds what an earlier sequence left.
"""
import functools
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS = 1e-6


def listed():
    return [
        # three 480p clips of one, two and three latent frames packed into one forward of the 12-head model
        dict(name="attn clips 12h", op="attn", dtype="bf16", heads=12, kv_heads=12, dim=128, seqs=3, lo=1560, hi=4680,
             causal=True, cached=False, q=0, cap=0),
        # one 720p chunk (3 latent frames, 10,800 tokens) as a causal prompt, 40 query heads sharing 8 kv heads
        dict(name="attn prompt 10800", op="attn", dtype="bf16", heads=40, kv_heads=8, dim=128, seqs=1, lo=10800,
             hi=10800, causal=True, cached=False, q=0, cap=0),
        # text prompts of very different lengths packed together, fp16
        dict(name="attn short prompts", op="attn", dtype="fp16", heads=32, kv_heads=8, dim=128, seqs=48, lo=1, hi=509,
             causal=True, cached=False, q=0, cap=0),
        # images at their own resolutions, every patch sees its whole image, narrow heads
        dict(name="attn images d64", op="attn", dtype="bf16", heads=16, kv_heads=16, dim=64, seqs=16, lo=196, hi=1023,
             causal=False, cached=False, q=0, cap=0),
        # the next 500 tokens of four prompts whose beginnings are in the cache
        dict(name="attn continued prompts", op="attn", dtype="bf16", heads=32, kv_heads=8, dim=128, seqs=4, lo=3000,
             hi=9001, causal=True, cached=True, q=500, cap=9216),
        # one token for each of 32 sequences over caches of up to 16k tokens
        dict(name="attn decode 32x16k", op="attn", dtype="bf16", heads=32, kv_heads=8, dim=128, seqs=32, lo=2048,
             hi=16384, causal=True, cached=True, q=1, cap=16384),
        # one token of one short sequence: latency
        dict(name="attn decode 1x1000", op="attn", dtype="bf16", heads=12, kv_heads=12, dim=128, seqs=1, lo=1000,
             hi=1000, causal=True, cached=True, q=1, cap=1024),
        # q/k norm and rotation of a 720p chunk, read out of the fused q|k|v projection
        dict(name="norm 720p chunk", op="norm", dtype="bf16", heads=40, kv_heads=40, dim=128, seqs=1, lo=10800,
             hi=10800, sections="22,21,21", layout="interleaved", cached=False, cap=0),
        # the decode step's q/k norm: 32 tokens, keys and values written to their cache rows
        dict(name="norm decode 32", op="norm", dtype="bf16", heads=32, kv_heads=8, dim=128, seqs=32, lo=1, hi=1,
             sections="64", layout="half", cached=True, cap=256),
        # packed prompts with narrow heads of which three quarters are rotated, fp16
        dict(name="norm prompts d64", op="norm", dtype="fp16", heads=16, kv_heads=4, dim=64, seqs=9, lo=17, hi=1201,
             sections="8,8,8", layout="half", cached=False, cap=0),
        # rotation alone: a 720p chunk
        dict(name="rope 720p chunk", op="rope", dtype="bf16", heads=40, kv_heads=0, dim=128, seqs=1, lo=10800,
             hi=10800, sections="22,21,21", layout="interleaved", cached=False, cap=0),
        # rotation alone: two axes over the patches of a few images, fp32
        dict(name="rope images fp32", op="rope", dtype="fp32", heads=12, kv_heads=0, dim=64, seqs=5, lo=49, hi=577,
             sections="16,16", layout="half", cached=False, cap=0),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["prompt", "prompt", "whole", "decode", "decode", "continued", "norm", "norm", "rope"])
    dim = rng.choice([64, 128, 128])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    kv_heads = rng.choice([1, 2, 4, 5, 8])
    heads = kv_heads * rng.choice([1, 1, 2, 3, 4, 5, 7, 8])
    if kind in ("prompt", "whole"):
        seqs = _log_int(rng, 1, 40)
        most = 10000 if kind == "prompt" else 6600
        hi = _log_int(rng, 16, min(most, most * math.sqrt(40 / (heads * seqs))))
        return dict(op="attn", dtype=dtype, heads=heads, kv_heads=kv_heads, dim=dim, seqs=seqs, lo=max(1, hi // 7),
                    hi=hi, causal=kind == "prompt", cached=False, q=0, cap=0)
    if kind in ("decode", "continued"):
        seqs = _log_int(rng, 1, 64) if kind == "decode" else _log_int(rng, 1, 6)
        hi = _log_int(rng, 64, min(60000, 4_000_000 // (seqs * kv_heads)))
        if kind == "continued":
            hi = min(hi, 16000)
        q = rng.choice([1, 1, 1, 2, 4]) if kind == "decode" else min(rng.randrange(9, 700), 1_900_000_000 // (hi * heads * seqs))
        return dict(op="attn", dtype=dtype, heads=heads, kv_heads=kv_heads, dim=dim, seqs=seqs, lo=max(q, hi // 5),
                    hi=max(q, hi), causal=True, cached=True, q=q, cap=max(q, hi) + rng.randrange(0, 100))
    dim = rng.choice([64, 80, 96, 128, 128, 256])
    pairs = dim // 2 if rng.random() < 0.7 else dim // 4 // 4 * 4
    axes = rng.choice([1, 2, 3])
    each = pairs // axes
    sections = [pairs - each * (axes - 1)] + [each] * (axes - 1)
    cached = kind == "norm" and rng.random() < 0.5
    seqs = _log_int(rng, 1, 64)
    hi = 1 if cached else _log_int(rng, 1, max(1, 3_000_000 // (seqs * heads * 4)))
    return dict(op=kind, dtype=rng.choice(["bf16", "fp16", "fp32"]), heads=heads, kv_heads=kv_heads if kind == "norm" else 0,
                dim=dim, seqs=seqs, lo=max(1, hi // 9), hi=hi, sections=",".join(map(str, sections)),
                layout=rng.choice(["interleaved", "half"]), cached=cached, cap=rng.randrange(100, 400) if cached else 0)


def _lengths(case):
    """Lengths of the case's sequences between lo and hi, both met when there are two or more."""
    n, lo, hi = case["seqs"], case["lo"], case["hi"]
    r = random.Random("%d %d %d" % (n, lo, hi))
    lens = [lo, hi][-n:] + [r.randrange(lo, hi + 1) for _ in range(n - 2)]
    r.shuffle(lens)
    return lens


def _starts(lens, device):
    return torch.tensor([0] + lens, device=device).cumsum(0).to(torch.int32)


def _grid_positions(lens, axes, gen, device):
    """[T, axes] int32 positions: each sequence walks a grid (frame, row, column) from its own start."""
    n = torch.tensor(lens, device=device)
    start = torch.randint(0, 2000, (len(lens),), generator=gen, device=device)
    seq = torch.repeat_interleave(torch.arange(len(lens), device=device), n)
    at = torch.arange(seq.numel(), device=device) - (n.cumsum(0) - n)[seq]
    if axes == 1:
        return (at + start[seq]).to(torch.int32)[:, None].contiguous()
    wide = 80 if axes == 3 else 31
    cols = [at % wide, at // wide] if axes == 2 else [at % wide, at // wide % 45, at // (wide * 45) + start[seq]]
    return torch.stack(cols[::-1], dim=1).to(torch.int32)


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    dt, d, hq, hk = DTYPES[case["dtype"]], case["dim"], case["heads"], case["kv_heads"]
    lens = _lengths(case)

    def randn(*shape, scale=1.0):
        return (torch.randn(*shape, generator=gen, device=dev) * scale).to(dt)

    if case["op"] == "attn":
        q_lens = [min(case["q"], n) for n in lens] if case["cached"] else lens
        s = dict(case=case, cu_q=_starts(q_lens, dev), max_q=max(q_lens), max_k=max(lens), k_lens=None)
        s["q"] = randn(sum(q_lens), hq, d, scale=1.5)
        if case["cached"]:
            s["cu_k"] = torch.arange(len(lens) + 1, device=dev, dtype=torch.int32) * case["cap"]
            s["k_lens"] = torch.tensor(lens, device=dev, dtype=torch.int32)
            s["k"], s["v"] = (randn(len(lens) * case["cap"], hk, d) for _ in range(2))
        else:  # keys normalised into a buffer of their own, values still inside the projection's output
            s["cu_k"] = s["cu_q"]
            s["k"] = randn(sum(lens), hk, d)
            s["v"] = randn(sum(lens), hq + 2 * hk, d)[:, hq + hk:]
        return s
    sections = [int(v) for v in case["sections"].split(",")]
    total = sum(lens)
    s = dict(case=case, sections=sections, positions=_grid_positions(lens, len(sections), gen, dev))
    x = randn(total, hq + 2 * hk, d)
    if case["op"] == "rope":
        s["x"] = x
        return s
    s["q"], s["k"], s["v"] = x[:, :hq], x[:, hq:hq + hk], x[:, hq + hk:]
    s["gamma_q"], s["gamma_k"] = ((1 + 0.2 * torch.randn(d, generator=gen, device=dev)).to(dt) for _ in range(2))
    if case["cached"]:
        s["k_cache"], s["v_cache"] = (randn(total * case["cap"], hk, d) for _ in range(2))
        at = torch.randint(0, case["cap"], (total,), generator=gen, device=dev)
        s["k_rows"] = torch.arange(total, device=dev) * case["cap"] + at
    return s


# ---- plain forms -------------------------------------------------------------------------------------------------


def _plain_attention(q, k, v, cu_q, cu_k, k_lens, max_q, max_k, causal):
    """Every sequence padded to the longest, one product of scores, a masked softmax, one product with the values."""
    hq, d, hk = q.shape[1], q.shape[2], k.shape[1]
    group = hq // hk
    n_q = (cu_q[1:] - cu_q[:-1]).long()
    n_k = (cu_k[1:] - cu_k[:-1] if k_lens is None else k_lens).long()
    i, j = torch.arange(max_q, device=q.device), torch.arange(max_k, device=q.device)
    rows = (cu_q[:-1, None] + i).clamp(max=q.shape[0] - 1).long()                    # [B, max_q]
    keys = (cu_k[:-1, None] + j).clamp(max=k.shape[0] - 1).long()                    # [B, max_k]
    qp = q[rows].float().view(-1, max_q, hk, group, d).permute(0, 2, 3, 1, 4).reshape(-1, hk, group * max_q, d)
    kp = k[keys].float().permute(0, 2, 3, 1)                                        # [B, hk, d, max_k]
    vp = v[keys].float().permute(0, 2, 1, 3)                                        # [B, hk, max_k, d]
    hidden = (j >= n_k[:, None])[:, None, :]                                        # [B, 1, max_k]
    if causal:
        hidden = hidden | (j > i[:, None] + (n_k - n_q)[:, None, None])             # [B, max_q, max_k]
    s = torch.matmul(qp, kp).view(-1, hk, group, max_q, max_k)
    s.mul_(1.0 / math.sqrt(d)).masked_fill_(hidden[:, None, None], float("-inf"))
    s.sub_(s.amax(-1, keepdim=True).clamp(min=-3e38)).exp_()
    total = s.sum(-1, keepdim=True)
    o = torch.matmul(s.view(-1, hk, group * max_q, max_k), vp).view(-1, hk, group, max_q, d)
    o = (o / total.clamp(min=1e-38)).permute(0, 3, 1, 2, 4).reshape(-1, max_q, hq, d)
    return o[i < n_q[:, None]].to(q.dtype)


def _frequencies(sections, device, theta=10000.0):
    """(axis, angular frequency) of every pair: theta^(-j / pairs of the axis), 64 bits."""
    n = torch.tensor(sections, device=device)
    axis = torch.repeat_interleave(torch.arange(len(sections), device=device), n)
    j = torch.arange(axis.numel(), device=device) - (n.cumsum(0) - n)[axis]
    return axis, torch.pow(theta, -j.double() / n[axis].double())


def _plain_rotate(x, positions, sections, layout):
    """x [T, H, D] fp32 with its leading 2 * sum(sections) dims rotated."""
    axis, f = _frequencies(sections, x.device)
    angle = positions[:, axis].double() * f
    c, s = angle.cos().float()[:, None], angle.sin().float()[:, None]
    n = f.numel()
    if layout == "half":
        a, b = x[..., :n], x[..., n:2 * n]
        return torch.cat([a * c - b * s, a * s + b * c, x[..., 2 * n:]], dim=-1)
    a, b = x[..., 0:2 * n:2], x[..., 1:2 * n:2]
    return torch.cat([torch.stack([a * c - b * s, a * s + b * c], dim=-1).flatten(-2), x[..., 2 * n:]], dim=-1)


def _plain_norm(x, gamma):
    x = x.float()
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * gamma.float()


# ---- one call ----------------------------------------------------------------------------------------------------


@functools.lru_cache(None)
def _kernels():
    import __graft_entry__

    __graft_entry__.load_package()
    import lbw_b200.kernels as kernels

    return kernels


@functools.lru_cache(None)
def _rope(sections, layout):
    """The rotation of a model's heads: made once, kept with the model."""
    _kernels()
    import lbw_b200.rope as rope

    return rope.AxialRope(sections, theta=10000.0, layout=layout)


def run(state):
    c = state["case"]
    if c["op"] == "attn":
        args = state["q"], state["k"], state["v"], state["cu_q"], state["cu_k"]
        if own:
            return _kernels().packed_attention(*args, k_lens=state["k_lens"], causal=c["causal"], max_q=state["max_q"])
        return _plain_attention(*args, state["k_lens"], state["max_q"], state["max_k"], c["causal"])
    positions, sections, layout = state["positions"], state["sections"], c["layout"]
    if c["op"] == "rope":
        if own:
            return _kernels().axial_rope(state["x"], positions, _rope(tuple(sections), layout))
        return _plain_rotate(state["x"].float(), positions, sections, layout).to(state["x"].dtype)
    q, k, v = state["q"], state["k"], state["v"]
    if own:
        kw = {}
        if c["cached"]:
            kw = dict(k_out=state["k_cache"], v=v, v_out=state["v_cache"], k_rows=state["k_rows"])
        qo, ko = _kernels().qk_headnorm_rope(q, k, state["gamma_q"], state["gamma_k"], EPS, positions,
                                             _rope(tuple(sections), layout), **kw)
    else:
        qo = _plain_rotate(_plain_norm(q, state["gamma_q"]), positions, sections, layout).to(q.dtype)
        ko = _plain_rotate(_plain_norm(k, state["gamma_k"]), positions, sections, layout).to(k.dtype)
        if c["cached"]:
            ko = state["k_cache"].index_copy_(0, state["k_rows"], ko)
            state["v_cache"].index_copy_(0, state["k_rows"], v)
    return (qo, ko, state["v_cache"]) if c["cached"] else (qo, ko)


def work(case):
    lens, d, hq, hk = _lengths(case), case["dim"], case["heads"], case["kv_heads"]
    size = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "attn":
        nq = [min(case["q"], n) for n in lens] if case["cached"] else lens
        seen = [a * n - a * (a - 1) // 2 if case["causal"] else a * n for a, n in zip(nq, lens)]
        return {"bytes": 2 * size * d * (hq * sum(nq) + hk * sum(lens)), "flops": 4 * d * hq * sum(seen)}
    total, axes = sum(lens), case["sections"].count(",") + 1
    moved = hq + hk + (hk if case["cached"] else 0)
    normed = 0 if case["op"] == "rope" else 4
    return {"bytes": total * (2 * moved * d * size + 4 * axes + (8 if case["cached"] else 0)),
            "flops": total * (hq + hk) * d * (3 + normed)}


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------


def exact(case, seed):
    if work(case)["flops"] > 2e13:
        return None
    s = prepare(case, seed)

    def attend(q, k, v, cu_q, cu_k, k_lens):
        """Head by head of sequence by sequence: softmax(q k^T / sqrt(dim)) v over the keys that a row sees."""
        out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
        cq, ck = cu_q.tolist(), cu_k.tolist()
        lens = [b - a for a, b in zip(ck, ck[1:])] if k_lens is None else k_lens.tolist()
        share = q.shape[1] // k.shape[1]
        for b, n in enumerate(lens):
            m = cq[b + 1] - cq[b]
            last = torch.full((m,), n - 1, device=q.device)
            if case["causal"]:
                last -= torch.arange(m - 1, -1, -1, device=q.device)
            for h in range(q.shape[1]):
                kk, vv = (x[ck[b]:ck[b] + n, h // share].double() for x in (k, v))
                z = q[cq[b]:cq[b + 1], h].double() @ kk.T / q.shape[2] ** 0.5
                z[torch.arange(n, device=q.device)[None] > last[:, None]] = -math.inf
                out[cq[b]:cq[b + 1], h] = torch.softmax(z, dim=1) @ vv
        return out

    def turned(x):
        """x with its pairs as complex numbers times e^(i angle)."""
        widths = [int(v) for v in case["sections"].split(",")]
        angles = [s["positions"][:, a:a + 1].double() * 10000.0 ** (-torch.arange(w, device=x.device).double() / w)
                  for a, w in enumerate(widths)]
        turn = torch.polar(torch.ones((), dtype=torch.float64, device=x.device), torch.cat(angles, dim=1))[:, None]
        n, y = sum(widths), x.clone()
        first = slice(0, n) if case["layout"] == "half" else slice(0, 2 * n, 2)
        second = slice(n, 2 * n) if case["layout"] == "half" else slice(1, 2 * n, 2)
        z = torch.complex(x[..., first].contiguous(), x[..., second].contiguous()) * turn
        y[..., first], y[..., second] = z.real, z.imag
        return y

    if case["op"] == "attn":
        return attend(s["q"], s["k"], s["v"], s["cu_q"], s["cu_k"], s["k_lens"])
    if case["op"] == "rope":
        return turned(s["x"].double())
    done = []
    for x, g in ((s["q"], s["gamma_q"]), (s["k"], s["gamma_k"])):
        x = x.double()
        done.append(turned(x / torch.sqrt((x * x).sum(-1, keepdim=True) / x.shape[-1] + EPS) * g.double()))
    if not case["cached"]:
        return tuple(done)
    k, v = s["k_cache"].double(), s["v_cache"].double()
    k[s["k_rows"]], v[s["k_rows"]] = done[1], s["v"].double()
    return done[0], k, v
