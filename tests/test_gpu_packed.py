"""Packed-sequence operators on a B200 against their 64-bit forms, every value within its own bound (packed_oracle)."""
import math

import pytest
import torch

import packed_oracle as po

pytestmark = pytest.mark.gpu
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def _gen(dev, seed):
    return torch.Generator(device=dev).manual_seed(seed)


def _randn(dev, seed, *shape, dtype=BF, scale=1.0):
    return (torch.randn(*shape, generator=_gen(dev, seed), device=dev) * scale).to(dtype)


def _cu(lens, dev):
    return torch.tensor([0] + list(lens), dtype=torch.int64).cumsum(0).to(torch.int32).to(dev)


# ---- rotation -----------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("tokens,heads,dim,sections", [(1, 1, 8, (4,)), (7, 3, 64, (16, 16)), (300, 5, 80, (20, 10, 10)),
                                                       (33, 40, 128, (22, 21, 21)), (5, 7, 256, (60, 4, 0, 64)),
                                                       (64, 2, 96, (12,)), (9, 33, 128, (64,))])
def test_axial_rope(cuda_dev, dtype, layout, tokens, heads, dim, sections):
    import lbw_b200.kernels as K
    from lbw_b200.rope import AxialRope
    r = AxialRope(sections, layout=layout, spectrum="head" if heads == 7 else "axis", scale=0.25 if heads == 5 else 1.0)
    x = _randn(cuda_dev, tokens + dim, tokens, heads, dim, dtype=dtype)
    pos = torch.randint(-3000, 3000, (tokens, len(sections)), generator=_gen(cuda_dev, 1), device=cuda_dev)
    if heads != 3:
        pos = pos.to(torch.int32)
    y, size = po.rotate(x.double(), pos, r)
    bound = po.head_bound(y, size, dtype, dim, False)
    out = K.axial_rope(x, pos, r)
    assert po.within(out, y, bound) <= 1
    assert torch.equal(out[..., 2 * sum(sections):], x[..., 2 * sum(sections):])
    yi, size = po.rotate(x.double(), pos, r, inverse=True)
    keep = x.clone()
    assert K.axial_rope(keep, pos, r, inverse=True, out=keep) is keep
    assert po.within(keep, yi, po.head_bound(yi, size, dtype, dim, False)) <= 1


def test_axial_rope_far_positions_strides_and_specials(cuda_dev):
    import lbw_b200.kernels as K
    from lbw_b200.rope import AxialRope
    r = AxialRope((32, 32))
    far = torch.tensor([[0, 1], [2 ** 31 - 1, -2 ** 31], [10 ** 6, 10 ** 7], [2 ** 40 + 12345, -2 ** 50]],
                       device=cuda_dev)
    wide = _randn(cuda_dev, 2, 4, 9, 256, dtype=F32)
    x = wide[:, 1::2, 64:192]                                             # every second head, inner dims
    y, size = po.rotate(x.double(), far, r)
    dst = torch.full((4, 4, 136), 7.0, device=cuda_dev)
    K.axial_rope(x, far.t().contiguous().t(), r, out=dst[..., :128])      # positions with swapped strides
    assert po.within(dst[..., :128], y, po.head_bound(y, size, F32, 128, False)) <= 1
    assert bool((dst[..., 128:] == 7).all())
    x = _randn(cuda_dev, 3, 3, 2, 96, dtype=BF)
    x[0, 0, 95], x[1, 1, 90] = float("inf"), float("nan")                 # in the dims that pass through
    out = K.axial_rope(x, torch.arange(3, device=cuda_dev), AxialRope((40,)))
    assert torch.equal(out[..., 80:].view(torch.int16), x[..., 80:].view(torch.int16))
    assert torch.isfinite(out[..., :80].float()).all()
    zero = torch.zeros(3, 1, dtype=torch.int32, device=cuda_dev)
    assert torch.equal(K.axial_rope(x[..., :80], zero, AxialRope((40,))), x[..., :80])


@pytest.mark.parametrize("kw", [dict(sections=(32, 32)), dict(sections=(24, 40), layout="half", spectrum="head", theta=5e5),
                                dict(sections=(4, 8), scale=(0.37, -3.0))])
def test_rotation_at_any_64_bit_position(cuda_dev, kw):
    """The angle is that of theta^-e itself, whatever the position: alone, turned back, and behind the norm."""
    import lbw_b200.kernels as K
    from lbw_b200.rope import AxialRope
    r = AxialRope(**kw)
    at = [0, 1, -1, 2 ** 31, -2 ** 40 - 7, 2 ** 50 + 1, -2 ** 50, 2 ** 62 + 12345, 2 ** 63 - 1, -2 ** 63, -2 ** 63 + 99]
    pos = torch.tensor([[a, b] for a in at for b in (at[3], at[-1])], dtype=torch.int64, device=cuda_dev)
    x = _randn(cuda_dev, 4, len(pos), 3, 128, dtype=F32)
    for inverse in (False, True):
        y, size = po.rotate(x.double(), pos, r, inverse=inverse)
        assert po.within(K.axial_rope(x, pos, r, inverse=inverse), y, po.head_bound(y, size, F32, 128, False)) <= 1
    y, size = po.rotate(po.norm(x, None, 1e-6), pos, r)
    for got in K.qk_headnorm_rope(x, x, None, None, 1e-6, pos, r):
        assert po.within(got, y, po.head_bound(y, size, F32, 128, True)) <= 1
    near = torch.randint(-2 ** 31, 2 ** 31, (40, 2), generator=_gen(cuda_dev, 1), device=cuda_dev)
    x = _randn(cuda_dev, 5, 40, 2, 128, dtype=F32)
    y, size = po.rotate(x.double(), near, r)
    back, _ = po.rotate(x.double(), near, r, inverse=True)
    for wide in (1, 0):                                                      # 64 bits of the step do for 32-bit positions
        r.c.wide = wide
        for p in (near, near.to(torch.int32)):
            assert po.within(K.axial_rope(x, p, r), y, po.head_bound(y, size, F32, 128, False)) <= 1
            assert po.within(K.axial_rope(x, p, r, inverse=True), back, po.head_bound(back, size, F32, 128, False)) <= 1


# ---- per-head norm + rotation -------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("tokens,hq,hk,dim,sections,layout", [
    (1, 1, 1, 64, (32,), "half"), (5, 12, 12, 128, (22, 21, 21), "interleaved"), (37, 7, 1, 80, (20, 20), "half"),
    (400, 8, 2, 96, (10, 10, 12), "interleaved"), (3, 40, 8, 128, (64,), "half"), (11, 3, 3, 256, (64, 32), "half"),
    (2000, 4, 2, 16, (4,), "interleaved"), (6, 5, 5, 128, None, "interleaved")])
def test_qk_headnorm_rope(cuda_dev, dtype, tokens, hq, hk, dim, sections, layout):
    import lbw_b200.kernels as K
    from lbw_b200.rope import AxialRope
    rope = AxialRope(sections, layout=layout) if sections else None
    qkv = _randn(cuda_dev, tokens + hq, tokens, hq + 2 * hk, dim, dtype=dtype, scale=2.0)
    qkv[0, 0] = 0                                                          # a head of zeros stays zeros
    q, k = qkv[:, :hq], qkv[:, hq:hq + hk]
    gq = _randn(cuda_dev, 3, dim, dtype=dtype)
    gk = None if hq == 7 else _randn(cuda_dev, 4, dim, dtype=F32)
    pos = torch.randint(0, 90000, (tokens, len(sections)), generator=_gen(cuda_dev, 5), device=cuda_dev) if sections else None
    before = qkv.clone()
    qo, ko = K.qk_headnorm_rope(q, k, gq, gk, 1e-6, pos, rope)
    assert torch.equal(qkv, before)
    for got, x, g in ((qo, q, gq), (ko, k, gk)):
        n = po.norm(x, g, 1e-6)
        y, size = po.rotate(n, pos, rope) if rope else (n, n.abs())
        assert po.within(got, y, po.head_bound(y, size, dtype, dim, True)) <= 1
    assert bool((qo[0, 0] == 0).all())
    K.qk_headnorm_rope(q, k, gq, gk, 1e-6, pos, rope, q_out=q, k_out=k)     # in place, inside the fused tensor
    assert torch.equal(q, qo) and torch.equal(k, ko) and torch.equal(qkv[:, hq + hk:], before[:, hq + hk:])


@pytest.mark.parametrize("index", [torch.int32, torch.int64])
@pytest.mark.parametrize("tokens,hq,hk,dim", [(1, 8, 2, 128), (9, 3, 3, 64), (130, 32, 8, 128), (20, 1, 5, 80)])
def test_qk_headnorm_rope_writes_cache_rows(cuda_dev, index, tokens, hq, hk, dim):
    """Rows in any order; padding (-1) and rows past the cache are not written; every other row stays."""
    import lbw_b200.kernels as K
    from lbw_b200.rope import AxialRope
    rope = AxialRope((dim // 2,), layout="half")
    qkv = _randn(cuda_dev, 1, tokens, hq + 2 * hk, dim)
    q, k, v = qkv[:, :hq], qkv[:, hq:hq + hk], qkv[:, hq + hk:]
    pos = torch.arange(tokens, device=cuda_dev, dtype=torch.int32) + 100
    cap = tokens * 2 + 3
    rows = torch.randperm(cap, generator=torch.Generator().manual_seed(2))[:tokens]
    rows[tokens // 2] = -1
    if tokens > 5:
        rows[5], rows[3] = cap, -2 ** 31
    rows = rows.to(index).to(cuda_dev)
    kc, vc = (torch.full((cap, hk, 2 * dim), 9.0, dtype=BF, device=cuda_dev)[..., :dim] for _ in range(2))
    want_k, want_v = kc.clone(), vc.clone()
    qo, ko = K.qk_headnorm_rope(q, k, None, None, 1e-5, pos, rope)
    keep = (rows >= 0) & (rows < cap)
    want_k[rows[keep].long()], want_v[rows[keep].long()] = ko[keep], v[keep]
    got_q, got_k = K.qk_headnorm_rope(q, k, None, None, 1e-5, pos, rope, k_out=kc, v=v, v_out=vc, k_rows=rows)
    assert torch.equal(got_q, qo) and got_k is kc
    assert torch.equal(kc, want_k) and torch.equal(vc, want_v)


def test_head_operators_refuse(cuda_dev):
    import lbw_b200.kernels as K
    from lbw_b200.rope import AxialRope
    r = AxialRope((32,))
    x = torch.zeros(4, 2, 64, dtype=BF, device=cuda_dev)
    pos = torch.zeros(4, dtype=torch.int32, device=cuda_dev)
    g = torch.ones(64, dtype=BF, device=cuda_dev)
    bad = [
        lambda: K.axial_rope(x.double(), pos, r), lambda: K.axial_rope(x[..., ::2], pos, r),
        lambda: K.axial_rope(x, pos[:3], r), lambda: K.axial_rope(x, pos.float(), r),
        lambda: K.axial_rope(x, pos, AxialRope((8, 8))), lambda: K.axial_rope(x[..., :56], pos, r),
        lambda: K.axial_rope(x, pos, r, out=x[:1].expand(4, 2, 64)), lambda: K.axial_rope(x, pos.cpu(), r),
        lambda: K.axial_rope(x[..., 4:], pos, AxialRope((28,))),            # 60 wide
        lambda: K.axial_rope(torch.zeros(4, 2, 68, dtype=BF, device=cuda_dev)[..., :64], pos, r),   # stride 68
        lambda: K.axial_rope(x.clone().requires_grad_(), pos, r),
        lambda: K.qk_headnorm_rope(x, x[:3], g, g, 1e-6, pos, r), lambda: K.qk_headnorm_rope(x, x, g[:32], g, 1e-6, pos, r),
        lambda: K.qk_headnorm_rope(x, x, g.half(), g, 1e-6, pos, r), lambda: K.qk_headnorm_rope(x, x.half(), g, g, 1e-6, pos, r),
        lambda: K.qk_headnorm_rope(x, x, g, g, 1e-6, pos), lambda: K.qk_headnorm_rope(x, x, g, g, -1.0, pos, r),
        lambda: K.qk_headnorm_rope(x, x, g, g, 1e-6, pos, r, v=x, v_out=x),
        lambda: K.qk_headnorm_rope(x, x, g, g, 1e-6, pos, r, k_rows=pos),
        lambda: K.qk_headnorm_rope(x, x, g, g, 1e-6, pos, r, k_out=x.clone(), k_rows=pos[:2]),
        lambda: K.qk_headnorm_rope(x, x, g, g, 1e-6, pos, r, k_out=x.clone(), k_rows=pos, v=x, v_out=x[:2].clone())]
    for call in bad:
        with pytest.raises(ValueError):
            call()
    assert K.axial_rope(x[:0], pos[:0], r).shape == (0, 2, 64)
    qo, ko = K.qk_headnorm_rope(x[:0], x[:0], g, g, 1e-6, pos[:0], r)
    assert qo.shape == ko.shape == (0, 2, 64)


# ---- attention ----------------------------------------------------------------------------------------------------


def _attention_case(dev, seed, q_lens, k_lens, hq, hk, dim, dtype, qk_scale=1.5):
    q = _randn(dev, seed, sum(q_lens), hq, dim, dtype=dtype, scale=qk_scale)
    k = _randn(dev, seed + 1, sum(k_lens), hk, dim, dtype=dtype)
    v = _randn(dev, seed + 2, sum(k_lens), hk, dim, dtype=dtype)
    return q, k, v, _cu(q_lens, dev), _cu(k_lens, dev)


LENGTHS = [
    ([1], [1]), ([128], [128]), ([129], [129]), ([257], [257]), ([64, 1, 200], [64, 1, 200]), ([3, 0, 5], [3, 0, 5]),
    ([700], [700]), ([1, 1, 1], [300, 1, 77]), ([5, 130], [400, 131]), ([200, 40], [100, 0]), ([0, 0], [10, 3]),
    (list(range(1, 70)), list(range(1, 70))), ([2, 260], [1000, 1300]), ([16, 17], [129, 127]),
]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("heads", [(1, 1), (4, 2), (6, 2), (8, 1), (10, 2), (14, 2), (34, 2)])
@pytest.mark.parametrize("lens", LENGTHS, ids=lambda v: "-".join(map(str, v[0][:4])) + "_" + "-".join(map(str, v[1][:4])))
def test_packed_attention(cuda_dev, lens, heads, causal):
    import lbw_b200._lib as L
    import lbw_b200.kernels as K
    dim, dtype = (64, 128)[len(lens[0]) % 2], (BF, HF)[sum(lens[0]) % 2]
    q, k, v, cu_q, cu_k = _attention_case(cuda_dev, 7, *lens, *heads, dim, dtype)
    want, bound = po.attention(q, k, v, cu_q, cu_k, causal=causal)
    for max_q in (None, max(lens[0])):
        out = K.packed_attention(q, k, v, cu_q, cu_k, causal=causal, max_q=max_q)
        assert po.within(out, want, bound) <= 1
    L.check_device_status()


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("causal", [True, False])
def test_packed_attention_long(cuda_dev, dtype, dim, causal):
    import lbw_b200.kernels as K
    q, k, v, cu_q, cu_k = _attention_case(cuda_dev, 3, [2500, 900], [2500, 1777], 6, 2, dim, dtype, qk_scale=3.0)
    want, bound = po.attention(q, k, v, cu_q, cu_k, causal=causal, scale=0.2)
    out = K.packed_attention(q, k, v, cu_q, cu_k, causal=causal, softmax_scale=0.2)
    assert po.within(out, want, bound) <= 1


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("q_len", [1, 3, 9, 40])
@pytest.mark.parametrize("heads", [(4, 4), (8, 2), (5, 1), (32, 1)])
def test_packed_attention_over_a_cache(cuda_dev, dtype, dim, q_len, heads):
    """Slabs with room to spare; what lies past a sequence's length is NaN and must not matter."""
    import lbw_b200.kernels as K
    lens, cap = [5000, q_len, 129, 1023, 0, 128], 5001
    hq, hk = heads
    n = len(lens)
    q = _randn(cuda_dev, 1, n * q_len, hq, dim, dtype=dtype)
    k, v = (torch.full((n * cap, hk, dim), float("nan"), dtype=dtype, device=cuda_dev) for _ in range(2))
    for b, m in enumerate(lens):
        k[b * cap:b * cap + m] = _randn(cuda_dev, 10 + b, m, hk, dim, dtype=dtype)
        v[b * cap:b * cap + m] = _randn(cuda_dev, 20 + b, m, hk, dim, dtype=dtype)
    cu_q, cu_k = _cu([q_len] * n, cuda_dev), _cu([cap] * n, cuda_dev)
    k_lens = torch.tensor(lens, dtype=torch.int32, device=cuda_dev)
    want, bound = po.attention(q, k, v, cu_q, cu_k, k_lens)
    for max_q in (None, q_len):
        out = K.packed_attention(q, k, v, cu_q, cu_k, k_lens=k_lens, max_q=max_q)
        assert po.within(out, want, bound) <= 1


def test_packed_attention_mixed_batch_and_rows_behind(cuda_dev):
    """Prompts and single tokens in one call; query rows of no sequence keep what they held; strided tensors."""
    import lbw_b200.kernels as K
    hq, hk, d = 8, 2, 128
    q_lens, k_lens = [300, 1, 1, 17, 2, 0, 129], [300, 2000, 5, 40, 2, 9, 4000]
    qkv = _randn(cuda_dev, 1, sum(q_lens) + 30, hq + 2, d)
    q = qkv[:, 1:hq + 1]
    kv = _randn(cuda_dev, 2, 2, hk, sum(k_lens) + 50, d)                   # head-major keys and values
    k, v = kv[0].transpose(0, 1), kv[1].transpose(0, 1)
    v[sum(k_lens):] = float("nan")
    cu_q, cu_k = _cu(q_lens, cuda_dev) + 4, _cu(k_lens, cuda_dev)           # the first rows belong to nobody either
    buf = torch.full((q.shape[0], 2 * hq, d), 5.0, dtype=BF, device=cuda_dev)
    out = buf[:, ::2]
    want, bound = po.attention(q, k, v, cu_q, cu_k)
    K.packed_attention(q, k, v, cu_q, cu_k, out=out)
    rows = slice(4, 4 + sum(q_lens))
    assert po.within(out[rows], want[rows], bound[rows]) <= 1
    assert bool((out[:4] == 5).all()) and bool((out[4 + sum(q_lens):] == 5).all()) and bool((buf[:, 1::2] == 5).all())


def test_packed_attention_peaked_and_huge_scores(cuda_dev):
    """Scores far from zero (the running maximum moves by thousands), and one key that takes everything."""
    import lbw_b200.kernels as K
    q, k, v, cu_q, cu_k = _attention_case(cuda_dev, 5, [300, 1], [900, 700], 4, 2, 128, BF)
    k[::37] *= 40
    q *= 4
    want, bound = po.attention(q, k, v, cu_q, cu_k)
    assert po.within(K.packed_attention(q, k, v, cu_q, cu_k), want, bound) <= 1
    k[:] = -60.0
    q[:] = 60.0                                                            # every score the same: -40,729
    want, bound = po.attention(q, k, v, cu_q, cu_k)
    assert po.within(K.packed_attention(q, k, v, cu_q, cu_k), want, bound) <= 1


def test_packed_attention_nan_stays_with_its_sequence(cuda_dev):
    """A NaN key or value reaches every row that sees it and no other sequence; NaN keys ahead of a row do not."""
    import lbw_b200.kernels as K
    for at in range(0, 128, 5):                                             # every place of a whole key tile
        q, k, v, cu_q, cu_k = _attention_case(cuda_dev, 5, [300, 20], [300, 300], 4, 2, 64, BF)
        clean = K.packed_attention(q, k, v, cu_q, cu_k)
        k[128 + at], k[300 + at] = float("nan"), float("nan")
        out = K.packed_attention(q, k, v, cu_q, cu_k)
        assert torch.equal(out[:128 + at], clean[:128 + at]) and torch.isnan(out[128 + at:].float()).all()
    for lens in ([130, 200, 60], [1, 1, 1]):
        ks = [130, 200, 60]
        q, k, v, cu_q, cu_k = _attention_case(cuda_dev, 5, lens, ks, 4, 2, 128, BF)
        clean = K.packed_attention(q, k, v, cu_q, cu_k)
        k[130 + 150] = float("nan")
        out = K.packed_attention(q, k, v, cu_q, cu_k)
        first = sum(lens[:2]) - 50 if lens[1] > 1 else 1                    # first query that sees key 150
        last = sum(lens[:2])
        assert torch.isnan(out[first:last].float()).all()
        assert torch.equal(out[:first], clean[:first]) and torch.equal(out[last:], clean[last:])
        k, v = k.nan_to_num(0.5), v.clone()
        v[130 + 3] = float("inf")
        out = K.packed_attention(q, k, v, cu_q, cu_k)
        assert torch.isfinite(out[:lens[0]].float()).all() and torch.isfinite(out[last:].float()).all()


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("heads,q_lens,k_lens", [
    ((4, 2), [300, 20], [300, 300]), ((6, 2), [130, 257], [200, 257]), ((4, 4), [200], [3000]),   # (keys in ranges)
    ((2, 2), [1000, 700], [1000, 600]), ((4, 2), [5, 2, 1], [400, 131, 90]), ((1, 1), [16, 3], [16, 2]),
    ((8, 2), list(range(1, 60)), list(range(1, 60)))])
def test_packed_attention_values_that_are_not_finite(cuda_dev, heads, q_lens, k_lens, causal, dim, dtype):
    """An infinite or NaN value makes its column of the rows that see it what the sum says, and changes nothing else."""
    import lbw_b200.kernels as K
    q, k, v, cu_q, cu_k = _attention_case(cuda_dev, 5, q_lens, k_lens, *heads, dim, dtype, qk_scale=0.5)
    gen = torch.Generator().manual_seed(dim + len(q_lens))
    n = 60
    at = [torch.randint(0, hi, (n,), generator=gen) for hi in (v.shape[0], heads[1], dim)]
    at[0][: n // 2] = v.shape[0] - 1 - torch.randint(0, min(150, v.shape[0]), (n // 2,), generator=gen)
    kinds = torch.randint(0, 3, (n,), generator=gen)
    at = tuple(at)
    v[at] = 0
    want, bound = po.attention(q, k, v, cu_q, cu_k, causal=causal)
    add = torch.zeros(q.shape, dtype=torch.float64)
    for row, head, col, kind in zip(*(x.tolist() for x in at), kinds.tolist()):
        v[row, head, col] = (math.nan, math.inf, -math.inf)[kind]
    group = heads[0] // heads[1]
    for row, head, col in set(zip(*(x.tolist() for x in at))):
        b = next(b for b in range(len(k_lens)) if row < sum(k_lens[:b + 1]))
        key = row - sum(k_lens[:b])
        first = max(0, key - (k_lens[b] - q_lens[b])) if causal else 0      # the first query that sees the key
        rows = slice(sum(q_lens[:b]) + first, sum(q_lens[:b + 1]))
        add[rows, head * group:(head + 1) * group, col] += float(v[row, head, col])
    add = add.to(cuda_dev)
    out = K.packed_attention(q, k, v, cu_q, cu_k, causal=causal).double()
    hit = add != 0                                                          # (NaN too)
    assert torch.equal(out[hit].isnan(), add[hit].isnan())
    assert torch.equal(out[hit].nan_to_num(7.0, 1e9, -1e9), add[hit].nan_to_num(7.0, 1e9, -1e9))
    assert po.within(out[~hit], want[~hit], bound[~hit]) <= 1


def test_packed_attention_bad_starts_stay_inside(cuda_dev):
    """Starts and lengths that do not fit are cut to the tensors: no row of another sequence is lost, none invented."""
    import lbw_b200._lib as L
    import lbw_b200.kernels as K
    q, k, v, cu_q, cu_k = _attention_case(cuda_dev, 5, [40, 40], [40, 40], 4, 2, 64, BF)
    want, bound = po.attention(q, k, v, cu_q, cu_k, causal=False)
    big = torch.tensor([1 << 30, 40], dtype=torch.int32, device=cuda_dev)
    out = K.packed_attention(q, k, v, cu_q, cu_k, k_lens=big, causal=False)
    assert po.within(out, want, bound) <= 1
    far_q = torch.tensor([0, 40, 1 << 30], dtype=torch.int32, device=cuda_dev)
    far_k = torch.tensor([-7, 40, 1 << 30], dtype=torch.int32, device=cuda_dev)
    out = K.packed_attention(q, k, v, far_q, far_k, causal=False)
    assert po.within(out, want, bound) <= 1
    low = torch.tensor([-5, 0], dtype=torch.int32, device=cuda_dev)
    out = K.packed_attention(q, k, v, cu_q, cu_k, k_lens=low, causal=False)
    assert bool((out == 0).all())
    L.check_device_status()


def test_packed_attention_offsets_past_32_bits(cuda_dev):
    """Keys whose element offset is beyond 2^32: a cache of 34 million rows, of which the last are used."""
    import lbw_b200.kernels as K
    rows, d = (1 << 25) + 3000, 128
    k, v = (torch.empty(rows, 1, d, dtype=BF, device=cuda_dev) for _ in range(2))
    k[-3000:], v[-3000:] = _randn(cuda_dev, 1, 3000, 1, d), _randn(cuda_dev, 2, 3000, 1, d)
    q = _randn(cuda_dev, 3, 21, 2, d)
    start = rows - 3000
    cu_k = torch.tensor([start, start + 1000, rows], dtype=torch.int32, device=cuda_dev)
    for q_lens in ([1, 20], [1, 1]):
        cu_q = _cu(q_lens, cuda_dev)
        want, bound = po.attention(q, k[start:], v[start:], cu_q, cu_k - start)
        out = K.packed_attention(q, k, v, cu_q, cu_k)
        n = sum(q_lens)
        assert po.within(out[:n], want[:n], bound[:n]) <= 1


def test_packed_attention_over_many_short_sequences(cuda_dev):
    """3,000 sequences, most of them empty or of one token, in both kernels' hands; the output in the query's place."""
    import lbw_b200.kernels as K
    gen = torch.Generator().manual_seed(3)
    q_lens = (torch.randint(0, 3, (3000,), generator=gen) * torch.randint(0, 2, (3000,), generator=gen)).tolist()
    k_lens = [n + int(i % 7 == 0) * (i % 40) for i, n in enumerate(q_lens)]
    q_lens[1500], k_lens[1500], q_lens[2999], k_lens[2999] = 70, 150, 9, 9
    q, k, v, cu_q, cu_k = _attention_case(cuda_dev, 5, q_lens, k_lens, 4, 2, 64, BF)
    want, bound = po.attention(q, k, v, cu_q, cu_k)
    assert po.within(K.packed_attention(q, k, v, cu_q, cu_k), want, bound) <= 1
    for lens in (None, 70, 1 << 40):
        x = q.clone()
        assert K.packed_attention(x, k, v, cu_q, cu_k, out=x, max_q=lens) is x
        assert po.within(x, want, bound) <= 1


@pytest.mark.parametrize("q_lens", [[96, 96, 96], [1, 191, 96], [288, 0, 0], [2, 2, 284]])
def test_packed_attention_where_max_q_says_all_are_alike(cuda_dev, q_lens):
    """max_q times the sequences is the number of rows: true or not, every row is computed."""
    import lbw_b200.kernels as K
    for k_lens in ([550, 110, 429], [300, 200, 300]):
        q, k, v, cu_q, cu_k = _attention_case(cuda_dev, 5, q_lens, k_lens, 8, 2, 128, BF)
        ws = K.packed_attention_workspace(288, sum(k_lens), 8, 2, 128, 3, cuda_dev, max_q=96)
        want, bound = po.attention(q, k, v, cu_q, cu_k)
        assert po.within(K.packed_attention(q, k, v, cu_q, cu_k, max_q=96, workspace=ws), want, bound) <= 1


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dim,q_lens,k_lens", [(64, [40], [40000]), (128, [20, 33], [20000, 25000]), (128, [25], [2049])])
def test_packed_attention_in_up_to_32_key_ranges(cuda_dev, dim, q_lens, k_lens, causal):
    """Few rows over many keys: 32 ranges, ranges of two sequences, ranges of two tiles; one range all NaN in its keys."""
    import lbw_b200.kernels as K
    q, k, v, cu_q, cu_k = _attention_case(cuda_dev, 5, q_lens, k_lens, 2, 1, dim, BF, qk_scale=0.5)
    want, bound = po.attention(q, k, v, cu_q, cu_k, causal=causal)
    assert po.within(K.packed_attention(q, k, v, cu_q, cu_k, causal=causal), want, bound) <= 1
    k[300:1800] = float("nan")
    out = K.packed_attention(q, k, v, cu_q, cu_k, causal=causal)
    assert torch.isnan(out[:q_lens[0]].float()).all()
    assert po.within(out[q_lens[0]:], want[q_lens[0]:], bound[q_lens[0]:]) <= 1


@pytest.mark.parametrize("heads,q_lens,k_lens", [((4, 4), [200], [3000]), ((8, 1), [2], [9000]), ((8, 2), [1] * 3, [5000, 64, 1])])
def test_packed_attention_in_place_where_keys_are_split(cuda_dev, heads, q_lens, k_lens):
    """Blocks that share a query's keys all read it before any of them writes its row."""
    import lbw_b200.kernels as K
    q, k, v, cu_q, cu_k = _attention_case(cuda_dev, 5, q_lens, k_lens, *heads, 128, BF)
    want = K.packed_attention(q, k, v, cu_q, cu_k)
    for _ in range(5):
        x = q.clone()
        assert torch.equal(K.packed_attention(x, k, v, cu_q, cu_k, out=x), want)


def test_packed_attention_takes_a_batch_dimension_of_one(cuda_dev):
    import lbw_b200.kernels as K
    q, k, v, cu_q, cu_k = _attention_case(cuda_dev, 5, [30, 1], [30, 50], 4, 2, 64, BF)
    out = K.packed_attention(q[None], k[None], v[None], cu_q, cu_k)
    assert out.shape == (1, 31, 4, 64) and torch.equal(out[0], K.packed_attention(q, k, v, cu_q, cu_k))


def test_packed_attention_refuses(cuda_dev):
    import lbw_b200.kernels as K
    x = torch.zeros(4, 2, 64, dtype=BF, device=cuda_dev)
    cu = _cu([4], cuda_dev)
    bad = [
        lambda: K.packed_attention(x.float(), x.float(), x.float(), cu, cu), lambda: K.packed_attention(x, x.half(), x, cu, cu),
        lambda: K.packed_attention(x, x, x[:3], cu, cu), lambda: K.packed_attention(x[:, :1], x, x, cu, cu),
        lambda: K.packed_attention(x[..., :32], x[..., :32], x[..., :32], cu, cu),
        lambda: K.packed_attention(x, x, x, cu.long(), cu), lambda: K.packed_attention(x, x, x, cu, cu[:1]),
        lambda: K.packed_attention(x, x, x, cu, cu, k_lens=cu), lambda: K.packed_attention(x, x, x, cu, cu.cpu()),
        lambda: K.packed_attention(x, x, x, cu, cu, softmax_scale=-1.0), lambda: K.packed_attention(x, x, x, cu, cu, max_q=-1),
        lambda: K.packed_attention(x, x[:1].expand(4, 2, 64), x, cu, cu),
        lambda: K.packed_attention(x, x, x, cu, cu, out=x[:, :1].expand(4, 2, 64)),
        lambda: K.packed_attention(x.clone().requires_grad_(), x, x, cu, cu),
        lambda: K.packed_attention(torch.zeros(4, 2, 68, dtype=BF, device=cuda_dev)[..., 2:66], x, x, cu, cu)]
    for call in bad:
        with pytest.raises(ValueError):
            call()
    assert K.packed_attention(x[:0], x, x, cu * 0, cu).shape == (0, 2, 64)
    none = torch.full_like(x, 3.0)
    K.packed_attention(x, x, x, cu[:1], cu[:1], out=none)                   # no sequences: nothing is written
    assert bool((none == 3).all())
    assert bool((K.packed_attention(x, x[:0], x[:0], cu, cu * 0) == 0).all())


# ---- together -----------------------------------------------------------------------------------------------------


def _layer(K, rope, qkv, hq, hk, gq, gk, pos, rows, kc, vc, cu_q, cu_k, k_lens, out=None, max_q=None):
    q, k, v = qkv[:, :hq], qkv[:, hq:hq + hk], qkv[:, hq + hk:]
    qo, _ = K.qk_headnorm_rope(q, k, gq, gk, 1e-6, pos, rope, k_out=kc, v=v, v_out=vc, k_rows=rows)
    return K.packed_attention(qo, kc, vc, cu_q, cu_k, k_lens=k_lens, out=out, max_q=max_q)


def test_prompt_then_tokens_over_the_cache(cuda_dev):
    """A serving loop: two prompts fill their cache slabs, then single tokens; each step against 64 bits over the
    rounded q, k, v that it really has."""
    import lbw_b200.kernels as K
    from lbw_b200.rope import AxialRope
    hq, hk, d, cap, lens = 8, 2, 128, 400, [300, 77]
    rope = AxialRope((22, 21, 21))
    gq, gk = _randn(cuda_dev, 1, d), _randn(cuda_dev, 2, d)
    kc, vc = (torch.full((2 * cap, hk, d), float("nan"), dtype=BF, device=cuda_dev) for _ in range(2))
    cu_k = _cu([cap, cap], cuda_dev)
    done = [0, 0]
    for step, new in enumerate((lens, [1, 1], [1, 1], [5, 1], [0, 1])):
        qkv = _randn(cuda_dev, 50 + step, sum(new), hq + 2 * hk, d)
        at = torch.cat([torch.arange(done[b], done[b] + new[b]) for b in range(2)])
        seq = torch.repeat_interleave(torch.arange(2), torch.tensor(new))
        pos = torch.stack([at // 50, at // 10 % 5, at % 10], 1).to(cuda_dev)
        rows = (at + seq * cap).to(cuda_dev)
        done = [a + n for a, n in zip(done, new)]
        k_lens = torch.tensor(done, dtype=torch.int32, device=cuda_dev)
        cu_q = _cu(new, cuda_dev)
        out = _layer(K, rope, qkv, hq, hk, gq, gk, pos, rows, kc, vc, cu_q, cu_k, k_lens)
        qn, size = po.rotate(po.norm(qkv[:, :hq], gq, 1e-6), pos, rope)
        kn, ksize = po.rotate(po.norm(qkv[:, hq:hq + hk], gk, 1e-6), pos, rope)
        q16, _ = K.qk_headnorm_rope(qkv[:, :hq], qkv[:, hq:hq + hk], gq, gk, 1e-6, pos, rope)
        assert po.within(q16, qn, po.head_bound(qn, size, BF, d, True)) <= 1
        assert po.within(kc[rows], kn, po.head_bound(kn, ksize, BF, d, True)) <= 1
        assert torch.equal(vc[rows], qkv[:, hq + hk:])
        want, bound = po.attention(q16, kc, vc, cu_q, cu_k, k_lens)
        assert po.within(out, want, bound) <= 1


def test_captured_step_follows_new_lengths_and_rows(cuda_dev):
    """One graph of the norm + cache write + attention, replayed with other lengths, rows and a padded batch entry."""
    import lbw_b200.kernels as K
    from lbw_b200.rope import AxialRope
    hq, hk, d, cap, n = 8, 2, 64, 600, 5
    rope = AxialRope((32,), layout="half")
    kc, vc = (_randn(cuda_dev, s, n * cap, hk, d) for s in (1, 2))
    qkv = _randn(cuda_dev, 3, n, hq + 2 * hk, d)
    pos, rows = (torch.zeros(n, dtype=torch.int64, device=cuda_dev) for _ in range(2))
    k_lens = torch.zeros(n, dtype=torch.int32, device=cuda_dev)
    cu_q, cu_k = _cu([1] * n, cuda_dev), _cu([cap] * n, cuda_dev)
    out = torch.empty(n, hq, d, dtype=BF, device=cuda_dev)

    def step():
        return _layer(K, rope, qkv, hq, hk, None, None, pos, rows, kc, vc, cu_q, cu_k, k_lens, out=out, max_q=1)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for lens in ([600, 1, 300, 129, 0], [1, 599, 2, 256, 77]):
        at = torch.tensor(lens) - 1
        pos.copy_(at)
        rows.copy_(torch.where(at < 0, at, at + torch.arange(n) * cap))
        k_lens.copy_(torch.tensor(lens, dtype=torch.int32))
        qkv.copy_(_randn(cuda_dev, sum(lens), n, hq + 2 * hk, d))
        before = kc.clone()
        graph.replay()
        torch.cuda.synchronize()
        q16, k16 = K.qk_headnorm_rope(qkv[:, :hq], qkv[:, hq:hq + hk], None, None, 1e-6, pos, rope)
        used = rows[rows >= 0]
        before[used] = k16[rows >= 0]
        assert torch.equal(kc, before)
        want, bound = po.attention(q16, kc, vc, cu_q, cu_k, k_lens)
        assert po.within(out, want, bound) <= 1


@pytest.mark.parametrize("tq,max_q", [(200, None), (2000, None), (2000, 700)])
def test_captured_prompts_follow_new_lengths(cuda_dev, tq, max_q):
    """Graphs of the tile kernel with the keys in ranges (tq 200) and without, next to the kernel for single tokens; two
    graphs with a workspace each, replayed side by side."""
    import lbw_b200.kernels as K
    hq, hk, d, tk, n = 8, 2, 128, 6000, 3
    q, k, v = _randn(cuda_dev, 1, tq, hq, d), _randn(cuda_dev, 2, tk, hk, d), _randn(cuda_dev, 3, tk, hk, d)
    sets = []
    for _ in range(2):
        cu_q, cu_k = (torch.zeros(n + 1, dtype=torch.int32, device=cuda_dev) for _ in range(2))
        ws = K.packed_attention_workspace(tq, tk, hq, hk, d, n, cuda_dev, max_q=max_q)
        out, side, graph = torch.empty_like(q), torch.cuda.Stream(), torch.cuda.CUDAGraph()
        with torch.cuda.stream(side):
            K.packed_attention(q, k, v, cu_q, cu_k, out=out, max_q=max_q, workspace=ws)
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            K.packed_attention(q, k, v, cu_q, cu_k, out=out, max_q=max_q, workspace=ws)
        sets.append((cu_q, cu_k, out, side, graph, ws))
    for lens in (([150, 1, 2], [150, 3000, 2]), ([1, 130, 60], [2500, 1300, 2000]), ([0, 3, 197], [0, 5000, 200])):
        want, bound = po.attention(q, k, v, _cu(lens[0], cuda_dev), _cu(lens[1], cuda_dev))
        for cu_q, cu_k, out, *_ in sets:
            cu_q.copy_(_cu(lens[0], cuda_dev))
            cu_k.copy_(_cu(lens[1], cuda_dev))
            out.zero_()
        torch.cuda.synchronize()
        for _, _, _, side, graph, _ in sets:
            with torch.cuda.stream(side):
                graph.replay()
        torch.cuda.synchronize()
        rows = sum(lens[0])
        for _, _, out, *_ in sets:
            assert po.within(out[:rows], want[:rows], bound[:rows]) <= 1 and bool((out[rows:] == 0).all())


def test_two_streams_at_once(cuda_dev):
    import lbw_b200.kernels as K
    cases = [_attention_case(cuda_dev, s, [1, 1], [5000, 300 + s], 8, 2, 128, BF) for s in (1, 40)]
    cases += [_attention_case(cuda_dev, s, [130, 60], [2130, 60 + s], 8, 2, 128, BF) for s in (2, 41)]
    want = [K.packed_attention(*c) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    got = [[] for _ in cases]
    for _ in range(20):
        for i, (c, s) in enumerate(zip(cases, streams)):
            with torch.cuda.stream(s):
                got[i].append(K.packed_attention(*c))
    torch.cuda.synchronize()
    for w, g in zip(want, got):
        assert all(torch.equal(w, x) for x in g)


def test_compiled_graph_equals_eager(cuda_dev):
    import lbw_b200.kernels as K
    import lbw_b200.ops  # noqa: F401
    from lbw_b200.rope import AxialRope
    rope = AxialRope((16, 16), layout="half")
    qkv = _randn(cuda_dev, 1, 50, 6, 64)
    pos = torch.arange(100, device=cuda_dev).view(50, 2)
    cu = _cu([20, 30], cuda_dev)

    def f(qkv, pos, cu):
        q, k = K.qk_headnorm_rope(qkv[:, :2], qkv[:, 2:4], None, None, 1e-6, pos, rope)
        return K.packed_attention(K.axial_rope(q, pos, rope), k, qkv[:, 4:], cu, cu)

    assert torch.equal(torch.compile(f, fullgraph=True, backend="aot_eager")(qkv, pos, cu), f(qkv, pos, cu))


def test_strides_of_a_dimension_of_one(cuda_dev):
    """Whatever stride torch leaves on a dimension of size 1 (here: 1), it is never used and nothing is refused for it."""
    import lbw_b200.kernels as K
    from lbw_b200.rope import AxialRope
    rope = AxialRope((32,))
    flat = _randn(cuda_dev, 1, 9, 64)
    for x in (flat[:, :, None].transpose(1, 2), flat[:1, :, None].permute(2, 0, 1), flat.t().contiguous().t()[:, None][:1].contiguous()):
        x = x if x.shape[1:] == (1, 64) else x.transpose(0, 1)
        n = x.shape[0]
        plain = x.contiguous().view(-1).clone().view(n, 1, 64)
        pos, cu = torch.arange(n, device=cuda_dev), _cu([n], cuda_dev)
        want = K.axial_rope(plain, pos, rope)
        assert torch.equal(K.axial_rope(x, pos, rope), want)
        out = torch.empty(n, 64, 1, dtype=BF, device=cuda_dev).transpose(1, 2)
        assert out.stride(1) == 1 and torch.equal(K.axial_rope(x, pos, rope, out=out), want)
        for a, b in zip(K.qk_headnorm_rope(x, x, None, None, 1e-6, pos, rope), K.qk_headnorm_rope(plain, plain, None, None, 1e-6, pos, rope)):
            assert torch.equal(a, b)
        want = K.packed_attention(plain, plain, plain, cu, cu)
        assert torch.equal(K.packed_attention(x, x, x, cu, cu, out=out), want)
        for q in (x[:1], x[-1:].as_strided((1, 1, 64), (3, 1, 1), x[-1:].storage_offset())):
            one = _cu([1], cuda_dev)
            assert torch.equal(K.packed_attention(q, x, x, one, cu), K.packed_attention(q.contiguous().clone(), plain, plain, one, cu))


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("q_len,n", [(1, 700), (4, 300), (4, 40), (300, 300), (40, 6000)])
def test_packed_attention_infinite_scores(cuda_dev, q_len, n, dim, dtype):
    """A score of -inf takes no part, a row of nothing else is zeros, a score of +inf makes its row NaN."""
    import lbw_b200.kernels as K
    q, k, v, cu_q, cu_k = _attention_case(cuda_dev, 5, [q_len], [n], 4, 2, dim, dtype)
    q[..., 3] = q[..., 3].abs() + 0.1
    gone = torch.zeros(n, dtype=torch.bool, device=cuda_dev)
    gone[1::3], gone[n // 2:n // 2 + 150] = True, True                      # (a whole key tile among them)
    k[gone, :, 3] = -math.inf
    want, bound = po.attention(q, k[~gone], v[~gone], cu_q, _cu([int((~gone).sum())], cuda_dev), causal=False)
    out = K.packed_attention(q, k, v, cu_q, cu_k, causal=False)
    assert po.within(out, want, bound) <= 1
    k[n // 3 // 3 * 3, 1, 3] = math.inf                                     # seen by the heads of the second kv head
    out = K.packed_attention(q, k, v, cu_q, cu_k, causal=False)
    assert torch.isnan(out[:, 2:].float()).all() and po.within(out[:, :2], want[:, :2], bound[:, :2]) <= 1
    k[..., 3] = -math.inf
    assert bool((K.packed_attention(q, k, v, cu_q, cu_k, causal=False) == 0).all())


AXES = ([16, 16], 10000.0, "half", "axis", [1.0, 1.0])


def _opcheck_args(name, dev):
    qkv = _randn(dev, 1, 50, 6, 64)
    q, k, v = (qkv[:, :2].contiguous(), qkv[:, 2:4].contiguous(), qkv[:, 4:].contiguous())
    pos, cu = torch.arange(100, device=dev).view(50, 2), _cu([20, 30], dev)
    if name == "axial_rope":
        return q, pos, *AXES, False, torch.empty_like(q)
    if name == "packed_attention":
        return q, k, v, cu, cu.clone(), torch.tensor([15, 30], dtype=torch.int32, device=dev), True, 0.125, torch.empty_like(q), 30
    caches = [torch.zeros(70, 2, 64, dtype=BF, device=dev) for _ in range(2)]
    return (q, k, _randn(dev, 2, 64), _randn(dev, 3, 64, dtype=F32), 1e-6, pos, *AXES, torch.empty_like(q), caches[0], v, caches[1],
            torch.arange(50, device=dev) + 10)


@pytest.mark.parametrize("name", ["axial_rope", "qk_headnorm_rope", "packed_attention"])
def test_packed_operators_opcheck(cuda_dev, name):
    """The tensors that an operator declares it writes are the ones it writes; compiled with dynamic shapes it does the same."""
    import lbw_b200.ops as O
    assert name in O.OPS
    res = torch.library.opcheck(getattr(torch.ops.lbw, name), _opcheck_args(name, cuda_dev),
                                test_utils=("test_schema", "test_faketensor", "test_aot_dispatch_dynamic"), raise_exception=False)
    assert all(v == "SUCCESS" for v in res.values()), res


def test_compiled_step_over_a_cache_equals_eager(cuda_dev):
    """A layer's middle in one graph: norm and rotation in place inside the fused tensor or to cache rows, lengths of the
    sequences in use, the output in the query's place; caches, rows and lengths that change between the calls."""
    import lbw_b200.kernels as K
    import lbw_b200.ops  # noqa: F401
    from lbw_b200.rope import AxialRope
    hq, hk, d, cap = 8, 2, 64, 90
    rope = AxialRope((16, 16))
    gain = _randn(cuda_dev, 9, d)

    def step(qkv, pos, rows, kc, vc, cu_q, cu_k, k_lens):
        q, k, v = qkv[:, :hq], qkv[:, hq:hq + hk], qkv[:, hq + hk:]
        qo, _ = K.qk_headnorm_rope(q, k, gain, None, 1e-6, pos, rope, q_out=q, k_out=kc, v=v, v_out=vc, k_rows=rows)
        return K.packed_attention(qo, kc, vc, cu_q, cu_k, k_lens=k_lens, out=qo, max_q=40)

    def prompt(qkv, pos, cu):
        q, k, v = qkv[:, :hq], qkv[:, hq:hq + hk], qkv[:, hq + hk:]
        K.qk_headnorm_rope(q, k, gain, gain, 1e-6, pos, rope, q_out=q, k_out=k)
        return K.axial_rope(K.packed_attention(q, k, v, cu, cu, causal=False), pos, rope, inverse=True)

    torch._dynamo.reset()
    compiled = torch.compile(step, fullgraph=True, backend="aot_eager")
    both = [[torch.zeros(2 * cap, hk, d, dtype=BF, device=cuda_dev) for _ in range(2)] for _ in range(2)]
    done = [0, 0]
    for i, new in enumerate(([40, 7], [1, 1], [1, 1], [3, 1])):
        at = torch.cat([torch.arange(done[b], done[b] + n) + b * cap for b, n in enumerate(new)]).to(cuda_dev)
        done = [a + n for a, n in zip(done, new)]
        pos = torch.stack([at, at * 3], 1)
        cu_q, cu_k = _cu(new, cuda_dev), _cu([cap, cap], cuda_dev)
        k_lens = torch.tensor(done, dtype=torch.int32, device=cuda_dev)
        qkv = [_randn(cuda_dev, i, sum(new), hq + 2 * hk, d) for _ in range(2)]
        with torch.no_grad():
            out = [f(x, pos, at, *c, cu_q, cu_k, k_lens) for f, x, c in zip((step, compiled), qkv, both)]
        assert torch.equal(*out) and torch.equal(*qkv)
        assert torch.equal(both[0][0], both[1][0]) and torch.equal(both[0][1], both[1][1])
    qkv = [_randn(cuda_dev, 8, 47, hq + 2 * hk, d) for _ in range(2)]
    pos, cu = torch.arange(94, device=cuda_dev).view(47, 2), _cu([40, 7], cuda_dev)
    assert torch.equal(prompt(qkv[0], pos, cu), torch.compile(prompt, fullgraph=True, backend="aot_eager")(qkv[1], pos, cu))
    assert torch.equal(*qkv)


def test_an_empty_operand_overlaps_nothing(cuda_dev):
    """Keys and values of no rows at the output's own address: nothing to read there."""
    import lbw_b200.kernels as K
    x, cu = _randn(cuda_dev, 1, 4, 2, 64), _cu([4], cuda_dev)
    assert bool((K.packed_attention(x, x[:0], x[:0], cu, cu * 0, out=x) == 0).all())
