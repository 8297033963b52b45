"""Packed-sequence operators without a GPU: the rotation's description, refusals, and the C entries' argument checks."""
import copy
import ctypes
import math
import pickle

import pytest
import torch

import lbw_b200._lib as L
import lbw_b200.kernels as K
import lbw_b200.rope as rope
import packed_oracle as po

BF = torch.bfloat16


@pytest.fixture(scope="module")
def lib():
    import __graft_entry__
    __graft_entry__.build()
    return L.load()


def test_axial_rope_frequencies_are_the_three_axis_tables():
    r = rope.AxialRope((22, 21, 21))
    freqs = rope.rope_freqs(max_frames=2)[1].double()          # angles at position 1
    assert torch.allclose(torch.tensor(r.inv_freq, dtype=torch.float64), freqs, rtol=1e-6)
    assert r.axis_of_pair == [0] * 22 + [1] * 21 + [2] * 21
    for i, f in enumerate(r.inv_freq):
        assert abs(r.c.step[i] / 2.0 ** 64 * 2 * math.pi - f) <= f * 2.0 ** -52 + 2.0 ** -64 * 7


def test_axial_rope_head_spectrum_and_scale():
    r = rope.AxialRope((3, 5), theta=100.0, spectrum="head", layout="half", scale=(0.5, 2.0))
    want = [100.0 ** (-i / 8) * (0.5 if i < 3 else 2.0) for i in range(8)]
    assert r.inv_freq == pytest.approx(want, rel=1e-15)
    assert (r.c.pairs, r.c.axes, r.c.layout) == (8, 2, 1)


@pytest.mark.parametrize("kw", [dict(sections=()), dict(sections=(3,)), dict(sections=(5, -1)), dict(sections=(132,)),
                                dict(sections=(8,), layout="pairs"), dict(sections=(8,), spectrum="x"),
                                dict(sections=(8,), scale=(1.0, 1.0)), dict(sections=(8,), scale=math.inf),
                                dict(sections=(8,), theta=0.0), dict(sections=(4,) * 9)])
def test_axial_rope_refuses(kw):
    with pytest.raises(ValueError):
        rope.AxialRope(**kw)


def test_cpu_tensors_are_refused():
    x = torch.zeros(4, 2, 64, dtype=BF)
    pos = torch.zeros(4, 1, dtype=torch.int32)
    cu = torch.tensor([0, 4], dtype=torch.int32)
    r = rope.AxialRope((32,))
    for call in (lambda: K.axial_rope(x, pos, r), lambda: K.qk_headnorm_rope(x, x, None, None, 1e-6, pos, r),
                 lambda: K.packed_attention(x, x, x, cu, cu)):
        with pytest.raises(ValueError, match="CUDA"):
            call()


def _axial(lib, a):
    seg = L.HEAD_ROWS.pack(_at(a["x"]), _at(a["out"]), 0, a["x_tok"], a["x_head"], a["out_tok"], a["out_head"], a["heads"], 0)
    return lib.lbw_axial_rope(seg, *(a[n] for n in ("tokens", "dim", "dtype", "pos", "bits", "pos_tok", "pos_axis", "rope",
                                                    "inverse")), None)


def _packed(lib, a):
    first = "q q_tok q_head k k_tok k_head v v_tok v_head out out_tok out_head cu_q cu_k k_lens".split()
    batch = L.PACKED_BATCH.pack(*(_at(a[n]) for n in first), *(a[n] for n in ("tq", "tk", "n", "hq", "hk", "dim", "dtype",
                                                                            "causal", "max_q", "scale")))
    return lib.lbw_packed_attention(batch, a["ws"], a["ws_bytes"], None)


def _at(p):
    return (p.value if isinstance(p, ctypes.c_void_p) else p) or 0


def _rope(pairs=32, axes=1, layout=0, axis=0):
    r = rope.RopeAxes(pairs, axes, layout, 0)
    r.axis[0] = axis
    return ctypes.byref(r)


P = ctypes.c_void_p(4096)


@pytest.mark.parametrize("change,status", [
    (dict(x=None), L.LBW_ERR_INVALID), (dict(out=None), L.LBW_ERR_INVALID), (dict(rope=None), L.LBW_ERR_INVALID),
    (dict(pos=None), L.LBW_ERR_INVALID), (dict(bits=16), L.LBW_ERR_INVALID), (dict(dtype=3), L.LBW_ERR_INVALID),
    (dict(dim=100), L.LBW_ERR_SHAPE), (dict(dim=264), L.LBW_ERR_SHAPE), (dict(dim=56), L.LBW_ERR_SHAPE),
    (dict(heads=0), L.LBW_ERR_SHAPE), (dict(tokens=-1), L.LBW_ERR_SHAPE), (dict(x_tok=1001), L.LBW_ERR_ALIGN),
    (dict(x=ctypes.c_void_p(4104)), L.LBW_ERR_ALIGN), (dict(rope=_rope(30)), L.LBW_ERR_SHAPE),
    (dict(rope=_rope(32, 0)), L.LBW_ERR_SHAPE), (dict(rope=_rope(32, 1, 2)), L.LBW_ERR_INVALID),
    (dict(rope=_rope(32, 1, 0, 1)), L.LBW_ERR_INVALID), (dict(rope=_rope(132)), L.LBW_ERR_SHAPE),
    (dict(tokens=0, x=None, out=None, pos=None), L.LBW_OK)])
def test_axial_rope_entry_checks(lib, change, status):
    a = dict(x=P, x_tok=1024, x_head=64, out=P, out_tok=1024, out_head=64, tokens=5, heads=2, dim=64, dtype=0, pos=P,
             bits=32, pos_tok=1, pos_axis=1, rope=_rope(), inverse=0)
    a.update(change)
    rc = _axial(lib, a)
    assert rc == status
    if status:
        assert "axial_rope" in L.last_error()


def _rows(**kw):
    r = dict(x=4096, out=4096, gamma=0, x_tok=1024, x_head=64, out_row=1024, out_head=64, heads=2, gamma_f32=0)
    r.update(kw)
    return L.HEAD_ROWS.pack(*r.values())


@pytest.mark.parametrize("change,status", [
    (dict(q=None), L.LBW_ERR_INVALID), (dict(k=None), L.LBW_ERR_INVALID), (dict(q=_rows(x=0)), L.LBW_ERR_INVALID),
    (dict(k=_rows(out=4098)), L.LBW_ERR_ALIGN), (dict(k=_rows(out_row=1020)), L.LBW_ERR_ALIGN),
    (dict(v=_rows(heads=0)), L.LBW_ERR_SHAPE), (dict(q=_rows(gamma=4097)), L.LBW_ERR_ALIGN),
    (dict(eps=-1.0), L.LBW_ERR_INVALID), (dict(eps=math.nan), L.LBW_ERR_INVALID), (dict(rows_bits=8), L.LBW_ERR_INVALID),
    (dict(out_rows=-1), L.LBW_ERR_SHAPE), (dict(dim=12), L.LBW_ERR_SHAPE), (dict(tokens=0, q=_rows(x=0)), L.LBW_OK)])
def test_qk_headnorm_rope_entry_checks(lib, change, status):
    a = dict(q=_rows(), k=_rows(), v=None, tokens=5, dim=64, dtype=0, eps=1e-6, pos=P, bits=32, pos_tok=1, pos_axis=1,
             rope=_rope(), rows=P, rows_bits=64, out_rows=9)
    a.update(change)
    assert lib.lbw_qk_headnorm_rope(*a.values(), None) == status


CALL = dict(q=P, q_tok=1024, q_head=64, k=P, k_tok=1024, k_head=64, v=P, v_tok=1024, v_head=64, out=P, out_tok=1024,
            out_head=64, cu_q=P, cu_k=P, k_lens=None, n=2, tq=100, tk=100, hq=8, hk=2, dim=64, dtype=0, causal=1, scale=0.1,
            max_q=0, ws=P, ws_bytes=1 << 40)


@pytest.mark.parametrize("change,status", [
    (dict(q=None), L.LBW_ERR_INVALID), (dict(v=None), L.LBW_ERR_INVALID), (dict(out=None), L.LBW_ERR_INVALID),
    (dict(cu_q=None), L.LBW_ERR_INVALID), (dict(dim=96), L.LBW_ERR_SHAPE), (dict(hk=3), L.LBW_ERR_SHAPE),
    (dict(hk=0), L.LBW_ERR_SHAPE), (dict(n=-1), L.LBW_ERR_SHAPE), (dict(tk=1 << 31), L.LBW_ERR_SHAPE),
    (dict(tq=1 << 28), L.LBW_ERR_SHAPE), (dict(tq=1 << 62), L.LBW_ERR_SHAPE), (dict(n=1 << 30), L.LBW_ERR_SHAPE),
    (dict(dtype=2), L.LBW_ERR_INVALID), (dict(scale=0.0), L.LBW_ERR_INVALID), (dict(scale=math.nan), L.LBW_ERR_INVALID),
    (dict(scale=math.inf), L.LBW_ERR_INVALID), (dict(out_tok=1028), L.LBW_ERR_ALIGN),
    (dict(out=ctypes.c_void_p(4104)), L.LBW_ERR_ALIGN), (dict(cu_k=ctypes.c_void_p(4098)), L.LBW_ERR_ALIGN),
    (dict(tq=0), L.LBW_OK), (dict(n=0), L.LBW_OK)])
def test_packed_attention_entry_checks(lib, change, status):
    assert _packed(lib, {**CALL, **change}) == status


def test_packed_attention_refuses_a_small_workspace(lib):
    n = ctypes.c_longlong(-1)
    assert lib.lbw_packed_attention_workspace(1, 100000, 8, 2, 128, 1, 1, 0, ctypes.byref(n), None) == L.LBW_OK
    assert n.value > 0
    rc = _packed(lib, {**CALL, "q_head": 128, "k_head": 128, "v_head": 128, "out_head": 128, "n": 1, "tq": 1, "tk": 100000,
                       "dim": 128, "max_q": 1, "ws_bytes": n.value - 1})
    assert rc == L.LBW_ERR_INVALID and "workspace" in L.last_error()
    assert lib.lbw_packed_attention_workspace(1, 100, 8, 3, 128, 1, 1, 0, ctypes.byref(n), None) == L.LBW_ERR_SHAPE
    assert lib.lbw_packed_attention_workspace(1, 100, 8, 2, 128, 1, 1, 0, None, None) == L.LBW_ERR_INVALID
    assert lib.lbw_packed_attention(None, P, 0, None) == lib.lbw_axial_rope(None, 1, 64, 0, P, 32, 1, 1, _rope(), 0, None) \
        == L.LBW_ERR_INVALID


def test_in_place_calls_that_would_race_are_refused(lib):
    """x as its own output with other strides or rows, keys or values as the output of the attention."""
    axial = dict(x=P, x_tok=1024, x_head=64, out=P, out_tok=2048, out_head=64, tokens=5, heads=2, dim=64, dtype=0, pos=P,
                 bits=32, pos_tok=1, pos_axis=1, rope=_rope(), inverse=0)
    assert _axial(lib, axial) == L.LBW_ERR_INVALID and "in place" in L.last_error()
    there = _rows(out=8192)
    for q, k, v, rows in ((_rows(out_head=128), there, None, None), (there, _rows(), None, P), (there, there, _rows(), P)):
        assert lib.lbw_qk_headnorm_rope(q, k, v, 5, 64, 0, 1e-6, P, 32, 1, 1, _rope(), rows, 64, 9, None) == L.LBW_ERR_INVALID
        assert "in place" in L.last_error()
    far = ctypes.c_void_p(1 << 20)
    for q, k, v, out_tok in ((far, P, far, 1024), (far, far, P, 1024), (P, far, far, 2048)):
        assert _packed(lib, {**CALL, "q": q, "k": k, "v": v, "out_tok": out_tok}) == L.LBW_ERR_INVALID
        assert "out is" in L.last_error()


def test_packed_attention_refuses_a_scale_out_of_range(lib):
    for scale in (3e38, 1e-46):                                             # times log2 e: infinite, zero
        assert _packed(lib, {**CALL, "scale": scale}) == L.LBW_ERR_INVALID
        assert "softmax_scale" in L.last_error()


def test_axial_rope_can_be_copied_and_pickled():
    """A model that holds one is deep-copied and saved whole."""
    r = rope.AxialRope((8, 4, 4), theta=500.0, layout="half", spectrum="head", scale=(1.0, 0.5, 2.0))
    for c in (copy.deepcopy(r), pickle.loads(pickle.dumps(r))):
        assert bytes(c.c) == bytes(r.c) and c.scale == r.scale and c.axis_of_pair == r.axis_of_pair


@pytest.mark.parametrize("kw", [dict(sections=(22, 21, 21)), dict(sections=(64,), theta=1e6), dict(sections=(3, 5), spectrum="head"),
                                dict(sections=(8, 4, 4), theta=500.0, scale=(1.0, 0.3, -2.0)),
                                dict(sections=(8,), theta=0.01, scale=1e9)])
def test_axial_rope_steps_hold_128_bits_of_the_frequency(kw):
    """Against theta^-e in 150 digits: the error of an angle is that of the step times the position."""
    r = rope.AxialRope(**kw)
    want = po.turns_per_position(r.sections, r.theta, r.spectrum, r.scale)
    for i, t in enumerate(want):
        got = r.c.step[i] << 64 | r.c.step_low[i]
        off = ((got << 64) - t + (1 << 191)) % (1 << 192) - (1 << 191)
        assert abs(off) <= 1 << 63                                          # half a step of 2^-128 turns
    assert r.c.wide == 1


def test_outputs_that_overlap_an_operand_are_refused(lib):
    """Not only at the same address: later rows, other heads, rows of the cache, and the other operands' outputs."""
    axial = dict(x=P, x_tok=128, x_head=64, out=ctypes.c_void_p(4096 + 256), out_tok=128, out_head=64, tokens=5, heads=2, dim=64,
                 dtype=0, pos=P, bits=32, pos_tok=1, pos_axis=1, rope=_rope(), inverse=0)
    for change in ({}, dict(out=ctypes.c_void_p(4096 - 256)), dict(x_tok=256, out_tok=256, out=ctypes.c_void_p(4096 + 128))):
        assert _axial(lib, {**axial, **change}) == L.LBW_ERR_INVALID and "overlaps x" in L.last_error()
    near = lambda at, out, **kw: _rows(x=at, out=out, x_tok=128, out_row=128, **kw)   # noqa: E731 (5 rows: 1,280 bytes)
    a, b, c, d = (1 << 20 + i for i in range(4))
    for q, k, v, rows, say in (
            (near(a, b), near(b, c), None, None, "q overlaps k"), (near(a, a), near(a, c), None, None, "q overlaps k"),
            (near(a, c), near(b, c + 256), None, None, "outputs of q and k"), (near(a, c), near(b, a + 1024), None, None, "k overlaps q"),
            (near(a, a), near(b + 256 * 8, b), None, P, "k overlaps k"),          # a cache row in use as the new keys
            (near(a, a), near(b, c), near(c + 256 * 39, d), P, "k overlaps v"), (near(a, a), near(b, c), near(d, c + 512), P, "outputs of k")):
        assert lib.lbw_qk_headnorm_rope(q, k, v, 5, 64, 0, 1e-6, P, 32, 1, 1, _rope(), rows, 64, 40, None) == L.LBW_ERR_INVALID
        assert say in L.last_error(), L.last_error()
    far = ctypes.c_void_p(1 << 30)
    at = ctypes.c_void_p((1 << 20) + 2 * 1024 * 99)                                # the last of the 100 rows
    for name in "qkv":
        one = {**dict(q=far, k=far, v=far), name: ctypes.c_void_p(1 << 20), "out": at}
        assert _packed(lib, {**CALL, **one}) == L.LBW_ERR_INVALID and "overlaps" in L.last_error()


def test_strides_of_a_dimension_of_one_are_not_passed_on():
    x = torch.zeros(5, 64, 1).transpose(1, 2)
    assert x.stride() == (64, 1, 1) and K._rows3("op", "x", K._form(x)) == (5, 1, 64, 64, 0)
    x = torch.zeros(2, 64).as_strided((1, 2, 64), (3, 64, 1))
    assert K._rows3("op", "x", K._form(x)) == (1, 2, 64, 0, 64)
