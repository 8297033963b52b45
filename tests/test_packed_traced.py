"""The packed-sequence operators inside a compiled graph and called as torch.ops.lbw: what eager calls refuse is refused
there too. Without a GPU: a refusal comes before any kernel."""
import pytest
import torch

import lbw_b200.kernels as K
import lbw_b200.ops  # noqa: F401
import lbw_b200.rope as rope

BF = torch.bfloat16
ROPE = rope.AxialRope((32,))
AXES = ([32], 10000.0, "interleaved", "axis", [1.0])


def _x(grad=False):
    return torch.zeros(4, 2, 64, dtype=BF).requires_grad_(grad)


POS = torch.zeros(4, 1, dtype=torch.int32)
CU = torch.tensor([0, 4], dtype=torch.int32)
GAIN = torch.ones(64)


def _direct(name, at):
    """torch.ops.lbw.<name> with a gradient required of one operand."""
    g = [i == at for i in range(9)]
    gain = GAIN.clone().requires_grad_(g[2])
    if name == "axial_rope":
        torch.ops.lbw.axial_rope(_x(g[0]), POS, *AXES, False, _x(g[1]))
    elif name == "qk_headnorm_rope":
        torch.ops.lbw.qk_headnorm_rope(_x(g[0]), _x(g[1]), gain, GAIN, 1e-6, POS, *AXES, _x(g[3]), _x(g[4]), None, None, None)
    else:
        torch.ops.lbw.packed_attention(_x(g[0]), _x(g[1]), _x(g[2]), CU, CU, None, True, 0.125, _x(g[3]), 0)


CASES = [("axial_rope", i) for i in range(2)] + [("qk_headnorm_rope", i) for i in range(5)] \
    + [("packed_attention", i) for i in range(4)]


@pytest.mark.parametrize("name,at", CASES)
def test_operator_refuses_a_gradient(name, at):
    with pytest.raises(ValueError, match="has no gradient"):
        _direct(name, at)
    with torch.no_grad(), pytest.raises(ValueError, match="CUDA"):           # allowed: it goes on to the kernel's checks
        _direct(name, at)


@pytest.mark.parametrize("fullgraph", [True, False])
@pytest.mark.parametrize("call", [
    lambda x, g: K.axial_rope(x, POS, ROPE), lambda x, g: K.qk_headnorm_rope(x, x, None, None, 1e-6, POS, ROPE),
    lambda x, g: K.qk_headnorm_rope(x.detach(), x.detach(), g, g, 1e-6), lambda x, g: K.packed_attention(x, x, x, CU, CU)])
def test_compiled_graph_refuses_a_gradient(call, fullgraph):
    torch._dynamo.reset()
    f = torch.compile(call, fullgraph=fullgraph, backend="aot_eager")
    with pytest.raises(Exception, match="has no gradient"):
        f(_x(True), GAIN.clone().requires_grad_())


@pytest.mark.parametrize("fullgraph", [True, False])
def test_compiled_graph_refuses_cache_rows_without_a_cache(fullgraph):
    """k_rows name rows of k_out: without it there is no cache that they could be rows of."""
    rows = torch.arange(4)

    def call(x):
        return K.qk_headnorm_rope(x, x, None, None, 1e-6, POS, ROPE, k_rows=rows)[1]

    with pytest.raises(ValueError, match="k_rows name rows of k_out"):
        call(_x())
    torch._dynamo.reset()
    with pytest.raises(Exception, match="k_rows name rows of k_out"):
        torch.compile(call, fullgraph=fullgraph, backend="aot_eager")(_x())
