"""The bound of the packed attention's 64-bit form (packed_oracle.attention) on the CPU: arithmetic like the kernels' stays
within it, and the faults that tests are there for - a row that was not written, a key tile that was left out - do not."""
import pytest
import torch

import packed_oracle as po

BF, HF = torch.bfloat16, torch.float16


def _emulated(q, k, v, drop=None):
    """One sequence, causal, fp32: 128 keys at a time, the running maximum moved when it grows by more than 2^8, probabilities
    rounded to the tensors' type for the second product. drop: a key tile that is left out."""
    tq, hq, d = q.shape
    n, group = k.shape[0], hq // k.shape[1]
    out = torch.zeros(q.shape)
    for h in range(hq):
        kk, vv = (x[:, h // group].float() for x in (k, v))
        s = q[:, h].float() @ kk.T
        hide = torch.arange(n)[None] > torch.arange(tq)[:, None] + (n - tq)
        s = s.masked_fill(hide, -torch.inf) * torch.tensor(1.4426950408889634 * d ** -0.5)
        m, l, o = torch.full((tq, 1), -torch.inf), torch.zeros(tq, 1), torch.zeros(tq, d)
        for t in range(0, n, 128):
            if t == drop:
                continue
            top = s[:, t:t + 128].amax(1, keepdim=True)
            new = torch.where(top > m + 8, top, m)
            a = torch.where(new > m, torch.exp2(m - new), torch.ones(()))
            p = torch.exp2(s[:, t:t + 128] - new.clamp(min=-1e30))
            m, l, o = new, l * a + p.sum(1, keepdim=True), o * a + p.to(q.dtype).float() @ vv[t:t + 128]
        out[:, h] = o / l
    return out.to(q.dtype)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("n", [1000, 2000, 5000])
def test_attention_bound_tells_a_fault_from_rounding(n, dim, dtype):
    g = torch.Generator().manual_seed(n + dim)
    q = (torch.randn(9, 4, dim, generator=g) * 1.5).to(dtype)
    k, v = (torch.randn(n, 2, dim, generator=g).to(dtype) for _ in range(2))
    cu_q, cu_k = torch.tensor([0, 9]), torch.tensor([0, n])
    want, bound = po.attention(q, k, v, cu_q, cu_k)
    out = _emulated(q, k, v)
    assert po.within(out, want, bound) <= 1
    none = out.clone()
    none[-1] = 0
    assert po.within(none, want, bound) > 4
    for drop in (0, 128 * (n // 256)):
        assert po.within(_emulated(q, k, v, drop), want, bound) > 1.5
