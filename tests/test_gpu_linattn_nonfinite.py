"""Infinities and NaN in linear attention: where they may go, and where not."""
import pytest
import torch

from sffft_amd import torch_ops  # noqa: F401

pytestmark = pytest.mark.gpu
NAN, INF = float("nan"), float("inf")
DTYPES = pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])


def inputs(dev, B, T, H, Hk, Dk, Dv, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)

    def r(*s, dt=dtype):
        return torch.randn(*s, generator=g).to(dt).to(dev)

    ld = torch.linspace(-0.5, -0.01, H).to(dev)
    return r(B, T, H, Dk), r(B, T, Hk, Dk), r(B, T, Hk, Dv), ld, r(B, H, Dk, Dv, dt=torch.float32), r(B, T, H, Dv), \
        r(B, H, Dk, Dv, dt=torch.float32)


def run(q, k, v, ld, s0, go, gs, lengths=None):
    """{name: output} of the forward and backward pass."""
    x = [t.detach().requires_grad_() for t in (q, k, v, s0)]
    o, s = torch.ops.sffft.linear_attention(*x[:3], ld, 0.2, x[3], lengths)
    return dict(zip(("o", "state", "dq", "dk", "dv", "dstate"), (o.detach(), s.detach(), *torch.autograd.grad((o, s), x, (go, gs)))))


@DTYPES
@pytest.mark.parametrize("D", [16, 64, 128])
@pytest.mark.parametrize("T,lengths", [(1, [0, 1]), (70, [3, 70]), (700, [150, 64])])
def test_tokens_that_do_not_count_give_zero_whatever_the_states_hold(dev, T, lengths, D, dtype):
    q, k, v, ld, s0, go, gs = inputs(dev, 2, T, 4, 2, D, D, dtype, seed=T)
    n = torch.tensor(lengths, dtype=torch.int32, device=dev)
    s0[0, 1, 3, 5], s0[1, 2, 0, 0] = INF, NAN
    gs[0, 0, 1, 2], gs[1, 3, 7, 7] = NAN, -INF
    got = run(q, k, v, ld, s0, go, gs, n)
    for name in ("o", "dq", "dk", "dv"):
        for b, m in enumerate(lengths):
            assert not bool(got[name][b, m:].any()), (name, b)
    for b, m in enumerate(lengths):
        if m == 0:
            assert torch.equal(got["state"][b], s0[b]) and torch.equal(got["dstate"][b].nan_to_num(1), gs[b].nan_to_num(1))
