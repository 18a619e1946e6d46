"""Calls whose queries have no heads but whose keys do: every output is made, none is left as it was allocated."""
import pytest
import torch

import mixer_oracle as mo
from sffft_amd import mixers, torch_ops  # noqa: F401

pytestmark = pytest.mark.gpu


def leave_marks(dev, *shapes):
    """Memory that the allocator hands out next for these shapes holds NaN."""
    marks = [torch.full(s, float("nan"), dtype=dt, device=dev) for s in shapes for dt in (torch.float32, torch.bfloat16) for _ in range(3)]
    del marks


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("interleaved", [False, True], ids=["half", "interleaved"])
def test_rotary_of_keys_alone(dev, interleaved, dtype):
    g = torch.Generator().manual_seed(1)
    k, gk = (torch.randn(2, 9, 3, 64, generator=g).to(dtype).to(dev) for _ in range(2))
    none = k[:, :, :0]
    table = mixers.rotary_table(16, 32, device=dev)
    want, _ = torch.ops.sffft.rotary(k, none, table, None, interleaved)
    leave_marks(dev, k.shape)
    x = k.clone().requires_grad_()
    q, got = torch.ops.sffft.rotary(none, x, table, None, interleaved)
    assert q.shape == none.shape and torch.equal(got, want)
    grad, = torch.autograd.grad(got, x, gk)
    assert torch.equal(grad, torch.ops.sffft.rotary(gk, none, table, None, interleaved, True)[0])
    y = k.clone()
    torch.ops.sffft.rotary_(none, y, table, None, interleaved)
    assert torch.equal(y, want)
    assert mo.rel_l2(got, mo.rotary(k, table, None, interleaved)) < (2.0 ** -8 if dtype == torch.bfloat16 else 1e-6)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
def test_attention_without_queries(dev, dtype):
    """Nothing depends on the keys and values: their gradients are zero."""
    k, v = (torch.randn(2, 9, 3, 64).to(dtype).to(dev).requires_grad_() for _ in range(2))
    q, s0 = torch.zeros(2, 9, 0, 64, dtype=dtype, device=dev), torch.zeros(2, 0, 64, 64, device=dev).requires_grad_()
    leave_marks(dev, k.shape)
    o, s = torch.ops.sffft.linear_attention(q, k, v, torch.zeros(0, device=dev), 0.1, s0)
    assert o.shape == (2, 9, 0, 64) and s.shape == (2, 0, 64, 64)
    leave_marks(dev, k.shape)
    for g, x in zip(torch.autograd.grad((o, s), (k, v, s0), (torch.zeros_like(o), torch.zeros_like(s))), (k, v, s0)):
        assert torch.equal(g, torch.zeros_like(x))
