"""Rotary positions on the GPU against the 64-bit rotation, pair by pair.

Tolerances: an output is two products and a sum in fp32, each rounded (3 * 2^-24 of the pair's size), then for
bf16 rounded once more (half a unit in the last of 8 significant bits: up to 2^-8 of the value).
"""
import pytest
import torch

import mixer_oracle as mo
from sffft_amd import mixers, torch_ops  # noqa: F401

pytestmark = pytest.mark.gpu


def check(got, want):
    x, y = got.detach().double().cpu(), want
    if got.dtype == torch.bfloat16:
        assert bool(((x - y).abs() <= 2.0 ** -8 * y.abs() + 1e-5).all())
    else:
        assert float((x - y).abs().max()) <= 4 * 2.0 ** -24 * float(y.abs().max()) * 1.5


CASES = [  # B, T, H, Hk, D, R
    (1, 1, 1, 1, 2, 2), (2, 1, 12, 12, 64, 64), (3, 17, 4, 1, 32, 16), (1, 33, 3, 3, 96, 48), (2, 5, 2, 2, 128, 32),
    (2, 9, 5, 1, 20, 6), (1, 7, 2, 1, 64, 30), (1, 65, 1, 0, 256, 128), (2, 1000, 2, 2, 64, 64),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("interleaved", [False, True], ids=["half", "interleaved"])
@pytest.mark.parametrize("case", CASES, ids=str)
def test_forward_and_gradients(dev, case, interleaved, dtype):
    B, T, H, Hk, D, R = case
    g = torch.Generator().manual_seed(T + D)
    def r(*s):
        return torch.randn(*s, generator=g).to(dtype).to(dev)
    q, k, gq, gk = r(B, T, H, D), r(B, T, Hk, D), r(B, T, H, D), r(B, T, Hk, D)
    table = mixers.rotary_table(4096, R, 1e4, "parts", 4.0, 512, device=dev)
    for positions in (None, torch.randint(0, 4096, (B, T), generator=g).int().to(dev),
                      torch.randint(0, 4096, (B, T), generator=g).to(dev)):
        x = [t.detach().requires_grad_() for t in (q, k)]
        out = torch.ops.sffft.rotary(*x, table, positions, interleaved)
        grads = torch.autograd.grad(out, x, (gq, gk))
        for a, t in zip(out, (q, k)):
            if t.numel():
                check(a, mo.rotary(t, table, positions, interleaved))
                assert torch.equal(a[..., R:], t[..., R:])
        for a, t in zip(grads, (gq, gk)):
            if t.numel():
                check(a, mo.rotary(t, table, positions, interleaved, inverse=True))
        # in place, and the binding: the same bits
        y = q.clone(), k.clone()
        torch.ops.sffft.rotary_(*y, table, positions, interleaved)
        assert torch.equal(y[0], out[0]) and torch.equal(y[1], out[1])
        if Hk:
            z = mixers.rotary(q, k, table, positions, interleaved)
            assert torch.equal(z[0], out[0]) and torch.equal(z[1], out[1])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
def test_strides(dev, dtype):
    B, T, H, D = 2, 19, 3, 64
    g = torch.Generator().manual_seed(7)
    table = mixers.rotary_table(64, 32, device=dev)
    fused = torch.randn(B, T, 2, H, D, generator=g).to(dtype).to(dev)
    wide = torch.randn(2, B, T, H, D + 1, generator=g).to(dtype).to(dev)
    turned = torch.randn(2, B, T, D, H, generator=g).to(dtype).to(dev)
    major = torch.randn(2, B, H, T, D, generator=g).to(dtype).to(dev)
    for q, k in (fused.unbind(2), wide[..., 1:].unbind(0), turned.transpose(3, 4).unbind(0),
                 major.transpose(2, 3).unbind(0), (fused[:, :, 0], fused[:, :1, 1].expand(B, T, H, D))):
        a = torch.ops.sffft.rotary(q, k, table)
        b = torch.ops.sffft.rotary(q.contiguous(), k.contiguous(), table)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    # in place in a view: what lies beside it stays
    before = fused.clone()
    q = fused[:, :, 0]
    torch.ops.sffft.rotary_(q, q[:, :, :0], table)
    assert torch.equal(fused[:, :, 1], before[:, :, 1])
    assert torch.equal(fused[:, :, 0], torch.ops.sffft.rotary(before[:, :, 0], before[:, :, 1], table)[0])


def test_positions_outside_the_table(dev):
    table = mixers.rotary_table(16, 32, device=dev)
    q = torch.randn(1, 4, 2, 64, device=dev)
    for dt in (torch.int32, torch.int64):
        pos = torch.tensor([[3, -1, 16, 15]], dtype=dt, device=dev)
        if dt == torch.int64:
            pos[0, 1] = 1 << 40
        out, _ = torch.ops.sffft.rotary(q, q, table, pos)
        assert bool(torch.isnan(out[0, 1:3, :, :32]).all()) and bool(torch.isfinite(out[0, [0, 3]]).all())
        assert torch.equal(out[..., 32:], q[..., 32:])


def test_gradient_against_differences(dev):
    """Linear: <g, f(x + d)> - <g, f(x)> = <f*(g), d>, to the rounding of fp32 sums."""
    g = torch.Generator().manual_seed(0)
    q, k, d, gq = (torch.randn(2, 30, 3, 64, generator=g).to(dev) for _ in range(4))
    table = mixers.rotary_table(30, 48, device=dev)
    x = q.clone().requires_grad_()
    out, _ = torch.ops.sffft.rotary(x, k, table)
    grad, = torch.autograd.grad(out, x, gq)
    moved, _ = torch.ops.sffft.rotary(q + d, k, table)
    want = float(((moved.double() - out.detach().double()) * gq).sum())
    assert abs(float((grad.double() * d).sum()) - want) < 1e-4 * float(gq.norm() * d.norm()) / d.numel() ** 0.5
    # and its gradient again
    x = q.clone().requires_grad_()
    y = gq.clone().requires_grad_()
    grad, = torch.autograd.grad(torch.ops.sffft.rotary(x, k, table)[0], x, y, create_graph=True)
    again, = torch.autograd.grad(grad, y, d)
    assert torch.equal(again, torch.ops.sffft.rotary(d, k, table)[0])


def test_refusals(dev):
    f, inplace = torch.ops.sffft.rotary, torch.ops.sffft.rotary_
    q, k, table = torch.zeros(2, 3, 4, 16, device=dev), torch.zeros(2, 3, 2, 16, device=dev), torch.zeros(8, 8, device=dev)
    pos = torch.zeros(2, 3, dtype=torch.int32, device=dev)
    bad = [lambda: f(q.half(), k.half(), table), lambda: f(q, k.bfloat16(), table), lambda: f(q, k[:, :2], table),
           lambda: f(q, k[..., :8], table), lambda: f(q, k, table[:, :7]), lambda: f(q, k, torch.zeros(8, 18, device=dev)),
           lambda: f(q, k, table.double()), lambda: f(q, k, table.cpu()), lambda: f(q, k, table, pos[:1]),
           lambda: f(q, k, table, pos.float()), lambda: f(q, k, table, pos.cpu()),
           lambda: f(q, k, table.clone().requires_grad_()), lambda: f(q[..., :15], k[..., :15], table),
           lambda: inplace(q.transpose(2, 3), k, table), lambda: inplace(q[:, :1].expand(2, 3, 4, 16), k, table),
           lambda: inplace(q.clone().requires_grad_(), k, table)]
    for i, call in enumerate(bad):
        with pytest.raises(RuntimeError):
            call()
            raise AssertionError(i)
