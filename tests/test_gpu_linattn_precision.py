"""How far linear attention's bf16 outputs are from the once-rounded 64-bit ones.

On the way to an output of 16 bits nothing is held in fewer than 16: weights within a chunk, entering states and
decayed values are sums of two bf16 parts, each off by up to 2^-17 of its size. The terms of an output are off
independently, so it is too, relative to outputs of usual size, and rounds to the other neighbour where it lies
that near the middle of two: for a share of at most 2 * 2^-17 / 2^-8 of them (neighbours are 2^-8 or more apart),
which are then off by 2^-7 at most. Relative L2 between the outputs and the rounded 64-bit ones: sqrt(2^-8) * 2^-7
= 2^-11; twice that is allowed.
"""
import pytest
import torch

import mixer_oracle as mo
from sffft_amd import torch_ops  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B,T,H,Hk,Dk,Dv", [(1, 1, 3, 3, 64, 64), (2, 61, 4, 4, 64, 64), (1, 650, 4, 4, 128, 128), (2, 500, 6, 2, 32, 64),
                                            (2, 1237, 12, 12, 64, 64), (1, 900, 4, 2, 96, 128), (8, 300, 12, 12, 128, 64)], ids=str)
def test_outputs_are_rounded_once(dev, B, T, H, Hk, Dk, Dv):
    g = torch.Generator().manual_seed(T)

    def r(*s, dt=torch.bfloat16):
        return torch.randn(*s, generator=g).to(dt).to(dev)

    q, k, v, go = r(B, T, H, Dk), r(B, T, Hk, Dk), r(B, T, Hk, Dv), r(B, T, H, Dv)
    s0, gs = (r(B, H, Dk, Dv, dt=torch.float32) * 4 for _ in range(2))
    ld = torch.linspace(-1.0, -0.001, H).to(dev)
    want = mo.attention_pairs(q, k, v, ld, Dk ** -0.5, go, s0, gs)
    x = [t.requires_grad_() for t in (q, k, v, s0)]
    o, s = torch.ops.sffft.linear_attention(q, k, v, ld, Dk ** -0.5, s0)
    got = (o, s, *torch.autograd.grad((o, s), x, (go, gs)))
    for name, a, w in zip(("o", "state", "dq", "dk", "dv"), got, want):
        if name != "state":
            assert mo.rel_l2(a, w.bfloat16()) < 2.0 ** -10, (name, mo.rel_l2(a, w.bfloat16()))
