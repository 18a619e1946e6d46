"""Heads that forget very slowly, over thousands of chunks: the error of a decay does not add up.

A state that is decayed by factors that are each rounded to fp32 is off by up to 2^-24 for each of them, in the same
direction: 1e-4 over 2048 chunks. With that made up for there remain roundings that are independent of each other. A
chunk rounds the state once when it decays it and, at bf16's three parts of two halves or fp32's six products, in six
matrix instructions of 32 products, whose partial sums may be rounded for each 8 of them: 25 roundings of 2^-25, over
2048 chunks 2^-25 sqrt(51200) = 7e-6 of the size of a head's state; 2e-5 is allowed. Of that the part along the
state itself, which is what a wrong decay leaves, is an eighth (64 elements), and the decay's argument adds 2^-23 of
itself, at most 6.6: 1e-5 is allowed, for 2e-6 expected.
"""
import pytest
import torch

from sffft_amd import torch_ops  # noqa: F401

pytestmark = pytest.mark.gpu


def oracle(q, k, v, ld, s0, scale):
    """(o of the last 64 tokens, final state) in 64 bits, by the sums over all tokens, on the inputs' device."""
    T = q.shape[1]
    t = torch.arange(T, dtype=torch.float64, device=q.device)
    ld = ld.double()
    k, v = (x.double().permute(0, 2, 1, 3).contiguous() for x in (k, v))  # [B, H, T, D]
    w = torch.exp(ld[:, None] * (T - 1 - t))[None, :, :, None]
    last = torch.matmul((k * w).transpose(2, 3).contiguous(), v) + torch.exp(ld * T)[None, :, None, None] * s0.double()
    o = []
    for i in range(T - 64, T):
        w = torch.exp(ld[:, None] * (i - t[:i + 1]))[None, :, :, None]
        s = torch.matmul((k[:, :, :i + 1] * w).transpose(2, 3).contiguous(), v[:, :, :i + 1]) + \
            torch.exp(ld * (i + 1))[None, :, None, None] * s0.double()
        o.append(scale * torch.matmul(q[:, i].double()[:, :, None], s)[:, :, 0])
    return torch.stack(o, 1), last


@pytest.mark.parametrize("dtype,T", [(torch.float32, 65536), (torch.bfloat16, 131072)], ids=["fp32", "bf16"])
@pytest.mark.parametrize("heads", [1024, 2], ids=["one march", "many segments"])
def test_states_after_many_chunks(dev, heads, dtype, T):
    """Enough heads for one march over all tokens, and few, whose segments a scan joins. The initial state outweighs
    what the tokens add, so that its decay is what is seen; every head is looked at by itself."""
    H, D = min(heads, 256), 8
    B = heads // H
    g = torch.Generator(device=dev).manual_seed(0)

    def r(*s):
        return torch.randn(*s, generator=g, device=dev)

    ld = -torch.logspace(-6.2, -4.3, H, device=dev)
    q, k, v = (r(B, T, H, D).to(dtype) for _ in range(3))
    s0 = r(B, H, D, D) * 1e5
    o, s = torch.ops.sffft.linear_attention(q, k, v, ld, 0.3, s0)
    for b in range(B):
        want, last = oracle(q[b:b + 1], k[b:b + 1], v[b:b + 1], ld, s0[b:b + 1], 0.3)
        d = (s[b:b + 1].double() - last).flatten(2).norm(dim=2) / last.flatten(2).norm(dim=2)
        assert float(d.max()) < 2e-5, float(d.max())
        along = (s[b:b + 1].double() * last).flatten(2).sum(2) / (last * last).flatten(2).sum(2) - 1
        assert float(along.abs().max()) < 1e-5, float(along.abs().max())
        d = (o[b:b + 1, -64:].double() - want).permute(0, 2, 1, 3).flatten(2).norm(dim=2) / want.permute(0, 2, 1, 3).flatten(2).norm(dim=2)
        assert float(d.max()) < (3 * 2.0 ** -9 if dtype == torch.bfloat16 else 2e-5), float(d.max())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
def test_decays_of_every_speed(dev, dtype):
    """A large initial state seen through decays from none to one that leaves 1e-30 of it: relative to what is left."""
    decays = [0.0, -1e-7, -1e-4, -0.003, -0.0107, -0.0109, -0.02, -0.03, -0.1, -0.3, 1e-4, 0.02]
    B, T, H, D = 100, 224, len(decays), 8
    ld = torch.tensor(decays, device=dev)
    k = torch.zeros(B, T, H, D, dtype=dtype, device=dev)
    s0 = torch.rand(B, H, D, D, device=dev) + 1
    _, s = torch.ops.sffft.linear_attention(k, k, k, ld, 1.0, s0)
    want = torch.exp(ld.double() * T)[None, :, None, None] * s0.double()
    # products of decays in the exponent: 2^-24 of 0.3 * 224 = 67
    assert float(((s.double() - want).abs() / want.abs()).max()) < 1e-5


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
def test_states_after_many_single_tokens(dev, dtype):
    """The decay of a token, rounded, would be off by up to 2^-24 in one direction each time: 2.4e-4 after 4096. A token
    rounds the state once or twice: 2^-25 sqrt(8192) = 3e-6 of a head's state, an eighth of it along the state, and
    the decay 2^-23 of its argument, 0.2 in all; 1e-5 and 2e-6 are allowed."""
    H, D, n = 64, 8, 4096
    g = torch.Generator(device=dev).manual_seed(3)
    ld = -torch.logspace(-6.2, -4.3, H, device=dev)
    q, k, v = (torch.randn(n, 1, H, D, generator=g, device=dev).to(dtype) for _ in range(3))
    s0 = torch.randn(1, H, D, D, generator=g, device=dev) * 1e5
    s = s0.clone()
    for t in range(n):
        torch.ops.sffft.linear_attention_step(q[t], k[t], v[t], ld, s, 0.3)
    _, last = oracle(*(x.transpose(0, 1) for x in (q, k, v)), ld, s0, 0.3)
    d = (s.double() - last).flatten(2).norm(dim=2) / last.flatten(2).norm(dim=2)
    along = (s.double() * last).flatten(2).sum(2) / (last * last).flatten(2).sum(2) - 1
    assert float(d.max()) < 1e-5 and float(along.abs().max()) < 2e-6, (float(d.max()), float(along.abs().max()))
