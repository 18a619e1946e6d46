"""Counts of gates, tokens and sequences that once asked for launches of 2^32 threads."""
import pytest
import torch

from sffft_amd import mixers, torch_ops  # noqa: F401

pytestmark = pytest.mark.gpu


def norm_oracle(x, y, gate, w_pre, w_post, scale, gr, gh, eps):
    """(r, h, dx, dy, dgate, dw_pre, dw_post, dscale) in 64 bits for silu gates [B, 1, C], on the inputs' device."""
    d = [t.double().requires_grad_() for t in (x, y, gate, w_pre, w_post, scale)]

    def norm(z):
        return z / torch.sqrt((z * z).mean(-1, keepdim=True) + eps)

    r = d[0] + d[5] * (d[2] / (1 + torch.exp(-d[2]))) * norm(d[1]) * d[4]
    h = norm(r) * d[3]
    return (r.detach(), h.detach(), *torch.autograd.grad((r, h), d, (gr.double(), gh.double())))


@pytest.mark.parametrize("B,C", [(8200, 16384), (87400, 1536), (33000, 40)])
def test_more_shared_gates_than_one_launch_took(dev, B, C):
    """One gate for every two tokens. fp32: sums over 2 B rows, 2^-24 sqrt(2 B) < 3e-5; bf16 would hide it."""
    T = 2
    g = torch.Generator(device=dev).manual_seed(C)

    def r(*s):
        return torch.randn(*s, generator=g, device=dev)

    x, y, gr, gh = (r(B, T, C) for _ in range(4))
    gate, w_pre, w_post, scale = r(B, 1, C), r(C) + 1, r(C) + 1, r(C)
    leaves = [t.requires_grad_() for t in (x, y, w_pre, w_post, gate, scale)]
    r_, h = torch.ops.sffft.block_norm(*leaves, "silu", 1e-6)
    dx, dy, dwq, dwp, dg, ds = torch.autograd.grad((r_, h), leaves, (gr, gh))
    got = [t.detach() for t in (r_, h, dx, dy, dg)]
    sums = [torch.zeros(C, dtype=torch.float64, device=dev) for _ in range(3)]
    step = max(1, (1 << 25) // (T * C))
    for a in range(0, B, step):
        z = slice(a, a + step)
        want = norm_oracle(*(t.detach() for t in (x[z], y[z], gate[z], w_pre, w_post, scale, gr[z], gh[z])), 1e-6)
        for name, p, w in zip(("r", "h", "dx", "dy", "dgate"), got, want):
            assert float((p[z].double() - w).norm() / w.norm()) < 1e-5, (name, a)
        for s, w in zip(sums, want[5:]):
            s += w
    for name, p, w in zip(("dw_pre", "dw_post", "dscale"), (dwq, dwp, ds), sums):
        assert float((p.double() - w).norm() / w.norm()) < 3e-5, name


def test_rotary_of_2_to_the_24_tokens(dev):
    """Two tokens to a workgroup: the same bits as in calls of fewer."""
    T, D = (1 << 24) + 5, 258
    table = mixers.rotary_table(1000, 256, device=dev)
    q = torch.randn(1, T, 1, D, dtype=torch.bfloat16, device=dev)
    pos = (torch.arange(T, device=dev) % 1000).int()[None]
    out, _ = torch.ops.sffft.rotary(q, q[:, :, :0], table, pos)
    for a in range(0, T, 1 << 20):
        z = slice(a, a + (1 << 20))
        assert torch.equal(out[:, z], torch.ops.sffft.rotary(q[:, z], q[:, z, :0], table, pos[:, z])[0]), a


def test_attention_beyond_2_to_the_32_bytes(dev):
    """Arrays of 4.8 GB: their last sequence gives, forward and backward, what it gives alone (in another cut: to the
    rounding of bf16, root mean square under 2^-9 on both sides)."""
    B, T, H, D = 48, 65536, 12, 64
    g = torch.Generator(device=dev).manual_seed(4)
    q, k, v, go = (torch.randn(B, T, H, D, generator=g, device=dev, dtype=torch.bfloat16) for _ in range(4))
    ld = torch.linspace(-0.1, -0.0001, H, device=dev)

    def run(z):
        x = [t[z].requires_grad_() for t in (q, k, v)]
        o, s = torch.ops.sffft.linear_attention(*x, ld, 0.125)
        return (o.detach(), s.detach(), *torch.autograd.grad(o, x, go[z]))

    for name, a, b in zip(("o", "state", "dq", "dk", "dv"), run(slice(0, B)), run(slice(B - 1, B))):
        a, b = a[-1:].double(), b.double()
        assert float((a - b).norm() / b.norm()) < (1e-5 if name == "state" else 2.0 ** -8), name


def test_norms_beyond_2_to_the_32_bytes(dev):
    """Rows of odd width, 4.7 GB of them: the last ones as by themselves."""
    B, C = 1535 * 1000, 1531
    g = torch.Generator(device=dev).manual_seed(5)
    x, y = (torch.randn(B, C, generator=g, device=dev, dtype=torch.bfloat16) for _ in range(2))
    gate, w = y.flip(1), torch.rand(C, generator=g, device=dev) + 0.5

    def run(z):
        t = [u[z].requires_grad_() for u in (x, y, gate)]
        r, h = torch.ops.sffft.block_norm(t[0], t[1], w, w, t[2], None, "silu")
        return (r.detach(), h.detach(), *torch.autograd.grad((r, h), t, (x[z], y[z])))

    for name, a, b in zip(("r", "h", "dx", "dy", "dgate"), run(slice(0, B)), run(slice(B - 1000, B))):
        a, b = a[-1000:].double(), b.double()
        assert float((a - b).norm() / b.norm()) < 2.0 ** -8, name
