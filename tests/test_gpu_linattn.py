"""Linear attention with a decay for each head on the GPU, against the 64-bit recurrence.

Tolerances (relative L2 error of a whole output), from the arithmetic:
- bf16 outputs: the result is rounded once (a root mean square under 2^-9 relative over many values), and on
  the way the weights of the tokens of a chunk and the entering state once each (2^-9 of the part that they
  carry): 3 * 2^-9.
- fp32 outputs, states and their gradients among them: products and sums in fp32, of up to 128 channels
  and about 1000 tokens, 2^-24 * sqrt(1128) = 2e-6 if their errors are independent; 1e-5 for chains of
  three such sums and decays evaluated as powers.
"""
import numpy as np
import pytest
import torch

import mixer_oracle as mo
from sffft_amd import mixers, torch_ops  # noqa: F401

pytestmark = pytest.mark.gpu

BF16, FP32 = 3 * 2.0 ** -9, 1e-5


def tol(t):
    return BF16 if t.dtype == torch.bfloat16 else FP32


def inputs(dev, B, T, H, Hk, Dk, Dv, dtype, seed=0, decays=None):
    g = torch.Generator().manual_seed(seed)
    def r(*s, dt=dtype):
        return torch.randn(*s, generator=g).to(dt).to(dev)
    ld = torch.linspace(-2.0, -0.001, H) if decays is None else torch.tensor(decays)
    return r(B, T, H, Dk), r(B, T, Hk, Dk), r(B, T, Hk, Dv), ld.float().to(dev), r(B, H, Dk, Dv, dt=torch.float32), \
        r(B, T, H, Dv), r(B, H, Dk, Dv, dt=torch.float32)


CASES = [  # B, T, H, Hk, Dk, Dv
    (1, 1, 1, 1, 8, 8), (2, 1, 3, 3, 64, 64), (1, 2, 2, 1, 16, 24), (2, 31, 2, 2, 32, 32), (1, 32, 2, 2, 64, 64),
    (1, 33, 2, 1, 128, 128), (2, 63, 4, 2, 64, 128), (1, 64, 1, 1, 128, 64), (3, 65, 2, 2, 72, 40), (1, 127, 3, 1, 96, 64),
    (1, 128, 2, 2, 128, 128), (2, 129, 2, 2, 64, 64), (1, 257, 6, 2, 120, 8), (1, 700, 2, 2, 128, 128), (2, 641, 3, 3, 64, 64),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("case", CASES, ids=str)
def test_forward_and_gradients(dev, case, dtype):
    q, k, v, ld, s0, go, gs = inputs(dev, *case, dtype, seed=sum(case))
    scale = case[4] ** -0.5
    want = mo.attention_grads(q, k, v, ld, scale, go, gs, s0)
    for t in (q, k, v, s0):
        t.requires_grad_(True)
    o, s = torch.ops.sffft.linear_attention(q, k, v, ld, scale, s0)
    got = (o, s, *torch.autograd.grad((o, s), (q, k, v, s0), (go, gs)))
    for name, a, w in zip(("o", "state", "dq", "dk", "dv", "dstate"), got, want):
        assert a.shape == w.shape
        assert mo.rel_l2(a, w) < tol(a), (name, mo.rel_l2(a, w))
    # without states: zero in, none wanted out
    want = mo.attention_grads(q, k, v, ld, scale, go, None)
    o, s = torch.ops.sffft.linear_attention(q, k, v, ld, scale)
    got = (o, s, *torch.autograd.grad(o, (q, k, v), go))
    for name, a, w in zip(("o", "state", "dq", "dk", "dv"), got, want):
        assert mo.rel_l2(a, w) < tol(a), (name, mo.rel_l2(a, w))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("B,T,H,Hk,Dk,Dv", [(3, 2001, 12, 12, 64, 64), (3, 2047, 12, 12, 128, 128), (2, 2500, 12, 12, 128, 64),
                                            (2, 2500, 12, 4, 64, 128), (3, 2047, 12, 1, 96, 96)])
def test_full_chip(dev, B, T, H, Hk, Dk, Dv, dtype):
    """More workgroups than the chip has CUs, so that several share one, for every size of the tiles: no element off
    by more than its row's size allows, and the same bits each time. (Stores of a workgroup that shared its CU once
    sent registers that were overwritten behind them, and a barrier once let outputs be read from LDS too early.)"""
    q, k, v, ld, s0, go, gs = inputs(dev, B, T, H, Hk, Dk, Dv, dtype, seed=T)
    scale = Dk ** -0.5
    want = mo.attention_pairs(q, k, v, ld, scale, go, s0, gs)
    for t in (q, k, v, s0):
        t.requires_grad_(True)
    first = None
    for _ in range(8):
        o, s = torch.ops.sffft.linear_attention(q, k, v, ld, scale, s0)
        got = (o, s, *torch.autograd.grad((o, s), (q, k, v, s0), (go, gs)))
        first = first or got
        assert all(torch.equal(a, b) for a, b in zip(got, first))
        for name, a, w in zip(("o", "state", "dq", "dk", "dv", "dstate"), got, want):
            a = a.detach().double()
            assert float((a - w).norm() / w.norm()) < (BF16 if got[0].dtype == torch.bfloat16 and name not in ("state", "dstate") else FP32), name
            # the largest single error: 2^-6 (bf16) or 1e-4 of the largest value
            assert float((a - w).abs().max()) < (2.0 ** -6 if dtype == torch.bfloat16 else 1e-4) * float(w.abs().max()), name


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("B,T,H,Hk,Dk,Dv", [(6, 1500, 12, 12, 32, 32), (3, 1800, 12, 4, 24, 96), (3, 1600, 12, 6, 72, 128), (3, 1700, 12, 12, 96, 64)])
def test_full_chip_of_other_tiles(dev, B, T, H, Hk, Dk, Dv, dtype):
    test_full_chip(dev, B, T, H, Hk, Dk, Dv, dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("T,lengths", [(5, [0, 5, 1]), (130, [64, 0, 130]), (200, [199, 65, 63]), (64, [0, 0, 0])], ids=str)
def test_lengths_and_what_lies_beyond_them(dev, T, lengths, dtype):
    """Tokens from lengths[b] on hold NaN and infinities: nothing of them reaches an output, their own are 0."""
    H, Hk, D = 4, 2, 64
    q, k, v, ld, s0, go, gs = inputs(dev, 3, T, H, Hk, D, D, dtype, seed=T)
    n = torch.tensor(lengths, dtype=torch.int32, device=dev)
    want = mo.attention_grads(q, k, v, ld, 0.2, go, gs, s0, lengths)
    for b, m in enumerate(lengths):
        for t, bad in ((q, float("nan")), (k, float("inf")), (v, float("-inf")), (go, float("nan"))):
            t[b, m:] = bad
    for t in (q, k, v, s0):
        t.requires_grad_(True)
    o, s = torch.ops.sffft.linear_attention(q, k, v, ld, 0.2, s0, n)
    got = (o, s, *torch.autograd.grad((o, s), (q, k, v, s0), (go, gs)))
    for name, a, w in zip(("o", "state", "dq", "dk", "dv", "dstate"), got, want):
        assert bool(torch.isfinite(a).all()), name
        assert mo.rel_l2(a, w) < tol(a), (name, mo.rel_l2(a, w))
        if name in ("o", "dq", "dk", "dv"):
            for b, m in enumerate(lengths):
                assert not bool(a[b, m:].any()), (name, b)
    for b, m in enumerate(lengths):
        if m == 0:  # an empty sequence hands its state on unchanged
            assert torch.equal(s[b], s0[b]) and torch.equal(got[5][b], gs[b])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("B,T,H,Hk,Dk,Dv,lengths", [(4, 1210, 2, 1, 64, 64, [1210, 0, 1, 601]), (4, 530, 3, 3, 96, 64, [200, 530, 0, 385]),
                                                    (3, 700, 16, 8, 72, 96, [700, 64, 333]), (2, 900, 1, 1, 128, 128, [899, 129])])
def test_lengths_that_end_before_some_segments(dev, B, T, H, Hk, Dk, Dv, lengths, dtype):
    """Long enough for segments of tokens, joined by the workgroups or by a scan, some of them without a token that counts."""
    q, k, v, ld, s0, go, gs = inputs(dev, B, T, H, Hk, Dk, Dv, dtype, seed=T)
    n = torch.tensor(lengths, dtype=torch.int32, device=dev)
    want = mo.attention_grads(q, k, v, ld, Dk ** -0.5, go, gs, s0, lengths)
    for b, m in enumerate(lengths):
        for t in (q, k, v, go):
            t[b, m:] = float("nan")
    for t in (q, k, v, s0):
        t.requires_grad_(True)
    o, s = torch.ops.sffft.linear_attention(q, k, v, ld, Dk ** -0.5, s0, n)
    got = (o, s, *torch.autograd.grad((o, s), (q, k, v, s0), (go, gs)))
    for name, a, w in zip(("o", "state", "dq", "dk", "dv", "dstate"), got, want):
        assert mo.rel_l2(a, w) < tol(a), (name, mo.rel_l2(a, w))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
def test_extreme_decays(dev, dtype):
    """No memory at all (-inf), a decay that underflows within a chunk, none (0), and a slow one."""
    case = (2, 150, 4, 4, 64, 32)
    decays = [float("-inf"), -30.0, 0.0, -1e-5]
    q, k, v, ld, s0, go, gs = inputs(dev, *case, dtype, seed=5, decays=decays)
    # the oracle's gradient of exp at -inf is not needed: its decays are powers of 0 there
    want = mo.attention_grads(q, k, v, ld, 0.125, go, gs, s0, [150, 77])
    n = torch.tensor([150, 77], dtype=torch.int32, device=dev)
    for t in (q, k, v, s0):
        t.requires_grad_(True)
    o, s = torch.ops.sffft.linear_attention(q, k, v, ld, 0.125, s0, n)
    got = (o, s, *torch.autograd.grad((o, s), (q, k, v, s0), (go, gs)))
    for name, a, w in zip(("o", "state", "dq", "dk", "dv", "dstate"), got, want):
        for h in range(4):
            x, y = (t[:, h] if name in ("state", "dstate") else t[:, :, h] for t in (a, w))
            assert mo.rel_l2(x, y) < tol(a), (name, h)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
def test_prompt_then_tokens(dev, dtype):
    """A prompt cut anywhere gives what one call gives, also token by token with the state in place."""
    B, T, H, Hk, Dk, Dv = 3, 150, 4, 2, 72, 64
    q, k, v, ld, s0, _, _ = inputs(dev, B, T, H, Hk, Dk, Dv, dtype, seed=9)
    want, last = mo.attention(q, k, v, ld, 0.1, s0)
    state, o = s0, []
    for a, z in ((0, 1), (1, 66), (66, 140)):
        x, state = torch.ops.sffft.linear_attention(q[:, a:z], k[:, a:z], v[:, a:z], ld, 0.1, state)
        o.append(x)
    cache = torch.full((7, H, Dk, Dv), 5.0, device=dev)
    slots = torch.tensor([4, 0, 6], dtype=torch.int32, device=dev)
    cache[slots.long()] = state
    version = cache._version
    for t in range(140, T):
        o.append(torch.ops.sffft.linear_attention_step(q[:, t], k[:, t], v[:, t], ld, cache, 0.1, slots)[:, None])
    assert cache._version > version
    o = torch.cat(o, 1)
    assert mo.rel_l2(o, want) < tol(o)
    assert mo.rel_l2(cache[slots.long()], last) < FP32
    others = [i for i in range(7) if i not in (4, 0, 6)]
    assert bool((cache[others] == 5.0).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("B,H,Hk,Dk,Dv", [(1, 1, 1, 8, 8), (3, 2, 1, 128, 128), (5, 4, 4, 64, 72), (2, 3, 3, 24, 96)])
def test_step(dev, B, H, Hk, Dk, Dv, dtype):
    q, k, v, ld, s0, _, _ = inputs(dev, B, 1, H, Hk, Dk, Dv, dtype, seed=B)
    want, last = mo.attention(q, k, v, ld, 0.3, s0)
    s = s0.clone()
    o = torch.ops.sffft.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], ld, s, 0.3)
    assert mo.rel_l2(o, want[:, 0]) < (2.0 ** -8 if dtype == torch.bfloat16 else FP32)
    assert mo.rel_l2(s, last) < FP32
    # a slot outside the cache: no state, output 0, nothing written
    s = s0.clone()
    slots = torch.arange(B, dtype=torch.int32, device=dev)
    slots[B - 1] = -1 if B % 2 else B
    o = torch.ops.sffft.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], ld, s, 0.3, slots)
    assert not bool(o[B - 1].any()) and torch.equal(s[B - 1], s0[B - 1])
    if B > 1:
        assert mo.rel_l2(s[:B - 1], last[:B - 1]) < FP32


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
def test_strides_and_orders(dev, dtype):
    """Views of one fused projection, head-major storage, a transposed channel order, an unaligned view and
    expanded inputs give what their contiguous copies give."""
    B, T, H, D = 2, 77, 3, 64
    g = torch.Generator().manual_seed(1)
    fused = torch.randn(B, T, 3, H, D, generator=g).to(dtype).to(dev)
    ld = torch.linspace(-1.0, -0.01, H, device=dev)
    views = [tuple(fused.unbind(2)),
             tuple(torch.randn(B, H, T, D, generator=g).to(dtype).to(dev).transpose(1, 2) for _ in range(3)),
             tuple(torch.randn(B, T, D, H, generator=g).to(dtype).to(dev).transpose(2, 3) for _ in range(3)),
             tuple(torch.randn(B, T, H, D + 1, generator=g).to(dtype).to(dev)[..., 1:] for _ in range(3)),
             tuple(torch.randn(B, 1, H, D, generator=g).to(dtype).to(dev).expand(B, T, H, D) for _ in range(3))]
    go = torch.randn(B, T, 1, D, generator=g).to(dtype).to(dev).expand(B, T, H, D)
    for q, k, v in views:
        a = [t.detach().requires_grad_() for t in (q, k, v)]
        c = [t.detach().contiguous().requires_grad_() for t in (q, k, v)]
        out = []
        for x, grad in ((a, go), (c, go.contiguous())):
            o, s = torch.ops.sffft.linear_attention(*x, ld, 0.2)
            out.append((o, s, *torch.autograd.grad((o, s.sum()), x, (grad, torch.ones((), device=dev)))))
        for x, y in zip(*out):
            assert torch.equal(x, y)


def test_gradient_against_differences(dev):
    """The kernel's gradients against central differences of the kernel's own outputs in fp32. Each input enters
    linearly, so a difference over a step of 1 is exact but for rounding: 1e-5 of the sums' sizes."""
    B, T, H, Hk, D = 1, 140, 4, 2, 64
    q, k, v, ld, s0, go, gs = inputs(dev, B, T, H, Hk, D, D, torch.float32, seed=2)
    x = [t.requires_grad_() for t in (q, k, v, s0)]
    def loss(y):
        o, s = torch.ops.sffft.linear_attention(y[0], y[1], y[2], ld, 0.125, y[3])
        return o, s
    grads = torch.autograd.grad(loss(x), x, (go, gs))
    for i in range(4):
        d = torch.randn(x[i].shape, generator=torch.Generator().manual_seed(i)).to(dev)
        def value(sign):
            with torch.no_grad():
                o, s = loss([t + sign * d if j == i else t for j, t in enumerate(x)])
            return float((o.double() * go).sum() + (s.double() * gs).sum())
        up, down = value(1), value(-1)
        got = float((grads[i].double() * d).sum())
        size = float(grads[i].double().norm() * d.double().norm())
        assert abs(got - (up - down) / 2) < 1e-4 * (size + abs(up) + abs(down)), i


def test_equal_calls_give_equal_bits_on_any_stream(dev):
    q, k, v, ld, s0, go, gs = inputs(dev, 2, 700, 4, 2, 64, 64, torch.bfloat16, seed=4)
    def run():
        x = [t.detach().requires_grad_() for t in (q, k, v, s0)]
        o, s = torch.ops.sffft.linear_attention(*x[:3], ld, 0.1, x[3])
        return (o, s, *torch.autograd.grad((o, s), x, (go, gs)))
    first = run()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        second = run()
    side.synchronize()
    for a, b in zip(first, second):
        assert torch.equal(a, b)


def test_graph_replays(dev):
    """Captured on its first call in this shape, replayed with other inputs between eager work."""
    B, T, H, D = 1, 333, 2, 64
    q, k, v, ld, s0, _, _ = inputs(dev, B, T, H, H, D, D, torch.bfloat16, seed=6)
    state = s0.clone()
    torch.ops.sffft.linear_attention(q[:, :8], k[:, :8], v[:, :8], ld, 0.1, s0)  # loads the library
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o, s = torch.ops.sffft.linear_attention(q, k, v, ld, 0.1, s0)
        one = torch.ops.sffft.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], ld, state, 0.1)
    for i in range(3):
        q.copy_(torch.randn(q.shape, generator=torch.Generator().manual_seed(i)).to(dev))
        state.copy_(s0)
        want = torch.ops.sffft.linear_attention(q, k, v, ld, 0.1, s0)
        st = s0.clone()
        want_one = torch.ops.sffft.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], ld, st, 0.1)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in ((o, want[0]), (s, want[1]), (one, want_one), (state, st)):
            assert torch.equal(a, b), i


def test_empty_calls(dev):
    q, k, v, ld, s0, _, _ = inputs(dev, 2, 3, 2, 2, 16, 16, torch.float32)
    o, s = torch.ops.sffft.linear_attention(q[:, :0], k[:, :0], v[:, :0], ld, 0.1, s0)
    assert o.shape == (2, 0, 2, 16) and torch.equal(s, s0)
    o, s = torch.ops.sffft.linear_attention(q[:0], k[:0], v[:0], ld, 0.1)
    assert o.shape == (0, 3, 2, 16) and s.shape == (0, 2, 16, 16)


def test_refusals(dev):
    q, k, v, ld, s0, _, _ = inputs(dev, 2, 5, 4, 2, 16, 16, torch.bfloat16)
    f, step = torch.ops.sffft.linear_attention, torch.ops.sffft.linear_attention_step
    i32 = torch.zeros(2, dtype=torch.int32, device=dev)
    bad = [lambda: f(q.half(), k.half(), v.half(), ld, 1.0), lambda: f(q, k.float(), v, ld, 1.0),
           lambda: f(q, k[:, :4], v, ld, 1.0), lambda: f(q[:, :, :3], k, v, ld[:3], 1.0),
           lambda: f(q[..., :12], k[..., :12], v, ld, 1.0), lambda: f(q, k, v, ld[:2], 1.0),
           lambda: f(q, k, v, ld.double(), 1.0), lambda: f(q, k, v, ld.cpu(), 1.0), lambda: f(q, k, v, ld, 1.0, s0[:1]),
           lambda: f(q, k, v, ld, 1.0, s0.bfloat16()), lambda: f(q, k, v, ld, 1.0, s0, i32.long()),
           lambda: f(q, k, v, ld, 1.0, s0, i32[:1]), lambda: f(q, k, v, ld.requires_grad_(), 1.0),
           lambda: step(q[:, 0], k[:, 0], v[:, 0], ld.detach(), s0[:, :, :, :8], 1.0),
           lambda: step(q[:, 0], k[:, 0], v[:, 0], ld.detach(), s0[:1], 1.0),
           lambda: step(q[:, 0], k[:, 0], v[:, 0], ld.detach(), s0.transpose(2, 3), 1.0),
           lambda: step(q[:, 0], k[:, 0].requires_grad_(), v[:, 0], ld.detach(), s0, 1.0)]
    for i, call in enumerate(bad):
        with pytest.raises(RuntimeError):
            call()
            raise AssertionError(i)
    ld = ld.detach()
    x = q.float().requires_grad_()
    o, _ = f(x, k.float(), v.float(), ld, 1.0)
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(o.sum(), x, create_graph=True)


def test_binding_matches_the_operators(dev):
    q, k, v, ld, s0, go, gs = inputs(dev, 2, 70, 4, 2, 64, 32, torch.bfloat16, seed=8)
    n = torch.tensor([70, 33], dtype=torch.int32, device=dev)
    x = [t.detach().requires_grad_() for t in (q, k, v, s0)]
    o, s = torch.ops.sffft.linear_attention(*x[:3], ld, 0.1, x[3], n)
    want = (o, s, *torch.autograd.grad((o, s), x, (go, gs)))
    got = mixers.linear_attention(q, k, v, ld, 0.1, s0, n) + mixers.linear_attention_backward(
        q, k, v, ld, 0.1, go, s0, n, gs)
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("T", [1, 64, 130, 500, 1500])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
def test_final_state_in_place_of_the_initial(dev, T, dtype):
    """sffft_linattn_fwd may write the final state over the initial one, however many segments read that."""
    B, H, D = 3, 12, 64
    q, k, v, ld, s0, _, _ = inputs(dev, B, T, H, H, D, D, dtype, seed=T)
    want = mixers.linear_attention(q, k, v, ld, 0.125, s0)
    p = mixers.linattn_params(q, k, v, 0.125)
    L, stream = mixers.lib(), torch.cuda.current_stream().cuda_stream
    need = L.sffft_linattn_work_bytes(p, 0)
    work = torch.empty(max(need, 16), dtype=torch.uint8, device=dev)
    for _ in range(4):
        s, o = s0.clone(), torch.empty_like(want[0])
        assert L.sffft_linattn_fwd(p, q.data_ptr(), k.data_ptr(), v.data_ptr(), ld.data_ptr(), s.data_ptr(), None, o.data_ptr(),
                                   s.data_ptr(), work.data_ptr(), work.numel(), stream) == 0
        assert mo.rel_l2(s, want[1].cpu()) < FP32 and mo.rel_l2(o, want[0].cpu()) < tol(o)


def test_state_beyond_two_gib(dev):
    """A state cache whose offsets pass 32 bits: the last slot is the one used."""
    H, D = 16, 128
    slots = (1 << 32) // (H * D * D * 4) + 2
    cache = torch.zeros(slots, H, D, D, device=dev)
    q, k, v, ld, s0, _, _ = inputs(dev, 1, 1, H, H, D, D, torch.float32, seed=3)
    cache[slots - 1] = s0[0]
    slot = torch.tensor([slots - 1], dtype=torch.int32, device=dev)
    o = torch.ops.sffft.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], ld, cache, 0.1, slot)
    want, last = mo.attention(q, k, v, ld, 0.1, s0)
    assert mo.rel_l2(o, want[:, 0]) < FP32 and mo.rel_l2(cache[slots - 1], last[0]) < FP32
    assert not bool(cache[:slots - 1].any())
