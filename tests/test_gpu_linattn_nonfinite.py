"""Infinities and NaN in linear attention: where they may go, and where not."""
import pytest
import torch

import mixer_oracle as mo
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


@DTYPES
@pytest.mark.parametrize("value", [NAN, INF, -INF])
@pytest.mark.parametrize("where", ["q", "k", "v", "go"])
@pytest.mark.parametrize("B,T,H,Hk,Dk,Dv,token,lengths", [(1, 1, 1, 1, 8, 8, 0, None), (2, 150, 2, 1, 64, 64, 70, [150, 100]),
                                                         (1, 90, 2, 2, 24, 128, 33, None), (1, 640, 2, 2, 128, 128, 300, None),
                                                         (1, 70, 2, 1, 96, 72, 64, None), (1, 130, 1, 1, 128, 40, 127, [129])])
def test_one_value_reaches_what_the_definition_lets_it_reach(dev, B, T, H, Hk, Dk, Dv, token, lengths, where, value, dtype):
    """The finite places are those of the 64-bit recurrence and its gradients, with values as near as ever: a value
    that is not finite stays away from the tokens before its own (after it, in the gradients of keys and values), and
    from channels that it has no part in."""
    q, k, v, ld, s0, go, gs = inputs(dev, B, T, H, Hk, Dk, Dv, dtype, seed=token)
    x = {"q": q, "k": k, "v": v, "go": go}[where]
    x[0, token, 0, 5] = value
    want = mo.attention_grads(q, k, v, ld, 0.2, go, gs, s0, lengths)
    got = run(q, k, v, ld, s0, go, gs, None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device=dev))
    for (name, a), w in zip(got.items(), want):
        a = a.double().cpu()
        assert torch.equal(torch.isfinite(a), torch.isfinite(w)), name
        bound = 3 * 2.0 ** -9 if dtype == torch.bfloat16 and name not in ("state", "dstate") else 1e-5
        assert mo.rel_l2(torch.where(torch.isfinite(w), a, 0.0), torch.where(torch.isfinite(w), w, 0.0)) < bound, name


@DTYPES
@pytest.mark.parametrize("B,T,lengths", [(2, 1, [1, 0]), (2, 90, [90, 33]), (2, 900, [900, 0]), (1, 4000, [3999])])
def test_a_decay_of_nan_is_not_hidden(dev, B, T, lengths, dtype):
    """It makes NaN of what its head's decay reaches, and of nothing else: the other heads keep their bits."""
    H, D = 4, 64
    q, k, v, ld, s0, go, gs = inputs(dev, B, T, H, H, D, D, dtype, seed=T)
    n = torch.tensor(lengths, dtype=torch.int32, device=dev)
    want = run(q, k, v, ld, s0, go, gs, n)
    bad = ld.clone()
    bad[2] = NAN
    got = run(q, k, v, bad, s0, go, gs, n)
    others = [0, 1, 3]
    for name in got:
        h = 1 if name in ("state", "dstate") else 2
        assert torch.equal(got[name].index_select(h, torch.tensor(others, device=dev)),
                           want[name].index_select(h, torch.tensor(others, device=dev))), name
    for b, m in enumerate(lengths):
        assert bool(torch.isnan(got["o"][b, :m, 2]).all()) and bool(torch.isnan(got["dq"][b, :m, 2]).all())
        assert not bool(got["o"][b, m:].any())
        if m:
            assert bool(torch.isnan(got["state"][b, 2]).all()) and bool(torch.isnan(got["dstate"][b, 2]).all())
            # the last token's key and value do not pass a decay on their way to the final state
            assert bool(torch.isnan(got["dk"][b, :m - 1, 2]).all()) and bool(torch.isfinite(got["dk"][b, m - 1, 2]).all())
            assert bool(torch.isnan(got["dv"][b, :m - 1, 2]).all()) and bool(torch.isfinite(got["dv"][b, m - 1, 2]).all())
        else:
            assert torch.equal(got["state"][b], s0[b]) and torch.equal(got["dstate"][b], gs[b])


@DTYPES
def test_a_decay_of_nan_is_not_hidden_from_single_tokens(dev, dtype):
    q, k, v, ld, s0, _, _ = inputs(dev, 3, 1, 4, 2, 64, 32, dtype)
    want, bad = s0.clone(), s0.clone()
    o = torch.ops.sffft.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], ld, want, 0.2)
    ld[1] = NAN
    p = torch.ops.sffft.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], ld, bad, 0.2)
    for x, y in ((p, o), (bad, want)):
        assert bool(torch.isnan(x[:, 1]).all()) and torch.equal(x[:, [0, 2, 3]], y[:, [0, 2, 3]])


@DTYPES
@pytest.mark.parametrize("B,T,H,Hk,Dk,Dv", [(60, 330, 12, 12, 128, 128), (60, 330, 12, 4, 128, 128), (60, 330, 12, 4, 96, 128), (100, 330, 12, 12, 64, 64),
                                            (100, 330, 12, 6, 32, 64), (60, 200, 12, 12, 64, 128)])
def test_chunks_after_one_that_is_not_finite(dev, B, T, H, Hk, Dk, Dv, dtype):
    """In a march of several chunks the others come out as without it, wherever the value has no part."""
    q, k, v, ld, s0, go, gs = inputs(dev, B, T, H, Hk, Dk, Dv, dtype, seed=7)
    clean, t = run(q, k, v, ld, s0, go, gs), 70
    channels = [c for c in range(Dv) if c != 5]

    def near(a, b):  # two roundings to bf16 (2^-9 each, root mean square); fp32 in another order of the sums
        a, b = a.double(), b.double()
        return bool(torch.isfinite(a).all()) and float((a - b).norm() / b.norm()) < (2.0 ** -8 if dtype == torch.bfloat16 else 1e-5)

    w = v.clone()
    w[:, t, :, 5] = INF
    got = run(q, k, w, ld, s0, go, gs)
    assert near(got["o"][..., channels], clean["o"][..., channels]) and near(got["o"][:, :t], clean["o"][:, :t])
    assert near(got["state"][..., channels], clean["state"][..., channels])
    assert near(got["dq"][:, :t], clean["dq"][:, :t]) and near(got["dv"], clean["dv"]) and near(got["dstate"], clean["dstate"])
    others = [i for i in range(T) if i != t]
    assert near(got["dk"][:, others], clean["dk"][:, others])
    assert not bool(torch.isfinite(got["o"][:, t:, :, 5]).any())
    w = go.clone()
    w[:, t, :, 5] = NAN
    got = run(q, k, v, ld, s0, w, gs)
    assert near(got["o"], clean["o"]) and near(got["dq"][:, others], clean["dq"][:, others])
    assert near(got["dk"][:, t + 1:], clean["dk"][:, t + 1:]) and near(got["dv"][:, t + 1:], clean["dv"][:, t + 1:])
    assert near(got["dv"][..., channels], clean["dv"][..., channels]) and near(got["dstate"][..., channels], clean["dstate"][..., channels])
    assert bool(torch.isnan(got["dv"][:, :t + 1, :, 5]).all())
