"""The norms around a block with its gate and residual scale, on the GPU, against 64 bits.

Tolerances (relative L2): fp32 results are a handful of products, two means of C squares and, for the
gradients of weights, sums over the rows in fp32: 2^-24 * sqrt(rows) is 2e-6 at 1000 rows; 1e-5. bf16 results
are rounded once: half a unit in the last of 8 significant bits, 2^-8 of a value just over a power of two.
"""
import pytest
import torch

import mixer_oracle as mo
from sffft_amd import mixers, torch_ops  # noqa: F401

pytestmark = pytest.mark.gpu

NAMES = ("x", "y", "w_pre", "w_post", "gate", "scale")


def tol(t):
    return 2.0 ** -8 if t.dtype == torch.bfloat16 else 1e-5


def inputs(dev, shape, dtype, gate, post=True, scale=True, seed=0):
    g = torch.Generator().manual_seed(seed)
    C = shape[-1]
    def r(*s, dt=dtype, add=0.0):
        return (torch.randn(*s, generator=g) + add).to(dt).to(dev)
    f = torch.float32
    gates = {"token": shape, "sequence": (*shape[:-2], 1, C), "none": None}[gate]
    return {"x": r(*shape), "y": r(*shape), "w_pre": r(C, dt=f, add=1.0), "w_post": r(C, dt=f, add=1.0) if post else None,
            "gate": r(*gates) if gates else None, "scale": r(C, dt=f) if scale else None}, r(*shape), r(*shape)


def oracle(t, act, gr, gh, eps=1e-6):
    d = {n: None if x is None else x.detach().double().cpu().requires_grad_() for n, x in t.items()}
    r, h = mo.block_norm(d["x"], d["y"], d["w_pre"], d["w_post"], d["gate"], d["scale"], act, eps)
    loss = sum((o * g.double().cpu()).sum() for o, g in ((r, gr), (h, gh)) if g is not None)
    leaves = [d[n] for n in NAMES if d[n] is not None]
    grads = torch.autograd.grad(loss, leaves, allow_unused=True)
    return (r.detach(), h.detach()), [torch.zeros_like(x) if g is None else g for g, x in zip(grads, leaves)]


def run(t, act, gr, gh, eps=1e-6):
    d = {n: None if x is None else x.detach().requires_grad_() for n, x in t.items()}
    out = torch.ops.sffft.block_norm(*(d[n] for n in NAMES), act, eps)
    leaves = [d[n] for n in NAMES if d[n] is not None]
    pairs = [(o, g) for o, g in zip(out, (gr, gh)) if g is not None]
    grads = torch.autograd.grad([o for o, _ in pairs], leaves, [g for _, g in pairs], allow_unused=True)
    return out, [torch.zeros_like(x) if g is None else g for g, x in zip(grads, leaves)]


SHAPES = [(1, 1), (3, 5), (1, 1, 64), (2, 7, 96), (5, 768), (2, 33, 255), (3, 40, 256), (2, 9, 1000), (1, 5, 1024),
          (2, 6, 1028), (2, 11, 1531), (3, 70, 1536), (2, 5, 2047), (1, 3, 4096), (2, 2, 6001), (1, 3, 8192), (1, 2, 16384),
          (4, 300, 64), (1, 2500, 96)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("gate,act", [("token", "silu"), ("sequence", "sigmoid"), ("none", "none")])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_forward_and_gradients(dev, shape, gate, act, dtype):
    t, gr, gh = inputs(dev, shape, dtype, gate, seed=sum(shape))
    want, wgrads = oracle(t, act, gr, gh)
    out, grads = run(t, act, gr, gh)
    for name, a, w in zip(("r", "h"), out, want):
        assert mo.rel_l2(a, w) < tol(a), name
    if shape[-1] == 1:
        return  # norm(y) of one channel is +-1: its gradient is a difference of equal numbers
    for name, a, w in zip([n for n in NAMES if t[n] is not None], grads, wgrads):
        assert a.shape == w.shape and mo.rel_l2(a, w) < tol(a), (name, mo.rel_l2(a, w))


@pytest.mark.parametrize("post", [False, True])
@pytest.mark.parametrize("scale", [False, True])
@pytest.mark.parametrize("gate,act", [("none", "none"), ("token", "none"), ("sequence", "silu"), ("token", "sigmoid")])
@pytest.mark.parametrize("grads", ["both", "r", "h"])
def test_absent_parts(dev, post, scale, gate, act, grads):
    t, gr, gh = inputs(dev, (2, 13, 96), torch.float32, gate, post, scale, seed=1)
    gr, gh = (gr if grads != "h" else None), (gh if grads != "r" else None)
    want, wgrads = oracle(t, act, gr, gh, 1e-3)
    out, got = run(t, act, gr, gh, 1e-3)
    for a, w in list(zip(out, want)) + list(zip(got, wgrads)):
        assert mo.rel_l2(a, w) < 1e-5


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("shape", [(7, 768), (3, 4, 1531), (2, 3, 4096)], ids=str)
def test_pre_norm(dev, shape, dtype):
    t, _, gh = inputs(dev, shape, dtype, "none", seed=2)
    x, w = t["x"].requires_grad_(), t["w_pre"].requires_grad_()
    h = torch.ops.sffft.pre_norm(x, w)
    dx, dw = torch.autograd.grad(h, (x, w), gh)
    d = [z.detach().double().cpu().requires_grad_() for z in (x, w)]
    _, want = mo.block_norm(d[0], None, d[1])
    wx, ww = torch.autograd.grad(want, d, gh.double().cpu())
    for a, b in ((h, want.detach()), (dx, wx), (dw, ww)):
        assert mo.rel_l2(a, b) < tol(a)


def test_rows_of_zeros_and_of_extremes(dev):
    """A row of zeros gives zeros through eps; values whose squares are near the ends of fp32 keep their norm; NaN
    stays in its row."""
    C = 256
    x = torch.zeros(5, C, device=dev)
    y = torch.zeros(5, C, device=dev)
    x[1], y[1] = 1e-12, -1e-12
    x[2], y[2] = 1e15, 3e15
    x[3, 7] = float("nan")
    x[4], y[4] = 1.0, 2.0
    w = torch.ones(C, device=dev)
    r, h = torch.ops.sffft.block_norm(x, y, w, w)
    assert not bool(r[0].any()) and not bool(h[0].any())
    want, _ = mo.block_norm(x.double().cpu(), y.double().cpu(), w.double().cpu(), w.double().cpu())[0], None
    assert mo.rel_l2(r[[1, 2, 4]], want[[1, 2, 4]]) < 1e-5
    assert bool(torch.isnan(h[3]).all()) and bool(torch.isfinite(h[[0, 1, 2, 4]]).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
def test_strides(dev, dtype):
    """Halves of a fused projection, unaligned, transposed and expanded inputs give what contiguous copies give."""
    B, T, C = 2, 9, 96
    g = torch.Generator().manual_seed(3)
    def r(*s):
        return torch.randn(*s, generator=g).to(dtype).to(dev)
    w, post = torch.rand(C, device=dev) + 0.5, (torch.rand(C + 1, device=dev) + 0.5)[1:]
    both, wide, turned, one = r(B, T, 2 * C), r(B, T, C + 1), r(T, B, C), r(B, 1, C)
    halves = both.chunk(2, -1)
    sets = [(halves[0], halves[1], None), (wide[..., 1:], halves[0], halves[1]), (turned.transpose(0, 1), halves[0], one),
            (r(B, C, T).transpose(1, 2), one.expand(B, T, C), halves[1])]
    gr, gh = r(B, 1, C).expand(B, T, C), r(B, T, 2 * C)[..., C:]
    for x, y, gate in sets:
        a = run({"x": x, "y": y, "w_pre": w, "w_post": post, "gate": gate, "scale": None}, "silu", gr, gh)
        b = run({"x": x.contiguous(), "y": y.contiguous(), "w_pre": w, "w_post": post.clone(),
                 "gate": None if gate is None else gate.contiguous(), "scale": None}, "silu", gr.contiguous(), gh.contiguous())
        for p, q in zip(a[0], b[0]):
            assert mo.rel_l2(p, q) < 1e-6  # loads of another width: the same sums in another order
        for p, q in zip(a[1], b[1]):
            assert mo.rel_l2(p, q) < (1e-2 if dtype == torch.bfloat16 else 1e-5)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("gate", ["token", "sequence"])
@pytest.mark.parametrize("B,T,C", [(1, 1, 9), (2, 2, 13), (3, 6, 20), (2, 7000, 255), (3, 1500, 1531), (1, 3, 4099), (1, 2, 9001)])
def test_rows_between_boundaries(dev, B, T, C, gate, dtype):
    """Rows that start anywhere: every array at the same odd place in a buffer of NaN, of which nothing outside the array is
    taken in or written over; with one array at another place too."""
    rows, io, f = B * T, dtype == torch.bfloat16, torch.float32
    gates = rows if gate == "token" else B
    g = torch.Generator().manual_seed(C)

    def put(n, at, fill=True, dt=dtype):
        buffer = torch.full((n * C + 32,), float("nan"), dtype=dt, device=dev)
        if fill:
            buffer[at:at + n * C] = torch.randn(n * C, generator=g).to(dt).to(dev)
        return buffer, buffer[at:at + n * C].view(n, C)

    for at, odd in ((3, 3), (0, 0), (3, 2)):
        x, y, gr, gh = (put(rows, at)[1] for _ in range(4))
        z = put(gates, odd)[1]
        w_pre, w_post, scale = (put(1, 5, dt=f)[1][0] for _ in range(3))
        outs = {n: put(k, at, False) for n, k in (("r", rows), ("h", rows), ("dx", rows), ("dy", rows), ("dgate", gates))}
        sums = {n: put(1, 5, False, f) for n in ("dw_pre", "dw_post", "dscale")}
        p = mixers.BlockNorm(io=int(io), rows=rows, C=C, act=mixers.ACTIVATIONS["silu"], gate_rows=1 if gate == "token" else T,
                             eps=1e-6, x=C, y=C, gate=C, gr=C, gh=C)
        ptr, stream = (lambda t: t.data_ptr()), torch.cuda.current_stream().cuda_stream
        L, inputs_ = mixers.lib(), [ptr(t) for t in (x, y, z, w_pre, w_post, scale)]
        assert L.sffft_blocknorm_fwd(p, *inputs_, ptr(outs["r"][1]), ptr(outs["h"][1]), stream) == 0
        work = torch.full((L.sffft_blocknorm_work_bytes(p, 1, 1) // 4,), float("nan"), device=dev)
        assert L.sffft_blocknorm_bwd(p, *inputs_, ptr(gr), ptr(gh), *(ptr(outs[n][1]) for n in ("dx", "dy", "dgate")),
                                     *(ptr(sums[n][1]) for n in sums), ptr(work), 4 * work.numel(), stream) == 0
        t = {"x": x, "y": y, "w_pre": w_pre, "w_post": w_post, "gate": z, "scale": scale}
        shaped = {n: v if v.dim() == 1 else v.view(B, -1, C) for n, v in t.items()}
        want, grads = oracle(shaped, "silu", gr.view(B, T, C), gh.view(B, T, C))
        got = [outs["r"], outs["h"]] + [{**outs, **sums}["d" + n] for n in NAMES]
        for name, (buffer, a), w in zip(("r", "h") + NAMES, got, (*want, *grads)):
            assert mo.rel_l2(a, w.reshape(a.shape)) < tol(a), (at, odd, name, mo.rel_l2(a, w.reshape(a.shape)))
            assert int(torch.isnan(buffer).sum()) == 32, (at, odd, name)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("T,C", [(700, 1531), (9000, 100), (9000, 37), (30, 2047)])
def test_odd_rows_within_wider_ones(dev, T, C, dtype):
    """Columns of wider arrays, NaN beside them: rows that start at the same distance from a boundary as the outputs', and others."""
    t, gr, gh = inputs(dev, (1, T, C), dtype, "token", seed=C)
    want, wgrads = oracle(t, "silu", gr, gh)

    def within(x, more, at):
        wide = torch.full((1, T, C + more), float("nan"), dtype=dtype, device=dev)
        wide[..., at:at + C] = x
        return wide[..., at:at + C]

    for more, at in ((16, 0), (8, 8), (5, 2)):
        m = dict(t, **{n: within(t[n], more, at) for n in ("x", "y", "gate")})
        out, grads = run(m, "silu", within(gr, more, at), within(gh, more, at))
        for name, a, w in zip(("r", "h") + NAMES, (*out, *grads), (*want, *wgrads)):
            assert mo.rel_l2(a, w) < tol(a), (more, at, name, mo.rel_l2(a, w))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("gate", ["token", "sequence", "none"])
@pytest.mark.parametrize("B,T,C", [(1, 1, 2), (5, 3, 8), (2, 77, 37), (3, 41, 64), (2, 5, 100), (1, 1001, 121), (2, 333, 128), (3, 35, 129),
                                   (1, 9, 200), (2, 50, 249), (1, 70, 256), (2, 70000, 64)])
def test_several_rows_to_a_wavefront(dev, B, T, C, gate, dtype):
    """Narrow rows, and counts of them that leave some lanes without one; eps = 0, where the norm of nothing is not defined."""
    t, gr, gh = inputs(dev, (B, T, C), dtype, gate, seed=C)
    want, wgrads = oracle(t, "sigmoid", gr, gh, 0.0)
    out, grads = run(t, "sigmoid", gr, gh, 0.0)
    names = ("r", "h", *[n for n in NAMES if t[n] is not None])
    for name, a, w in zip(names, (*out, *grads), (*want, *wgrads)):
        assert a.shape == w.shape and mo.rel_l2(a, w) < tol(a), (name, mo.rel_l2(a, w))
    h = torch.ops.sffft.pre_norm(t["x"], t["w_pre"], 0.0)
    assert mo.rel_l2(h, mo.block_norm(t["x"].double().cpu(), None, t["w_pre"].double().cpu(), None, None, None, "none", 0.0)[1]) < tol(h)


def test_gradient_against_differences(dev):
    """Central differences of the fp32 kernel's own outputs over a step of 1e-2 of the values: the curvature leaves
    (1e-2)^2 relative, rounding 2^-24 * 1e2 of the sums' sizes: 1e-3 of the gradient's size along the direction."""
    t, gr, gh = inputs(dev, (2, 20, 96), torch.float32, "sequence", seed=4)
    _, grads = run(t, "silu", gr, gh)
    for i, name in enumerate(NAMES):
        d = torch.randn(t[name].shape, generator=torch.Generator().manual_seed(i)).to(dev)
        def value(sign):
            m = dict(t, **{name: t[name] + sign * 1e-2 * d})
            r, h = torch.ops.sffft.block_norm(*(m[n] for n in NAMES), "silu", 1e-6)
            return float((r.double() * gr).sum() + (h.double() * gh).sum())
        with torch.no_grad():
            want = (value(1) - value(-1)) / 2e-2
        got = float((grads[i].double() * d).sum())
        assert abs(got - want) < 1e-3 * float(grads[i].double().norm() * d.double().norm()), name


def test_equal_calls_give_equal_bits_and_graphs_replay(dev):
    t, gr, gh = inputs(dev, (2, 700, 768), torch.bfloat16, "sequence", seed=5)
    a = run(t, "silu", gr, gh)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b = run(t, "silu", gr, gh)
    side.synchronize()
    for p, q in zip((*a[0], *a[1]), (*b[0], *b[1])):
        assert torch.equal(p, q)
    p = {n: None if x is None else x.reshape(-1, 768) if x.dim() == 3 else x for n, x in t.items()}
    args = (p["x"], p["y"], p["w_pre"], p["w_post"], p["gate"], p["scale"], gr.reshape(-1, 768), gh.reshape(-1, 768), "silu")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = mixers.block_norm_backward(*args)
    for i in range(3):
        p["x"].copy_(torch.randn(p["x"].shape, generator=torch.Generator().manual_seed(i)).to(dev))
        want = mixers.block_norm_backward(*args)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(out, want):
            assert torch.equal(x, y), i


def test_refusals(dev):
    f = torch.ops.sffft.block_norm
    x, w = torch.zeros(2, 3, 8, device=dev), torch.ones(8, device=dev)
    bad = [lambda: f(x.half(), x.half(), w), lambda: f(x, x.bfloat16(), w), lambda: f(x, x[:, :2], w), lambda: f(x, x, w[:7]),
           lambda: f(x, x, w.bfloat16()), lambda: f(x, x, w.cpu()), lambda: f(x, x, w, w[None]),
           lambda: f(x, x, w, w, x[:, :2]), lambda: f(x, x, w, w, x[:1]), lambda: f(x, x, w, w, x.bfloat16()),
           lambda: f(x, x, w, w, x, x), lambda: f(x, x, w, w, x, None, "gelu"), lambda: f(x, x, w, w, x, None, "silu", -1.0),
           lambda: torch.ops.sffft.pre_norm(x, w, float("nan")),
           lambda: torch.ops.sffft.pre_norm(torch.zeros(1, 16385, device=dev), torch.ones(16385, device=dev))]
    for i, call in enumerate(bad):
        with pytest.raises(RuntimeError):
            call()
            raise AssertionError(i)
    y = x.clone().requires_grad_()
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(f(y, x, w)[1].sum(), y, create_graph=True)
    e = torch.zeros(0, 8, device=dev, requires_grad=True)
    r, h = f(e, e.detach(), w)
    assert r.shape == (0, 8) and torch.autograd.grad(h.sum(), e)[0].shape == (0, 8)
