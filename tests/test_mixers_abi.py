"""The C ABI and the PyTorch schemas of the operators beside the convolution, as far as they need no
GPU: exports, argument refusals, workspace sizes, the rotary tables, fake tensors; and the 64-bit
oracle's own gradients against differences."""
import ctypes
import math
import re

import numpy as np
import pytest
import torch

import mixer_oracle as mo
import sffft_amd as sf
from sffft_amd import mixers, torch_ops  # noqa: F401

NULL = ctypes.c_void_p(0)


def at(i):
    return ctypes.c_void_p((1 << 40) + i * (1 << 36))  # device addresses that no check reads


def strides(*s):
    return (ctypes.c_longlong * 3)(*s)


def test_every_declared_symbol_is_exported():
    text = open(mixers.OPS_HEADER_PATH).read()
    names = set(re.findall(r"^\s*(?:const\s+)?[a-z_0-9]+\s*\*?\s*(sffft_[a-z0-9_]+)\s*\(", text, re.M))
    assert len(names) == 10
    for n in names:
        assert hasattr(mixers.lib(), n), n


def attn(**kw):
    d = dict(io=1, B=2, T=100, H=4, Hk=2, Dk=64, Dv=32, scale=0.125)
    d.update(kw)
    p = mixers.LinAttn(*(d[n] for n in ("io", "B", "T", "H", "Hk", "Dk", "Dv", "scale")))
    p.q, p.go = strides(d["T"] * d["H"] * d["Dk"], d["H"] * d["Dk"], d["Dk"]), strides(d["T"] * d["H"] * d["Dv"], d["H"] * d["Dv"], d["Dv"])
    p.k, p.v = strides(d["T"] * d["Hk"] * d["Dk"], d["Hk"] * d["Dk"], d["Dk"]), strides(d["T"] * d["Hk"] * d["Dv"], d["Hk"] * d["Dv"], d["Dv"])
    return p


BAD_SHAPES = [dict(io=2), dict(B=0), dict(T=0), dict(H=0), dict(Hk=3), dict(Dk=0), dict(Dk=60), dict(Dk=136),
              dict(Dv=4), dict(Dv=256), dict(B=1 << 20, T=1 << 12)]


@pytest.mark.parametrize("bad", BAD_SHAPES, ids=str)
def test_linattn_refuses_shapes(bad):
    p, L = attn(**bad), mixers.lib()
    big = 1 << 40
    assert L.sffft_linattn_fwd(p, at(0), at(1), at(2), at(3), NULL, NULL, at(4), at(5), at(6), big, NULL) == 1
    assert L.sffft_linattn_bwd(p, at(0), at(1), at(2), at(3), NULL, NULL, at(4), NULL, at(5), at(6), at(7), NULL, at(8),
                               big, NULL) == 1
    assert L.sffft_linattn_step(p, at(0), at(1), at(2), at(3), at(4), 4, NULL, at(5), NULL) == 1
    assert L.sffft_linattn_work_bytes(p, 0) == 0 and L.sffft_linattn_work_bytes(p, 1) == 0


def test_linattn_refuses_pointers():
    L, p, big = mixers.lib(), attn(), 1 << 34
    def fwd(*a):
        return L.sffft_linattn_fwd(p, *a, big, NULL)
    good = [at(0), at(1), at(2), at(3), NULL, NULL, at(4), at(5), at(6)]
    for i in (0, 1, 2, 3, 6):  # q, k, v, log_decay, o may not be NULL
        assert fwd(*[NULL if j == i else g for j, g in enumerate(good)]) == 1, i
    off = ctypes.c_void_p(at(9).value + 8)
    for i in (0, 1, 2, 4, 6, 7):  # 16-byte rows
        assert fwd(*[off if j == i else g for j, g in enumerate(good)]) == 1, i
    assert fwd(*[at(0) if j == 6 else g for j, g in enumerate(good)]) == 1           # o over q
    assert fwd(*[at(1) if j == 7 else g for j, g in enumerate(good)]) == 1           # final state over k
    p.q = strides(100 * 4 * 64, 4 * 64 + 4, 64)                                      # rows not aligned
    assert fwd(*good) == 1
    p.q = strides(-100 * 4 * 64, 4 * 64, 64)
    assert fwd(*good) == 1
    p = attn()
    p1 = attn(T=1)
    assert L.sffft_linattn_step(p, at(0), at(1), at(2), at(3), at(4), 4, NULL, at(5), NULL) == 1    # T is not 1
    assert L.sffft_linattn_step(p1, at(0), at(1), at(2), at(3), at(4), 0, NULL, at(5), NULL) == 1   # no slot
    assert L.sffft_linattn_step(p1, at(0), at(1), at(2), at(3), at(0), 4, NULL, at(5), NULL) == 1   # state over q
    b = [at(0), at(1), at(2), at(3), NULL, NULL, at(4), NULL, at(5), at(6), at(7), NULL]
    def bwd(args, work=at(8), n=big):
        return L.sffft_linattn_bwd(p, *args, work, n, NULL)
    for i in (0, 1, 2, 3, 6, 8, 9, 10):
        assert bwd([NULL if j == i else g for j, g in enumerate(b)]) == 1, i
    need = L.sffft_linattn_work_bytes(p, 1)
    assert need >= 2 * 100 * 4 * (64 + 32) * 4  # shared heads: dk and dv of each query head
    assert bwd(b, NULL) == 1 and bwd(b, at(8), need - 1) == 1 and bwd(b, at(5)) == 1
    assert bwd([at(8) if j == 8 else g for j, g in enumerate(b)]) == 1               # dq over the workspace


def rotary(**kw):
    d = dict(io=1, B=2, T=10, H=4, Hk=2, D=64, R=32, interleaved=0, inverse=0, positions=100, pos_bits=32)
    d.update(kw)
    p = mixers.Rotary(*d.values())
    p.q = p.qo = strides(d["T"] * d["H"] * d["D"], d["H"] * d["D"], d["D"])
    p.k = p.ko = strides(d["T"] * d["Hk"] * d["D"], d["Hk"] * d["D"], d["D"])
    return p


def test_rotary_refusals():
    f = mixers.lib().sffft_rotary_apply
    a = [at(0), at(1), at(2), at(3), at(4), at(5), NULL]
    for bad in (dict(io=3), dict(B=0), dict(T=0), dict(H=0), dict(Hk=-1), dict(D=63), dict(R=0), dict(R=31), dict(R=66),
                dict(interleaved=2), dict(inverse=-1), dict(positions=0), dict(pos_bits=16), dict(B=1 << 30, T=1 << 10)):
        assert f(rotary(**bad), *a) == 1, bad
    p = rotary()
    for i in (0, 1, 2, 4, 5):
        assert f(p, *[NULL if j == i else g for j, g in enumerate(a)]) == 1, i
    assert f(rotary(Hk=0), *a) == 1                                                # k given, no key heads
    assert f(p, at(0), at(1), at(2), at(3), at(1), at(5), NULL) == 1               # q' over k is not in place
    assert f(p, at(0), at(1), at(2), at(3), ctypes.c_void_p(at(0).value + 64), at(5), NULL) == 1  # a partial overlap
    assert f(p, at(0), at(1), at(2), at(3), at(2), at(5), NULL) == 1               # over the table
    assert f(p, ctypes.c_void_p(at(0).value + 1), *a[1:]) == 1
    p.qo = strides(10 * 4 * 64, 4 * 64, 128)
    assert f(p, at(0), at(1), at(2), at(3), at(0), at(5), NULL) == 1               # in place at other strides


def norm(**kw):
    d = dict(io=1, rows=12, C=40, act=2, gate_rows=1, eps=1e-6, x=40, y=40, gate=40, gr=40, gh=40)
    d.update(kw)
    return mixers.BlockNorm(*d.values())


def test_norm_refusals():
    L = mixers.lib()
    f = [at(i) for i in range(8)] + [NULL]
    b = [at(i) for i in range(14)]
    for bad in (dict(io=2), dict(rows=0), dict(C=0), dict(C=16385), dict(act=3), dict(gate_rows=0), dict(gate_rows=5),
                dict(eps=-1.0), dict(eps=math.inf), dict(eps=math.nan), dict(x=39), dict(x=-40)):
        p = norm(**bad)
        assert L.sffft_blocknorm_fwd(p, *f) == 1, bad
        assert L.sffft_blocknorm_bwd(p, *b, at(14), 1 << 34, NULL) == 1, bad
    p = norm()
    def fwd(**kw):
        names = ("x", "y", "gate", "w_pre", "w_post", "scale", "r", "h")
        return L.sffft_blocknorm_fwd(p, *[kw.get(n, g) for n, g in zip(names, f)], NULL)
    for kw in (dict(x=NULL), dict(w_pre=NULL), dict(h=NULL), dict(r=NULL), dict(y=NULL), dict(h=at(0)), dict(r=at(7)),
               dict(y=NULL, r=NULL), dict(x=ctypes.c_void_p(at(0).value + 1))):
        assert fwd(**kw) == 1, kw
    need = L.sffft_blocknorm_work_bytes(p, 1, 1)
    assert need > 0
    def bwd(work=at(14), n=1 << 34, **kw):
        names = ("x", "y", "gate", "w_pre", "w_post", "scale", "gr", "gh", "dx", "dy", "dgate", "dw_pre", "dw_post", "dscale")
        return L.sffft_blocknorm_bwd(p, *[kw.get(m, g) for m, g in zip(names, b)], work, n, NULL)
    for kw in (dict(work=NULL), dict(n=need - 1), dict(gr=NULL, gh=NULL), dict(dx=NULL), dict(dy=NULL), dict(dgate=NULL),
               dict(dw_post=NULL), dict(scale=NULL), dict(dx=at(6)), dict(work=at(0)), dict(dw_pre=at(8))):
        assert bwd(**kw) == 1, kw


@pytest.mark.parametrize("scaling", sorted(mixers.SCALINGS))
@pytest.mark.parametrize("R", [2, 10, 64])
def test_rotary_table(scaling, R):
    P, base, factor, trained = 700, 500.0, 4.0, 256
    t = mixers.rotary_table(P, R, base, scaling, factor, trained, 1.25).numpy().astype(np.float64)
    i = np.arange(R // 2)
    f = base ** (-2.0 * i / R)
    if scaling == "linear":
        f = f / factor
    if scaling == "stretched" and R > 2:
        f = (base * factor ** (R / (R - 2))) ** (-2.0 * i / R)
        assert np.isclose(f[0], 1.0) and np.isclose(f[-1] * factor, base ** (-2.0 * i[-1] / R))
    if scaling == "parts":
        keep = np.clip((trained * f / (2 * np.pi) - 1) / 31, 0, 1)
        f = f * keep + f / factor * (1 - keep)
    a = np.arange(P)[:, None] * f
    want = 1.25 * np.concatenate([np.cos(a), np.sin(a)], 1)
    # one rounding to fp32 (2^-24 relative), and the two hosts' cos and angle: 700 * 2^-52 and less
    assert np.abs(t - want).max() <= 1.25 * (2.0 ** -24 + 1e-12)


def test_rotary_table_refusals():
    for kw in (dict(positions=0, R=8), dict(positions=4, R=7), dict(positions=4, R=0), dict(positions=4, R=8, base=0.0),
               dict(positions=4, R=8, base=math.inf), dict(positions=4, R=8, factor=0.0),
               dict(positions=4, R=8, scaling="parts", trained=0), dict(positions=4, R=8, magnitude=math.nan)):
        with pytest.raises(mixers.MixerError):
            mixers.rotary_table(**kw)
    with pytest.raises(ValueError):
        mixers.rotary_table(4, 8, scaling="other")


def test_schemas_and_dispatch():
    s = {n: str(getattr(torch.ops.sffft, n).default._schema) for n in ("linear_attention_step", "rotary_", "block_norm")}
    assert "Tensor(a!) state" in s["linear_attention_step"]
    assert "Tensor(a!) q, Tensor(b!) k" in s["rotary_"]
    assert 'str activation="none", float eps=' in s["block_norm"]
    for n in ("linear_attention", "linear_attention_step", "rotary", "rotary_", "block_norm", "pre_norm"):
        for key in ("CUDA", "Autograd"):
            assert torch._C._dispatch_has_kernel_for_dispatch_key(f"sffft::{n}", key), (n, key)


def test_fake_shapes():
    from torch._subclasses.fake_tensor import FakeTensorMode

    ops = torch.ops.sffft
    with FakeTensorMode():
        def t(*s, dtype=torch.bfloat16):
            return torch.empty(*s, device="cuda", dtype=dtype)
        ld = t(6, dtype=torch.float32)
        o, s = ops.linear_attention(t(2, 9, 6, 64), t(2, 9, 3, 64), t(2, 9, 3, 32), ld, 0.1)
        assert o.shape == (2, 9, 6, 32) and o.dtype == torch.bfloat16
        assert s.shape == (2, 6, 64, 32) and s.dtype == torch.float32
        assert ops.linear_attention_step(t(2, 6, 64), t(2, 3, 64), t(2, 3, 32), ld, s, 0.1).shape == (2, 6, 32)
        q, k = ops.rotary(t(2, 9, 6, 64), t(2, 9, 3, 64), t(50, 32, dtype=torch.float32))
        assert q.shape == (2, 9, 6, 64) and k.shape == (2, 9, 3, 64)
        r, h = ops.block_norm(t(2, 9, 48), t(2, 9, 48), t(48, dtype=torch.float32))
        assert r.shape == h.shape == (2, 9, 48) and h.dtype == torch.bfloat16
        assert ops.pre_norm(t(5, 48), t(48, dtype=torch.float32)).shape == (5, 48)
        for bad in (lambda: ops.linear_attention(t(2, 9, 6, 60), t(2, 9, 3, 60), t(2, 9, 3, 32), ld, 0.1),
                    lambda: ops.linear_attention(t(2, 9, 6, 64), t(2, 8, 3, 64), t(2, 8, 3, 32), ld, 0.1),
                    lambda: ops.rotary(t(2, 9, 6, 64), t(2, 9, 3, 64), t(50, 66, dtype=torch.float32)),
                    lambda: ops.block_norm(t(2, 9, 48), t(2, 9, 48), t(47, dtype=torch.float32))):
            with pytest.raises(RuntimeError):
                bad()


def test_oracle_attention_gradient_against_differences():
    """The oracle's gradient, used for the kernels', against central differences of its recurrence. It is
    linear in each input, so a difference is exact but for rounding: 1e-16 of values of order 10 over steps of 1."""
    g = torch.Generator().manual_seed(3)
    B, T, H, Hk, Dk, Dv = 2, 7, 4, 2, 8, 8
    def r(*s):
        return torch.randn(*s, generator=g, dtype=torch.float64)
    q, k, v, s0, go, gs = r(B, T, H, Dk), r(B, T, Hk, Dk), r(B, T, Hk, Dv), r(B, H, Dk, Dv), r(B, T, H, Dv), r(B, H, Dk, Dv)
    ld, n = torch.tensor([-0.1, -1.0, 0.0, -3.0], dtype=torch.float64), [7, 4]
    grads = mo.attention_grads(q, k, v, ld, 0.3, go, gs, s0, n)[2:]
    x = [q, k, v, s0]
    for i in range(4):
        d = torch.randn(x[i].shape, generator=g, dtype=torch.float64)
        def loss(sign):
            y = [t + sign * d if j == i else t for j, t in enumerate(x)]
            o, s = mo.attention(y[0], y[1], y[2], ld, 0.3, y[3], n)
            return float((o * go).sum() + (s * gs).sum())
        want = (loss(1) - loss(-1)) / 2
        assert abs(float((grads[i] * d).sum()) - want) < 1e-9 * max(1.0, abs(want)), i
    # a plausible mistake (the decay of a shared head's neighbour) fails the same check
    wrong = mo.attention_grads(q, k, v, ld.flip(0), 0.3, go, gs, s0, n)[2]
    assert mo.rel_l2(wrong, grads[0]) > 1e-2
