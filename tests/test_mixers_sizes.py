"""Sizes whose launches would have 2^32 threads or more: refused before the first launch, with a workspace of 0 bytes; the
largest below them pass the checks (without a GPU the launch itself then fails)."""
import ctypes

import pytest
import torch

from sffft_amd import mixers

NULL = ctypes.c_void_p(0)
EINVAL = 1
pytestmark = pytest.mark.skipif(torch.cuda.is_available(), reason="addresses that no kernel may follow")


def at(i):
    return ctypes.c_void_p((i + 1) << 55)  # far apart: nothing overlaps


def attn(B, H, Hk, Dk=8, Dv=8, T=1, io=1):
    p = mixers.LinAttn(io, B, T, H, Hk, Dk, Dv, 1.0)
    for n, h, d in (("q", H, Dk), ("k", Hk, Dk), ("v", Hk, Dv), ("go", H, Dv)):
        setattr(p, n, (ctypes.c_longlong * 3)(T * h * d, h * d, d))
    return p


def calls(p):
    L, big = mixers.lib(), 1 << 50
    return {"fwd": L.sffft_linattn_fwd(p, at(0), at(1), at(2), at(3), NULL, NULL, at(4), at(5), at(6), big, NULL) != EINVAL,
            "bwd": L.sffft_linattn_bwd(p, at(0), at(1), at(2), at(3), NULL, NULL, at(4), NULL, at(5), at(6), at(7), NULL,
                                       at(8), big, NULL) != EINVAL,
            "step": L.sffft_linattn_step(p, at(0), at(1), at(2), at(3), at(4), 4, NULL, at(5), NULL) != EINVAL}


@pytest.mark.parametrize("B,H,Hk,Dk,Dv,io,fits", [
    ((1 << 24) - 1, 1, 1, 8, 8, 1, "step"), ((1 << 24) - 8, 1, 1, 8, 8, 1, "step fwd"), (1 << 24, 1, 1, 8, 8, 1, ""),
    ((1 << 23) - 8, 1, 1, 8, 72, 1, "step fwd bwd"), (1 << 23, 1, 1, 8, 72, 1, "step"),  # two tiles of values; two marches
    (5592400, 1, 1, 8, 8, 1, "step fwd bwd"), (5592406, 1, 1, 8, 8, 1, "step fwd"),   # three marches
    (2796200, 1, 1, 128, 128, 0, "step fwd bwd"), (2796203, 1, 1, 128, 128, 0, "step fwd"),  # in two tiles
    (4194296, 2, 1, 8, 8, 1, "step fwd bwd"), (4194304, 2, 1, 8, 8, 1, "step fwd"),   # two of shared heads
    ((1 << 23) - 8, 2, 1, 8, 16, 1, "step fwd bwd"), (1 << 23, 2, 1, 8, 16, 1, ""),   # one at a time
])
def test_attention(B, H, Hk, Dk, Dv, io, fits):
    p = attn(B, H, Hk, Dk, Dv, io=io)
    assert {n for n, ok in calls(p).items() if ok} == set(fits.split())
    if "bwd" not in fits:
        assert mixers.lib().sffft_linattn_work_bytes(p, 1) == 0


def test_attention_sums_of_shared_heads():
    # 2^34 elements of dk and dv, four to a thread
    for T, ok in (((1 << 20) - 1, True), (1 << 20, False)):
        p = attn(8, 16, 8, 128, 128, T)
        assert calls(p)["bwd"] is ok and calls(p)["fwd"]
        assert (mixers.lib().sffft_linattn_work_bytes(p, 1) > 0) is ok


def norm(rows, C, gate_rows, io=1):
    return mixers.BlockNorm(io, rows, C, 2, gate_rows, 1e-6, C, C, C, C, C)


@pytest.mark.parametrize("rows,C,gate_rows,ok", [
    (2 * ((1 << 26) - 1), 64, 2, True), (2 << 26, 64, 2, False),            # a wavefront a gate
    (2 * ((1 << 22) - 1), 16384, 2, True), (2 << 22, 16384, 2, False),      # 16 of them
    (2 << 22, 16384, 1, True), (1 << 40, 8, 1, True),                       # a gate a row: parts of many rows
    (2 * 87380 * 100, 1536, 2, True),
])
def test_norms(rows, C, gate_rows, ok):
    L, p = mixers.lib(), norm(rows, C, gate_rows)
    fwd = L.sffft_blocknorm_fwd(p, *[at(i) for i in range(8)], NULL)
    bwd = L.sffft_blocknorm_bwd(p, *[at(i) for i in range(14)], at(14), 1 << 54, NULL)
    assert (fwd != EINVAL) is ok and (bwd != EINVAL) is ok


def test_rotary():
    """A workgroup takes several tokens where there are 2^24 and more."""
    for T, H, D, R, ok in (((1 << 24) - 1, 1, 258, 258, True), (1 << 24, 1, 258, 258, True), ((1 << 31) - 1, 3, 258, 256, True),
                           (1 << 24, 1, 131070, 2, False)):
        p = mixers.Rotary(1, 1, T, H, 0, D, R, 0, 0, 10, 32)
        p.q = p.qo = (ctypes.c_longlong * 3)(T * H * D, H * D, D)
        rc = mixers.lib().sffft_rotary_apply(p, at(0), NULL, at(1), NULL, at(2), NULL, NULL)
        assert (rc != EINVAL) is ok, (T, H, D)
