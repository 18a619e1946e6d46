"""Linear attention refuses outputs over any of its inputs, the decays, lengths and slots among them. At the C ABI, without a GPU."""
import ctypes

import pytest
import torch

from sffft_amd import mixers

EINVAL = 1
pytestmark = pytest.mark.skipif(torch.cuda.is_available(), reason="addresses that no kernel may follow")
B, T, H, Hk, D = 3, 700, 4, 2, 64


def at(i):
    return ctypes.c_void_p((1 << 40) + i * (1 << 36))


def params(T):
    p = mixers.LinAttn(0, B, T, H, Hk, D, D, 0.1)
    p.q = p.go = (ctypes.c_longlong * 3)(T * H * D, H * D, D)
    p.k = p.v = (ctypes.c_longlong * 3)(T * Hk * D, Hk * D, D)
    return p


CALLS = {  # inputs, then outputs, in the call's order
    "fwd": (("q", "k", "v", "log_decay", "initial_state", "lengths"), ("o", "final_state", "work")),
    "bwd": (("q", "k", "v", "log_decay", "initial_state", "lengths", "go", "d_final_state"),
            ("dq", "dk", "dv", "d_initial_state", "work")),
    "step": (("q", "k", "v", "log_decay", "state", "slots"), ("o",)),
}


def call(name, **over):
    ins, outs = CALLS[name]
    a = {n: at(i) for i, n in enumerate(ins + outs)}
    a.update({n: a[m] for n, m in over.items()})
    L, args = mixers.lib(), [a[n] for n in ins + outs]
    if name == "step":
        return L.sffft_linattn_step(params(1), *args[:5], 8, args[5], args[6], None)
    return getattr(L, "sffft_linattn_" + name)(params(T), *args, 1 << 35, None)


@pytest.mark.parametrize("name,out,inp", [(n, o, i) for n, (ins, outs) in CALLS.items() for o in outs + (("state",) if n == "step" else ())
                                          for i in ins if i != o])
def test_outputs_over_inputs(name, out, inp):
    in_place = name == "fwd" and (out, inp) == ("final_state", "initial_state")
    assert (call(name, **{out: inp}) == EINVAL) != in_place


@pytest.mark.parametrize("name", CALLS)
def test_apart(name):
    assert call(name) != EINVAL
