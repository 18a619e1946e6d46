"""Python binding of libsffft_ops.so (include/sffft_ops.h): the sequence-mixing operators beside the
long convolution.

- linear attention with a decay for each head: ``linear_attention`` (prompts, any length),
  ``linear_attention_backward`` and ``linear_attention_step`` (one token, state in place);
- rotary positions: ``rotary`` and ``rotary_table``;
- the norms around a block with its gate and residual scale: ``block_norm``,
  ``block_norm_backward``.

A thin ctypes layer, as ``sffft_amd`` is over libsffft.so: torch supplies device memory and the current
stream, and there is no fallback. For training use ``torch.ops.sffft.linear_attention`` /
``rotary`` / ``block_norm`` / ``pre_norm`` (``sffft_amd.torch_ops``), which are differentiable.
"""
from __future__ import annotations

import ctypes
import os

from . import SFFFT_EHIP, SFFFT_OK, _HERE, _ptr, _stream, strerror

OPS_LIB_PATH = os.path.join(_HERE, "libsffft_ops.so")
OPS_HEADER_PATH = os.path.join(os.path.dirname(_HERE), "include", "sffft_ops.h")
IO_F32, IO_BF16 = 0, 1
ACTIVATIONS = {"none": 0, "sigmoid": 1, "silu": 2}
SCALINGS = {"none": 0, "linear": 1, "stretched": 2, "parts": 3}

_Strides = ctypes.c_longlong * 3


class LinAttn(ctypes.Structure):
    """sffft_linattn"""

    _fields_ = [(n, ctypes.c_int) for n in ("io", "B", "T", "H", "Hk", "Dk", "Dv")] + [("scale", ctypes.c_float)] + \
        [(n, _Strides) for n in ("q", "k", "v", "go")]


class Rotary(ctypes.Structure):
    """sffft_rotary"""

    _fields_ = [(n, ctypes.c_int) for n in ("io", "B", "T", "H", "Hk", "D", "R", "interleaved", "inverse", "positions",
                                            "pos_bits")] + [(n, _Strides) for n in ("q", "k", "qo", "ko")]


class BlockNorm(ctypes.Structure):
    """sffft_blocknorm"""

    _fields_ = [("io", ctypes.c_int), ("rows", ctypes.c_longlong), ("C", ctypes.c_int), ("act", ctypes.c_int),
                ("gate_rows", ctypes.c_longlong), ("eps", ctypes.c_float)] + \
        [(n, ctypes.c_longlong) for n in ("x", "y", "gate", "gr", "gh")]


_lib = None


def lib() -> ctypes.CDLL:
    """Loads libsffft_ops.so (built in-tree by `make -C sffft_amd -f ops.mk`)."""
    global _lib
    if _lib is None:
        if not os.path.exists(OPS_LIB_PATH):
            raise RuntimeError(f"{OPS_LIB_PATH} is missing: build it with `make -C sffft_amd -f ops.mk` "
                               "(or __graft_entry__.build())")
        try:
            import torch  # noqa: F401  (its HIP runtime is the one to bind, as in load_library)
        except ImportError:
            pass
        L = ctypes.CDLL(OPS_LIB_PATH)
        vp, ci, sz, cd = ctypes.c_void_p, ctypes.c_int, ctypes.c_size_t, ctypes.c_double
        A, R, N = (ctypes.POINTER(t) for t in (LinAttn, Rotary, BlockNorm))
        sigs = {
            "sffft_linattn_work_bytes": (sz, [A, ci]),
            "sffft_linattn_fwd": (ci, [A] + [vp] * 9 + [sz, vp]),
            "sffft_linattn_bwd": (ci, [A] + [vp] * 13 + [sz, vp]),
            "sffft_linattn_step": (ci, [A] + [vp] * 5 + [ci, vp, vp, vp]),
            "sffft_rotary_apply": (ci, [R] + [vp] * 7),
            "sffft_rotary_table": (ci, [ci, ci, cd, ci, cd, ci, cd, vp]),
            "sffft_blocknorm_work_bytes": (sz, [N, ci, ci]),
            "sffft_blocknorm_fwd": (ci, [N] + [vp] * 9),
            "sffft_blocknorm_bwd": (ci, [N] + [vp] * 15 + [sz, vp]),
            "sffft_ops_last_error": (ctypes.c_char_p, []),
        }
        for name, (res, args) in sigs.items():
            f = getattr(L, name)
            f.restype, f.argtypes = res, args
        _lib = L
    return _lib


class MixerError(RuntimeError):
    def __init__(self, code: int, what: str):
        detail = lib().sffft_ops_last_error().decode() if code == SFFFT_EHIP else ""
        super().__init__(f"{what}: {strerror(code)} (code {code}) {detail}".rstrip())
        self.code = code


def _check(code: int, what: str) -> None:
    if code != SFFFT_OK:
        raise MixerError(code, what)


def _io(t) -> int:
    import torch

    if not t.is_cuda or t.dtype not in (torch.float32, torch.bfloat16):
        raise TypeError(f"float32 or bfloat16 GPU tensors expected, got {t.dtype} on {t.device}")
    return IO_BF16 if t.dtype == torch.bfloat16 else IO_F32


def _opt(t):
    return ctypes.c_void_p(0) if t is None else _ptr(t)


def _strides(t, token: bool = True):
    s = t.stride()
    return _Strides(s[0], s[1] if token else 0, s[-2])


def _same(what, ref, *tensors):
    for t in tensors:
        if t is not None and (t.device != ref.device or t.stride(-1) != 1):
            raise ValueError(f"{what}: every tensor must be on {ref.device} with contiguous channels")


def linattn_params(q, k, v, scale: float, token: bool = True, go=None) -> LinAttn:
    """The sffft_linattn of q [B, T, H, Dk], k [B, T, Hk, Dk], v [B, T, Hk, Dv] (without T: token False)."""
    T = q.shape[1] if token else 1
    if k.shape[:-2] != q.shape[:-2] or v.shape[:-1] != k.shape[:-1] or k.shape[-1] != q.shape[-1] or \
            not q.dtype == k.dtype == v.dtype:
        raise ValueError(f"k and v must be the keys and values of q's tokens, in its type: got {tuple(q.shape)}, "
                         f"{tuple(k.shape)}, {tuple(v.shape)}")
    p = LinAttn(_io(q), q.shape[0], T, q.shape[-2], k.shape[-2], q.shape[-1], v.shape[-1], scale)
    p.q, p.k, p.v = _strides(q, token), _strides(k, token), _strides(v, token)
    if go is not None:
        p.go = _strides(go)
    return p


def _vectors(what, p, log_decay, state, lengths, ref, rows):
    import torch

    if log_decay.dtype != torch.float32 or tuple(log_decay.shape) != (p.H,) or not log_decay.is_contiguous():
        raise ValueError(f"{what}: log_decay must be float32 [{p.H}]")
    if state is not None and (state.dtype != torch.float32 or not state.is_contiguous()
                              or tuple(state.shape[1:]) != (p.H, p.Dk, p.Dv) or rows is not None and len(state) != rows):
        raise ValueError(f"{what}: the state must be contiguous float32 [.., {p.H}, {p.Dk}, {p.Dv}]")
    if lengths is not None and (lengths.dtype != torch.int32 or tuple(lengths.shape) != (p.B,)
                                or not lengths.is_contiguous()):
        raise ValueError(f"{what}: lengths or slots must be int32 [{p.B}]")
    _same(what, ref, log_decay, state, lengths)


def linear_attention(q, k, v, log_decay, scale: float, initial_state=None, lengths=None, work=None):
    """(o [B, T, H, Dv], final state [B, H, Dk, Dv] fp32) of sffft_linattn_fwd."""
    import torch

    _same("linear_attention", q, q, k, v)
    p = linattn_params(q, k, v, scale)
    _vectors("linear_attention", p, log_decay, initial_state, lengths, q, p.B)
    o = torch.empty((p.B, p.T, p.H, p.Dv), dtype=q.dtype, device=q.device)
    s = torch.empty((p.B, p.H, p.Dk, p.Dv), dtype=torch.float32, device=q.device)
    need = lib().sffft_linattn_work_bytes(ctypes.byref(p), 0)
    if work is None:
        work = torch.empty(max(need, 16), dtype=torch.uint8, device=q.device)
    _check(lib().sffft_linattn_fwd(ctypes.byref(p), _ptr(q), _ptr(k), _ptr(v), _ptr(log_decay), _opt(initial_state),
                                   _opt(lengths), _ptr(o), _ptr(s), _ptr(work), work.numel() * work.element_size(),
                                   _stream()), "sffft_linattn_fwd")
    return o, s


def linear_attention_backward(q, k, v, log_decay, scale: float, go, initial_state=None, lengths=None,
                              d_final_state=None, work=None):
    """(dq, dk, dv, d_initial_state) of sffft_linattn_bwd from o's gradient go [B, T, H, Dv]."""
    import torch

    _same("linear_attention_backward", q, q, k, v, go)
    p = linattn_params(q, k, v, scale, go=go)
    if tuple(go.shape) != (p.B, p.T, p.H, p.Dv) or go.dtype != q.dtype:
        raise ValueError("linear_attention_backward: go must be [B, T, H, Dv] in q's type")
    _vectors("linear_attention_backward", p, log_decay, initial_state, lengths, q, p.B)
    _vectors("linear_attention_backward", p, log_decay, d_final_state, lengths, q, p.B)
    dq, dk, dv = (torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k, v))
    ds = torch.empty((p.B, p.H, p.Dk, p.Dv), dtype=torch.float32, device=q.device)
    need = lib().sffft_linattn_work_bytes(ctypes.byref(p), 1)
    if work is None:
        work = torch.empty(max(need, 16), dtype=torch.uint8, device=q.device)
    _check(lib().sffft_linattn_bwd(ctypes.byref(p), _ptr(q), _ptr(k), _ptr(v), _ptr(log_decay), _opt(initial_state),
                                   _opt(lengths), _ptr(go), _opt(d_final_state), _ptr(dq), _ptr(dk), _ptr(dv),
                                   _ptr(ds), _ptr(work), work.numel() * work.element_size(), _stream()),
           "sffft_linattn_bwd")
    return dq, dk, dv, ds


def linear_attention_step(q, k, v, log_decay, state, scale: float, slots=None):
    """o [B, H, Dv] of one token, q [B, H, Dk], k [B, Hk, Dk], v [B, Hk, Dv]; state [slots, H, Dk, Dv] in place."""
    import torch

    _same("linear_attention_step", q, q, k, v)
    p = linattn_params(q, k, v, scale, token=False)
    _vectors("linear_attention_step", p, log_decay, state, slots, q, None)
    if slots is None and len(state) < p.B:
        raise ValueError(f"linear_attention_step: {p.B} sequences need as many rows of state or slots")
    o = torch.empty((p.B, p.H, p.Dv), dtype=q.dtype, device=q.device)
    _check(lib().sffft_linattn_step(ctypes.byref(p), _ptr(q), _ptr(k), _ptr(v), _ptr(log_decay), _ptr(state),
                                    len(state), _opt(slots), _ptr(o), _stream()), "sffft_linattn_step")
    return o


def rotary_table(positions: int, R: int, base: float = 10000.0, scaling: str = "none", factor: float = 1.0,
                 trained: int = 1, magnitude: float = 1.0, device=None):
    """The table [positions, R] fp32 (cos, then sin) of sffft_rotary_table, on `device`. `scaling`:
    "none", "linear" (positions divided by factor), "stretched" (a larger base) or "parts" (pairs that
    turn less than once over `trained` tokens divided by factor, fast ones kept)."""
    import torch

    if scaling not in SCALINGS:
        raise ValueError(f"scaling must be one of {sorted(SCALINGS)}, got {scaling!r}")
    table = torch.empty((max(positions, 1), max(R, 1)), dtype=torch.float32)
    _check(lib().sffft_rotary_table(positions, R, base, SCALINGS[scaling], factor, trained, magnitude, _ptr(table)),
           "sffft_rotary_table")
    return table if device is None else table.to(device)


def rotary(q, k, table, positions=None, interleaved: bool = False, inverse: bool = False, inplace: bool = False):
    """(q', k') of sffft_rotary_apply for q [B, T, H, D], k [B, T, Hk, D]; in place: q and k themselves."""
    import torch

    _same("rotary", q, q, k, table, positions)
    B, T, H, D = q.shape
    if k.dim() != 4 or k.shape[:2] != q.shape[:2] or k.shape[3] != D or k.dtype != q.dtype:
        raise ValueError("rotary: k must be [B, T, Hk, D] in q's type")
    if table.dtype != torch.float32 or table.dim() != 2 or not table.is_contiguous():
        raise ValueError("rotary: table must be contiguous float32 [positions, R]")
    if positions is not None and (positions.dtype not in (torch.int32, torch.int64) or not positions.is_contiguous()
                                  or tuple(positions.shape) != (B, T)):
        raise ValueError("rotary: positions must be contiguous int32 or int64 [B, T]")
    qo, ko = (q, k) if inplace else (torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k))
    bits = 64 if positions is not None and positions.dtype == torch.int64 else 32
    p = Rotary(_io(q), B, T, H, k.shape[2], D, table.shape[1], int(interleaved), int(inverse), table.shape[0], bits,
               _strides(q), _strides(k), _strides(qo), _strides(ko))
    _check(lib().sffft_rotary_apply(ctypes.byref(p), _ptr(q), _ptr(k), _ptr(table), _opt(positions), _ptr(qo),
                                    _ptr(ko), _stream()), "sffft_rotary_apply")
    return qo, ko


def _norm_params(x, y, gate, activation, eps, gr=None, gh=None) -> BlockNorm:
    import torch

    C = x.shape[-1]
    for t in (x, y, gate, gr, gh):
        if t is not None and (t.dim() != 2 or t.shape[1] != C or t.dtype != x.dtype):
            raise ValueError("block_norm: x, y, gate and gradients must be [rows, C] in one type")
    rows = x.shape[0]
    for t in (y, gr, gh):
        if t is not None and t.shape[0] != rows:
            raise ValueError("block_norm: y and gradients must have x's rows")
    if gate is not None and (gate.shape[0] < 1 or rows % gate.shape[0]):
        raise ValueError("block_norm: the gate's rows must divide x's")
    _same("block_norm", x, x, y, gate, gr, gh)
    assert isinstance(x, torch.Tensor)
    return BlockNorm(_io(x), rows, C, ACTIVATIONS[activation], rows // gate.shape[0] if gate is not None else 1, eps,
                     *(t.stride(0) if t is not None else 0 for t in (x, y, gate, gr, gh)))


def _norm_vectors(C, ref, *ws):
    import torch

    for w in ws:
        if w is not None and (w.dtype != torch.float32 or tuple(w.shape) != (C,) or not w.is_contiguous()):
            raise ValueError(f"block_norm: weights must be contiguous float32 [{C}]")
    _same("block_norm", ref, *ws)


def block_norm(x, y, w_pre, w_post=None, gate=None, scale=None, activation: str = "none", eps: float = 1e-6):
    """(r, h) of sffft_blocknorm_fwd for x, y [rows, C]; gate [rows, C] or a row for every rows / n. y None:
    (None, norm(x) . w_pre)."""
    import torch

    p = _norm_params(x, y, gate, activation, eps)
    _norm_vectors(p.C, x, w_pre, w_post, scale)
    r = None if y is None else torch.empty(x.shape, dtype=x.dtype, device=x.device)
    h = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    _check(lib().sffft_blocknorm_fwd(ctypes.byref(p), _ptr(x), _opt(y), _opt(gate), _ptr(w_pre), _opt(w_post),
                                     _opt(scale), _opt(r), _ptr(h), _stream()), "sffft_blocknorm_fwd")
    return r, h


def block_norm_backward(x, y, w_pre, w_post, gate, scale, gr, gh, activation: str = "none", eps: float = 1e-6,
                        work=None):
    """(dx, dy, dgate, dw_pre, dw_post, dscale) of sffft_blocknorm_bwd; None for absent inputs."""
    import torch

    p = _norm_params(x, y, gate, activation, eps, gr, gh)
    _norm_vectors(p.C, x, w_pre, w_post, scale)
    out = [None if t is None else torch.empty(t.shape, dtype=t.dtype, device=x.device)
           for t in (x, y, gate, w_pre, w_post, scale)]
    need = lib().sffft_blocknorm_work_bytes(ctypes.byref(p), int(y is not None), int(gate is not None))
    if work is None:
        work = torch.empty(max(need, 16), dtype=torch.uint8, device=x.device)
    _check(lib().sffft_blocknorm_bwd(ctypes.byref(p), _ptr(x), _opt(y), _opt(gate), _ptr(w_pre), _opt(w_post),
                                     _opt(scale), _opt(gr), _opt(gh), *(_opt(t) for t in out), _ptr(work),
                                     work.numel() * work.element_size(), _stream()), "sffft_blocknorm_bwd")
    return tuple(out)
