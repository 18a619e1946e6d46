"""Forward-mode derivatives of the operators beside the convolution: none has one, and each says so, whatever input carries the
tangent and whether or not a gradient is recorded. On meta tensors, so no GPU is needed."""
import pytest
import torch
import torch.autograd.forward_ad as fw

from sffft_amd import torch_ops  # noqa: F401

ops = torch.ops.sffft
f32 = torch.float32


def t(*shape):
    return torch.empty(*shape, dtype=f32, device="meta")


# name: (the call, its tensors)
CALLS = {
    "linear_attention": (lambda q, k, v, d, s: ops.linear_attention(q, k, v, d, 1.0, s),
                         lambda: [t(2, 5, 4, 16), t(2, 5, 2, 16), t(2, 5, 2, 8), t(4), t(2, 4, 16, 8)]),
    "linear_attention_step": (lambda q, k, v, d, s: ops.linear_attention_step(q, k, v, d, s, 1.0),
                              lambda: [t(2, 4, 16), t(2, 2, 16), t(2, 2, 8), t(4), t(2, 4, 16, 8)]),
    "rotary": (lambda q, k, table: ops.rotary(q, k, table), lambda: [t(2, 5, 4, 16), t(2, 5, 2, 16), t(9, 8)]),
    "rotary_": (lambda q, k, table: ops.rotary_(q, k, table), lambda: [t(2, 5, 4, 16), t(2, 5, 2, 16), t(9, 8)]),
    "block_norm": (lambda x, y, wq, wp, g, s: ops.block_norm(x, y, wq, wp, g, s, "silu"),
                   lambda: [t(2, 5, 8), t(2, 5, 8), t(8), t(8), t(2, 5, 8), t(8)]),
    "pre_norm": (lambda x, w: ops.pre_norm(x, w), lambda: [t(5, 8), t(8)]),
}


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("name,i", [(n, i) for n, (_, args) in CALLS.items() for i in range(len(args()))])
def test_a_tangent_is_refused(name, i, grad):
    call, args = CALLS[name]
    x = args()
    with torch.set_grad_enabled(grad), fw.dual_level():
        x[i] = fw.make_dual(x[i], torch.empty_like(x[i]))
        with pytest.raises(RuntimeError, match="forward-mode"):
            call(*x)
    call(*args())  # and none without one


@pytest.mark.parametrize("name", [n for n in CALLS if n not in ("linear_attention_step", "rotary_")])
def test_a_tangent_of_a_gradient_is_refused(name):
    call, args = CALLS[name]
    x = args()
    x[0].requires_grad_(True)
    out = call(*x)
    out = out if isinstance(out, torch.Tensor) else out[0]
    with fw.dual_level():
        go = fw.make_dual(torch.empty_like(out), torch.empty_like(out))
        with pytest.raises(RuntimeError, match="forward-mode"):
            torch.autograd.grad(out, x[0], go)


def test_jvp_is_refused():
    with pytest.raises(RuntimeError, match="forward-mode"):
        torch.func.jvp(lambda x: ops.pre_norm(x, t(8)), (t(5, 8),), (t(5, 8),))
