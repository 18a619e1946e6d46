"""rotary_ refuses views whose elements alias, which several lanes would turn in no order, and turns those that do not."""
import pytest
import torch

from sffft_amd import mixers, torch_ops  # noqa: F401

pytestmark = pytest.mark.gpu


def test_views_in_place(dev):
    B, T, H, Hk, D = 2, 33, 4, 2, 64
    table = mixers.rotary_table(64, D, device=dev)
    x = torch.randn(B, T, (H + 2 * Hk) * D, device=dev)
    for view in (lambda t: t[..., :H * D].unflatten(-1, (H, D)), lambda t: t.view(B, -1)[:, :H * T * D].unflatten(-1, (H, T, D)).transpose(1, 2)):
        for other in (lambda t: t[..., H * D:(H + Hk) * D].unflatten(-1, (Hk, D)),
                      lambda t: t.view(B, -1)[:, H * T * D:(H + Hk) * T * D].unflatten(-1, (Hk, T, D)).transpose(1, 2)):
            y = x.clone()
            q, k = view(y), other(y)
            if q.stride() != k.stride():
                with pytest.raises(RuntimeError, match="overlap"):
                    torch.ops.sffft.rotary_(q, k, table)
                continue
            want = torch.ops.sffft.rotary(view(x), other(x), table)
            torch.ops.sffft.rotary_(q, k, table)
            assert torch.equal(q, want[0]) and torch.equal(k, want[1])
    z = torch.randn(B, T, H, D, device=dev)
    for q, k in ((z, z[:, :, 1:]), (z, z), (z[:, :, 1:], z), (z.as_strided((B, T, 3, D), (D, D, D, 1)), z[:, :, :0]),
                 (z.as_strided((1, T, 3, D), (0, D, D, 1)), z[:1, :, :0]), (z[:, :1].expand(B, T, H, D), z[:, :, :0])):
        before = z.clone()
        with pytest.raises(RuntimeError, match="overlap"):
            torch.ops.sffft.rotary_(q, k, table)
        assert torch.equal(z, before)
