"""How attention calls are cut into segments, as their workspaces tell: no GPU is needed."""
import ctypes

import pytest

from sffft_amd import mixers

CUS = 256


def segments(heads, T, D, io):
    p = mixers.LinAttn(io, heads, T, 1, 1, D, D, 1.0)
    n = mixers.lib().sffft_linattn_work_bytes(ctypes.byref(p), 0) // (heads * D * D * 4)
    return max(n, 1)


@pytest.mark.parametrize("io", [0, 1])
@pytest.mark.parametrize("D", [64, 128])
def test_eight_segments_only_where_they_run_well(D, io):
    """A call gets fewer segments than would fill the chip, to have at most 8, only if these make 5 workgroups for 8 CUs, and no more
    than one on each (above 64 channels) or two (fp32); else the finest cut up to `fill` workgroups."""
    chunk, fill = (64 if io else 32), (512 if D > 64 else 1024)
    joined = 0
    for heads in range(1, 200):
        for T in range(chunk, 200 * chunk, 13 * chunk):
            chunks = T // chunk
            per = -(-chunks // min(chunks, max(1, fill // heads)))
            n = segments(heads, T, D, io)
            if n != -(-chunks // per):
                assert n <= 8, (heads, T)
                assert n * heads >= CUS * 5 // 8, (heads, T, n)
                assert n * heads <= (CUS if D > 64 else 2 * CUS if not io else 8 * 200), (heads, T, n)
                joined += 1
    assert joined
