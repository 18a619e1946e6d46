"""Registers that the norm kernels of more than 512 lanes spill: rows of more than 4096 channels leave each lane 128 registers, and
the gradients need more. Bounds of what stands, so that it does not grow unseen; none elsewhere (test_mixer_resources.py)."""
import pytest

from test_mixer_resources import kernels

# forward or backward, channels a lane (16 beyond 8192 channels), with y: registers a lane at most
BOUNDS = {("fwd", "8", "0"): 0, ("fwd", "8", "1"): 0, ("fwd", "16", "0"): 0, ("fwd", "16", "1"): 9,
          ("bwd", "8", "0"): 0, ("bwd", "8", "1"): 87, ("bwd", "16", "0"): 8, ("bwd", "16", "1"): 312}


@pytest.mark.parametrize("which,n,y", BOUNDS)
def test_spills_of_wide_rows(which, n, y):
    found = [r for key, r in kernels("ops_api", r"(fwd|bwd)_kernelI[ft]Li\d+ELi(\d+)ELi1024ELb[01]ELb([01])E") if key == (which, n, y)]
    assert found
    assert max(int(r["VGPRs Spill"]) for r in found) <= BOUNDS[which, n, y]
