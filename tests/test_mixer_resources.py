"""The compiler's resource report of linear attention, rotary positions and block norms: the wavefronts a SIMD that the
launches count on, and no spills but those of the largest tiles.

As for the convolution's kernels (test_kernel_resources.py) the build keeps the report beside each object; no
GPU is needed.
"""
import re

import pytest

from test_kernel_resources import reports


def kernels(objects, pattern):
    rep = reports(objects=objects)
    if not rep:
        pytest.skip("no resource reports: build with `make -C sffft_amd -f ops.mk` first")
    out = [(re.search(pattern, name).groups(), r) for name, r in rep.items() if re.search(pattern, name)]
    assert out
    return out


def test_march_kernels():
    # march_kernel<T, TO, K, V, writes outputs, planes>
    for (t, k, v, out), r in kernels("linattn", r"march_kernelI([ft])[ft]Li(\d+)ELi(\d+)ELb([01])"):
        groups = 3 if int(k) <= 64 and v == "64" else 2
        assert int(r["Occupancy"]) >= groups, (t, k, v, out)
        assert int(r["VGPRs Spill"]) <= (24 if v == "128" and out == "1" else 0), (t, k, v, out)
        # workgroups on a CU by its 160 KB of LDS: as many as by the registers
        assert int(r["LDS Size"]) * groups <= 160 * 1024, (t, k, v, out)


def test_norm_kernels():
    # fwd_kernel/bwd_kernel<T, vector, channels a lane, lanes, shifted, with y>; 1024 lanes leave 128 registers each
    for (which, vec, lanes), r in kernels("ops_api", r"(fwd|bwd)_kernelI[ft]Li(\d+)ELi\d+ELi(\d+)E"):
        if int(lanes) <= 512:
            assert int(r["VGPRs Spill"]) == 0, (which, vec, lanes)
            if which == "fwd" and vec != "1" and int(lanes) >= 256:
                assert int(r["Occupancy"]) >= 6, (vec, lanes)  # what the count of its workgroups assumes


def test_the_others_do_not_spill():
    for objects, pattern in (("linattn", r"(step|scan|head_sum)_kernel"), ("ops_api", r"(rotary|sum)_kernel")):
        for name, r in kernels(objects, pattern):
            assert int(r["VGPRs Spill"]) == 0 and int(r["ScratchSize"]) == 0, name
