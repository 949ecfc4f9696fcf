"""The kernels over a paged cache in the library that is built: those that read fragments through inline assembly with counted waits
spill nothing, and what is meant to run beside others fits."""
import importlib
import json
import os

import pytest

B = importlib.import_module("fgrpo.build")


@pytest.fixture(scope="module")
def usage():
    path = os.path.join(B.CSRC, "resource_usage.json")
    if not (os.path.exists(path) and os.path.exists(B.LIB_PATH)):
        B.build(verbose=False)
    with open(path) as f:
        return json.load(f)["kernels"]


@pytest.mark.parametrize("family", ["paged_tiles_kernel", "paged_rows_kernel", "paged_rows16_kernel"])
@pytest.mark.parametrize("shape", ["ILi128ELb0E", "ILi128ELb1E", "ILi64ELb0E", "ILi64ELb1E"])
def test_attention_kernels_keep_their_registers(usage, family, shape):
    found = [u for name, u in usage.items() if family + shape in name]
    assert len(found) == 1
    assert found[0]["vgpr_spill"] == 0 and found[0]["scratch"] == 0 and found[0]["agprs"] == 0 and found[0]["vgprs"] <= 256
    # work-groups a CU of 160 KiB of LDS: two of tiles, four of one wavefront
    assert found[0]["lds"] * (2 if family == "paged_tiles_kernel" else 4) <= 160 * 1024


def test_guard_knows_them():
    name = "_ZN5fgrpoL18paged_tiles_kernelILi128ELb1EEEvNS_9PagedAttnENS_10PagedSplitE"
    clean = dict(sgprs=96, vgprs=250, agprs=0, scratch=0, occupancy=2, sgpr_spill=90, vgpr_spill=0, lds=70000)
    assert not any(name in x for x in B.check_resource_usage({name: clean}))
    assert any(name in x for x in B.check_resource_usage({name: dict(clean, vgpr_spill=1, scratch=8)}))
