"""What the sliding-window, rotary and joining kernels ask of the device: no registers in memory, no private segment, and the backward's two workgroups a CU."""
import os
import re
import subprocess

import pytest

from ultraattn_amd.build import CSRC, HIPCC_FLAGS, hipcc_path

SOURCES = ["swa_fwd.hip", "swa_bwd.hip", "swa_decode.hip", "rope.hip", "rows.hip"]


@pytest.fixture(scope="module")
def kernels(tmp_path_factory):
    """{kernel: {field: value}} of all sources."""
    out = tmp_path_factory.mktemp("asm")
    try:
        runs = [(out / f"{s}.s", subprocess.Popen([hipcc_path(), *HIPCC_FLAGS, "--cuda-device-only", "-S", os.path.join(CSRC, s), "-o", str(out / f"{s}.s")],
                                                  stdout=subprocess.DEVNULL, stderr=subprocess.DEVNULL)) for s in SOURCES]
    except FileNotFoundError:
        pytest.skip("no hipcc")
    found = {}
    for path, run in runs:
        assert run.wait() == 0, path
        for k in re.findall(r"^ +- \.agpr_count:.*?\.wavefront_size", path.read_text(), flags=re.M | re.S):
            found[re.search(r"\.name:\s*(\w+)", k).group(1)] = {f: int(re.search(rf"\.{f}:\s*(\d+)", k).group(1)) for f in (
                "vgpr_count", "vgpr_spill_count", "sgpr_spill_count", "private_segment_fixed_size", "group_segment_fixed_size")}
    return found


def test_nothing_spills(kernels):
    assert sum("swa_bwd_kernel" in k for k in kernels) == 4 and sum("swa_fwd_kernel" in k for k in kernels) == 4 and sum(bool(re.search(r"\d+rows_\w+_kernel", k)) for k in kernels) == 16
    for name, k in kernels.items():
        assert k["vgpr_spill_count"] == k["sgpr_spill_count"] == k["private_segment_fixed_size"] == 0, (name, k)


def test_two_workgroups_share_a_cu(kernels):
    """Of 512 vector registers a lane and 160 KiB of LDS, with one wave of a workgroup on each of a CU's four SIMDs."""
    for name, k in kernels.items():
        if "swa_fwd_kernel" in name or "swa_bwd_kernel" in name:
            assert k["vgpr_count"] <= 256 and k["group_segment_fixed_size"] <= 80 << 10, (name, k)
            if "Li64E" in name:
                assert k["vgpr_count"] <= 168 and k["group_segment_fixed_size"] <= (160 << 10) // 3, (name, k)
