"""What the paged cache's kernels ask of the device: no registers in memory, no private segment, and where they are meant to, two workgroups a CU."""
import os
import re
import subprocess

import pytest

from ultraattn_amd.build import CSRC, HIPCC_FLAGS, hipcc_path


@pytest.fixture(scope="module")
def kernels(tmp_path_factory):
    """{kernel: {field: value}}"""
    out = tmp_path_factory.mktemp("asm")
    try:
        runs = [(out / f"{s}.s", subprocess.Popen([hipcc_path(), *HIPCC_FLAGS, "--cuda-device-only", "-S", os.path.join(CSRC, s), "-o", str(out / f"{s}.s")],
                                                  stdout=subprocess.DEVNULL, stderr=subprocess.DEVNULL)) for s in ("paged_decode.hip", "paged_keep.hip")]
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
    assert sum("paged_few_kernel" in k for k in kernels) == 16 and sum("paged_many_kernel" in k for k in kernels) == 8
    assert sum("paged_join_kernel" in k for k in kernels) == 4 and sum("paged_keep_kernel" in k for k in kernels) == 3
    for name, k in kernels.items():
        assert k["vgpr_spill_count"] == k["sgpr_spill_count"] == k["private_segment_fixed_size"] == 0, (name, k)


def test_two_workgroups_share_a_cu(kernels):
    """Of 512 vector registers a lane and 160 KiB of LDS, with one wave of a workgroup on each of a CU's four SIMDs; few rows of 128 entries fill it with one."""
    for name, k in kernels.items():
        if "paged_many_kernel" in name or ("paged_few_kernel" in name and "Li64E" in name):
            assert k["vgpr_count"] <= 256 and k["group_segment_fixed_size"] <= 80 << 10, (name, k)
        assert k["group_segment_fixed_size"] <= 160 << 10, (name, k)


def test_three_workgroups_of_many_rows_of_64_share_a_cu(kernels):
    """Three waves a SIMD have 168 registers each (of 512 in eights)."""
    found = [k for name, k in kernels.items() if "paged_many_kernel" in name and "Li64E" in name]
    assert len(found) == 4
    for k in found:
        assert k["vgpr_count"] <= 168 and 3 * k["group_segment_fixed_size"] <= 160 << 10, k
