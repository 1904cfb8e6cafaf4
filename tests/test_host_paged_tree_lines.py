"""The lines of a tree in LDS, from the assembly of ``paged_decode.hip`` as it is built.

In the kernel of few rows all four waves of a workgroup resolve the tree and store the same words, with no barrier before they are read.  That holds only if a word is
stored once, with its final value: a line that is stored whole and then cut to its window in a loop is, for a while, another one, and a slower wave puts it back
behind a faster one that reads it already."""
import os
import re
import subprocess

import pytest

from ultraattn_amd.build import CSRC, HIPCC_FLAGS, hipcc_path


@pytest.fixture(scope="module")
def few_rows_of_trees(tmp_path_factory):
    """{kernel: basic blocks, in order, as (label, instructions)}"""
    out = tmp_path_factory.mktemp("asm") / "paged_decode.s"
    try:
        r = subprocess.run([hipcc_path(), *HIPCC_FLAGS, "--cuda-device-only", "-S", os.path.join(CSRC, "paged_decode.hip"), "-o", str(out)], capture_output=True, text=True)
    except FileNotFoundError:
        pytest.skip("no hipcc")
    assert r.returncode == 0, r.stderr
    kernels = {}
    for m in re.finditer(r"^(_ZN2ua16paged_few_kernel\w*Lb1E\w*):.*?^\.Lfunc_end", out.read_text(), flags=re.M | re.S):
        parts = re.split(r"^(\.LBB\w+|; %bb\.\d+):.*$", m.group(0), flags=re.M)
        kernels[m.group(1)] = [(label, re.findall(r"^[ \t]+([a-z]\w+)[ \t]*(.*)$", body, flags=re.M)) for label, body in zip(parts[1::2], parts[2::2])]
    return kernels


def loops(blocks):
    """Runs of blocks from a label to a branch back to it."""
    place = {label: i for i, (label, _) in enumerate(blocks)}
    for i, (_, instructions) in enumerate(blocks):
        for op, args in instructions:
            if "branch" in op and place.get(args.strip(), i + 1) <= i:
                yield [x for _, block in blocks[place[args.strip()]:i + 1] for x in block]


def test_no_loop_before_the_walk_stores_to_lds(few_rows_of_trees):
    assert len(few_rows_of_trees) == 8
    for kernel, blocks in few_rows_of_trees.items():
        found = list(loops(blocks))
        assert any("mfma" in op for loop in found for op, _ in loop) and any("bpermute" in op for loop in found for op, _ in loop), kernel       # the walk; the branches
        for loop in found:
            if not any("mfma" in op for op, _ in loop):
                assert not [op for op, _ in loop if op.startswith(("ds_write", "ds_store"))], kernel
