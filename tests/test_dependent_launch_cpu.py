"""Kernels that are launched while the kernel before them still runs (launch_dependent in
common.cuh) must not read through the read-only path, which is for memory that nobody
writes while the kernel lives: no __ldg, no ld.global.nc, no const __restrict__ pointers, from
which the compiler makes the same loads."""
import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "obsidian-memory-transformer_b200" / "csrc"
CODE = {f.name: re.sub(r"//[^\n]*|/\*.*?\*/", "", f.read_text(), flags=re.S)
        for f in CSRC.glob("*.cu")}
FILES = sorted(n for n, s in CODE.items() if "launch_dependent(" in s)


def kernels(s):
    """Names launched by launch_dependent, by themselves or through a variable."""
    names = set(re.findall(r"launch_dependent\(\s*([a-z_]+kernel)", s))
    for var in re.findall(r"launch_dependent\(\s*([a-z]+),", s):
        names |= set(re.findall(rf"auto {var} = ([a-z_]+kernel)", s))
    return names


def test_there_are_such_kernels():
    assert {k for n in FILES for k in kernels(CODE[n])} >= {
        "cache_append_kernel", "cache_read_kernel", "cache_reorder_kernel", "beam_chunk_kernel",
        "beam_merge_kernel", "tree_mma_kernel", "tree_tc_kernel", "tree_combine_kernel"}


@pytest.mark.parametrize("name", FILES)
def test_no_read_only_loads(name):
    s = CODE[name]
    assert "__ldg(" not in s and "ld.global.nc" not in s
    for k in kernels(s):
        params = re.search(rf"\b{k}\(((?:[^()]|\([^()]*\))*)\)\s*{{", s)
        assert params, k
        for p in params.group(1).split(","):
            assert not ("const" in p.split("*")[0] and "__restrict__" in p), (k, p.strip())
