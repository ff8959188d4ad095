"""Shared memory that a launch sizes begins where its type wants it, and behind the kernel's own: a kernel that takes it in
larger pieces says so (no GPU: the sources are looked at)."""

from __future__ import annotations

import re

import pytest

from dominusultra_b200 import build

WIDE = re.compile(r"uint4|int4|float4|\bv4\b|uint2|int2\b|float2|cluster_load4|join_slices")


def _kernels():
    for path in build.sources():
        text = re.sub(r"//[^\n]*", "", path.read_text())
        for part in (x.split("\n}\n")[0] for x in text.split("__global__")[1:]):
            array = re.search(r"extern __shared__ (?:__align__\((\d+)\) )?(\w+) (\w+)\[\];", part)
            if array:
                yield path.name + ":" + re.search(r"(\w+_kernel)\(", part).group(1), part, array


@pytest.mark.parametrize("body,array", [pytest.param(b, a, id=n) for n, b, a in _kernels()])
def test_wide_accesses_are_aligned(body, array):
    align, kind, name = array.groups()
    by_hand = re.search(name + r"\w*.{0,40}\n?.*\+ (127|1023)u?\) & ~", body)  # (rounded up to where a TMA tile begins)
    if int(align or 4) < 16 and not by_hand:
        assert kind in ("int", "float", "uint32_t") and not WIDE.search(body), name


def test_there_are_such_kernels():
    assert {n.split(":")[1] for n, *_ in _kernels()} >= {"paged_fork_kernel", "paged_compact_kernel", "extend_paged_kernel", "paged_tables_kernel"}
