"""Kernels that start beside the kernel before them and read its output by TMA (no GPU).

A wait for that kernel makes its writes visible to ordinary loads. TMA reads through another proxy, and
needs a proxy fence between the two. Nothing goes wrong visibly without one, so the sources are looked at."""

from __future__ import annotations

import re

import pytest

from dominusultra_b200 import build

WAIT = re.compile(r"griddep_wait\(\);")
FENCED = re.compile(r"griddep_wait\(\);\s*(?:if \([^;]*\) )?fence_proxy_async_global\(\);")


def _kernels():
    found = []
    for path in build.sources():
        text = re.sub(r"//[^\n]*", "", path.read_text())
        parts = re.split(r"__global__", text)[1:]
        for part in parts:
            name = re.search(r"(\w+_kernel)\(", part).group(1)
            if re.search(r"tma_load_\dd\(|bulk_load\(", part) and WAIT.search(part):
                found.append((f"{path.name}:{name}", part))
    return found


def test_there_are_such_kernels():
    names = [n for n, _ in _kernels()]
    for want in ("decode_kernel", "decode_tc_kernel", "decode_paged_kernel", "prefill_fa_kernel", "prefill_fa1_kernel"):
        assert any(n.endswith(":" + want) for n in names), (want, names)


@pytest.mark.parametrize("name,body", _kernels(), ids=[n for n, _ in _kernels()])
def test_the_wait_is_followed_by_a_proxy_fence(name, body):
    assert len(WAIT.findall(body)) == len(FENCED.findall(body))
