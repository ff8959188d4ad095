"""Calls of several launches over one workspace (no GPU: the source is looked at). Host threads that call on one stream
share a workspace, and kernels of one's call must not come between those of another's."""

from __future__ import annotations

import re

import pytest

from dominusultra_b200 import build

HELD = "const LaunchOrder order(g_launch_mu);"


def _body(name):
    text = re.sub(r"//[^\n]*", "", (build.CSRC / "du_api.cu").read_text())
    return re.search(r"\nint " + name + r"\([^;{]*\) \{\n(.*?)\n\}\n", text, re.S).group(1)


@pytest.mark.parametrize(
    "name", ["du_extend_paged", "du_paged_compact", "du_decode_paged", "du_prefill", "decode_impl", "decode_kvcache_impl"]
)
def test_launches_over_a_workspace_are_held_together(name):
    body = _body(name)
    assert body.count(HELD) == 1
    assert not re.search(r"\blaunch_\w+(<[^;]*?>)?\(", body[: body.index(HELD)])
    assert re.search(r"\blaunch_\w+(<[^;]*?>)?\(", body[body.index(HELD) :])
