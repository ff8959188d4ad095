"""Prefills and decodes of several sizes from several host threads on one stream, which share its workspaces (GPU)."""

from __future__ import annotations

import threading

import pytest
import torch

from dominusultra_b200 import _lib, dominus_ultra_decode, dominus_ultra_decode_kvcache, dominus_ultra_prefill, precompute_rope_cos_sin

pytestmark = pytest.mark.gpu


def _prefill(B, Hq, Hkv, T, D, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    q, k, v = (torch.randn(B, h, T, D, generator=g, device="cuda").bfloat16() for h in (Hq, Hkv, Hkv))
    cos, sin = precompute_rope_cos_sin(T, D, "cuda", torch.bfloat16)
    return lambda: dominus_ultra_prefill(q, k, v, cos, sin, Hkv)[0]


def _decode(B, Hq, Hkv, L, D, seed, lens=None):
    g = torch.Generator(device="cuda").manual_seed(seed)
    q = torch.randn(B, Hq, 1, D, generator=g, device="cuda").bfloat16()
    k, v = (torch.randn(B, Hkv, L, D, generator=g, device="cuda").bfloat16() for _ in range(2))
    cos, sin = precompute_rope_cos_sin(L + 1, D, "cuda", torch.bfloat16)
    if lens is None:
        return lambda: dominus_ultra_decode(q, k, v, cos, sin, Hkv)
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    return lambda: dominus_ultra_decode_kvcache(q, k, v, cos, sin, n, num_kv_heads=Hkv)


@pytest.mark.parametrize("kind", ["prefill", "decode", "decode_kvcache"])
def test_from_threads_on_one_stream(cuda_device, kind):
    _lib.read_status(reset=True)
    if kind == "prefill":
        calls = [_prefill(1, 8, 2, 3000, 64, 1), _prefill(2, 4, 4, 777, 128, 2), _prefill(1, 2, 1, 5000, 32, 3)]
    elif kind == "decode":
        calls = [_decode(1, 8, 2, 20000, 64, 1), _decode(2, 8, 8, 9000, 128, 2), _decode(1, 4, 1, 40000, 32, 3), _decode(3, 6, 2, 7000, 256, 4)]
    else:
        calls = [_decode(2, 8, 2, 20000, 64, 1, [20000, 77]), _decode(5, 8, 8, 4000, 128, 2, [1, 4000, 300, 0, 2222]), _decode(1, 4, 1, 30000, 32, 3, [29000])]
    want = [f() for f in calls]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        got = []
        for j in range(120):
            at = (i * 5 + j) % len(calls)
            got.append((at, calls[at]()))
            if len(got) == 12:
                bad.extend(n for n, x in got if not torch.equal(x, want[n]))
                got.clear()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad
    assert _lib.read_status(reset=True)[0] == 0
