"""Which sizes of attention over the paged cache reach the launch, on the CPU: where a
machine has no GPU the launch itself then fails, with a status of its own."""

import pytest
import torch

from qsa_vllm_amd import _lib

from .test_paged_host import _attention

HIP, UNSUPPORTED = -3, -2
NAMES = ["qsa_window_attention", "qsa_int4_kv_attention"]


@pytest.mark.skipif(torch.cuda.is_available(), reason="the addresses are no tensors'")
@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("change", [
    dict(rows=1 << 20, hq=16, most=1 << 20),                                  # one long prompt
    dict(rows=4096 * 16, requests=4096, hq=64, hkv=64, dim=64, most=16),      # few rows, not joined
    dict(rows=(1 << 26) - 1, hq=16, hkv=1, dim=64, most=1 << 26),             # 2^30 (row, head)s
    dict(rows=1 << 22, requests=1 << 22, hq=1, hkv=1, most=1),                # as many single tokens
    dict(rows=(1 << 23) + 99, requests=1 << 22, hq=2, hkv=1, most=100),       # and chunks beside them
])
def test_sizes_that_are_launched(name, change):
    assert _attention(name, **change) == HIP
    assert b"launch" in _lib.load().qsa_last_error()


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("change", [
    dict(rows=1 << 26, hq=16, hkv=1, dim=64, most=1 << 26),
    dict(rows=1 << 24, requests=1 << 24, hq=1, hkv=1, most=1),     # 2^32 threads of few rows
    dict(rows=1 << 23, requests=1 << 23, hq=68, hkv=4, most=1),    # the same of tiles
])
def test_sizes_past_the_largest(name, change):
    assert _attention(name, **change) == UNSUPPORTED
    assert b"too many" in _lib.load().qsa_last_error()


def test_a_join_past_the_largest():
    """Rows of no request count where pieces are joined: a launch over all rows."""
    f = _lib.load().qsa_paged_attention_workspace_bytes
    args = dict(rows=1 << 24, hq=20, hkv=1, dim=128, most=100, longest=1 << 20)
    need = f(1 << 24, 1, 20, 1, 128, 0, 0, 100, 1 << 20)
    assert need > 0
    for name in NAMES:
        assert _attention(name, ws=16, ws_bytes=need, **args) == UNSUPPORTED


def test_more_requests_than_rows():
    """A join counts all requests, of rows or not, in 64 bits."""
    args = dict(rows=8, requests=1 << 29, hq=4, hkv=2, most=8, longest=1 << 20)
    need = _lib.load().qsa_paged_attention_workspace_bytes(8, 1 << 29, 4, 2, 128, 0, 0, 8, 1 << 20)
    assert need > 0
    for name in NAMES:
        assert _attention(name, ws=16, ws_bytes=need, **args) == UNSUPPORTED
