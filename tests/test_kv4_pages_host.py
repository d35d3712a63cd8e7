"""Pages of a 4-bit cache at the largest, on the CPU: what is refused before a launch."""

from qsa_vllm_amd import _lib

from .test_paged_host import _attention


def test_a_page_past_64_gib_is_refused():
    """A cache of one block has no block stride that could speak for it."""
    change = dict(blocks=1, kb=0, kh=0, hkv=1, width=1, window=64)
    for page, dim in ((1 << 29, 128), (1 << 30, 64), ((1 << 36) // 144 + 1, 128)):
        assert _lib.load().qsa_kv4_page_bytes(page, dim) >= 1 << 36
        assert _attention("qsa_int4_kv_attention", page=page, dim=dim, **change) == -2
        assert b"64 GiB" in _lib.load().qsa_last_error()
    # Neither has one whose blocks lie between another head's.
    assert _attention("qsa_int4_kv_attention", page=1 << 28, blocks=2, kb=1 << 35, kh=1 << 20) == -2
