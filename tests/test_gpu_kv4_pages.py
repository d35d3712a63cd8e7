"""A 4-bit cache of one page whose words lie past 2^31 bytes of them: rows written and
read there, as in a cache of small pages."""

import pytest
import torch

from qsa_vllm_amd.ops import Int4KVCache, qk_norm_rope, qsa_int4_paged_attention

from .paged_cases import DEV

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bad", [False, True])
@pytest.mark.parametrize("new", [1, 3, 40])
def test_a_page_of_2_to_the_28_tokens(new, bad):
    """The first tokens (sinks), and 100 about position 2^28; beside it the same tokens at
    positions as far from a multiple of 64. ``bad``: one group of V has no code."""
    gen = torch.Generator().manual_seed(new)
    kv = torch.randn(104, 1, 256, generator=gen).bfloat16().to(DEV)
    if bad:
        kv[64, 0, 128 + 70] = float("inf")
    q = torch.randn(new, 4, 128, generator=gen).bfloat16().to(DEV)
    page = (1 << 28) + 64
    big = Int4KVCache(torch.empty(1, 1, Int4KVCache.page_bytes(page, 128), dtype=torch.uint8,
                                  device=DEV), page, 128)
    small = Int4KVCache.allocate(16, 16, 1, 128, DEV)
    results = []
    for cache, middle in ((big, 1 << 28), (small, 128)):
        slots = torch.cat((torch.arange(4), torch.arange(middle - 50, middle + 50))).to(DEV)
        held = [torch.empty(104, 1, 128, dtype=torch.bfloat16, device=DEV) for _ in range(2)]
        qk_norm_rope(None, kv[..., :128], None, None, None, None, 1e-6, value=kv[..., 128:],
                     cache=cache, slot_mapping=slots, k_out=held[0], v_out=held[1])
        table = torch.arange(-(-(middle + 50) // cache.page_size), dtype=torch.int32, device=DEV)[None]
        got = qsa_int4_paged_attention(
            q, cache, table, torch.tensor([middle + 50], dtype=torch.int32, device=DEV),
            torch.tensor([0, new], dtype=torch.int32, device=DEV), window=50, sink_tokens=3,
            max_query_len=new, max_seq_len=1 << 29)
        results.append((got, *held))
    nan = torch.zeros(new, 4, 128, dtype=torch.bool, device=DEV)
    nan[max(0, new - 40):, :, 64:96] = bad
    assert torch.equal(torch.isnan(results[0][0]), nan)
    for a, b in zip(*results):
        assert torch.equal(torch.nan_to_num(a, 77.0), torch.nan_to_num(b, 77.0))
