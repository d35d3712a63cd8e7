"""Attention over the paged cache in calls of very many rows and requests: a small case,
held against 64 bits (tolerance: ``paged_cases``), over and over."""

import pytest
import torch

from .paged_cases import DEV, Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [16, 4])
def test_a_million_rows(bits):
    """A prompt of 2^20 tokens whose pages, and queries, come again every 1024: past the
    first window every row's result is that of the row 1024 before."""
    n, times = 1024, 1024
    c = Case([0], [n], heads=16, kv_heads=1, dim=64, window=64, bits=bits)
    q = c.q.to(DEV).repeat(times, 1, 1)
    got = c.run(q=q, table=c.table.repeat(1, times),
                lens=torch.tensor([n * times], dtype=torch.int32, device=DEV),
                qsl=torch.tensor([0, n * times], dtype=torch.int32, device=DEV),
                max_query_len=n * times, max_seq_len=n * times).view(times, n, 16, 64)
    c.check(got[0])
    assert torch.equal(got[0, 64:], got[1, 64:])
    for i in range(2, times, 64):
        part = got[i:i + 64]
        assert torch.equal(part, got[1:2].expand_as(part))


@pytest.mark.parametrize("bits", [16, 4])
def test_many_requests_of_a_few_rows(bits):
    """4096 requests of 16 rows of 64 heads each, all over the same pages."""
    times = 4096
    c = Case([21], [16], heads=64, kv_heads=64, dim=64, bits=bits)
    q = c.q.to(DEV).repeat(times, 1, 1)
    got = c.run(q=q, table=c.table.repeat(times, 1),
                lens=torch.full((times,), c.lens[0], dtype=torch.int32, device=DEV),
                qsl=torch.arange(0, 16 * times + 1, 16, dtype=torch.int32, device=DEV))
    got = got.view(times, 16, 64, 64)
    c.check(got[0])
    for i in range(0, times, 256):
        assert torch.equal(got[i:i + 256], got[:1].expand(256, -1, -1, -1))
