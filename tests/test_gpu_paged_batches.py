"""Attention over the paged cache: requests in any order, and each way of sharing out
prompt chunks (tolerance: ``paged_cases``)."""

import pytest
import torch

from .paged_cases import DEV, Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("ctx,new,heads,kv_heads,dim,window,sinks", [
    ([3000, 50, 700, 0, 2100, 333], [1, 2, 1, 1, 1, 2], 16, 2, 128, None, 0),      # pieces of few rows
    ([int(61 * i % 2900) for i in range(90)], [1] * 88 + [0, 1], 8, 2, 64, None, 0),
    ([2000, 3000, 90, 1200], [20, 33, 17, 70], 8, 1, 128, None, 0),                # pieces of tiles
    ([2500, 100, 1800, 0, 900], [1, 150, 1, 60, 2], 16, 2, 128, 900, 5),           # both
    ([400, 300, 200, 0], [64, 64, 64, 64], 4, 2, 64, 150, 3),                      # alike chunks
])
def test_same_bits_in_any_order_of_requests(ctx, new, heads, kv_heads, dim, window, sinks, bits):
    """Each request's rows are the same bits wherever it stands in the call."""
    c = Case(ctx, new, heads, kv_heads, dim, window=window, sinks=sinks, gate=True, bits=bits,
             seed=len(ctx))
    first, cache = c.run(), c.device_cache()
    c.check(first)
    own = [slice(c.starts[b], c.starts[b + 1]) for b in range(len(ctx))]
    orders = [list(reversed(range(len(ctx))))]
    orders += [torch.randperm(len(ctx), generator=c.gen).tolist() for _ in range(3)]
    q, gate = c.q, c.gate
    for order in orders:
        assert order != sorted(order)
        c.gate = torch.cat([gate[own[b]] for b in order])
        starts = torch.tensor([0] + [new[b] for b in order]).cumsum(0).to(torch.int32)
        got = c.run(q=torch.cat([q[own[b]] for b in order]).to(DEV), table=c.table[order],
                    lens=torch.tensor([c.lens[b] for b in order], dtype=torch.int32, device=DEV),
                    qsl=starts.to(DEV), cache=cache)
        assert torch.equal(got, torch.cat([first[own[b]] for b in order]))


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("ctx,new,heads,kv_heads,dim", [
    ([900], [150], 4, 2, 128),             # a chunk on four times its tokens and more
    ([1300], [70], 8, 2, 64),
    ([2000, 2100], [130, 130], 2, 1, 128),     # two such
    ([1000, 700, 400, 100], [140, 140, 140, 139], 2, 1, 128),   # chunks of almost one length
    ([300, 0], [140, 1], 4, 1, 64),            # a chunk beside a single token
])
def test_chunks_of_prompts(ctx, new, heads, kv_heads, dim, bits):
    c = Case(ctx, new, heads, kv_heads, dim, gate=True, bits=bits, seed=sum(new))
    c.check(c.run())
    c.check(c.run(max_seq_len=40000))
    table = c.table.clone()
    table[:, 2::7] = -1
    c.check(c.run(table=table), table=table)
