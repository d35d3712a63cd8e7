"""Windowed attention and attention over a 4-bit cache on the GPU against a 64-bit
statement of them, row by row (tolerance: ``paged_cases``)."""

import numpy as np
import pytest
import torch

from qsa_vllm_amd.ops import (Int4KVCache, qsa_int4_paged_attention, qsa_sparse_paged_attention,
                              qsa_tree_paged_attention, qsa_window_paged_attention, tree_ancestors)

from .paged_cases import DEV, Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("ctx,new,heads,kv_heads,page,window,sinks", [
    ([0], [1], 1, 1, 16, None, 0),                    # the token itself is all there is
    ([1], [1], 8, 1, 16, 1, 0),                       # a window of the token itself
    ([37], [5], 4, 2, 16, 3, 2),                      # under one stage
    ([127, 128, 126, 63, 64], [1] * 5, 16, 2, 16, None, 0),   # single tokens about stages' ends
    ([127, 128, 126, 300], [1] * 4, 16, 2, 16, 64, 1),
    ([300], [3], 16, 2, 272, 100, 4),
    ([64, 0, 63, 200], [2, 4, 1, 7], 8, 4, 48, 65, 3),
    ([500, 20], [8, 8], 16, 2, 16, 128, 130),         # sinks over several stages
    ([130, 700, 0], [17, 33, 90], 4, 1, 16, 200, 5),  # several tiles
    ([90], [64], 8, 1, 1, 70, 1),                     # pages of one token
    ([0, 5, 2], [40, 0, 70], 6, 2, 16, 33, 0),        # an empty request
    ([33], [100], 3, 3, 16, None, 0),                 # no sharing of kv heads
    ([0], [300], 16, 1, 16, 90, 10),                  # a prompt of many tiles
    ([200], [1], 40, 1, 16, 150, 2),                  # more query heads than a tile's rows
    ([5, 9], [3, 1], 4, 2, 16, 1000, 1000),           # window and sinks past everything
])
def test_matches_64_bits(ctx, new, heads, kv_heads, page, window, sinks, dim, bits):
    print(ctx, new, heads, kv_heads, page, window, sinks, dim, bits, flush=True)
    c = Case(ctx, new, heads, kv_heads, dim, page, window, sinks, gate=len(ctx) % 2 == 1,
             seed=sum(ctx) + dim, bits=bits)
    c.check(c.run())


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("max_seq_len", [5000, 0, 100000])
@pytest.mark.parametrize("new,window,sinks", [
    ([1, 1, 1], None, 0), ([1, 2, 1], 1500, 70), ([9, 2, 20], None, 0), ([12, 64, 1], 2000, 4)])
def test_long_contexts_split(new, window, sinks, max_seq_len, bits):
    """Several pieces a request, of ragged lengths; the bound on the length only shapes
    the launch."""
    c = Case([4000, 17, 1999], new, heads=8, kv_heads=2, window=window, sinks=sinks, gate=True,
             seed=max_seq_len + sum(new), bits=bits)
    c.check(c.run(max_seq_len=max_seq_len))


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("ctx,new", [([5000], [1]), ([600] * 70, [1] * 70),
                                     ([100, 900, 30, 2000], [1, 1, 130, 60]),
                                     ([700] * 3, [40] * 3)])
def test_batches(ctx, new, bits):
    """Many requests, single tokens and chunks in one call."""
    c = Case(ctx, new, heads=16, kv_heads=2, window=700, sinks=4, seed=len(ctx), bits=bits)
    c.check(c.run())


@pytest.mark.parametrize("bits,layout", [(16, "head_major"), (16, "separate"), (4, "strided")])
def test_layouts(bits, layout):
    c = Case([300, 40], [3, 70], heads=8, kv_heads=2, window=120, sinks=3, bits=bits, layout=layout)
    c.check(c.run())


@pytest.mark.parametrize("bits", [16, 4])
def test_strided_rows_gate_and_out(bits):
    """Queries and gates interleaved by head, as a projection leaves them; out a view."""
    c = Case([300, 40, 9], [1, 7, 1], heads=4, kv_heads=2, window=120, sinks=3, gate=True, bits=bits)
    rows = c.starts[-1]
    both = torch.cat((c.q, c.gate), -1).to(DEV)
    out = torch.full((rows, 4, 2 * 128), 7.0, dtype=torch.bfloat16, device=DEV)
    call = qsa_int4_paged_attention if bits == 4 else qsa_window_paged_attention
    cache = c.device_cache()
    got = call(both[..., :128], *((cache,) if bits == 4 else cache), c.table.to(DEV),
               torch.tensor(c.lens, dtype=torch.int32, device=DEV), c.qsl.to(DEV), out[..., 128:],
               window=120, sink_tokens=3, output_gate=both[..., 128:], max_query_len=7,
               max_seq_len=309)
    c.check(got)
    assert (out[..., :128] == 7).all()
    # A gate whose dims are not contiguous, and one value for a whole head.
    c.gate = c.gate[..., :1].expand(-1, -1, 128)
    c.check(c.run())
    wide = torch.randn(rows, 4, 128, 3, generator=c.gen).bfloat16()
    c.gate = wide[..., 1]
    c.check(c.run())


@pytest.mark.parametrize("bits", [16, 4])
def test_rows_of_no_request_stay(bits):
    c = Case([100, 30], [3, 40], window=50, sinks=2, bits=bits)
    rows = c.starts[-1]
    q = torch.cat((c.q, c.q[:9])).to(DEV)
    out = torch.full(q.shape, 3.0, dtype=torch.bfloat16, device=DEV)
    got = c.run(out=out, q=q)
    c.check(got[:rows])
    assert (got[rows:] == 3).all()
    # Rows past the announced most are not computed either; the others keep their positions.
    out.fill_(3.0)
    got = c.run(out=out, max_query_len=33)
    c.check(torch.cat((got[:36], c.run()[36:])))
    assert (got[36:rows] == 3).all()


@pytest.mark.parametrize("bits", [16, 4])
def test_freed_and_missing_pages(bits):
    """Pages that left every window may be taken away; pages that are missing inside it,
    or whose entry is no block, are not seen."""
    c = Case([900, 400, 64], [1, 3, 1], heads=8, window=200, sinks=20, bits=bits)
    full = c.run()
    table = c.table.clone()
    table[0, 2:43] = -1       # positions 32 .. 687 of a row that sees 0 .. 19 and 701 on
    table[1, 2:12] = 1 << 30
    got = c.run(table=table)
    assert torch.equal(got, full)
    table[0, 50] = -7
    table[1, 24:] = -1        # the rows' own pages too
    table[2] = -1             # nothing left at all
    got = c.run(table=table)
    c.check(got, table=table)
    assert (got[4] == 0).all()


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("ctx,new,heads,kv_heads,dim,page,window,sinks", [
    ([50, 2000, 0, 700, 3, 4100, 90], [1, 40, 1, 2, 300, 1, 0], 16, 2, 128, 16, 600, 3),
    ([900, 5000, 17], [1, 1, 200], 8, 1, 64, 48, None, 0),       # a long piece beside tiles
    ([3000, 0, 64], [3, 129, 20], 4, 4, 64, 16, None, 0),        # heads of their own
    ([700, 800], [1, 33], 16, 1, 128, 272, 300, 70),             # 16 heads: one row is all of a few
    ([10, 20], [2, 5], 20, 1, 128, 16, None, 0),                 # 20 heads: none is of few rows
    ([int(37 * i % 1500) for i in range(70)], [1] * 66 + [0, 30, 2, 5], 16, 2, 128, 16, None, 0),
])
def test_steps_of_both(ctx, new, heads, kv_heads, dim, page, window, sinks, bits):
    """Chunks and single tokens in one call: tiles and few rows side by side, pieces of
    both, more requests than lanes, empty ones among them."""
    print(ctx[:7], new[:7], heads, kv_heads, dim, page, window, bits, flush=True)
    c = Case(ctx, new, heads, kv_heads, dim, page, window, sinks, gate=True, seed=sum(new), bits=bits)
    c.check(c.run())
    table = c.table.clone()       # and with pages missing from all of them
    table[:, 1::5] = -1
    c.check(c.run(table=table), table=table)


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("requests,heads,dim", [(1, 16, 128), (1, 8, 64), (20, 16, 128), (150, 16, 64)])
def test_single_tokens_in_pieces(requests, heads, dim, bits):
    """Each way of joining pieces, by the number of heads in the call."""
    gen = torch.Generator().manual_seed(requests)
    ctx = torch.randint(1500, 3000, (requests,), generator=gen).tolist()
    c = Case(ctx, [1] * requests, heads, 2, dim, gate=True, seed=heads, bits=bits)
    c.check(c.run(max_seq_len=max(c.lens)))


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("new", [[1], [2], [1, 50]])
def test_values_that_are_not_finite_in_pieces(new, bits):
    """V of a token that all rows see, in a whole block and in the last one: its dims and
    no others, whichever piece holds it. In the last row's own token: that row alone."""
    c = Case([3000, 2500][:len(new)], new, heads=8, kv_heads=2, bits=bits, seed=8)
    clean = c.run()
    for pos in (700, c.lens[0] - new[0] - 1, c.lens[0] - 1):
        block, place = int(c.table[0, pos // 16]), pos % 16
        saved, words = c.kv.clone(), [w.copy() for w in c.words] if bits == 4 else None
        if bits == 4:
            c.words[1][block, place, 0, 2] = 0x7FC0
        c.kv[block, place, 0, 128 + 64:128 + 96] = float("nan")
        got = c.run()
        c.kv = saved
        if bits == 4:
            c.words = words
        for r in range(c.starts[-1]):
            if r >= new[0] or pos > c.lens[0] - new[0] + r:
                assert torch.equal(got[r], clean[r])
                continue
            assert torch.isnan(got[r, :4, 64:96]).all()
            assert torch.equal(got[r, 4:], clean[r, 4:])
            rest = torch.cat((got[r, :4, :64], got[r, :4, 96:]), -1)
            assert torch.equal(rest, torch.cat((clean[r, :4, :64], clean[r, :4, 96:]), -1))


def test_lengths_that_do_not_fit():
    """Lengths past the table, under the rows, zero and negative: what is there is seen."""
    c = Case([100, 40, 3, 0], [2, 5, 1, 2], heads=4, window=None)
    lens = torch.tensor([5000, 3, 0, -8], dtype=torch.int32, device=DEV)
    got = c.run(lens=lens)
    c.lens = [5000, 3, 0, -8]
    c.kv = torch.nan_to_num(c.kv)      # request 0 sees all of its pages
    got = c.run(lens=lens)
    c.check(got)
    assert (got[c.starts[1]:c.starts[1] + 2] == 0).all() and (got[c.starts[2]:] == 0).all()


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("new,window", [([1, 1], 64), ([40, 3], 64), ([2, 200], 100)])
def test_values_that_are_not_finite_reach_the_rows_that_see_them(new, window, bits):
    """Infinities and NaN in K or V of some tokens: rows outside their windows (before
    them, or after) are untouched."""
    c = Case([200, 150], new, heads=8, kv_heads=2, window=window, sinks=2, bits=bits, seed=3)
    clean = c.run()
    at = [c.lens[0] - new[0] - 3, c.lens[0] - 1, c.lens[0] - 1 - window]
    spots = [(0, at[0], "v"), (0, at[1], "k"), (1, c.lens[1] - new[1] // 2 - 1, "v"),
             (1, c.lens[1] - window, "v"), (1, 1, "v")]
    for b, pos, which in spots:
        block, place = int(c.table[b, pos // 16]), pos % 16
        saved, words = c.kv.clone(), [w.copy() for w in c.words] if bits == 4 else None
        side = 128 if which == "v" else 0
        if bits == 4:
            c.words[int(which == "v")][block, place, 1, 1] = 0x7FC0
            c.kv[block, place, 1, side + 32:side + 64] = float("nan")
            dims = slice(32, 64)
        else:
            c.kv[block, place, 1, side + 40] = float("inf") if pos % 2 else float("nan")
            dims = slice(40, 41)
        got = c.run()
        c.kv = saved
        if bits == 4:
            c.words = words
        for r in range(c.starts[-1]):
            rb = 0 if r < c.starts[1] else 1
            sees = rb == b and pos in c.seen(rb, r - c.starts[rb]).tolist()
            if not sees:
                assert torch.equal(got[r], clean[r]), (b, pos, which, r)
                continue
            assert torch.equal(got[r, :4], clean[r, :4])     # the other kv head
            if which == "v":
                assert not torch.isfinite(got[r, 4:, dims]).any(), (b, pos, r)
                rest = torch.ones(128, dtype=torch.bool)
                rest[dims] = False
                assert torch.isfinite(got[r, 4:, rest]).all()
            elif bits == 4 or pos % 2 == 0:
                assert torch.isnan(got[r, 4:]).all(), (b, pos, r)


def test_scores_of_infinity():
    """A score of plus infinity gives NaN; of minus infinity no weight, and zeros to a row
    that has no other."""
    c = Case([40], [1], heads=2, kv_heads=2, window=None)
    c.q[:] = 1.0
    c.kv[..., 0] = torch.where(torch.isnan(c.kv[..., 0]), c.kv[..., 0], torch.tensor(-float("inf")))
    assert (c.run() == 0).all()
    page = int(c.table[0, 0])
    c.kv[page, 3, :, 0] = 1.0
    got = c.run()
    want = c.kv[page, 3, :, 128:]
    assert torch.equal(got[0].cpu(), want)
    c.kv[page, 5, :, 0] = float("inf")
    assert torch.isnan(c.run()).all()


@pytest.mark.parametrize("bits", [16, 4])
def test_large_scores(bits):
    """Scores that pass the exponents' base again and again, and rows of one weight."""
    c = Case([700], [5], heads=8, kv_heads=2, window=None, bits=bits, scale=6.0, seed=5)
    c.check(c.run())
    c = Case([700], [90], heads=8, kv_heads=2, window=300, sinks=9, bits=bits, scale=6.0, seed=6)
    c.check(c.run())


@pytest.mark.parametrize("bits", [16, 4])
def test_same_bits_again_and_in_any_batch_order(bits):
    c = Case([900, 20, 300], [1, 30, 2], heads=8, window=400, sinks=4, bits=bits)
    first = c.run()
    for _ in range(3):
        assert torch.equal(c.run(), first)


def test_no_window_gives_what_the_siblings_give():
    """The whole context: as tree attention of a chain, and as sparse attention of a list
    of all slots, within both tolerances."""
    c = Case([300, 61], [4, 9], heads=8, kv_heads=2)
    want, tol = c.want()
    got = c.run()
    k, v = c.device_cache()
    parents = torch.tensor([j - 1 for n in c.new for j in range(n)])
    tree = qsa_tree_paged_attention(
        c.q.to(DEV), k, v, c.table.to(DEV), torch.tensor(c.ctx, dtype=torch.int32, device=DEV),
        c.qsl.to(DEV), tree_ancestors(parents, c.qsl, 9).to(DEV), max_query_len=9,
        max_context_len=300)
    assert ((got.double() - tree.double()).abs().cpu() <= 2 * tol).all()
    width = max(c.lens)
    idx = torch.full((c.starts[-1], width), -1, dtype=torch.int32)
    for b in range(2):
        for i in range(c.new[b]):
            j = c.seen(b, i)
            idx[c.starts[b] + i, :len(j)] = j.to(torch.int32)
    req = torch.repeat_interleave(torch.arange(2, dtype=torch.int32), torch.tensor(c.new))
    sparse = torch.empty_like(got)
    qsa_sparse_paged_attention(c.q.to(DEV), k, v, idx.to(DEV), c.table.to(DEV), req.to(DEV), sparse,
                               use_decode_kernel=False, indices_are_physical=False)
    assert ((got.double() - sparse.double()).abs().cpu() <= 2 * tol).all()


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("new", [[1, 1, 1], [3, 40, 1]])
def test_captured_call_follows_its_buffers(new, bits):
    """Lengths, tables, queries and the cache are read anew on every replay."""
    cases = [Case([700, 40, 90], new, heads=8, window=256, sinks=4, gate=True, bits=bits, seed=s)
             for s in (1, 2, 3)]
    for s, c in enumerate(cases[1:]):       # other lengths within the same pages
        c.lens = [n - 5 * (s + 1) for n in c.lens]
        c.ctx = [n - 5 * (s + 1) for n in c.ctx]
    c = cases[0]
    cache = c.device_cache()
    tensors = [cache.data] if bits == 4 else [cache[0]._base if cache[0]._base is not None else cache[0]]
    q, gate, table = c.q.to(DEV), c.gate.to(DEV), c.table.to(DEV)
    lens = torch.tensor(c.lens, dtype=torch.int32, device=DEV)
    qsl, out = c.qsl.to(DEV), torch.zeros(c.q.shape, dtype=torch.bfloat16, device=DEV)
    call = qsa_int4_paged_attention if bits == 4 else qsa_window_paged_attention

    def step():
        call(q, *((cache,) if bits == 4 else cache), table, lens, qsl, out, window=256,
             sink_tokens=4, output_gate=gate, max_query_len=max(new), max_seq_len=1024)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for c in cases + cases[:1]:
        source = c.device_cache()
        source = [source.data] if bits == 4 else [source[0]._base]
        for dst, src in zip(tensors, source):
            dst.copy_(src)
        q.copy_(c.q)
        gate.copy_(c.gate)
        table.copy_(c.table)
        lens.copy_(torch.tensor(c.lens, dtype=torch.int32))
        out.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        c.check(out)


@pytest.mark.parametrize("bits", [16, 4])
def test_calls_on_two_streams(bits):
    """Two calls in flight with partial results each."""
    cases = [Case([3000, 2000], [1, 2], heads=8, seed=s, bits=bits) for s in (1, 2)]
    caches = [c.device_cache() for c in cases]
    want = [c.run(cache=k) for c, k in zip(cases, caches)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(5):
        got = []
        for c, k, s in zip(cases, caches, streams):
            with torch.cuda.stream(s):
                got.append(c.run(cache=k))
        torch.cuda.synchronize()
        for g, w in zip(got, want):
            assert torch.equal(g, w)


def test_cache_past_4_gib():
    """Blocks whose offsets pass 32 bits."""
    c = Case([100, 30], [1, 20], heads=4, kv_heads=2, window=None)
    small = c.device_cache()[0]._base
    blocks = (5 << 30) // (16 * 2 * 256 * 2)
    big = torch.empty(blocks, 16, 2, 256, dtype=torch.bfloat16, device=DEV)
    move = torch.randperm(small.shape[0], generator=c.gen) * ((blocks - 1) // small.shape[0]) + (
        (blocks - 1) % small.shape[0])
    big[move.to(DEV)] = small
    table = torch.where(c.table >= 0, move[c.table.clamp(min=0).long()].to(torch.int32), c.table)
    assert int(table.max()) * 16 * 2 * 256 * 2 > 1 << 32
    got = c.run(table=table, cache=(big[..., :128], big[..., 128:]))
    c.check(got)


def test_4_bit_cache_past_4_gib():
    c = Case([100, 30], [1, 20], heads=4, kv_heads=2, window=None, bits=4)
    small = c.device_cache().data
    blocks = (5 << 30) // small[0].numel()
    big = torch.empty(blocks, *small.shape[1:], dtype=torch.uint8, device=DEV)
    move = torch.randperm(small.shape[0], generator=c.gen) * ((blocks - 1) // small.shape[0]) + (
        (blocks - 1) % small.shape[0])
    big[move.to(DEV)] = small
    table = torch.where(c.table >= 0, move[c.table.clamp(min=0).long()].to(torch.int32), c.table)
    assert int(table.max()) * small[0].numel() > 1 << 32
    c.check(c.run(table=table, cache=Int4KVCache(big, 16, 128)))


def test_empty_calls():
    c = Case([10], [2])
    k, v = c.device_cache()
    none = torch.empty(0, 4, 128, dtype=torch.bfloat16, device=DEV)
    lens = torch.tensor([12], dtype=torch.int32, device=DEV)
    got = qsa_window_paged_attention(none, k, v, c.table.to(DEV), lens, c.qsl.to(DEV),
                                     max_query_len=1, max_seq_len=12)
    assert got.shape == none.shape
    # No blocks, or no table: nothing is seen.
    q = c.q.to(DEV)
    got = qsa_window_paged_attention(q, k[:0], v[:0], c.table.to(DEV), lens, c.qsl.to(DEV),
                                     max_query_len=2, max_seq_len=12)
    assert (got == 0).all()
    got = qsa_window_paged_attention(q, k, v, c.table.to(DEV)[:, :0], lens, c.qsl.to(DEV),
                                     max_query_len=2, max_seq_len=12)
    assert (got == 0).all()


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("new", [[1], [2, 1], [40], [300]])
def test_no_blocks(new, bits):
    """Lengths and a table that speak of pages that the cache does not have."""
    c = Case([100] * len(new), new, bits=bits)
    cache = c.device_cache()
    cache = Int4KVCache(cache.data[:0], 16, 128) if bits == 4 else (cache[0][:0], cache[1][:0])
    assert (c.run(cache=cache) == 0).all()


def test_refusals():
    c = Case([10], [2])
    k, v = c.device_cache()
    q, table, qsl = c.q.to(DEV), c.table.to(DEV), c.qsl.to(DEV)
    lens = torch.tensor([12], dtype=torch.int32, device=DEV)
    kw = dict(max_query_len=2, max_seq_len=12)
    call = qsa_window_paged_attention
    for bad, match in [
        (lambda: call(q.float(), k, v, table, lens, qsl, **kw), "q must be"),
        (lambda: call(q, k.float(), v, table, lens, qsl, **kw), "k_cache must be"),
        (lambda: call(q, k, v[:, :8], table, lens, qsl, **kw), "one shape"),
        (lambda: call(q[..., :64], k, v, table, lens, qsl, **kw), "head dim"),
        (lambda: call(q[:, :3], k, v, table, lens, qsl, **kw), "multiple of kv heads"),
        (lambda: call(q, k, v, table.long(), lens, qsl, **kw), "block_table"),
        (lambda: call(q, k, v, table, lens[:0], qsl, **kw), "seq_lens has 0"),
        (lambda: call(q, k, v, table, lens, qsl[:1], **kw), "query_start_loc has 1"),
        (lambda: call(q, k, v, table, lens, qsl, window=0, **kw), "window must be positive"),
        (lambda: call(q, k, v, table, lens, qsl, sink_tokens=-1, **kw), "sink_tokens"),
        (lambda: call(q, k, v, table, lens, qsl, max_query_len=-1, max_seq_len=1), "max_query_len"),
        (lambda: call(q, k, v, table, lens, qsl, torch.empty_like(q)[:1], **kw), "out must be"),
        (lambda: call(q, k, v, table, lens, qsl, q[:1].expand(2, -1, -1), **kw), "overlap"),
        (lambda: call(q, k, v, table, lens, qsl, output_gate=q[:1], **kw), "output_gate"),
        (lambda: call(q.cpu(), k, v, table, lens, qsl, **kw), "expected a GPU tensor"),
        (lambda: call(torch.empty(2, 4, 129, dtype=torch.bfloat16, device=DEV)[..., 1:], k, v, table,
                      lens, qsl, **kw), "alignment"),
    ]:
        with pytest.raises(RuntimeError, match=match):
            bad()
    four = Int4KVCache.allocate(3, 16, 2, 128, DEV)
    for bad, match in [
        (lambda: qsa_int4_paged_attention(q[..., :64], four, table, lens, qsl, **kw), "head dim"),
        (lambda: qsa_int4_paged_attention(q, Int4KVCache(four.data, 32, 128), table, lens, qsl, **kw),
         "4-bit cache must be"),
        (lambda: qsa_int4_paged_attention(q, Int4KVCache(four.data.int(), 16, 128), table, lens, qsl,
                                          **kw), "4-bit cache must be"),
        (lambda: qsa_int4_paged_attention(q, Int4KVCache(four.data[:, :, 16:], 16, 128), table, lens,
                                          qsl, **kw), "4-bit cache must be"),
    ]:
        with pytest.raises(RuntimeError, match=match):
            bad()
