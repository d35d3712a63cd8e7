"""Norm and rotation of heads and the cache's rows on the GPU against 64 bits.

Tolerance. The norm's sum of D squares is off by at most 2^-24 (D / 8 + 4) of itself,
the inverse root by half that and 2^-22, the products by 2^-24 each: under 2^-19 of a
normed value y. A rotated one is a cos - b sin: 2^-19 (|a| + |b|) and the table's fp32
half step, 2^-25 of each. Then one rounding to bf16, 2^-8 of the value."""

import numpy as np
import pytest
import torch

from qsa_vllm_amd.ops import (Int4KVCache, indexer_norm_rope, IndexerRMSNorm, qk_norm_rope,
                              qsa_int4_paged_attention, qsa_window_paged_attention, rotary_cache,
                              rotary_table)

from .paged_cases import DEV, quantize4, values4

pytestmark = pytest.mark.gpu
EPS = 1e-6


def _want(x, weight, positions, table):
    y = x.double()
    if weight is not None:
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + EPS) * weight.double()
    size = y.abs()
    if table is not None and table.shape[1]:
        rotary = table.shape[1]
        inside = (positions >= 0) & (positions < table.shape[0])
        row = table.double()[positions.clamp(0, table.shape[0] - 1)] * inside[:, None]
        cos, sin = row[:, None].chunk(2, -1)
        a, b = y[..., :rotary // 2], y[..., rotary // 2:rotary]
        size = size.clone()
        size[..., :rotary] = (a.abs() + b.abs()).repeat(1, 1, 2)
        y = torch.cat((a * cos - b * sin, b * cos + a * sin, y[..., rotary:]), -1)
    return y, 2 ** -8 * y.abs() + 2 ** -18 * size + 2 ** -120


class Rows:
    def __init__(self, tokens, heads, kv_heads, dim, seed=0, scale=1.0):
        gen = torch.Generator().manual_seed(seed)
        self.gen = gen
        rows = (torch.randn(tokens, (2 * heads + 2 * kv_heads) * dim + 16, generator=gen) * scale)
        rows = rows.bfloat16()
        self.rows = rows.to(DEV)
        n = 2 * heads * dim

        def parts(t):   # queries with gates between them, keys, values: a projection's columns
            return (t[:, :n].view(tokens, heads, 2 * dim)[..., :dim],
                    t[:, n:n + kv_heads * dim].view(tokens, kv_heads, dim),
                    t[:, n + kv_heads * dim:n + 2 * kv_heads * dim].view(tokens, kv_heads, dim))

        self.q, self.k, self.v = parts(rows)
        self.dq, self.dk, self.dv = parts(self.rows)
        self.qw, self.kw = ((1 + 0.3 * torch.randn(dim, generator=gen)).bfloat16() for _ in range(2))


def _check(got, want):
    want, tol = want
    off = (got.cpu().double() - want).abs()
    assert (off <= tol).all(), f"{(off / tol).max().item():.2f} times the tolerance"


@pytest.mark.parametrize("tokens,heads,kv_heads,dim,rotary,norm,table", [
    (1, 1, 1, 128, 64, True, "fp32"), (1, 16, 2, 128, 64, True, "bf16"),
    (7, 6, 2, 64, 64, True, "fp32"), (33, 3, 3, 128, 128, True, "fp32"),
    (5, 4, 1, 64, 32, False, "bf16"), (9, 2, 2, 128, 16, True, "fp32"),
    (130, 5, 1, 128, 0, True, "fp32"), (3, 4, 4, 64, 0, False, "fp32"),
    (600, 16, 2, 128, 96, True, "fp32"),
])
def test_matches_64_bits(tokens, heads, kv_heads, dim, rotary, norm, table):
    r = Rows(tokens, heads, kv_heads, dim, tokens + dim)
    positions = torch.randint(0, 5000, (tokens,), generator=r.gen)
    t = None
    if rotary:
        t = rotary_table(5000, rotary, 1e7) if table == "fp32" else rotary_cache(5000, rotary, 1e7, "cpu")
    qw, kw = (r.qw, r.kw) if norm else (None, None)
    on = lambda x: None if x is None else x.to(DEV)  # noqa: E731
    q, k = qk_norm_rope(r.dq, r.dk, on(qw), on(kw), positions.to(DEV), on(t), EPS)
    _check(q, _want(r.q, qw, positions, t))
    _check(k, _want(r.k, kw, positions, t))
    assert q.is_contiguous() and k.is_contiguous()


def test_norm_of_one_side_in_place_and_without_queries():
    r = Rows(11, 4, 2, 128)
    positions = torch.arange(11)
    t = rotary_table(64, 64, 1e4)
    args = (positions.to(DEV), t.to(DEV), EPS)
    q, k = qk_norm_rope(r.dq, r.dk, None, r.kw.to(DEV), *args)
    _check(q, _want(r.q, None, positions, t))
    _check(k, _want(r.k, r.kw, positions, t))
    none, k2 = qk_norm_rope(None, r.dk, None, r.kw.to(DEV), *args)
    assert none is None and torch.equal(k2, k)
    gates = r.rows[:, :4 * 256].view(11, 4, 256)[..., 128:].clone()
    got = qk_norm_rope(r.dq, r.dk, None, r.kw.to(DEV), *args, q_out=r.dq, k_out=r.dk)
    assert got[0] is r.dq and torch.equal(r.dq, q) and torch.equal(r.dk, k)
    assert torch.equal(r.rows[:, :4 * 256].view(11, 4, 256)[..., 128:], gates)


def test_positions_outside_the_table_and_far_ones():
    r = Rows(5, 2, 1, 128)
    t = rotary_table(131072, 64, 1e7)
    positions = torch.tensor([131071, 131072, -1, 0, 1 << 40])
    q, _ = qk_norm_rope(r.dq, r.dk, r.qw.to(DEV), None, positions.to(DEV), t.to(DEV), EPS)
    _check(q, _want(r.q, r.qw, positions, t))
    assert (q[1, :, :64] == 0).all() and (q[4, :, :64] == 0).all()
    # As the indexer's heads, up to its roundings in between (a few of bf16's half steps).
    norm = IndexerRMSNorm(128, EPS).to(DEV)
    both = rotary_cache(131072, 64, 1e7, torch.device(DEV))
    x = r.dq.contiguous()
    old = indexer_norm_rope(x, norm, positions.to(DEV), both, 64)
    new, _ = qk_norm_rope(x, r.dk, norm.weight.data, None, positions.to(DEV), both, EPS)
    want, tol = _want(r.q, torch.ones(128), positions, both.cpu())
    size = want.abs().amax(-1, keepdim=True)
    assert ((old.double() - new.double()).cpu().abs() <= 2 ** -8 * 6 * size).all()


def test_table_of_far_positions():
    """Angles of 64 bits: each entry within an fp32 half step of its cosine or sine."""
    t = rotary_table(131072, 64, 1e7).double()
    pos = np.array([0, 1, 77, 65537, 131071])
    for c in (0, 1, 13, 31):
        angle = pos.astype(np.longdouble) * np.longdouble(1e7) ** (np.longdouble(-2 * c) / 64)
        # (the 64-bit angle itself is off by 2^-52 of up to 131071 radians)
        for got, want in ((t[pos, c], np.cos(angle)), (t[pos, 32 + c], np.sin(angle))):
            assert np.abs(got.numpy() - want.astype(np.float64)).max() <= 2 ** -25 + 2 ** -34


def test_zero_and_extreme_rows():
    """A row of zeros stays zeros; large and tiny values are normed in 32 bits."""
    r = Rows(4, 1, 1, 128)
    r.q, r.k = r.q.clone(), r.k.clone()
    r.q[0] = 0
    r.q[1] *= 1e15
    r.q[2] *= 1e-15
    q, _ = qk_norm_rope(r.q.to(DEV), r.dk, r.qw.to(DEV), r.kw.to(DEV), None, None, EPS)
    _check(q, _want(r.q, r.qw, None, None))
    assert (q[0] == 0).all()


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("dim,page,layout", [(128, 16, "pair"), (64, 48, "pair"), (128, 1, "pair"),
                                             (64, 272, "split"), (128, 16, "split")])
def test_cache_rows(bits, dim, page, layout):
    """Rows land in their slots and nowhere else; rows without a slot are not stored."""
    tokens, heads, kv_heads, blocks = 70, 4, 2, 90 if page == 1 else 12
    r = Rows(tokens, heads, kv_heads, dim, dim + page)
    positions = torch.randint(0, 900, (tokens,), generator=r.gen)
    t = rotary_table(1000, 32, 1e5)
    slots = torch.randperm(blocks * page, generator=r.gen)[:tokens]
    slots[5], slots[6], slots[7] = -1, blocks * page, -(1 << 40)
    slots[8] = 1 << 40
    if bits == 16:
        kv = torch.full((blocks, page, kv_heads, 2 * dim), 9.0, dtype=torch.bfloat16, device=DEV)
        if layout == "split":
            kv = torch.full((blocks, kv_heads, page, 2 * dim), 9.0, dtype=torch.bfloat16, device=DEV)
            kv = kv.transpose(1, 2)
        cache = kv[..., :dim], kv[..., dim:]
    else:
        cache = Int4KVCache.allocate(blocks, page, kv_heads, dim, DEV)
        if layout == "split":    # pages inside larger blocks
            wide = torch.zeros(blocks, kv_heads + 1, cache.data.shape[2] + 32, dtype=torch.uint8,
                               device=DEV)
            cache = Int4KVCache(wide[:, 1:, :cache.data.shape[2]], page, dim)
            assert cache.data.shape[1] == kv_heads
        cache.data.fill_(0xEE)
    k_out, v_out = (torch.empty(tokens, kv_heads, dim, dtype=torch.bfloat16, device=DEV)
                    for _ in range(2))
    q, k = qk_norm_rope(r.dq, r.dk, r.qw.to(DEV), r.kw.to(DEV), positions.to(DEV), t.to(DEV), EPS,
                        value=r.dv, cache=cache, slot_mapping=slots.to(DEV), k_out=k_out, v_out=v_out)
    _check(q, _want(r.q, r.qw, positions, t))
    want_k, tol = _want(r.k, r.kw, positions, t)
    live = (slots >= 0) & (slots < blocks * page)
    if bits == 16:
        _check(k, (want_k, tol))
        assert torch.equal(v_out, r.dv)
        got = [c.reshape(-1, kv_heads, dim).cpu() for c in cache]
    else:
        # V's codes and values bit by bit; K's from a row that is off by its own tolerance:
        # a step at most (the zero point's rounding and the value's, at the range's ends),
        # from a range that moved by twice the tolerance.
        codes, zero, scale = quantize4(r.v.float().numpy())
        assert torch.equal(v_out.cpu(), torch.from_numpy(values4(codes, zero, scale)).bfloat16())
        y = want_k.unflatten(-1, (-1, 32))
        most = tol.unflatten(-1, (-1, 32)).amax(-1)
        step = (y.amax(-1).clamp(min=0) - y.amin(-1).clamp(max=0) + 2 * most) / 15 * 1.125
        allowed = (step + most)[..., None].expand(-1, -1, -1, 32).flatten(-2)
        assert ((k.cpu().double() - want_k).abs() <= allowed).all()
        got = [c.reshape(-1, kv_heads, dim).cpu() for c in cache.dequantize()]
        # Every byte of other slots is as it was: codes 14, words 0xEEEE.
    untouched = torch.ones(blocks * page, dtype=torch.bool)
    untouched[slots[live]] = False
    for have, rows in zip(got, (k_out, v_out)):
        assert torch.equal(have[slots[live]], rows.cpu()[live])
        rest = have[untouched]
        assert (rest == rest[:1]).all()
    if bits == 4 and layout == "split":
        rest = wide.clone()
        rest[:, 1:, :cache.data.shape[2]] = 0
        assert (rest == 0).all()


def test_4_bit_rows_of_edges():
    """Ranges of one sign, constants, zeros, tiny and huge values bit by bit; groups that
    hold what has no code read as NaN, their neighbours do not."""
    gen = torch.Generator().manual_seed(0)
    v = torch.randn(16, 1, 128, generator=gen)
    v[0] = 0
    v[1] = 3.0
    v[2] = -1.5
    v[3] = v[3].abs() + 100
    v[4] = -v[4].abs() - 7
    v[5] *= 1e-30
    v[6] *= 2.0 ** 123 / v[6].abs().max()
    v[7, 0, :32] = torch.arange(32) - 16.0
    v[8] = torch.arange(128) * 0.25
    v[9, 0, ::2] = 0
    v = v.bfloat16()
    v[10, 0, 3] = float("inf")
    v[11, 0, 40] = float("nan")
    v[12, 0, 70] = -2.0 ** 126
    v[13, 0, 127] = 2.0 ** 125
    cache = Int4KVCache.allocate(1, 16, 1, 128, DEV)
    out = torch.empty_like(v, device=DEV)
    zeros = torch.zeros_like(v, device=DEV)
    qk_norm_rope(None, zeros, None, None, None, None, EPS, value=v.to(DEV), cache=cache,
                 slot_mapping=torch.arange(16, device=DEV), v_out=out)
    held = cache.dequantize()
    assert (held[0] == 0).all()
    assert torch.equal(torch.nan_to_num(held[1][0], 77.0), torch.nan_to_num(out, 77.0))
    bad = torch.zeros(16, 4, dtype=torch.bool)
    bad[10, 0] = bad[11, 1] = bad[12, 2] = True
    got = out.cpu().unflatten(-1, (4, 32))[:, 0]
    assert torch.equal(torch.isnan(got).all(-1), bad) and torch.equal(torch.isnan(got).any(-1), bad)
    codes, zero, scale = quantize4(torch.nan_to_num(v.float(), 0.0, 0.0, 0.0).numpy())
    want = torch.from_numpy(values4(codes, zero, scale)).bfloat16().unflatten(-1, (4, 32))[:, 0]
    assert torch.equal(got[~bad], want[~bad])
    # Within a step of the value, where the step is the range's 15th and at most an eighth.
    x = v.double().unflatten(-1, (4, 32))[:, 0]
    step = (x.amax(-1).clamp(min=0) - x.amin(-1).clamp(max=0)) / 15 * 1.125 + 2.0 ** -100
    assert ((got.double() - x).abs() <= step[..., None])[~bad].all()


@pytest.mark.parametrize("bits", [16, 4])
def test_layer_steps_together(bits):
    """A prompt in two chunks, then single tokens of two requests: norm, rotation and store,
    then windowed attention over the cache so far, against a 64-bit layer over the rows
    that the cache holds. The attention's tolerance is 2^-8 of the weights' (twice from 4
    bits) and of the result, with 2^-8 of q k's exponents for q's own rounding."""
    heads, kv_heads, dim, page, window, sinks = 8, 2, 128, 16, 40, 3
    t = rotary_table(400, 64, 1e6)
    table = torch.randperm(60, dtype=torch.int32).view(2, 30)
    if bits == 16:
        kv = torch.full((60, page, kv_heads, 2 * dim), float("nan"), dtype=torch.bfloat16, device=DEV)
        cache = kv[..., :dim], kv[..., dim:]
    else:
        cache = Int4KVCache.allocate(60, page, kv_heads, dim, DEV)
    have = [0, 0]
    seen = [[], []]
    for step, new in enumerate([(70, 20), (30, 50), (1, 1), (1, 1), (1, 1)]):
        r = Rows(sum(new), heads, kv_heads, dim, step)
        req = torch.repeat_interleave(torch.arange(2), torch.tensor(new))
        positions = torch.cat([torch.arange(have[b], have[b] + new[b]) for b in range(2)])
        slots = table[req, positions // page].long() * page + positions % page
        held = [torch.empty(sum(new), kv_heads, dim, dtype=torch.bfloat16, device=DEV)
                for _ in range(2)]
        q, k = qk_norm_rope(r.dq, r.dk, r.qw.to(DEV), r.kw.to(DEV), positions.to(DEV), t.to(DEV),
                            EPS, value=r.dv, cache=cache, slot_mapping=slots.to(DEV),
                            k_out=held[0], v_out=held[1])
        have = [have[b] + new[b] for b in range(2)]
        qsl = torch.tensor([0, new[0], sum(new)], dtype=torch.int32, device=DEV)
        lens = torch.tensor(have, dtype=torch.int32, device=DEV)
        kw = dict(window=window, sink_tokens=sinks, max_query_len=max(new), max_seq_len=max(have))
        if bits == 16:
            got = qsa_window_paged_attention(q, *cache, table.to(DEV), lens, qsl, **kw)
        else:
            got = qsa_int4_paged_attention(q, cache, table.to(DEV), lens, qsl, **kw)
        got = got.cpu().double()
        want_q, _ = _want(r.q, r.qw, positions, t)
        for b in range(2):
            seen[b] += [(held[0][i].cpu().double(), held[1][i].cpu().double())
                        for i in range(sum(new)) if req[i] == b]
        for i in range(sum(new)):
            b, p = int(req[i]), int(positions[i])
            at = [j for j in range(p + 1) if j > p - window or j < sinks]
            ks = torch.stack([seen[b][j][0] for j in at]).permute(1, 2, 0)
            vs = torch.stack([seen[b][j][1] for j in at]).permute(1, 0, 2)
            qi = want_q[i].view(kv_heads, -1, dim)
            w = torch.softmax(qi @ ks / dim ** 0.5, -1)
            o = w @ vs
            spread = (qi.abs() @ ks.abs()).amax(-1, keepdim=True) / dim ** 0.5
            off = (2 * 2 ** -8 * spread * 1.05 + (2 if bits == 4 else 1) * 2 ** -8 * 1.01 + 2 ** -12) * (
                w @ vs.abs() + o.abs())
            assert ((got[i].view(kv_heads, -1, dim) - o).abs() <= off + 2 ** -8 * (o.abs() + off)).all()


def test_captured_call_follows_its_buffers():
    r = Rows(6, 4, 2, 128)
    cache = Int4KVCache.allocate(4, 16, 2, 128, DEV)
    t, qw, kw = rotary_table(100, 64, 1e4, DEV), r.qw.to(DEV), r.kw.to(DEV)
    positions = torch.arange(6, device=DEV)
    slots = torch.arange(6, device=DEV)
    q_out = torch.empty(6, 4, 128, dtype=torch.bfloat16, device=DEV)

    def step():
        qk_norm_rope(r.dq, r.dk, qw, kw, positions, t, EPS, value=r.dv, cache=cache,
                     slot_mapping=slots, q_out=q_out)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in range(3):
        r.rows.copy_(torch.randn(r.rows.shape, generator=r.gen))
        positions.add_(7)
        slots.add_(9)
        graph.replay()
        torch.cuda.synchronize()
        got, data = q_out.clone(), cache.data.clone()
        cache.data.zero_()
        step()
        at = slots.cpu()
        assert torch.equal(got, q_out)
        new = cache.dequantize()
        old = Int4KVCache(data, 16, 128).dequantize()
        for a, b in zip(old, new):
            assert torch.equal(a.reshape(64, 2, 128)[at], b.reshape(64, 2, 128)[at])
        cache.data.copy_(data)


def test_empty_and_refused_calls():
    r = Rows(3, 4, 2, 128)
    pos, t = torch.arange(3, device=DEV), rotary_table(8, 64, 1e4, DEV)
    w = r.qw.to(DEV)
    q, k = qk_norm_rope(r.dq[:0], r.dk[:0], w, w, pos[:0], t, EPS)
    assert q.shape == (0, 4, 128) and k.shape == (0, 2, 128)
    four = Int4KVCache.allocate(2, 16, 2, 128, DEV)
    kv = torch.zeros(2, 16, 2, 256, dtype=torch.bfloat16, device=DEV)
    pair = kv[..., :128], kv[..., 128:]
    for bad, match in [
        (lambda: qk_norm_rope(r.dq.float(), r.dk, w, w, pos, t, EPS), "query must be"),
        (lambda: qk_norm_rope(r.dq[:2], r.dk, w, w, pos, t, EPS), "query must be"),
        (lambda: qk_norm_rope(r.dq, r.dk, w[:64], w, pos, t, EPS), "q_weight"),
        (lambda: qk_norm_rope(r.dq, r.dk, w, w.float(), pos, t, EPS), "k_weight"),
        (lambda: qk_norm_rope(r.dq, r.dk, w, w, pos[:2], t, EPS), "positions"),
        (lambda: qk_norm_rope(r.dq, r.dk, w, w, None, t, EPS), "positions"),
        (lambda: qk_norm_rope(r.dq, r.dk, w, w, pos.int(), t, EPS), "positions"),
        (lambda: qk_norm_rope(r.dq, r.dk, w, w, pos, t.half(), EPS), "cos_sin"),
        (lambda: qk_norm_rope(r.dq, r.dk, w, w, pos, t[:, :24].contiguous(), EPS), "multiple of 16"),
        (lambda: qk_norm_rope(r.dq, r.dk, w, w, pos, torch.cat((t, t, t), 1), EPS), "rotary_dim"),
        (lambda: qk_norm_rope(r.dq, r.dk, w, w, pos, t, EPS, cache=pair, slot_mapping=pos), "values"),
        (lambda: qk_norm_rope(r.dq, r.dk, w, w, pos, t, EPS, value=r.dv, cache=four), "slot"),
        (lambda: qk_norm_rope(r.dq, r.dk, w, w, pos, t, EPS, slot_mapping=pos), "needs a cache"),
        (lambda: qk_norm_rope(r.dq, r.dk, w, w, pos, t, EPS, value=r.dv, cache=pair,
                              slot_mapping=pos.int()), "slot_mapping"),
        (lambda: qk_norm_rope(r.dq, r.dk, w, w, pos, t, EPS, value=r.dv, slot_mapping=pos,
                              cache=(pair[0][:, :, :1], pair[1][:, :, :1])), "caches must be"),
        (lambda: qk_norm_rope(r.dq, r.dk, w, w, pos, t, EPS, value=r.dv, slot_mapping=pos,
                              cache=Int4KVCache(four.data, 32, 128)), "4-bit cache must be"),
        (lambda: qk_norm_rope(r.dq, r.dk, w, w, pos, t, EPS, value=r.dv, slot_mapping=pos,
                              cache=Int4KVCache(four.data, 16, 64)), "head dim"),
        (lambda: qk_norm_rope(r.dq, r.dk, w, w, pos, t, EPS, v_out=torch.empty_like(r.dv)), "values"),
        (lambda: qk_norm_rope(r.dq, r.dk, w, w, pos, t, EPS,
                              k_out=torch.empty_like(r.dk)[:1].expand(3, -1, -1)), "overlap"),
        (lambda: qk_norm_rope(r.rows[:, 4:516].view(3, 4, 128), r.dk, w, w, pos, t, EPS), "alignment"),
        (lambda: qk_norm_rope(r.dq[..., :32], r.dk[..., :32], None, None, pos, None, EPS), "head_dim"),
    ]:
        with pytest.raises(RuntimeError, match=match):
            bad()
    with pytest.raises(RuntimeError, match="page size"):
        Int4KVCache.allocate(2, 0, 2, 128)
    with pytest.raises(RuntimeError, match="head dim"):
        Int4KVCache.page_bytes(16, 96)
