"""Norm and rotation of heads, and the cache's rows, in calls of many tokens, where a
group of lanes takes several heads of a token, beside calls of few. Against 64 bits
(tolerance: ``test_gpu_head_rope``), in bytes of the whole cache, and against each other."""

import numpy as np
import pytest
import torch

from qsa_vllm_amd.ops import Int4KVCache, qk_norm_rope, rotary_cache, rotary_table

from .paged_cases import DEV, pack4, quantize4, values4
from .test_gpu_head_rope import EPS, Rows, _check, _want

pytestmark = pytest.mark.gpu

# Query heads and kv heads that fill groups of lanes and that do not, calls of more than
# 4096 rows (all but the first of each kind).
HEADS = [(30, 5, 3, 128), (700, 5, 3, 128), (900, 6, 1, 64), (30, 6, 1, 64), (600, 16, 2, 128),
         (1100, 1, 5, 64), (800, 7, 2, 64)]


def _on(x):
    return None if x is None else x.to(DEV)


@pytest.mark.parametrize("tokens,heads,kv_heads,dim,rotary,norm,table", [
    (900, 5, 1, 128, 0, True, "fp32"), (1000, 6, 3, 64, 32, True, "bf16"),
    (700, 5, 3, 128, 64, True, "fp32"), (1500, 3, 1, 64, 64, False, "fp32"),
    (600, 9, 7, 128, 128, True, "bf16"), (4500, 0, 1, 128, 96, True, "fp32"),
])
def test_many_rows_match_64_bits(tokens, heads, kv_heads, dim, rotary, norm, table):
    """Into new tensors, then in place."""
    assert tokens * (heads + kv_heads) > 4096
    r = Rows(tokens, heads, kv_heads, dim, tokens + dim)
    positions = torch.randint(-3, 5005, (tokens,), generator=r.gen)
    t = None
    if rotary:
        t = rotary_table(5000, rotary, 1e7) if table == "fp32" else rotary_cache(5000, rotary, 1e7, "cpu")
    qw, kw = (r.qw, r.kw) if norm else (None, None)
    query = r.dq if heads else None
    args = (r.dk, _on(qw), _on(kw), positions.to(DEV), _on(t), EPS)
    q, k = qk_norm_rope(query, *args)
    if heads:
        _check(q, _want(r.q, qw, positions, t))
    _check(k, _want(r.k, kw, positions, t))
    rows = r.rows.clone()
    qk_norm_rope(query, *args, q_out=query, k_out=r.dk)
    assert torch.equal(r.dk, k) and (not heads or torch.equal(r.dq, q))
    # Gates, values and what lies behind them are as they were.
    end = 2 * heads * dim
    gates = (rows[:, :end].view(tokens, heads, 2 * dim)[..., dim:],
             r.rows[:, :end].view(tokens, heads, 2 * dim)[..., dim:])
    assert torch.equal(*gates)
    assert torch.equal(rows[:, end + kv_heads * dim:], r.rows[:, end + kv_heads * dim:])


class _Stored:
    """A call into a cache of one fill, and all that the cache has to hold after it."""

    def __init__(self, tokens, heads, kv_heads, dim, page, bits, layout="pair"):
        r = self.r = Rows(tokens, heads, kv_heads, dim, tokens + dim + page)
        self.bits, self.page, self.dim, self.kv_heads = bits, page, dim, kv_heads
        self.blocks = -(-(tokens + 40) // page)
        self.positions = torch.randint(0, 900, (tokens,), generator=r.gen)
        self.table = rotary_table(1000, 32, 1e5)
        slots = torch.randperm(self.blocks * page, generator=r.gen)[:tokens]
        for at, slot in ((5, -1), (6, self.blocks * page), (7, -(1 << 40)), (8, 1 << 40),
                         (tokens - 1, -1)):
            slots[at] = slot
        self.slots = slots
        self.live = (slots >= 0) & (slots < self.blocks * page)
        self.whole, self.cache = self.fresh(layout)
        self.layout = layout

    def fresh(self, layout):
        """(the whole buffer, the cache in it), every byte 0xEE or every value 9."""
        blocks, page, heads, dim = self.blocks, self.page, self.kv_heads, self.dim
        if self.bits == 4:
            size = Int4KVCache.page_bytes(page, dim)
            if layout == "split":       # pages inside larger blocks
                whole = torch.full((blocks, heads + 1, size + 32), 0xEE, dtype=torch.uint8, device=DEV)
                return whole, Int4KVCache(whole[:, 1:, :size], page, dim)
            whole = torch.full((blocks, heads, size), 0xEE, dtype=torch.uint8, device=DEV)
            return whole, Int4KVCache(whole, page, dim)
        shape = (blocks, heads, page, 2 * dim + 8) if layout == "split" else (blocks, page, heads, 2 * dim)
        whole = torch.full(shape, 9.0, dtype=torch.bfloat16, device=DEV)
        kv = whole.transpose(1, 2) if layout == "split" else whole
        return whole, (kv[..., :dim], kv[..., dim:2 * dim])

    def call(self, cache, part=slice(None), **out):
        r = self.r
        return qk_norm_rope(r.dq[part], r.dk[part], r.qw.to(DEV), r.kw.to(DEV),
                            self.positions[part].to(DEV), self.table.to(DEV), EPS, value=r.dv[part],
                            cache=cache, slot_mapping=self.slots[part].to(DEV), **out)

    def rows(self):
        """(query, key) rows of a call without a cache."""
        r = self.r
        return qk_norm_rope(r.dq, r.dk, r.qw.to(DEV), r.kw.to(DEV), self.positions.to(DEV),
                            self.table.to(DEV), EPS)

    def held(self, key):
        """K and V rows as the cache has to hold them, and their codes and words."""
        if self.bits == 16:
            return [key.cpu(), self.r.v], None
        parts = [quantize4(x.float().cpu().numpy()) for x in (key, self.r.v)]
        return [torch.from_numpy(values4(*p)).bfloat16() for p in parts], parts

    def want(self, key):
        """The whole buffer after the call."""
        whole, cache = self.fresh(self.layout)
        whole = whole.cpu()
        values, parts = self.held(key)
        block, place = self.slots[self.live] // self.page, self.slots[self.live] % self.page
        if self.bits == 16:
            kv = whole.transpose(1, 2) if self.layout == "split" else whole
            for i, x in enumerate(values):
                kv[block, place, :, i * self.dim:(i + 1) * self.dim] = x[self.live]
            return whole
        shape = (self.blocks, self.page, self.kv_heads)
        data, mask = [], []
        for codes, zero, scale in parts:
            word = (scale.view(np.uint32) >> 16).astype(np.uint16) | zero.astype(np.uint16)
            for x, ones, width, kind in ((codes, 15, self.dim, np.float32),
                                         (word, 0xFFFF, self.dim // 32, np.uint16)):
                for dst, src in ((data, x[self.live.numpy()]), (mask, kind(ones))):
                    a = np.zeros((*shape, width), dtype=kind)
                    a[block.numpy(), place.numpy()] = src
                    dst.append(a)
        data, mask = pack4(*data), pack4(*mask)
        view = whole[:, 1:, :data.shape[2]] if self.layout == "split" else whole
        view.copy_((view & ~mask) | data)
        return whole


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("page,layout", [(16, "pair"), (1, "pair"), (48, "split")])
@pytest.mark.parametrize("tokens,heads,kv_heads,dim", HEADS)
def test_all_bytes_of_the_cache(tokens, heads, kv_heads, dim, page, layout, bits):
    """Rows in their slots, and every other byte as it was: other slots, what fills up a
    page's words, gaps between pages, rows without a slot."""
    s = _Stored(tokens, heads, kv_heads, dim, page, bits, layout)
    q, key = s.rows()
    _check(q, _want(s.r.q, s.r.qw, s.positions, s.table))
    _check(key, _want(s.r.k, s.r.kw, s.positions, s.table))
    values, _ = s.held(key)
    k_out, v_out = (torch.empty(tokens, kv_heads, dim, dtype=torch.bfloat16, device=DEV)
                    for _ in range(2))
    got, _ = s.call(s.cache, k_out=k_out, v_out=v_out)
    assert torch.equal(got, q)
    assert torch.equal(k_out.cpu(), values[0]) and torch.equal(v_out.cpu(), values[1])
    assert torch.equal(s.whole.cpu(), s.want(key))
    # Without the rows as held, and in place.
    whole, cache = s.fresh(layout)
    s.call(cache)
    assert torch.equal(whole, s.whole)
    whole, cache = s.fresh(layout)
    r = s.r
    s.call(cache, q_out=r.dq, k_out=r.dk, v_out=r.dv)
    assert torch.equal(whole, s.whole) and torch.equal(r.dq, q)
    assert torch.equal(r.dk, k_out) and torch.equal(r.dv, v_out)


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("tokens,heads,kv_heads,dim", HEADS)
def test_few_tokens_and_many_give_the_same_bits(tokens, heads, kv_heads, dim, bits):
    """One call, and the same rows in calls of up to 100 tokens."""
    s = _Stored(tokens, heads, kv_heads, dim, 16, bits)
    outs = [torch.empty(tokens, kv_heads, dim, dtype=torch.bfloat16, device=DEV) for _ in range(4)]
    q, _ = s.call(s.cache, k_out=outs[0], v_out=outs[1])
    whole, cache = s.fresh("pair")
    for i in range(0, tokens, 100):
        part = slice(i, min(i + 100, tokens))
        assert (heads + 2 * kv_heads) * 100 <= 4096
        got, _ = s.call(cache, part, k_out=outs[2][part], v_out=outs[3][part])
        assert torch.equal(got, q[part])
    assert torch.equal(outs[0], outs[2]) and torch.equal(outs[1], outs[3])
    assert torch.equal(whole, s.whole)


def test_edge_rows_among_many():
    """What has no code, constants, one sign, tiny values: the 4-bit rows of a call of few
    tokens, repeated past 4096 rows."""
    gen = torch.Generator().manual_seed(0)
    v = torch.randn(16, 3, 64, generator=gen)
    v[0], v[1], v[2] = 0, 3.0, -1.5
    v[3] = v[3].abs() + 100
    v[5] *= 1e-30
    v[6] *= 2.0 ** 123 / v[6].abs().max()
    v = v.bfloat16()
    v[10, 0, 3], v[11, 1, 40], v[12, 2, 33] = float("inf"), float("nan"), -2.0 ** 126
    times, size = 100, Int4KVCache.page_bytes(16, 64)
    many = v.repeat(times, 1, 1).to(DEV)
    outs = []
    for x in (v.to(DEV), many):
        cache = Int4KVCache.allocate(len(x) // 16, 16, 3, 64, DEV)
        out = torch.empty_like(x)
        qk_norm_rope(None, x, None, None, None, None, EPS, value=x, cache=cache,
                     slot_mapping=torch.arange(len(x), device=DEV), v_out=out)
        outs.append((cache.data, out))
    (data, out), (all_data, all_out) = outs
    assert torch.equal(all_data, data.expand(times, 3, size))
    assert torch.equal(all_out.view(torch.int16), out.repeat(times, 1, 1).view(torch.int16))
    codes, zero, scale = quantize4(torch.nan_to_num(v.float(), 0.0, 0.0, 0.0).numpy())
    want = torch.from_numpy(values4(codes, zero, scale)).bfloat16()
    good = ~torch.isnan(out.cpu())
    assert int((~good).sum()) == 3 * 32 and torch.equal(out.cpu()[good], want[good])
