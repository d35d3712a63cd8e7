"""Windowed attention as a layer of the hybrid decoder: the projection, its heads
normed, rotated and stored, attention over the cache, the output projection.

The layer's output equals its operators called one after the other, bit for bit, and
each of those is held against 64 bits on its own inputs with its own tolerance. The
norm's and rotation's: sums of 128 squares in fp32, a square root and a quotient, two
products and a sum, all under 2^-18 of |a cos| + |b sin|, and one rounding to bf16 of
2^-8. A 4-bit code is off by at most its scale (half a step of rounding, and as much
again where the group's zero point was rounded away from its end of the range)."""

from dataclasses import replace

import pytest
import torch
import torch.nn.functional as F

from qsa_vllm_amd.hybrid import HybridConfig, HybridDecodeGraph, make_hybrid_workload
from qsa_vllm_amd.ops import (qk_norm_rope, qsa_int4_paged_attention,
                              qsa_window_paged_attention)
from tests.paged_cases import Case

pytestmark = pytest.mark.gpu
DEV = "cuda:0"

CFG = HybridConfig(num_layers=4, hidden_size=512, vocab_size=256, tp_size=2, num_heads=16,
                   num_kv_heads=4, head_dim=128, intermediate_size=512, linear_num_key_heads=4,
                   linear_num_value_heads=8, indexer_heads=8, init_std=0.05, rope_dim=64,
                   window_layers=(0, 2), attention_window=200, sink_tokens=3)


def _workload(bits, seed=3, window=200):
    cfg = replace(CFG, window_kv_bits=bits, attention_window=window)
    return make_hybrid_workload(cfg, decode_lens=[700, 1500, 33, 260], chunk_prefixes=[0, 300],
                                chunk=100, device=DEV, seed=seed, state_std=0.05)


def _rotate(y, positions):
    """64-bit (result, |a cos| + |b sin|) of normed rows [tokens, heads, dim]."""
    half = CFG.rope_dim // 2
    angle = positions.double()[:, None] * CFG.rope_theta ** (
        -torch.arange(half).double() * 2 / CFG.rope_dim)
    c, s = angle.cos()[:, None], angle.sin()[:, None]
    a, b, rest = y[..., :half], y[..., half:2 * half], y[..., 2 * half:]
    return (torch.cat((a * c - b * s, b * c + a * s, rest), -1),
            torch.cat(((a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs(), rest.abs()), -1))


def _scales(cache):
    """K's and V's scales [blocks, page, heads, dim / 32] of a 4-bit cache."""
    page, dim = cache.page_size, cache.head_dim
    codes, words = page * dim // 2, page * dim // 16
    out = []
    for which in (0, 1):
        first = 2 * codes + which * (-(-words // 16) * 16)
        w = cache.data[:, :, first:first + words].cpu().reshape(*cache.data.shape[:2], page, -1, 2)
        w = w.to(torch.int32)
        out.append((((w[..., 0] | w[..., 1] << 8) & 0xFFF0) << 16).view(torch.float32).transpose(1, 2))
    return out


@pytest.mark.parametrize("window", [200, None])
@pytest.mark.parametrize("bits", [16, 4])
def test_layer_is_its_operators(bits, window):
    wl = _workload(bits, window=window)
    batch = wl.build()
    assert [layer.kind for layer in wl.model.layers] == [
        "sliding_attention", "linear_attention", "sliding_attention", "full_attention"]
    m = wl.model.layers[2].mixer
    gen = torch.Generator().manual_seed(1)
    m.q_norm = (1 + 0.2 * torch.randn(128, generator=gen)).bfloat16().to(DEV)
    m.k_norm = (1 + 0.2 * torch.randn(128, generator=gen)).bfloat16().to(DEV)
    t, d = batch.num_tokens, 128
    x = torch.randn(t, 512, generator=gen).bfloat16().to(DEV)
    before = m.state.clone()
    got = m(x, batch)
    written = m.state.clone()

    # The same, operator by operator, from the same cache.
    m.state.copy_(before)
    qkv = F.linear(x, m.qkv_weight, m.qkv_bias)
    qg = qkv[:, :m.q_size].view(t, m.heads, 2 * d)
    key = qkv[:, m.q_size:m.q_size + m.kv_size].view(t, m.kv_heads, d)
    value = qkv[:, m.q_size + m.kv_size:].view(t, m.kv_heads, d)
    pos, slots = batch.qsa.positions, batch.qsa.main.slot_mapping
    query, _ = qk_norm_rope(qg[..., :d], key, m.q_norm, m.k_norm, pos, m.cos_sin, m.eps, value=value,
                            cache=m.cache, slot_mapping=slots)
    assert torch.equal(m.state, written)
    held = m.cache.dequantize() if bits == 4 else m.cache
    held = [h.cpu() for h in held]
    at = slots.cpu() // 16, slots.cpu() % 16
    for rows, weight, out in ((qg[..., :d], m.q_norm, query.cpu()), (key, m.k_norm, held[0][at])):
        y = rows.cpu().double()
        y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + m.eps) * weight.cpu().double()
        want, size = _rotate(y, pos.cpu())
        off = 2.0 ** -18 * size + 2.0 ** -8 * want.abs()
        if bits == 4 and rows is key:
            off = off + _scales(m.cache)[0][at].double().repeat_interleave(32, -1) * (1 + 2 ** -7)
        assert ((out.double() - want).abs() <= off).all()
    if bits == 16:
        assert torch.equal(held[1][at], value.cpu())
    else:
        off = _scales(m.cache)[1][at].double().repeat_interleave(32, -1) * (1 + 2 ** -7)
        assert ((held[1][at].double() - value.cpu().double()).abs() <= off).all()
    kw = dict(window=window, sink_tokens=3, output_gate=qg[..., d:], max_query_len=100,
              max_seq_len=1501)
    call = qsa_int4_paged_attention if bits == 4 else qsa_window_paged_attention
    args = (m.cache,) if bits == 4 else m.cache
    core = call(query, *args, batch.qsa.main.block_table, batch.qsa.compressed.seq_lens,
                batch.query_start_loc, **kw)
    assert torch.equal(F.linear(core.view(t, -1), m.o_proj), got)

    c = Case.__new__(Case)
    c.ctx, c.new, c.page, c.dim = wl.computed, wl.scheduled, 16, d
    c.heads, c.kv_heads, c.window, c.sinks, c.bits = m.heads, m.kv_heads, window, 3, bits
    c.lens = [a + b for a, b in zip(c.ctx, c.new)]
    c.starts = batch.query_start_loc.cpu().tolist()
    c.table = batch.qsa.main.block_table.cpu()
    c.kv, c.q, c.gate = torch.cat(held, -1), query.cpu(), qg[..., d:].cpu()
    if bits == 4:
        c.parts = [(None, None, s.numpy()) for s in _scales(m.cache)]
    c.check(core)


@pytest.mark.parametrize("bits", [16, 4])
def test_decode_graph_equals_eager(bits):
    """Replayed on longer contexts and other tokens than the captured ones."""
    wl = _workload(bits, seed=9)
    start = [t.clone() for t in wl.layer_states()]

    def restore():
        for t, s in zip(wl.layer_states(), start):
            t.copy_(s)

    graph = HybridDecodeGraph(wl.model, wl.build_decode())
    base = list(wl.computed)
    for trial in (1, 2, 3):
        wl.computed[:4] = [c - 20 + 7 * trial for c in base[:4]]
        wl.token_ids[:4] = (wl.token_ids[:4] + 17 * trial) % 256
        restore()
        eager = wl.model.forward(wl.build_decode()).clone()
        states = [t.clone() for t in wl.layer_states()]
        restore()
        got = graph.replay(wl.build_decode()).clone()
        torch.cuda.synchronize()
        assert torch.isfinite(eager).all() and torch.equal(got, eager)
        assert all(torch.equal(a, b) for a, b in zip(wl.layer_states(), states))


def test_a_prompt_in_chunks_is_the_prompt():
    """A prompt of 260 tokens at once and in chunks (one of them a single token): the
    layer's cache is the same, its outputs agree to the rounding of the weights."""
    m_cfg = replace(CFG, num_layers=1, window_layers=(0,), attention_window=50)
    x = torch.randn(260, 512, generator=torch.Generator().manual_seed(5)).bfloat16().to(DEV)
    outs, states = [], []
    for chunks in ([260], [100, 1, 31, 128]):
        wl = make_hybrid_workload(m_cfg, decode_lens=[], chunk_prefixes=[0], chunk=260, device=DEV,
                                  seed=2)
        m, done, parts = wl.model.layers[0].mixer, 0, []
        for n in chunks:
            batch = wl.builder.build([done], [n], [0] * n, wl.main_table, wl.comp_table,
                                     wl.ring_blocks, wl.state_slots)
            core = _core(m, x[done:done + n], batch)
            parts.append(core)
            done += n
        outs.append(torch.cat(parts).cpu().double())
        states.append(m.state.clone())
    # (Libraries may sum a projection of other row counts in another order: what is
    # compared starts from the projection of the whole prompt.)
    assert torch.equal(*states)
    kv = m.state.cpu().double()
    size = kv[..., 128:].abs().max()
    # Each rounds its weights by 2^-8 of them, both ways, and its result by 2^-8.
    assert ((outs[0] - outs[1]).abs() <= 4 * 2.0 ** -8 * size * (1 + 2.0 ** -6)).all()


def _core(m, x, batch):
    """The layer's attention on rows whose projection is summed row by row."""
    qkv = (x.double().cpu() @ m.qkv_weight.double().cpu().T + m.qkv_bias.double().cpu()).bfloat16()
    qkv = qkv.to(DEV)
    t, d = len(x), 128
    qg = qkv[:, :m.q_size].view(t, m.heads, 2 * d)
    key = qkv[:, m.q_size:m.q_size + m.kv_size].view(t, m.kv_heads, d)
    value = qkv[:, m.q_size + m.kv_size:].view(t, m.kv_heads, d)
    query, _ = qk_norm_rope(qg[..., :d], key, m.q_norm, m.k_norm, batch.qsa.positions, m.cos_sin,
                            m.eps, value=value, cache=m.cache,
                            slot_mapping=batch.qsa.main.slot_mapping)
    return qsa_window_paged_attention(query, *m.cache, batch.qsa.main.block_table,
                                      batch.qsa.compressed.seq_lens, batch.query_start_loc,
                                      window=m.window, sink_tokens=m.sinks, output_gate=qg[..., d:],
                                      max_query_len=t, max_seq_len=260)
