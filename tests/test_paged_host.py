"""Windowed attention, the 4-bit cache and the heads' norm and rotation on the CPU: the
cache's layout, the position tables, and what the C entry points refuse (no launch)."""

import ctypes

import numpy as np
import pytest
import torch

from qsa_vllm_amd import _lib
from qsa_vllm_amd.ops import (Int4KVCache, qk_norm_rope, qsa_int4_paged_attention,
                              qsa_window_paged_attention, rotary_cache, rotary_table)

from .paged_cases import pack4, quantize4, values4


@pytest.mark.parametrize("page,dim,want", [(16, 128, 2304), (16, 64, 1152), (1, 64, 96), (1, 128, 160),
                                           (3, 64, 224), (272, 128, 39168)])
def test_page_bytes(page, dim, want):
    assert Int4KVCache.page_bytes(page, dim) == want
    assert Int4KVCache.allocate(2, page, 3, dim).data.shape == (2, 3, want)


@pytest.mark.parametrize("page,dim", [(16, 128), (3, 64), (1, 128)])
def test_values_of_packed_codes(page, dim):
    gen = np.random.default_rng(page)
    x = torch.from_numpy(gen.standard_normal((2, 4, page, 3, dim)).astype(np.float32)).bfloat16()
    parts = [quantize4(t.float().numpy()) for t in x]
    words = [(s.view(np.uint32) >> 16).astype(np.uint16) | z.astype(np.uint16) for _, z, s in parts]
    data = pack4(parts[0][0], words[0], parts[1][0], words[1])
    got = Int4KVCache(data, page, dim).dequantize()
    for have, p, t in zip(got, parts, x):
        exact = torch.from_numpy(values4(*p))
        assert torch.equal(have.float(), exact)      # bf16 holds every value
        step = torch.from_numpy(p[2]).repeat_interleave(32, -1)
        assert ((exact - t.float()).abs() <= step).all()


def test_every_value_of_a_word_is_a_bf16_value():
    codes = np.arange(16, dtype=np.float32)
    for z in range(16):
        for top in range(8):      # a scale's four significant bits
            s = np.float32((1 + top / 8) * 2.0 ** -3)
            x = (codes - np.float32(z)) * s
            assert (torch.from_numpy(x).bfloat16().float().numpy() == x).all()


def test_rotary_table_is_the_indexer_table_of_near_positions():
    a, b = rotary_table(64, 32, 1e4), rotary_cache(64, 32, 1e4, "cpu")
    assert a.dtype == torch.float32 and (a - b.float()).abs().max() <= 2 ** -8 * 1.01


def _attention(name, **change):
    args = dict(q=16, q_row=128, q_head=128, rows=2, hq=4, dim=128)
    if name == "qsa_window_attention":
        args |= dict(k=16, kb=4096, kt=256, kh=128, v=16, vb=4096, vt=256, vh=128)
    else:
        args |= dict(k=16, kb=4608, kh=2304)
    args |= dict(blocks=4, page=16, hkv=2, table=16, table_row=4, width=4, requests=1, lens=16, qsl=16,
                 window=0, sinks=0, out=16, o_row=512, o_head=128, gate=None, g_row=0, g_head=0,
                 g_dim=0, most=1, longest=64, ws=None, ws_bytes=0, stream=None)
    assert set(change) <= set(args)
    args |= change
    return getattr(_lib.load(), name)(*args.values())


@pytest.mark.parametrize("name", ["qsa_window_attention", "qsa_int4_kv_attention"])
def test_attention_refuses_before_a_launch(name):
    cases = [(dict(rows=-1), -1), (dict(window=-1), -1), (dict(sinks=-1), -1), (dict(most=-1), -1),
             (dict(dim=96), -2), (dict(hkv=3), -2), (dict(hkv=0), -2), (dict(page=0), -1),
             (dict(q=None), -1), (dict(out=None), -1), (dict(lens=None), -1), (dict(qsl=None), -1),
             (dict(table=None), -1), (dict(k=None), -1), (dict(q=8), -1), (dict(q_row=100), -1),
             (dict(out=2), -1), (dict(o_row=3), -1), (dict(k=24), -1), (dict(kb=4100), -1),
             (dict(rows=1 << 29, most=1 << 29), -2), (dict(kb=1 << 40), -2)]
    for change, status in cases:
        assert _attention(name, **change) == status, change
        assert name.encode() in _lib.load().qsa_last_error()
    # A call that splits needs its workspace, 16-byte aligned and whole.
    need = _lib.load().qsa_paged_attention_workspace_bytes(2, 1, 4, 2, 128, 0, 0, 1, 1 << 20)
    assert need > 0
    for ws, size in ((None, 0), (16, need - 1), (24, need)):
        assert _attention(name, longest=1 << 20, ws=ws, ws_bytes=size) == _lib.QSA_ERR_WORKSPACE
    # Nothing to do.
    for change in (dict(rows=0), dict(requests=0), dict(most=0)):
        assert _attention(name, **change) == 0


def test_workspace_of_odd_arguments():
    f = _lib.load().qsa_paged_attention_workspace_bytes
    assert f(0, 1, 4, 2, 128, 0, 0, 1, 99) == 0 and f(1, 0, 4, 2, 128, 0, 0, 1, 99) == 0
    assert f(1, 1, 4, 0, 128, 0, 0, 1, 99) == 0 and f(1, 1, 4, 2, 128, -1, 0, 1, 99) == 0
    # A window bounds what is split.
    assert f(1, 1, 4, 2, 128, 64, 4, 1, 1 << 30) == 0
    top = 2 ** 31 - 1
    assert f(1 << 20, top, 1024, 1, 128, top, top, top, top) >= 0


def _rope(**change):
    args = dict(q=16, q_t=512, q_h=128, hq=4, k=16, k_t=256, k_h=128, v=16, v_t=256, v_h=128, hkv=2,
                dim=128, tokens=3, qw=16, kw=16, eps=ctypes.c_float(1e-6), pos=16, table=16, fp32=1,
                most=100, rotary=64, qo=16, qo_t=512, qo_h=128, ko=None, ko_t=0, ko_h=0, vo=None,
                vo_t=0, vo_h=0, bits=16, slots=16, kc=16, kcb=4096, kct=256, kch=128, vc=16, vcb=4096,
                vct=256, vch=128, blocks=4, page=16, stream=None)
    assert set(change) <= set(args)
    args |= change
    return _lib.load().qsa_qk_norm_rope(*args.values())


def test_norm_rope_refuses_before_a_launch():
    for change, status in [
        (dict(tokens=-1), -1), (dict(hq=-1), -1), (dict(dim=32), -2), (dict(bits=8), -2),
        (dict(rotary=24), -2), (dict(rotary=144), -2), (dict(rotary=-16), -2), (dict(pos=None), -1),
        (dict(table=None), -1), (dict(most=0), -1), (dict(q=None), -1), (dict(qo=None), -1),
        (dict(k=None), -1), (dict(v=None), -1), (dict(slots=None), -1), (dict(kc=None), -1),
        (dict(vc=None), -1), (dict(page=0), -1), (dict(kc=24), -1), (dict(kct=100), -1),
        (dict(bits=4, kcb=100), -1), (dict(q_t=100), -1), (dict(k=24), -1), (dict(qw=8), -1),
        (dict(bits=0, v=None, vo=16), -1), (dict(tokens=1 << 30), -2),
    ]:
        assert _rope(**change) == status, change
        assert b"qsa_qk_norm_rope" in _lib.load().qsa_last_error()
    assert _rope(tokens=0) == 0
    # A launch of 2^32 threads and more, of fewer than 2^31 rows.
    for change in (dict(tokens=1 << 28, hq=1, hkv=0), dict(tokens=(1 << 28) // 3 + 1, hkv=1)):
        assert _rope(**change) == -2
        assert b"too many rows" in _lib.load().qsa_last_error()


def test_cpu_tensors_are_refused():
    q = torch.zeros(1, 4, 128, dtype=torch.bfloat16)
    kv = torch.zeros(2, 16, 2, 128, dtype=torch.bfloat16)
    one = torch.ones(1, dtype=torch.int32)
    qsl = torch.tensor([0, 1], dtype=torch.int32)
    table = torch.zeros(1, 2, dtype=torch.int32)
    four = Int4KVCache.allocate(2, 16, 2, 128)
    for call in (lambda: qsa_window_paged_attention(q, kv, kv, table, one, qsl, max_query_len=1,
                                                    max_seq_len=1),
                 lambda: qsa_int4_paged_attention(q, four, table, one, qsl, max_query_len=1,
                                                  max_seq_len=1),
                 lambda: qk_norm_rope(q, q, None, None, None, None, 1e-6)):
        with pytest.raises((RuntimeError, NotImplementedError)):
            call()


def test_window_layers_of_the_hybrid_decoder():
    from qsa_vllm_amd.hybrid import HybridConfig

    assert "sliding_attention" not in HybridConfig().layer_types()
    kinds = HybridConfig(num_layers=4, window_layers=(0, 3)).layer_types()
    assert kinds == ["sliding_attention", "linear_attention", "linear_attention", "sliding_attention"]
    with pytest.raises(ValueError, match="window_kv_bits"):
        HybridConfig(window_kv_bits=8)
    with pytest.raises(ValueError, match="window_layers"):
        HybridConfig(num_layers=4, window_layers=(4,))
