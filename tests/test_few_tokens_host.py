"""The operators of a step over a few tokens, on the CPU: the 4-bit weight's
layout and rounding, ancestor bits against a walk up the tree, and what the C
entry points refuse (no launch)."""

import contextlib
import gc
import types
import weakref

import numpy as np
import pytest
import torch

from qsa_vllm_amd import _lib
from qsa_vllm_amd.hybrid import HybridDecodeGraph
from qsa_vllm_amd.ops import (LogitsRules, int4_linear, int4_pack, int4_quantize, process_logits,
                              qsa_tree_paged_attention, tree_ancestors)


def test_packed_words_hold_each_code_at_its_place():
    """Lane 16 g + n, word j of tile (n tile, k tile): inputs 32 j + 8 g + i of
    output n, i even in bits 2 i, i odd in bits 14 + 2 i."""
    gen = torch.Generator().manual_seed(0)
    n, k = 21, 300
    codes = torch.randint(0, 16, (n, k), generator=gen, dtype=torch.uint8)
    scales = torch.rand(n, 10, generator=gen).bfloat16()
    zeros = torch.randint(0, 16, (n, 10), generator=gen, dtype=torch.uint8)
    w = int4_pack(codes, scales, zeros, group_size=32)
    assert tuple(w.codes.shape) == (2, 3, 64, 4) and tuple(w.scales.shape) == (2, 3, 16, 4)
    words = w.codes.numpy().view(np.uint32)
    for out in range(32):
        for inp in range(384):
            t, kt, j, g, i = out // 16, inp // 128, inp % 128 // 32, inp % 32 // 8, inp % 8
            shift = 2 * i if i % 2 == 0 else 14 + 2 * i
            got = (int(words[t, kt, 16 * g + out % 16, j]) >> shift) & 15
            if out < n:     # inputs past the width weigh nothing: the zero point
                assert got == (int(codes[out, inp]) if inp < k else
                               int(zeros[out, 9]) if inp < 320 else 0), (out, inp)
    for out in range(n):
        for group in range(10):
            place = (out // 16, group // 4, out % 16, group % 4)
            assert w.scales[place] == scales[out, group] and w.zeros[place] == zeros[out, group]
    want = (codes.float() - zeros.float().repeat_interleave(32, 1)[:, :k]) * (
        scales.float().repeat_interleave(32, 1)[:, :k])
    assert torch.equal(w.dequantize(), want)


def test_packing_takes_strided_codes():
    gen = torch.Generator().manual_seed(1)
    codes = torch.randint(0, 16, (80, 40), generator=gen, dtype=torch.uint8)
    scales = torch.rand(2, 40, generator=gen).half()
    a = int4_pack(codes.t(), scales.t(), group_size=64)
    b = int4_pack(codes.t().contiguous(), scales.t().contiguous(), group_size=64)
    assert torch.equal(a.codes, b.codes) and torch.equal(a.scales, b.scales)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("zero_points", [False, True])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_quantized_weight_is_the_nearest_code(dtype, zero_points, group):
    """Off by half a step of the group, plus what the code range's ends lose:
    the scale's own rounding moves the end of 7 (15 with zero points) steps by
    at most 7 (15) times half the type's step."""
    gen = torch.Generator().manual_seed(2)
    w = (torch.randn(19, 330, generator=gen) * 0.02).to(dtype)
    w[3, :group] = 0
    q = int4_quantize(w, group_size=group, zero_points=zero_points)
    nt = q.scales.shape[0]
    steps = q.scales.permute(0, 2, 1, 3).reshape(nt * 16, -1)[:19].float()
    step = steps.repeat_interleave(group, 1)[:, :330]
    off = (q.dequantize() - w.float()).abs()
    end = torch.finfo(dtype).eps / 2 * (15 if zero_points else 7)
    # with zero points the zero's own rounding shifts both ends by half a step
    assert (off <= step * ((1.0 if zero_points else 0.5) + end) * (1 + 1e-6)).all()
    assert (q.dequantize()[3, :group] == 0).all()


@pytest.mark.parametrize("zero_points", [False, True])
def test_quantizing_takes_finite_weights_and_no_others(zero_points):
    """Large values of both signs have a range past the type's; an infinity or NaN has
    no code, nor bf16 values whose range passes 32 bits."""
    for dtype, top in ((torch.bfloat16, 2.0 ** 127 - 2.0 ** 119), (torch.float16, 65504.0),
                       (torch.bfloat16, torch.finfo(torch.bfloat16).max)):
        w = torch.zeros(3, 130, dtype=dtype)
        w[0, 0], w[0, 1], w[1, 129] = top, -top, -top
        if top > 2.0 ** 127:
            with pytest.raises(RuntimeError, match="finite"):
                int4_quantize(w, group_size=64, zero_points=zero_points)
            continue
        q = int4_quantize(w, group_size=64, zero_points=zero_points)
        got = q.dequantize().double()
        step = top / (7.5 if zero_points else 7)
        # half a step, as much again for the zero point's own rounding, and what the
        # scale's rounding moves the range's end by
        off = step * ((1.0 if zero_points else 0.5) + 15 * torch.finfo(dtype).eps / 2)
        assert (got - w.double()).abs().max() <= off
        for bad in (float("nan"), float("inf"), -float("inf")):
            broken = w.clone()
            broken[2, 70] = bad
            with pytest.raises(RuntimeError, match="finite"):
                int4_quantize(broken, group_size=64, zero_points=zero_points)


def _walk(parents, starts, words):
    bits = np.zeros((len(parents), words), dtype=np.uint32)
    for b in range(len(starts) - 1):
        for r in range(starts[b], starts[b + 1]):
            j = r - starts[b]
            while True:
                bits[r, j // 32] |= np.uint32(1 << (j % 32))
                p = int(parents[starts[b] + j])
                if not 0 <= p < j:
                    break
                j = p
    return bits.view(np.int32)


@pytest.mark.parametrize("lens", [[1], [5, 0, 1, 33], [64, 7], [100], [0, 3], [32, 31, 65]])
def test_ancestors_match_a_walk(lens):
    gen = torch.Generator().manual_seed(sum(lens))
    starts = np.concatenate([[0], np.cumsum(lens)])
    parents = []
    for t in lens:
        for j in range(t):
            parents.append(int(torch.randint(-1, j, (1,), generator=gen)) if j else -1)
    chain = [j - 1 for t in lens for j in range(t)]
    for p in (parents, chain):
        got = tree_ancestors(torch.tensor(p, dtype=torch.int32),
                             torch.tensor(starts, dtype=torch.int32), max(lens))
        assert got.dtype == torch.int32
        assert np.array_equal(got.numpy(), _walk(p, starts, -(-max(lens) // 32)))


def test_a_parent_that_is_no_earlier_node_is_the_context():
    starts = torch.tensor([0, 3, 5], dtype=torch.int32)
    got = tree_ancestors(torch.tensor([5, 1, 2, 1, -7]), starts, 3)
    assert got.view(-1).tolist() == [1, 2, 4, 1, 2]
    assert tree_ancestors(torch.empty(0, dtype=torch.int64), starts * 0, 4).shape == (0, 1)


# --- refusals: nothing is launched ---------------------------------------------

def _int4_args(**over):
    a = dict(x=1 << 20, xs=256, codes=1 << 21, scales=1 << 22, zeros=None, bias=None, y=1 << 23,
             ys=64, rows=4, n=64, k=256, group=128, fp16=0, stream=None)
    a.update(over)
    return list(a.values())


def test_int4_linear_refuses():
    lib = _lib.load()
    f = lib.qsa_int4_linear
    assert f(*_int4_args(rows=0)) == 0 and f(*_int4_args(n=0)) == 0
    assert f(*_int4_args(group=48)) == -2 and b"group size" in lib.qsa_last_error()
    assert f(*_int4_args(group=256)) == -2
    assert f(*_int4_args(k=0)) == -2
    assert f(*_int4_args(rows=-1)) == -1 and f(*_int4_args(xs=-8)) == -1
    assert f(*_int4_args(x=None)) == -1 and f(*_int4_args(scales=None)) == -1
    assert f(*_int4_args(codes=(1 << 21) + 4)) == -1 and b"misaligned" in lib.qsa_last_error()
    assert f(*_int4_args(x=(1 << 20) + 1)) == -1
    assert f(*_int4_args(ys=32)) == -1 and b"overlap" in lib.qsa_last_error()
    assert f(*_int4_args(rows=1 << 30, n=1 << 24, ys=1 << 24)) == -2
    assert f(*_int4_args(rows=2**31 - 1, n=64)) == -2
    # more threads than a launch holds, offsets past 64 bits, a width past 2^30
    assert f(*_int4_args(rows=1 << 27, n=16, xs=256)) == -2
    assert f(*_int4_args(xs=2**61)) == -2 and f(*_int4_args(k=2**30 + 1)) == -2


@pytest.mark.parametrize("rows,n,k,x", [
    (1 << 26, 16, 256, 1 << 20), ((1 << 25) - 31, 16, 256, 1 << 20), (1 << 24, 1 << 20, 256, 1 << 20),
    (1 << 28, 16, 2048, (1 << 20) + 2), (2**31 - 1, 1, 64, (1 << 20) + 2), (2**31 - 64, 1, 8, 1 << 20),
    (1, 2**31 - 1, 256, 1 << 20), (5, (1 << 31) - 512, 1024, 1 << 20)])
def test_int4_linear_refuses_more_threads_than_a_launch_holds(rows, n, k, x):
    """By the blocks of the very launch, whatever they are rounded up to: a
    refusal, not a launch that fails. (32 rows x 8 blocks of 512 threads: 2^25 - 31
    rows are one block too many.)"""
    lib = _lib.load()
    assert lib.qsa_int4_linear(*_int4_args(rows=rows, n=n, k=k, x=x, ys=2**31)) == -2
    assert b"too many rows" in lib.qsa_last_error()


def _tree_args(**over):
    a = dict(q=1 << 20, qr=2048, qh=128, rows=8, hq=16, d=128, k=1 << 21, kb=8192, kt=512, kh=256,
             v=(1 << 21) + 256, vb=8192, vt=512, vh=256, blocks=64, page=16, hkv=2, table=1 << 23,
             tr=4, tw=4, nreq=2, ctx=1 << 24, qsl=1 << 25, anc=1 << 26, ar=1, words=1, out=1 << 27,
             outr=2048, outh=128, gate=None, gr=0, gh=0, gd=0, mq=4, mc=60, ws=None, wsb=0,
             stream=None)
    a.update(over)
    return list(a.values())


def test_tree_attention_refuses():
    lib = _lib.load()
    f = lib.qsa_tree_attention
    assert f(*_tree_args(rows=0)) == 0 and f(*_tree_args(nreq=0)) == 0
    assert f(*_tree_args(mq=0)) == 0                   # no request has a node
    assert f(*_tree_args(d=96)) == -2 and b"head_dim" in lib.qsa_last_error()
    assert f(*_tree_args(hq=15)) == -2 and f(*_tree_args(hkv=0)) == -2
    assert f(*_tree_args(page=0)) == -1
    assert f(*_tree_args(rows=-1)) == -1 and f(*_tree_args(mc=-1)) == -1
    assert f(*_tree_args(q=(1 << 20) + 8)) == -1 and f(*_tree_args(kt=516)) == -1
    assert f(*_tree_args(outr=2047)) == -1
    # 64 GiB of cache from the first row to the last is too far apart, a page
    # table and a batch whose stages pass 31 bits too much
    assert f(*_tree_args(kb=2**32, blocks=10)) == -2 and b"64 GiB" in lib.qsa_last_error()
    assert f(*_tree_args(vt=2**40)) == -2 and f(*_tree_args(vb=-8192)) == -2
    assert f(*_tree_args(kt=2**62)) == -2
    assert f(*_tree_args(nreq=1 << 20, tw=1 << 20, rows=1 << 20, mq=1)) == -2
    assert f(*_tree_args(nreq=1, rows=2**31 - 1, mq=2**31 - 1)) == -2
    for name in ("q", "k", "v", "table", "ctx", "qsl", "anc", "out"):
        assert f(*_tree_args(**{name: None})) == -1, name
    need = lib.qsa_tree_attention_workspace_bytes(8, 2, 16, 2, 128, 4, 60000)
    assert need > 0
    assert f(*_tree_args(mc=60000)) == -4 and b"workspace" in lib.qsa_last_error()
    assert f(*_tree_args(mc=60000, ws=1 << 28, wsb=need - 1)) == -4
    assert f(*_tree_args(mc=60000, ws=(1 << 28) + 4, wsb=need)) == -4
    assert lib.qsa_tree_attention_workspace_bytes(8, 2, 16, 2, 128, 4, 60) == 0


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("nreq,mq,hq,mc", [
    (1 << 24, 1, 16, 60000),        # joining: 2^24 requests of at least one workgroup each
    (1 << 18, 64, 32, 60000),       # 2^18 x 64 x 32 (row, head)s, 8 or 16 a workgroup
    (1 << 24, 1, 2, 0),             # attention: a workgroup for each request and kv head
])
def test_tree_attention_refuses_more_threads_than_a_launch_holds(d, nreq, mq, hq, mc):
    """Either launch's, before the first: a refused call writes nothing."""
    lib = _lib.load()
    args = dict(rows=min(nreq * mq, 2**31 - 1), hq=hq, hkv=2, d=d, tw=1, nreq=nreq, mq=mq, mc=mc,
                ws=1 << 30, wsb=1 << 40)
    assert lib.qsa_tree_attention(*_tree_args(**args)) == -2
    assert b"too many" in lib.qsa_last_error()


def test_tree_attention_workspace_stays_in_proportion():
    """Two pieces of at most 128 rows for each of at most 512 workgroups (and 8 for
    each 128 rows of a request and kv head), whatever the context and the batch."""
    f = _lib.load().qsa_tree_attention_workspace_bytes
    for rows, nreq, most, ctx in ((1, 1, 1, 2**30), (64, 1, 64, 131072), (64, 64, 1, 131072),
                                  (4096, 64, 64, 524288)):
        assert 0 < f(rows, nreq, 16, 2, 128, most, ctx) <= (
            2 * (512 + 8 * -(-most * 8 // 128)) * min(128, max(16, most * 8)) * 129 * 4)
    assert f(0, 1, 16, 2, 128, 1, 1000) == 0 and f(4, 1, 16, 0, 128, 1, 1000) == 0


def _logits_args(**over):
    a = dict(x=1 << 20, type=1, xr=1000, out=1 << 22, outr=1000, rows=4, vocab=1000, first=0,
             t2r=None, nreq=4, hist=None, hr=0, hw=0, lens=None, prompts=None, rep=None, freq=None,
             pres=None, bids=None, bir=0, bvals=None, bvr=0, nb=0, allowed=None, alr=0,
             draft=None, anc=None, ancr=0, words=0, qsl=None, stream=None)
    a.update(over)
    return list(a.values())


def test_process_logits_refuses():
    lib = _lib.load()
    f = lib.qsa_process_logits
    assert f(*_logits_args(rows=0)) == 0 and f(*_logits_args(vocab=0)) == 0
    assert f(*_logits_args(type=3)) == -2
    assert f(*_logits_args(x=None)) == -1 and f(*_logits_args(out=None)) == -1
    assert f(*_logits_args(rows=-1)) == -1 and f(*_logits_args(first=-5)) == -1
    assert f(*_logits_args(hist=1 << 23)) == -1 and b"lengths" in lib.qsa_last_error()
    assert f(*_logits_args(nb=3)) == -1
    assert f(*_logits_args(nb=1 << 20, bids=1 << 23, bvals=1 << 24)) == -2
    assert f(*_logits_args(anc=1 << 23)) == -1
    assert f(*_logits_args(anc=1 << 23, words=33, draft=1 << 24, qsl=1 << 25)) == -2
    assert f(*_logits_args(nb=1025, bids=1 << 23, bvals=1 << 24)) == -2
    assert f(*_logits_args(first=2**31 - 1000, vocab=1000)) == -1
    assert f(*_logits_args(rows=2**31 - 1)) == -2 and f(*_logits_args(rows=1 << 24, vocab=1)) == -2
    assert f(*_logits_args(x=(1 << 20) + 1)) == -1 and f(*_logits_args(out=(1 << 22) + 2)) == -1


def test_python_layer_refuses():
    codes = torch.zeros(16, 128, dtype=torch.uint8)
    scales = torch.ones(16, 1, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="group size"):
        int4_pack(codes, scales, group_size=16)
    with pytest.raises(RuntimeError, match="codes must be uint8"):
        int4_pack(codes.int(), scales)
    with pytest.raises(RuntimeError, match="scales must be"):
        int4_pack(codes, scales.float())
    with pytest.raises(RuntimeError, match="scales must be"):
        int4_pack(codes, scales, group_size=64)
    with pytest.raises(RuntimeError, match="zeros must be"):
        int4_pack(codes, scales, scales)
    with pytest.raises(RuntimeError, match="input features"):
        int4_pack(codes[:, :0], scales[:, :0])
    with pytest.raises(RuntimeError, match="weight must be"):
        int4_quantize(scales.float())
    # CPU tensors: there is no CPU kernel.
    w = int4_pack(codes, scales)
    with pytest.raises(RuntimeError):
        int4_linear(torch.zeros(1, 128, dtype=torch.bfloat16), w)
    with pytest.raises(RuntimeError):
        process_logits(torch.zeros(1, 8))
    i32 = torch.zeros(2, dtype=torch.int32)
    kv = torch.zeros(1, 16, 1, 64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError):
        qsa_tree_paged_attention(torch.zeros(1, 1, 64, dtype=torch.bfloat16), kv, kv, i32[:1, None],
                                 i32[:1], i32, i32[:1, None], max_query_len=1, max_context_len=1)
    with pytest.raises(RuntimeError, match="max_query_len"):
        tree_ancestors(i32, i32, 0)
    with pytest.raises(RuntimeError, match="parents"):
        tree_ancestors(i32.float(), i32, 1)


# --- a captured step keeps what its kernels read ---------------------------------

def test_a_captured_step_keeps_its_rules(monkeypatch):
    """The kernels of a graph hold addresses, not tensors: the rules' tensors
    must live as long as the graph, also where the caller's object is dropped or
    its fields get other tensors."""
    stream = types.SimpleNamespace(wait_stream=lambda other: None)
    for name, value in (("Stream", lambda: stream), ("current_stream", lambda: stream),
                        ("stream", lambda s: contextlib.nullcontext()),
                        ("synchronize", lambda: None), ("CUDAGraph", lambda: None),
                        ("graph", lambda g: contextlib.nullcontext())):
        monkeypatch.setattr(torch.cuda, name, value)
    batch = types.SimpleNamespace(
        num_tokens=2, qsa=types.SimpleNamespace(main=types.SimpleNamespace(max_query_len=1)))
    model = types.SimpleNamespace(cfg=types.SimpleNamespace(compress_ratio=4),
                                  forward=lambda batch, rules: torch.zeros(2, 8))
    rules = LogitsRules(frequency=torch.ones(2), presence=torch.ones(2), vocab_start=8)
    alive = [weakref.ref(rules.frequency), weakref.ref(rules.presence)]
    graph = HybridDecodeGraph(model, batch, rules=rules)
    rules.frequency = torch.zeros(2)
    del rules
    gc.collect()
    assert all(ref() is not None for ref in alive)
    del graph
    gc.collect()
    assert all(ref() is None for ref in alive)
    assert HybridDecodeGraph(model, batch).rules is None
