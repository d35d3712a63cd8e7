"""The operators of a step over a few tokens as they are used together, and in
the hybrid decoder.

The verification of drafted trees on one attention layer: 4-bit query/key/value
projection of the nodes, their K/V written to the cache, tree attention, 4-bit
output projection, 4-bit LM head, rules on the nodes' logits. Every stage is
checked against 64 bits on the stage's own inputs (so rounding does not
accumulate), with its operator's tolerance: fp32 sums as in the tests of each
operator, and half a step of the output type (bf16 2^-8)."""

import math

import pytest
import torch

from qsa_vllm_amd.hybrid import (HybridConfig, HybridDecodeGraph, make_hybrid_workload)
from qsa_vllm_amd.ops import (LogitsRules, int4_linear, int4_quantize, process_logits,
                              qsa_store_cache_rows, qsa_tree_paged_attention, tree_ancestors)

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24


def _check_linear(x, weight, got, bias=None):
    w = weight.dequantize().cpu().double()
    xd = x.cpu().double()
    y = xd @ w.t()
    if bias is not None:
        y = y + bias.cpu().double()
    scale = weight.scales.float().max().item()
    sums = U * (36 * 286 * scale * xd.abs().sum(1, keepdim=True)
                + (w.shape[1] / 32 + 12) * (xd.abs() @ w.abs().t()) + y.abs())
    off = (got.cpu().double() - y).abs()
    assert (off <= sums + 2.0 ** -8 * (y.abs() + sums)).all()


class Verify:
    heads, kv_heads, dim, hidden, vocab, page = 8, 2, 64, 256, 1000, 16

    def __init__(self, seed=0):
        gen = torch.Generator().manual_seed(seed)
        self.ctx, self.nodes = [90, 300, 7], [9, 1, 14]
        rows, d = sum(self.nodes), self.dim
        starts = torch.tensor([0] + self.nodes).cumsum(0)
        parents = torch.tensor([int(torch.randint(-1, j, (1,), generator=gen)) if j else -1
                                for t in self.nodes for j in range(t)])
        def weight(n, k):
            return int4_quantize((torch.randn(n, k, generator=gen) * 0.05).bfloat16().to(DEV),
                                 group_size=64, zero_points=True)
        qkv = (self.heads + 2 * self.kv_heads) * d
        self.w_qkv, self.w_o = weight(qkv, self.hidden), weight(self.hidden, self.heads * d)
        self.w_head = weight(self.vocab, self.hidden)
        self.bias = (torch.randn(qkv, generator=gen) * 0.1).bfloat16().to(DEV)
        pages = [-(-(c + t) // self.page) for c, t in zip(self.ctx, self.nodes)]
        order = torch.randperm(sum(pages) + 1, generator=gen)
        table = torch.full((3, max(pages)), -1, dtype=torch.int32)
        at = 0
        for b, p in enumerate(pages):
            table[b, :p] = order[at:at + p].int()
            at += p
        kv = torch.randn(len(order), self.page, self.kv_heads, 2 * d, generator=gen).bfloat16()
        slots = [int(table[b, (c + j) // self.page]) * self.page + (c + j) % self.page
                 for b, (c, t) in enumerate(zip(self.ctx, self.nodes)) for j in range(t)]
        req = torch.repeat_interleave(torch.arange(3), torch.tensor(self.nodes))
        i32 = dict(dtype=torch.int32, device=DEV)
        self.x = torch.randn(rows, self.hidden, generator=gen).bfloat16().to(DEV)
        self.kv, self.table = kv.to(DEV), table.to(DEV)
        self.slots = torch.tensor(slots, dtype=torch.int64, device=DEV)
        self.ctx_lens, self.qsl = torch.tensor(self.ctx, **i32), starts.to(**i32)
        self.parents, self.req = parents.to(DEV), req.to(**i32)
        self.draft = torch.randint(0, 40, (rows,), generator=gen).to(**i32)
        self.rules = LogitsRules(
            history=torch.randint(0, 60, (3, 300), generator=gen).to(**i32),
            history_lens=self.ctx_lens, prompt_lens=self.ctx_lens // 2,
            repetition=torch.tensor([1.2, 1.0, 1.4], device=DEV),
            frequency=torch.tensor([0.1, 0.0, 0.3], device=DEV),
            presence=torch.tensor([0.2, 0.5, 0.0], device=DEV),
            bias_ids=torch.randint(0, 60, (3, 4), generator=gen).to(**i32),
            bias_values=torch.randn(3, 4, generator=gen).to(DEV),
            allowed=torch.randint(-2**31, 2**31, (rows, 32), generator=gen).to(**i32))

    def step(self):
        d = self.dim
        anc = tree_ancestors(self.parents, self.qsl, max(self.nodes))
        qkv = int4_linear(self.x, self.w_qkv, self.bias)
        q, k, v = qkv.split((self.heads * d, self.kv_heads * d, self.kv_heads * d), dim=1)
        rows = torch.cat([k.view(-1, self.kv_heads, d), v.view(-1, self.kv_heads, d)], dim=-1)
        qsa_store_cache_rows(self.kv.view(self.kv.shape[0], self.page, 1, -1), self.slots,
                             rows.reshape(len(rows), -1))
        out = qsa_tree_paged_attention(q.view(-1, self.heads, d), self.kv[..., :d],
                                       self.kv[..., d:], self.table, self.ctx_lens, self.qsl, anc,
                                       max_query_len=max(self.nodes), max_context_len=300)
        hidden = int4_linear(out.view(len(out), -1), self.w_o)
        logits = int4_linear(hidden, self.w_head)
        final = process_logits(logits, token_to_req=self.req, draft_tokens=self.draft,
                               ancestors=anc, query_start_loc=self.qsl, **vars(self.rules))
        return anc, qkv, out, hidden, logits, final


def test_verification_step_stage_by_stage():
    s = Verify()
    anc, qkv, out, hidden, logits, final = (t.clone() for t in s.step())
    _check_linear(s.x, s.w_qkv, qkv, s.bias)
    _check_linear(out.view(len(out), -1), s.w_o, hidden)
    _check_linear(hidden, s.w_head, logits)
    # attention over the cache that holds the nodes' rows
    d, group = s.dim, s.heads // s.kv_heads
    kv, table, anc, parents = s.kv.cpu(), s.table.cpu(), anc.cpu(), s.parents.cpu()
    q = qkv.cpu()[:, :s.heads * d].view(-1, s.heads, d)
    row = 0
    for b, (c, t) in enumerate(zip(s.ctx, s.nodes)):
        first = row
        for j in range(t):
            path, p = [], j
            while p >= 0:
                path.append(p)
                p = int(parents[first + p])
            assert int(anc[row, 0]) == sum(1 << p for p in path)
            seen = list(range(c)) + [c + p for p in sorted(path)]
            rows = kv[[int(table[b, p // s.page]) for p in seen], [p % s.page for p in seen]].double()
            for h in range(s.heads):
                k, v = rows[:, h // group, :d], rows[:, h // group, d:]
                w = torch.softmax(k @ q[row, h].double() / math.sqrt(d), 0)
                o, mass = w @ v, w @ v.abs()
                spread = (k.abs() @ q[row, h].double().abs()).max().item() / math.sqrt(d)
                rel = 2 ** -8 + 72 * U * spread + 2 ** -18
                off = (out[row, h].cpu().double() - o).abs()
                assert (off <= rel * mass + 2 ** -8 * (o.abs() + rel * mass)).all()
            row += 1
    # rules: the node's path counts as said
    r = s.rules
    for row in range(len(out)):
        b = int(s.req[row])
        n, prompt = s.ctx[b], s.ctx[b] // 2
        said = {}
        for tok in r.history[b, prompt:n].tolist():
            said[tok] = said.get(tok, 0) + 1
        ever = set(r.history[b, :n].tolist())
        for j in range(s.nodes[b]):
            if (int(anc[row, 0]) >> j) & 1:
                tok = int(s.draft[int(s.qsl[b]) + j])
                said[tok] = said.get(tok, 0) + 1
                ever.add(tok)
        x, got = logits[row].cpu().double(), final[row].cpu().double()
        rep, f, p = (float(t[b]) for t in (r.repetition, r.frequency, r.presence))
        for tok in range(s.vocab):
            y = float(x[tok])
            m = abs(y) * max(rep, 1 / rep)
            if tok in ever:
                y = y / rep if y > 0 else y * rep
            if said.get(tok):
                y -= f * said[tok] + p
                m += f * said[tok] + p
            for i in range(4):
                if int(r.bias_ids[b, i]) == tok:
                    y += float(r.bias_values[b, i])
                    m += abs(float(r.bias_values[b, i]))
            if not (int(r.allowed[row, tok // 32]) >> (tok % 32)) & 1:
                assert got[tok] == -math.inf
            else:
                assert abs(got[tok] - y) <= 8 * U * m + 2.0 ** -149


def test_verification_step_in_a_graph():
    """Captured once; every replay, on new nodes, rules and lengths, equals the
    eager step, with eager work in between."""
    s = Verify(seed=1)
    s.step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = s.step()
    gen = torch.Generator().manual_seed(2)
    for i in range(4):
        s.x.copy_(torch.randn(s.x.shape, generator=gen).bfloat16())
        s.draft.copy_(torch.randint(0, 40, s.draft.shape, generator=gen))
        s.ctx_lens.sub_(1)
        s.rules.frequency.add_(0.05)
        kv = s.kv.clone()
        graph.replay()
        got = [t.clone() for t in captured]
        torch.cuda.synchronize()
        s.kv.copy_(kv)
        for a, b in zip(got, s.step()):
            assert torch.equal(a, b)


def test_two_graphs_share_nothing():
    """Two captured steps replayed in turn and on two streams at once: each has
    its own workspace."""
    steps = [Verify(seed=3), Verify(seed=4)]
    graphs, outs, want = [], [], []
    for s in steps:
        s.ctx_lens.fill_(0)
        s.ctx_lens.add_(torch.tensor(s.ctx, dtype=torch.int32, device=DEV))
        want.append([t.clone() for t in s.step()])
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(s.step())
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in steps]
    for _ in range(5):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    for o, w in zip(outs, want):
        for a, b in zip(o, w):
            assert torch.equal(a, b)


# --- in the hybrid decoder ----------------------------------------------------

CFG = dict(num_layers=4, hidden_size=512, vocab_size=512, tp_size=2, num_heads=32, num_kv_heads=4,
           head_dim=128, intermediate_size=1024, linear_num_key_heads=4, linear_num_value_heads=8,
           indexer_heads=8, token_topk=256, init_std=0.05)


def _workload(**over):
    return make_hybrid_workload(HybridConfig(**{**CFG, **over}), decode_lens=[700, 1500, 33, 260],
                                chunk_prefixes=[0, 300], chunk=100, device=DEV, seed=5,
                                state_std=0.05)


def _rules(requests, shard):
    gen = torch.Generator().manual_seed(6)
    i32 = dict(dtype=torch.int32, device=DEV)
    return LogitsRules(
        history=torch.randint(0, shard, (requests, 64), generator=gen).to(**i32),
        history_lens=torch.full((requests,), 64, **i32), prompt_lens=torch.full((requests,), 20, **i32),
        repetition=torch.full((requests,), 1.3, device=DEV),
        frequency=torch.full((requests,), 0.2, device=DEV),
        presence=torch.full((requests,), 0.4, device=DEV),
        allowed=torch.randint(-2**31, 2**31, (requests, -(-shard // 32)), generator=gen).to(**i32))


@pytest.mark.parametrize("group", [32, 128])
def test_decoder_with_4_bit_weights(group):
    """Every projection of a step is the product with its dequantized weight, on
    the step's own activations: prompts and decode rows in one batch."""
    import qsa_vllm_amd.hybrid as H

    wl = _workload(weight_bits=4, weight_group=group)
    seen = []
    plain = H._linear
    try:
        def watch(x, w, bias=None):
            y = plain(x, w, bias)
            seen.append((x.clone(), w, y.clone(), bias))
            return y
        H._linear = watch
        logits = wl.model.forward(wl.build())
    finally:
        H._linear = plain
    # four layers of two mixer and two MLP projections, and the LM head
    assert len(seen) == 17 and torch.isfinite(logits).all()
    assert logits.dtype == torch.float32 and logits.shape == (6, 256)
    for x, w, y, bias in seen:
        assert w.group_size == group
        _check_linear(x.reshape(-1, x.shape[-1]), w, y.reshape(-1, y.shape[-1]), bias)


@pytest.mark.parametrize("bits", [4, 16])
def test_decoder_applies_the_rules(bits):
    wl = _workload(weight_bits=bits)
    batch = wl.build_decode()
    states = [t.clone() for t in wl.layer_states()]

    def reset():
        for t, s in zip(wl.layer_states(), states):
            t.copy_(s)
    plain = wl.model.forward(batch).clone()
    reset()
    rules = _rules(4, wl.cfg.vocab_shard)
    ruled = wl.model.forward(batch, rules).clone()
    assert torch.equal(ruled, process_logits(plain, **vars(rules)))
    assert (ruled == -math.inf).any() and not torch.equal(ruled, plain)
    # captured: the rules' buffers are read anew
    reset()
    graph = HybridDecodeGraph(wl.model, batch, rules=rules)
    for step in range(3):
        reset()
        rules.frequency.add_(0.1)
        got = graph.replay().clone()
        torch.cuda.synchronize()
        assert torch.equal(got, process_logits(plain, **vars(rules)))


def test_weight_bits_are_checked():
    with pytest.raises(ValueError, match="weight_bits"):
        HybridConfig(weight_bits=8)


def test_a_graph_of_passing_rules():
    """The caller's rules are dropped after the capture and memory of their sizes
    is allocated and filled anew: the replays apply the rules all the same."""
    wl = _workload(weight_bits=4)
    batch = wl.build_decode()
    states = [t.clone() for t in wl.layer_states()]

    def reset():
        for t, s in zip(wl.layer_states(), states):
            t.copy_(s)
    want = wl.model.forward(batch, _rules(4, wl.cfg.vocab_shard)).clone()
    reset()
    graph = HybridDecodeGraph(wl.model, batch, rules=_rules(4, wl.cfg.vocab_shard))
    over = [torch.zeros_like(t) for _ in range(8) for t in vars(_rules(4, wl.cfg.vocab_shard)).values()
            if isinstance(t, torch.Tensor)]
    for step in range(3):
        reset()
        got = graph.replay().clone()
        torch.cuda.synchronize()
        assert torch.equal(got, want)
    del over
