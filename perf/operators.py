"""Operators of a serving step over a few tokens, as measurable cases.

Three operators of the step that verifies drafted tokens (or decodes single
ones) next to the sparse path, each on the sizes of the hybrid decoder (hidden
size 4096, 16 query and 2 key/value heads of 128 dims on one of two GPUs, pages
of 16 tokens, contexts up to 131072, a vocabulary of 99072 or a shard of it):

* ``int4``: a projection with 4-bit weights, group scales and, for some,
  zero points, on a few activation rows;
* ``tree``: attention of a request's drafted token tree over its committed
  context and its ancestors in the tree, all in the paged cache;
* ``logits``: penalties for repeated tokens, biases and grammar masks on the
  logits of decode rows or of drafted nodes.

``own`` chooses between the plain form (elementary torch operations in 32 bits)
and the package's entry points.
"""

from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda:0"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _int4(name, rows, n, k, group=128, zeros=False, bias=False, dtype="bf16"):
    return dict(name=name, kind="int4", rows=rows, n=n, k=k, group=group, zeros=zeros, bias=bias,
                dtype=dtype)


def _tree(name, requests, nodes_min, nodes_max, ctx_min, ctx_max, heads=16, kv_heads=2, dim=128,
          page=16, gate=False):
    return dict(name=name, kind="tree", requests=requests, nodes_min=nodes_min, nodes_max=nodes_max,
                ctx_min=ctx_min, ctx_max=ctx_max, heads=heads, kv_heads=kv_heads, dim=dim, page=page,
                gate=gate)


def _logits(name, requests, nodes, vocab, hist_min, hist_max, biases=0, grammar=True, dtype="bf16",
            shard=False):
    return dict(name=name, kind="logits", requests=requests, nodes=nodes, vocab=vocab,
                hist_min=hist_min, hist_max=hist_max, biases=biases, grammar=grammar, dtype=dtype,
                shard=shard)


def listed():
    return [
        # One user's next token through an attention output projection.
        _int4("int4_1_o_proj", 1, 4096, 2048),
        # The same token through the LM head shard.
        _int4("int4_1_lm_head", 1, 49536, 4096),
        # A verified tree of 61 drafted tokens through a gated MLP's first projection.
        _int4("int4_61_gate_up", 61, 11264, 4096),
        # Seven users through the MLP's second projection, small groups with zero points.
        _int4("int4_7_down_g32", 7, 4096, 5632, group=32, zeros=True, bias=True, dtype="fp16"),
        # 250 decode rows through a whole MLP's first projection, groups of 64 with zero points.
        _int4("int4_250_gate_up_g64", 250, 22528, 4096, group=64, zeros=True),
        # One user's small draft on a short chat.
        _tree("tree_1x8_on_500", 1, 8, 8, 500, 500),
        # Single tokens of 64 users over their whole context.
        _tree("tree_64x1_on_8k", 64, 1, 1, 1024, 8192),
        # 32 users with drafts of different sizes at 4k-32k, gated output.
        _tree("tree_32x16_on_32k", 32, 5, 24, 4096, 32768, gate=True),
        # One user's full tree on a very long context.
        _tree("tree_1x64_on_128k", 1, 64, 64, 131072, 131072),
        # One user's next token, the shard's logits.
        _logits("logits_1", 1, 0, 49536, 1000, 1000, biases=16, shard=True),
        # 128 users at once, the whole vocabulary in 32 bits.
        _logits("logits_128", 128, 0, 99072, 512, 32768, biases=64, dtype="fp32"),
        # The nodes of eight users' drafted trees, each with its own grammar state.
        _logits("logits_8x61", 8, 61, 49536, 512, 16384, biases=16, shard=True),
    ]


def _log(rng, low, high):
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng: random.Random):
    kind = rng.choice(["int4", "tree", "logits"])
    if kind == "int4":
        rows = _log(rng, 1, 256)
        n = _log(rng, 256, 49536)
        k = 8 * _log(rng, 32, 1408)
        while rows * n * k > 250 * 22528 * 4096:
            n = max(256, n // 2)
        case = _int4("", rows, n, k, group=rng.choice([32, 64, 128]), zeros=rng.random() < 0.5,
                     bias=rng.random() < 0.3, dtype=rng.choice(["bf16", "bf16", "fp16"]))
    elif kind == "tree":
        requests = _log(rng, 1, 64)
        ctx_max = _log(rng, 16, min(131072, 1048576 // requests))
        nodes = _log(rng, 1, 64)
        while requests * nodes * ctx_max > 64 * 131072:
            nodes = max(1, nodes // 2)
            if nodes == 1:
                break
        kv_heads = rng.choice([1, 2, 2, 4])
        case = _tree("", requests, rng.randint(1, nodes), nodes, rng.randint(0, ctx_max), ctx_max,
                     heads=kv_heads * rng.choice([1, 4, 8, 8] if kv_heads < 4 else [2, 4]),
                     kv_heads=kv_heads, dim=rng.choice([64, 128, 128]),
                     page=rng.choice([16, 16, 48, 272]), gate=rng.random() < 0.5)
    else:
        nodes = rng.choice([0, 0, _log(rng, 1, 64)])
        requests = _log(rng, 1, 128 if nodes == 0 else max(1, 512 // nodes))
        vocab = _log(rng, 1000, 99072)
        while requests * max(1, nodes) * vocab > 128 * 99072:
            vocab //= 2
        hist_max = _log(rng, 16, 32768)
        case = _logits("", requests, nodes, vocab, rng.randint(0, hist_max), hist_max,
                       biases=rng.choice([0, 5, 64, 300]), grammar=rng.random() < 0.7,
                       dtype=rng.choice(["bf16", "fp32", "fp16"]), shard=rng.random() < 0.5)
    del case["name"]
    return case


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------

def _ragged(gen, count, low, high):
    """``count`` lengths in [low, high], the longest among them."""
    n = torch.randint(low, high + 1, (count,), generator=gen)
    n[int(torch.randint(0, count, (1,), generator=gen))] = high
    return n.tolist()


def _tree_lengths(case):
    """Drafted nodes and committed tokens of each request: the case's own, the
    same whatever the inputs' seed."""
    gen = torch.Generator().manual_seed(case["requests"])
    nodes = _ragged(gen, case["requests"], case["nodes_min"], case["nodes_max"])
    return nodes, _ragged(gen, case["requests"], case["ctx_min"], case["ctx_max"])


def _random_trees(gen, nodes):
    """Per request, a random tree over its drafted tokens: parent of each node
    (an earlier one, -1 for the committed context) and the ancestor bits (its
    own among them) as 32-bit words."""
    words = -(-max(nodes, default=1) // 32)
    rows, bits = [], []
    for t in nodes:
        seen = []
        for j in range(t):
            parent = int(torch.randint(max(-1, j - 6), j, (1,), generator=gen)) if j else -1
            seen.append((seen[parent] if parent >= 0 else 0) | (1 << j))
            rows.append(parent)
        bits += seen

    def signed(word):
        return word - (1 << 32) if word >> 31 else word

    table = [[signed((b >> (32 * w)) & 0xFFFFFFFF) for w in range(words)] for b in bits]
    return rows, torch.tensor(table, dtype=torch.int32).reshape(len(bits), words)


def _starts(lengths):
    out = [0]
    for n in lengths:
        out.append(out[-1] + n)
    return out


def _prepare_int4(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    n, k, dtype = case["n"], case["k"], TYPES[case["dtype"]]
    groups = -(-k // case["group"])
    codes = torch.randint(0, 16, (n, k), generator=g, device=DEV, dtype=torch.uint8)
    scales = ((torch.rand(n, groups, generator=g, device=DEV) + 0.5) * 0.006).to(dtype)
    zeros = None
    if case["zeros"]:
        zeros = torch.randint(4, 12, (n, groups), generator=g, device=DEV, dtype=torch.uint8)
    bias = None
    if case["bias"]:
        bias = (torch.randn(n, generator=g, device=DEV) * 0.1).to(dtype)
    x = torch.randn(case["rows"], k, generator=g, device=DEV).to(dtype)
    state = dict(kind="int4", x=x, codes=codes, scales=scales, zeros=zeros, bias=bias,
                 group=case["group"])
    if own:
        from qsa_vllm_amd.ops import int4_pack
        state["weight"] = int4_pack(codes, scales, zeros, group_size=case["group"])
    return state


def _prepare_tree(case, seed):
    gen = torch.Generator().manual_seed(seed)
    g = torch.Generator(device=DEV).manual_seed(seed)
    nreq, page, dim = case["requests"], case["page"], case["dim"]
    nodes, ctx = _tree_lengths(case)
    _, ancestors = _random_trees(gen, nodes)
    pages = [-(-(c + t) // page) for c, t in zip(ctx, nodes)]
    order = torch.randperm(sum(pages) + 3, generator=gen).to(torch.int32)
    table = torch.full((nreq, max(pages)), -1, dtype=torch.int32)
    at = 0
    for i, p in enumerate(pages):
        table[i, :p] = order[at:at + p]
        at += p
    blocks = len(order)
    kv = torch.empty(blocks, page, case["kv_heads"], 2 * dim, dtype=torch.bfloat16, device=DEV)
    flat = kv.view(-1)
    step = 1 << 26
    for i in range(0, flat.numel(), step):
        n = min(step, flat.numel() - i)
        flat[i:i + n] = torch.randn(n, generator=g, device=DEV)
    rows = sum(nodes)
    q = (torch.randn(rows, case["heads"], dim, generator=g, device=DEV) * 2).to(torch.bfloat16)
    gate = None
    if case["gate"]:
        gate = torch.randn(rows, case["heads"], dim, generator=g, device=DEV).to(torch.bfloat16)
    starts = _starts(nodes)
    return dict(kind="tree", q=q, k_cache=kv[..., :dim], v_cache=kv[..., dim:], gate=gate,
                table=table.to(DEV), ctx=torch.tensor(ctx, dtype=torch.int32, device=DEV),
                starts=torch.tensor(starts, dtype=torch.int32, device=DEV),
                ancestors=ancestors.to(DEV), ctx_list=ctx, nodes_list=nodes)


def _prepare_logits(case, seed):
    gen = torch.Generator().manual_seed(seed)
    g = torch.Generator(device=DEV).manual_seed(seed)
    nreq, vocab = case["requests"], case["vocab"]
    total = 2 * vocab if case["shard"] else vocab      # ids of the whole vocabulary
    first = vocab if case["shard"] else 0               # this shard's first id
    nodes = [case["nodes"]] * nreq if case["nodes"] else [1] * nreq
    rows = sum(nodes)
    lens = _ragged(gen, nreq, case["hist_min"], case["hist_max"])
    prompt = [int(torch.randint(0, n + 1, (1,), generator=gen)) for n in lens]
    width = max(max(lens), 1)

    def words(*shape):  # token ids, the common ones often
        u = torch.rand(*shape, generator=g, device=DEV)
        return (u.pow(3) * total).long().clamp_(max=total - 1)

    logits = (torch.randn(rows, vocab, generator=g, device=DEV) * 3).to(TYPES[case["dtype"]])
    state = dict(
        kind="logits", logits=logits, first=first,
        history=words(nreq, width).to(torch.int32),
        history_lens=torch.tensor(lens, dtype=torch.int32, device=DEV),
        prompt_lens=torch.tensor(prompt, dtype=torch.int32, device=DEV),
        repetition=torch.rand(nreq, generator=g, device=DEV) * 0.5 + 1.0,
        frequency=torch.rand(nreq, generator=g, device=DEV) * 0.5,
        presence=torch.rand(nreq, generator=g, device=DEV) * 0.5,
        token_to_req=torch.repeat_interleave(
            torch.arange(nreq, dtype=torch.int32), torch.tensor(nodes)).to(DEV),
        bias_ids=None, bias_values=None, allowed=None, draft_tokens=None, ancestors=None,
        starts=None)
    if case["biases"]:
        ids = torch.stack([torch.randperm(total, generator=gen)[:case["biases"]]
                           for _ in range(nreq)])
        state["bias_ids"] = ids.to(torch.int32).to(DEV)
        state["bias_values"] = torch.randn(nreq, ids.shape[1], generator=g, device=DEV) * 4
    if case["grammar"]:
        # A third of the rows is free, a third allows about half of the words,
        # a third few of them.
        w = -(-vocab // 32)
        bits = torch.randint(-(1 << 31), 1 << 31, (rows, w), generator=g, device=DEV)
        few = bits & torch.randint(-(1 << 31), 1 << 31, (rows, w), generator=g, device=DEV)
        few &= torch.randint(-(1 << 31), 1 << 31, (rows, w), generator=g, device=DEV)
        state_of = torch.randint(0, 3, (rows, 1), generator=g, device=DEV)
        bits = torch.where(state_of == 0, torch.full_like(bits, -1),
                           torch.where(state_of == 1, bits, few))
        state["allowed"] = bits.to(torch.int32)
    if case["nodes"]:
        _, ancestors = _random_trees(gen, nodes)
        state["ancestors"] = ancestors.to(DEV)
        state["draft_tokens"] = words(rows).to(torch.int32)
        state["starts"] = torch.tensor(_starts(nodes), dtype=torch.int32, device=DEV)
    return state


def prepare(case, seed):
    return {"int4": _prepare_int4, "tree": _prepare_tree, "logits": _prepare_logits}[case["kind"]](
        case, seed)


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------

def _plain_int4(s):
    x, codes, group = s["x"], s["codes"], s["group"]
    n, k = codes.shape
    zero = s["zeros"].float() if s["zeros"] is not None else torch.full_like(s["scales"], 8.0,
                                                                             dtype=torch.float32)
    scale = s["scales"].float().repeat_interleave(group, dim=1)[:, :k]
    weight = (codes.float() - zero.repeat_interleave(group, dim=1)[:, :k]) * scale
    y = x.float() @ weight.t()
    if s["bias"] is not None:
        y = y + s["bias"].float()
    return y.to(x.dtype)


def _visible(ancestors, count):
    """[rows, count] truth values of the ancestor bits."""
    j = torch.arange(count, device=ancestors.device)
    return (ancestors[:, j // 32] >> (j % 32).to(torch.int32)) & 1 != 0


def _plain_tree(s):
    q, kc, vc = s["q"], s["k_cache"], s["v_cache"]
    _, page, kv_heads, dim = kc.shape
    heads = q.shape[1]
    group = heads // kv_heads
    out = torch.empty_like(q)
    row = 0
    for b, (ctx, t) in enumerate(zip(s["ctx_list"], s["nodes_list"])):
        used = s["table"][b, :-(-(ctx + t) // page)].long()
        seen = torch.ones(t, ctx + t, dtype=torch.bool, device=q.device)
        seen[:, ctx:] = _visible(s["ancestors"][row:row + t], t)
        seen = seen.repeat_interleave(group, dim=0)
        for h in range(kv_heads):
            k = kc[used, :, h].reshape(-1, dim)[:ctx + t].float()
            v = vc[used, :, h].reshape(-1, dim)[:ctx + t].float()
            mine = slice(h * group, (h + 1) * group)
            query = q[row:row + t, mine].float().reshape(t * group, dim)
            score = (query @ k.t()) * dim ** -0.5
            score = score.masked_fill(~seen, -math.inf)
            weight = (score - score.amax(dim=1, keepdim=True)).exp()
            o = (weight @ v) / weight.sum(dim=1, keepdim=True)
            o = o.view(t, group, dim)
            if s["gate"] is not None:
                o = o / (1 + (-s["gate"][row:row + t, mine].float()).exp())
            out[row:row + t, mine] = o.to(q.dtype)
        row += t
    return out


def _plain_logits(s):
    logits, req = s["logits"], s["token_to_req"].long()
    rows, vocab = logits.shape
    dev, first = logits.device, s["first"]
    nreq, width = s["history"].shape
    at = torch.arange(width, device=dev)
    ids = s["history"].long() - first
    here = (at < s["history_lens"][:, None]) & (ids >= 0) & (ids < vocab)
    slot = ids.clamp(0, vocab - 1)
    spoken = here & (at >= s["prompt_lens"][:, None])
    count = torch.zeros(nreq, vocab, dtype=torch.int32, device=dev)
    count.scatter_add_(1, slot, spoken.to(torch.int32))
    ever = torch.zeros(nreq, vocab, dtype=torch.int32, device=dev)
    ever.scatter_add_(1, slot, here.to(torch.int32))
    count, ever = count[req], ever[req]
    if s["draft_tokens"] is not None:
        most = int(s["ancestors"].shape[1]) * 32
        j = torch.arange(most, device=dev)
        node = s["starts"][req].long()[:, None] + j
        inside = node < s["starts"][req + 1].long()[:, None]
        token = s["draft_tokens"][node.clamp(max=rows - 1)].long() - first
        inside &= _visible(s["ancestors"], most) & (token >= 0) & (token < vocab)
        token = token.clamp(0, vocab - 1)
        count = count.scatter_add(1, token, inside.to(torch.int32))
        ever = ever.scatter_add(1, token, inside.to(torch.int32))
    y = logits.float()
    r = s["repetition"][req][:, None]
    y = torch.where(ever > 0, torch.where(y > 0, y / r, y * r), y)
    y = y - s["frequency"][req][:, None] * count
    y = y - s["presence"][req][:, None] * (count > 0)
    if s["bias_ids"] is not None:
        ids = s["bias_ids"].long() - first
        ok = (ids >= 0) & (ids < vocab)
        bias = torch.zeros(nreq, vocab, device=dev)
        bias.scatter_add_(1, ids.clamp(0, vocab - 1), s["bias_values"] * ok)
        y = y + bias[req]
    if s["allowed"] is not None:
        y = y.masked_fill(~_visible(s["allowed"], vocab), -math.inf)
    return y


def run(state):
    if not own:
        return {"int4": _plain_int4, "tree": _plain_tree, "logits": _plain_logits}[state["kind"]](
            state)
    from qsa_vllm_amd import ops

    s = state
    if s["kind"] == "int4":
        return ops.int4_linear(s["x"], s["weight"], s["bias"])
    if s["kind"] == "tree":
        return ops.qsa_tree_paged_attention(
            s["q"], s["k_cache"], s["v_cache"], s["table"], s["ctx"], s["starts"], s["ancestors"],
            output_gate=s["gate"], max_query_len=max(s["nodes_list"]),
            max_context_len=max(s["ctx_list"]))
    return ops.process_logits(
        s["logits"], token_to_req=s["token_to_req"], history=s["history"],
        history_lens=s["history_lens"], prompt_lens=s["prompt_lens"], repetition=s["repetition"],
        frequency=s["frequency"], presence=s["presence"], bias_ids=s["bias_ids"],
        bias_values=s["bias_values"], allowed=s["allowed"], vocab_start=s["first"],
        draft_tokens=s["draft_tokens"], ancestors=s["ancestors"], query_start_loc=s["starts"])


# ---------------------------------------------------------------------------
# Work and exact results
# ---------------------------------------------------------------------------

def work(case):
    if case["kind"] == "int4":
        n, k, rows = case["n"], case["k"], case["rows"]
        groups = -(-k // case["group"])
        size = n * k // 2 + 2 * n * groups + (n * groups // 2 if case["zeros"] else 0)
        size += 2 * rows * (k + n) + (2 * n if case["bias"] else 0)
        return {"bytes": size, "flops": 2 * rows * n * k}
    if case["kind"] == "tree":
        nodes, ctx = _tree_lengths(case)
        dim, heads, kv_heads = case["dim"], case["heads"], case["kv_heads"]
        tokens = sum(ctx) + sum(nodes)
        size = tokens * kv_heads * 2 * dim * 2
        size += sum(nodes) * heads * dim * 2 * (3 if case["gate"] else 2)
        flops = sum(4 * t * heads * dim * (c + t) for t, c in zip(nodes, ctx))
        return {"bytes": size, "flops": flops}
    rows = case["requests"] * max(1, case["nodes"])
    per = {"bf16": 2, "fp16": 2, "fp32": 4}[case["dtype"]] + 4
    size = rows * case["vocab"] * per + (rows * case["vocab"] // 8 if case["grammar"] else 0)
    size += case["requests"] * (case["hist_min"] + case["hist_max"]) // 2 * 4
    size += case["requests"] * case["biases"] * 8
    return {"bytes": size, "flops": rows * case["vocab"]}


def _exact_int4(s):
    """Group by group: sum of codes times activations, less the zero point
    times the activations' sum, times the scale."""
    x, codes = s["x"].double(), s["codes"]
    y = torch.zeros(x.shape[0], codes.shape[0], dtype=torch.float64, device=x.device)
    for i in range(s["scales"].shape[1]):
        part = slice(i * s["group"], min((i + 1) * s["group"], codes.shape[1]))
        xs = x[:, part]
        zero = s["zeros"][:, i].double() if s["zeros"] is not None else 8.0
        dots = xs @ codes[:, part].double().t().contiguous()
        y += (dots - xs.sum(dim=1, keepdim=True) * zero) * s["scales"][:, i].double()
    return y if s["bias"] is None else y + s["bias"].double()


def _exact_tree(s):
    """Node by node over its own list of positions, one kv head at a time."""
    q, kc, vc = s["q"].double(), s["k_cache"], s["v_cache"]
    _, page, kv_heads, dim = kc.shape
    group = q.shape[1] // kv_heads
    out = torch.zeros_like(q)
    ancestors = s["ancestors"].cpu()
    row = 0
    for b, (ctx, t) in enumerate(zip(s["ctx_list"], s["nodes_list"])):
        pos = torch.arange(ctx + t, device=q.device)
        page_of = s["table"][b].long()[pos // page]
        k = kc[page_of, pos % page].double().permute(1, 2, 0).contiguous()   # [kv, dim, len]
        v = vc[page_of, pos % page].double().permute(1, 0, 2).contiguous()   # [kv, len, dim]
        for j in range(t):
            bits = ancestors[row].tolist()
            mine = [i for i in range(t) if (bits[i // 32] >> (i % 32)) & 1]
            mine = torch.tensor([ctx + i for i in mine], device=q.device)
            for h in range(kv_heads):
                heads = slice(h * group, (h + 1) * group)
                score = q[row, heads] @ k[h] / math.sqrt(dim)
                score = torch.cat([score[:, :ctx], score[:, mine]], dim=1)
                p = torch.softmax(score, dim=1)
                out[row, heads] = p[:, :ctx] @ v[h, :ctx] + p[:, ctx:] @ v[h, mine]
            row += 1
    return out if s["gate"] is None else out * torch.sigmoid(s["gate"].double())


def _exact_logits(s):
    """Row by row, each from its own list of tokens."""
    y = s["logits"].double()
    vocab, first = y.shape[1], s["first"]
    history, lens, prompts = s["history"].cpu(), s["history_lens"].tolist(), s["prompt_lens"].tolist()
    reqs = s["token_to_req"].tolist()
    starts = s["starts"].tolist() if s["starts"] is not None else None
    drafts = s["draft_tokens"].cpu() if starts else None
    ancestors = s["ancestors"].tolist() if starts else None
    of_request = {}

    def counted(tokens):
        tokens = tokens.long() - first
        return torch.bincount(tokens[(tokens >= 0) & (tokens < vocab)], minlength=vocab)

    for row, b in enumerate(reqs):
        if b not in of_request:
            h = history[b, :lens[b]]
            of_request[b] = counted(h[:prompts[b]]), counted(h[prompts[b]:])
        prompt, spoken = of_request[b]
        if starts:
            bits = ancestors[row]
            path = [starts[b] + j for j in range(starts[b + 1] - starts[b])
                    if (bits[j // 32] >> (j % 32)) & 1]
            spoken = spoken + counted(drafts[torch.tensor(path, dtype=torch.long)])
        spoken = spoken.to(y.device).double()
        r = s["repetition"][b].double()
        old = (prompt.to(y.device) > 0) | (spoken > 0)
        z = y[row]
        z = torch.where(old & (z > 0), z / r, torch.where(old, z * r, z))
        z = z - spoken * s["frequency"][b].double() - (spoken > 0) * s["presence"][b].double()
        if s["bias_ids"] is not None:
            ids = s["bias_ids"][b].long() - first
            ok = (ids >= 0) & (ids < vocab)
            z = z.index_put((ids[ok],), s["bias_values"][b][ok].double(), accumulate=True)
        y[row] = z
    if s["allowed"] is not None:
        shifts = torch.arange(32, device=y.device, dtype=torch.int32)
        bits = ((s["allowed"][:, :, None] >> shifts) & 1).reshape(y.shape[0], -1)[:, :vocab]
        y = torch.where(bits == 1, y, torch.full_like(y, -math.inf))
    return y


def exact(case, seed):
    state = prepare(case, seed)
    return {"int4": _exact_int4, "tree": _exact_tree, "logits": _exact_logits}[case["kind"]](state)
