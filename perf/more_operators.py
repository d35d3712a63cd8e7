"""Operators of an attention layer beside the sparse ones, as measurable cases.

Three operators that write and read a layer's paged cache, on the sizes of the
hybrid decoder (16 query and 2 key/value heads of 128 dims on one of two GPUs,
64 rotated dims, pages of 16 tokens, serving steps of 112 decode requests and 16
prefill chunks of 512 tokens):

* ``rope``: queries and keys normed for each head and rotated by their position,
  keys and values stored into a bf16 or a 4-bit paged cache;
* ``window``: attention of single tokens and prompt chunks over the last tokens
  of a request and a few first ones that stay visible, bf16 cache;
* ``kv4``: attention over a cache held in 4 bits, the whole context or a window.

A 4-bit cache keeps, for every block and kv head, a page's K codes (page x
dim / 2 bytes), its V codes, and 16-bit words of groups of 32 dims for K and then
for V (each filled up to 16 bytes). A word's low four bits are the zero point z,
the others a bf16 scale s of four significant bits: x = (code - z) * s. Code words
of 8 dims: V's natural, 4 bits a dim; K's dim 2 i in bits 4 i, dim 2 i + 1 in bits
16 + 4 i, and the word of dims 32 a + 8 b .. at byte b * dim / 8 + 4 a of its row.

``own`` chooses between the plain form (elementary torch operations in 32 bits)
and the package's entry points.
"""

from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda:0"
EPS = 1e-6
THETA = 1.0e7


def _rope(name, decodes, chunks, chunk, heads=16, kv_heads=2, dim=128, rotary=64, page=16, bits=16,
          norm=True):
    return dict(name=name, kind="rope", decodes=decodes, chunks=chunks, chunk=chunk, heads=heads,
                kv_heads=kv_heads, dim=dim, rotary=rotary, page=page, bits=bits, norm=norm)


def _attn(name, kind, decodes, chunks, chunk, ctx_min, ctx_max, window=0, sinks=0, heads=16,
          kv_heads=2, dim=128, page=16, gate=False):
    return dict(name=name, kind=kind, decodes=decodes, chunks=chunks, chunk=chunk, ctx_min=ctx_min,
                ctx_max=ctx_max, window=window, sinks=sinks, heads=heads, kv_heads=kv_heads, dim=dim,
                page=page, gate=gate)


def listed():
    return [
        # One user's next token.
        _rope("rope_1", 1, 0, 0),
        # The next token of 112 users, into a 4-bit cache.
        _rope("rope_112_kv4", 112, 0, 0, bits=4),
        # A mixed serving step: 112 decode tokens and 16 chunks of 512.
        _rope("rope_8304", 112, 16, 512),
        # A prompt of 8191 tokens, small heads rotated whole, into a 4-bit cache.
        _rope("rope_8191_kv4_d64", 0, 1, 8191, heads=32, kv_heads=8, dim=64, rotary=64, bits=4),
        # One user's next token in a short chat.
        _attn("window_1_on_700", "window", 1, 0, 0, 700, 700, window=512, sinks=4),
        # The next token of 112 users on long contexts, gated output.
        _attn("window_112_on_32k", "window", 112, 0, 0, 4096, 32768, window=4096, sinks=4, gate=True),
        # A prompt of 8192 tokens at once.
        _attn("window_8192", "window", 0, 1, 8192, 0, 0, window=4096, sinks=4),
        # A mixed serving step: 112 decode tokens and 16 chunks of 512.
        _attn("window_mixed", "window", 112, 16, 512, 512, 16384, window=4096, sinks=4),
        # One user's next token over a 4-bit cache.
        _attn("kv4_1_on_2000", "kv4", 1, 0, 0, 2000, 2000),
        # The next token of 64 users over their whole contexts.
        _attn("kv4_64_on_8k", "kv4", 64, 0, 0, 1024, 8192),
        # One user's next token on a very long context.
        _attn("kv4_1_on_128k", "kv4", 1, 0, 0, 131071, 131071, gate=True),
        # Four chunks of 500 tokens of long prompts.
        _attn("kv4_4x500_on_16k", "kv4", 0, 4, 500, 8192, 16384),
    ]


def _log(rng, low, high):
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng: random.Random):
    kind = rng.choice(["rope", "window", "kv4"])
    kv_heads = rng.choice([1, 2, 2, 4, 8])
    group = rng.choice([1, 3, 4, 8, 8, 16] if kv_heads < 4 else [1, 2, 4])
    heads, dim = kv_heads * group, rng.choice([64, 128, 128])
    page = rng.choice([16, 16, 48, 272, 1])
    step = rng.choice(["decode", "decode", "chunks", "mixed"])
    decodes = 0 if step == "chunks" else _log(rng, 1, 128)
    if kind == "rope":
        chunks, chunk = (0, 0) if step == "decode" else (_log(rng, 1, 16), _log(rng, 2, 4096))
        while chunks * chunk * (heads + 2 * kv_heads) * dim > 8192 * 20 * 128:
            chunk = max(2, chunk // 2)
            chunks = max(1, chunks - 1)
        case = _rope("", decodes, chunks, chunk, heads, kv_heads, dim,
                     rng.choice([dim, dim // 2, 32, 0]), page, rng.choice([16, 4]),
                     rng.random() < 0.8)
    else:
        chunks, chunk = (0, 0) if step == "decode" else (_log(rng, 1, 16), _log(rng, 2, 8192))
        window = rng.choice([0, _log(rng, 1, 8192), _log(rng, 64, 8192)])
        sinks = rng.choice([0, 1, 4, 130]) if window else 0
        ctx_max = _log(rng, 1, min(131072, 1048576 // max(1, decodes + chunks)))

        def cost():  # (row, token) pairs of all heads
            return chunks * chunk * heads * dim * (min(window or 1 << 30, ctx_max + chunk) + sinks)

        while chunks and cost() > 8192 * 16 * 128 * 4096:
            if chunk > 64:
                chunk //= 2
            elif chunks > 1:
                chunks //= 2
            else:
                ctx_max //= 2
        case = _attn("", kind, decodes, chunks, chunk, rng.randint(0, ctx_max), ctx_max, window, sinks,
                     heads, kv_heads, dim, page, rng.random() < 0.5)
    del case["name"]
    return case


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------

def _lengths(case):
    """(tokens already cached, tokens of this step) of each request, the decode
    requests first: the case's own, the same whatever the inputs' seed."""
    count = case["decodes"] + case["chunks"]
    gen = torch.Generator().manual_seed(count)
    low, high = case.get("ctx_min", 0), case.get("ctx_max", 120000)
    ctx = torch.randint(low, high + 1, (count,), generator=gen)
    ctx[int(torch.randint(0, count, (1,), generator=gen))] = high
    return ctx.tolist(), [1] * case["decodes"] + [case["chunk"]] * case["chunks"]


def _starts(lengths):
    out = [0]
    for n in lengths:
        out.append(out[-1] + n)
    return out


def _pages(gen, lengths, page):
    """A page table of shuffled blocks and the number of blocks."""
    pages = [-(-n // page) for n in lengths]
    order = torch.randperm(sum(pages) + 3, generator=gen).to(torch.int32)
    table = torch.full((len(lengths), max(pages)), -1, dtype=torch.int32)
    at = 0
    for i, p in enumerate(pages):
        table[i, :p] = order[at:at + p]
        at += p
    return table, len(order)


def _randn(g, *shape, scale=1.0):
    """bf16 normal values, made in pieces."""
    out = torch.empty(shape, dtype=torch.bfloat16, device=DEV)
    flat, step = out.view(-1), 1 << 26
    for i in range(0, flat.numel(), step):
        n = min(step, flat.numel() - i)
        flat[i:i + n] = torch.randn(n, generator=g, device=DEV) * scale
    return out


def _pad16(n):
    return -(-n // 16) * 16


def _page_bytes(page, dim):
    return page * dim + 2 * _pad16(page * dim // 16)


def _angles(max_position, rotary):
    """fp32 [positions, rotary]: cosines, then sines, of 64-bit angles."""
    half = torch.arange(0, rotary, 2, dtype=torch.float64, device=DEV)
    phase = torch.arange(max_position, dtype=torch.float64, device=DEV)[:, None] * (
        THETA ** (-half / max(rotary, 1)))
    return torch.cat((phase.cos(), phase.sin()), dim=1).float()


def _codes4(x):
    """4-bit codes [..., dim], zero points and scales [..., dim / 32] of ``x``'s
    bf16 values: the step is the range (0 in it) over 15, raised to four
    significant bits."""
    y = x.float().unflatten(-1, (-1, 32))
    low, high = y.amin(-1).clamp(max=0), y.amax(-1).clamp(min=0)
    step = ((high - low) / torch.full_like(high, 15.0)).clamp(min=2.0 ** -100)
    scale = ((step.view(torch.int32) + 0xFFFFF) & ~0xFFFFF).view(torch.float32)
    zero = (-low / scale).round().clamp(0, 15)
    codes = ((y / scale[..., None]).round() + zero[..., None]).clamp(0, 15)
    return codes.flatten(-2), zero, scale


def _cache4(g, blocks, page, kv_heads, dim):
    """A filled 4-bit cache [blocks, kv_heads, page bytes] of normal K and V."""
    data = torch.zeros(blocks, kv_heads, _page_bytes(page, dim), dtype=torch.uint8, device=DEV)
    meta = page * dim // 16
    step = max(1, (1 << 25) // (page * kv_heads * dim))
    for at in range(0, blocks, step):
        n = min(step, blocks - at)
        part = data[at:at + n]
        for which in (0, 1):
            codes, zero, scale = _codes4(_randn(g, n, kv_heads, page, dim))
            c = codes.to(torch.uint8)
            if which == 0:   # pairs of nibbles (0, 2), (4, 6), (1, 3), (5, 7) of each word
                c = c.unflatten(-1, (dim // 32, 4, 8)).transpose(-3, -2)
                c = c[..., [0, 2, 4, 6, 1, 3, 5, 7]].flatten(-3)
            c = c[..., 0::2] | (c[..., 1::2] << 4)
            part[:, :, which * page * dim // 2:][:, :, :page * dim // 2] = c.flatten(2)
            word = (scale.view(torch.int32) >> 16) | zero.to(torch.int32)
            low, high = (word & 255).to(torch.uint8), ((word >> 8) & 255).to(torch.uint8)
            first = page * dim + which * _pad16(meta)
            part[:, :, first:first + meta] = torch.stack((low, high), -1).flatten(2)
    return data


def _prepare_rope(case, seed):
    gen = torch.Generator().manual_seed(seed)
    g = torch.Generator(device=DEV).manual_seed(seed)
    heads, kv_heads, dim, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    ctx, new = _lengths(case)
    # The pages that this step writes to, spread over a small cache.
    table, blocks = _pages(gen, [c % page + n for c, n in zip(ctx, new)], page)
    starts, cached = torch.tensor(_starts(new)), torch.tensor(ctx)
    req = torch.repeat_interleave(torch.arange(len(new)), torch.tensor(new))
    positions = torch.arange(len(req)) - starts[req] + cached[req]
    slots = table[req, positions // page - cached[req] // page].long() * page + positions % page
    # One projection's output: queries with gates between them, keys, values. A few
    # channels of the keys are large, as trained ones are.
    rows = _randn(g, len(req), (2 * heads + 2 * kv_heads) * dim)
    q = rows[:, :2 * heads * dim].view(-1, heads, 2 * dim)[..., :dim]
    k = rows[:, 2 * heads * dim:(2 * heads + kv_heads) * dim].view(-1, kv_heads, dim)
    v = rows[:, (2 * heads + kv_heads) * dim:].view(-1, kv_heads, dim)
    k[..., ::29] *= 2
    weight = [(1 + 0.1 * torch.randn(dim, generator=g, device=DEV)).bfloat16() if case["norm"] else None
              for _ in range(2)]
    state = dict(kind="rope", q=q, k=k, v=v, q_weight=weight[0], k_weight=weight[1],
                 positions=positions.to(DEV), slots=slots.to(DEV), page=page,
                 cos_sin=_angles(1 << 17, case["rotary"]) if case["rotary"] else None)
    if case["bits"] == 16:
        kv = torch.zeros(blocks, page, kv_heads, 2 * dim, dtype=torch.bfloat16, device=DEV)
        state["cache"] = kv[..., :dim], kv[..., dim:]
    else:
        state["cache"] = None
        state["data"] = torch.zeros(blocks, kv_heads, _page_bytes(page, dim), dtype=torch.uint8,
                                    device=DEV)
        state["k_held"] = torch.empty(len(req), kv_heads, dim, dtype=torch.bfloat16, device=DEV)
        state["v_held"] = torch.empty_like(state["k_held"])
        if own:
            from qsa_vllm_amd.ops import Int4KVCache
            state["cache"] = Int4KVCache(state["data"], page, dim)
    return state


def _prepare_attn(case, seed):
    gen = torch.Generator().manual_seed(seed)
    g = torch.Generator(device=DEV).manual_seed(seed)
    heads, kv_heads, dim, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    ctx, new = _lengths(case)
    total = [c + n for c, n in zip(ctx, new)]
    table, blocks = _pages(gen, total, page)
    state = dict(kind=case["kind"], page=page, dim=dim, table=table.to(DEV), new=new, total=total,
                 window=case["window"], sinks=case["sinks"],
                 lens=torch.tensor(total, dtype=torch.int32, device=DEV),
                 starts=torch.tensor(_starts(new), dtype=torch.int32, device=DEV))
    if case["kind"] == "kv4":
        state["cache"] = state["data"] = _cache4(g, blocks, page, kv_heads, dim)
        if own:
            from qsa_vllm_amd.ops import Int4KVCache
            state["cache"] = Int4KVCache(state["data"], page, dim)
    else:
        kv = _randn(g, blocks, page, kv_heads, 2 * dim)
        state["k_cache"], state["v_cache"] = kv[..., :dim], kv[..., dim:]
    state["q"] = _randn(g, sum(new), heads, dim, scale=2.0)
    state["gate"] = _randn(g, sum(new), heads, dim) if case["gate"] else None
    return state


def prepare(case, seed):
    return (_prepare_rope if case["kind"] == "rope" else _prepare_attn)(case, seed)


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------

def _plain_norm_rope(x, weight, positions, cos_sin):
    y = x.float()
    if weight is not None:
        y = y * (y.square().mean(-1, keepdim=True) + EPS).rsqrt() * weight.float()
    if cos_sin is None:
        return y.to(x.dtype)
    rotary = cos_sin.shape[1]
    cos, sin = cos_sin[positions][:, None].chunk(2, dim=-1)
    a, b = y[..., :rotary // 2], y[..., rotary // 2:rotary]
    return torch.cat((a * cos - b * sin, b * cos + a * sin, y[..., rotary:]), -1).to(x.dtype)


def _plain_rope(s):
    q = _plain_norm_rope(s["q"], s["q_weight"], s["positions"], s["cos_sin"])
    k = _plain_norm_rope(s["k"], s["k_weight"], s["positions"], s["cos_sin"])
    if s["cache"] is None:
        def held(x):
            codes, zero, scale = _codes4(x)
            return ((codes.unflatten(-1, (-1, 32)) - zero[..., None]) * scale[..., None]).flatten(-2)
        return q, held(k).to(k.dtype), held(s["v"]).to(k.dtype)
    block, place = s["slots"] // s["page"], s["slots"] % s["page"]
    s["cache"][0][block, place] = k
    s["cache"][1][block, place] = s["v"]
    return q, s["cache"][0], s["cache"][1]


def _rows4(data, which, blocks, places, page, dim):
    """fp32 K (0) or V (1) rows [n, kv_heads, dim] of a 4-bit cache."""
    kv_heads, row, meta = data.shape[1], dim // 2, page * dim // 16
    flat = data.view(-1)
    first = (blocks[:, None] * kv_heads + torch.arange(kv_heads, device=data.device)) * data.shape[2]
    at = first + which * page * row + places[:, None] * row
    c = flat[at[..., None] + torch.arange(row, device=data.device)]
    c = torch.stack((c & 15, c >> 4), -1).flatten(-2)
    if which == 0:   # K's order within a row
        c = c.unflatten(-1, (4, dim // 32, 8))[..., [0, 4, 1, 5, 2, 6, 3, 7]].transpose(-3, -2)
        c = c.flatten(-3)
    at = first + page * dim + which * _pad16(meta) + places[:, None] * (dim // 16)
    w = flat[at[..., None] + torch.arange(dim // 16, device=data.device)].int()
    w = w[..., 0::2] | (w[..., 1::2] << 8)
    scale = ((w & 0xFFF0) << 16).view(torch.float32)
    return ((c.unflatten(-1, (-1, 32)) - (w & 15).float()[..., None]) * scale[..., None]).flatten(-2)


def _plain_part(s, reqs, row0, rows):
    """Requests ``reqs`` of ``rows`` rows each, from row ``row0`` on, padded to the
    longest of them."""
    dev = s["q"].device
    n, heads, dim = len(reqs), s["q"].shape[1], s["dim"]
    lens = s["lens"][reqs[0]:reqs[0] + n].long()
    most = max(s["total"][b] for b in reqs)
    if s["window"]:
        most = min(most, s["window"] + rows - 1)
    # The positions that any row sees: the last ones, and the first ones before them.
    first = (lens - most).clamp(min=0)
    at = first[:, None] + torch.arange(most, device=dev)
    inside = at < lens[:, None]
    if s["window"] and s["sinks"]:
        early = torch.arange(s["sinks"], device=dev).expand(n, -1)
        inside = torch.cat((early < torch.minimum(first, lens)[:, None], inside), 1)
        at = torch.cat((early, at), 1)
    safe = torch.where(inside, at, torch.zeros_like(at))
    blocks = s["table"][reqs[0]:reqs[0] + n].long().gather(1, safe // s["page"]).flatten()
    places = (safe % s["page"]).flatten()
    if s["kind"] == "kv4":
        k, v = (_rows4(s["data"], which, blocks, places, s["page"], dim) for which in (0, 1))
    else:
        k, v = s["k_cache"][blocks, places].float(), s["v_cache"][blocks, places].float()
    kv_heads = k.shape[1]
    k, v = (x.view(n, -1, kv_heads, dim).transpose(1, 2).contiguous() for x in (k, v))
    q = s["q"][row0:row0 + n * rows].float().view(n, rows, kv_heads, -1, dim)
    group = q.shape[3]
    q = q.permute(0, 2, 1, 3, 4).reshape(n, kv_heads, rows * group, dim)
    pos = lens[:, None] - rows + torch.arange(rows, device=dev)
    seen = inside[:, None] & (at[:, None] <= pos[..., None])
    if s["window"]:
        seen &= (at[:, None] > pos[..., None] - s["window"]) | (at[:, None] < s["sinks"])
    score = q @ k.transpose(2, 3).contiguous() * dim ** -0.5
    score = score.view(n, kv_heads, rows, group, -1).masked_fill_(~seen[:, None, :, None], -math.inf)
    score = score.view(n, kv_heads, rows * group, -1)
    weight = score.sub_(score.amax(-1, keepdim=True)).exp_()
    o = weight @ v / weight.sum(-1, keepdim=True)
    return o.view(n, kv_heads, rows, group, dim).transpose(1, 2).reshape(n * rows, heads, dim)


def _plain_attn(s):
    count = s["new"].count(1) if s["new"][0] == 1 else 0
    # Single tokens together, 16 requests at a time; a prompt's rows by request.
    parts = [list(range(i, min(i + 16, count))) for i in range(0, count, 16)]
    parts += [[b] for b in range(count, len(s["new"]))]
    out, row = [], 0
    for reqs in parts:
        out.append(_plain_part(s, reqs, row, s["new"][reqs[0]]))
        row += len(reqs) * s["new"][reqs[0]]
    o = torch.cat(out)
    if s["gate"] is not None:
        o = o / (1 + (-s["gate"].float()).exp())
    return o.to(s["q"].dtype)


def run(state):
    s = state
    if not own:
        return _plain_rope(s) if s["kind"] == "rope" else _plain_attn(s)
    from qsa_vllm_amd import ops

    if s["kind"] == "rope":
        held = "k_held" in s
        q, _ = ops.qk_norm_rope(
            s["q"], s["k"], s["q_weight"], s["k_weight"], s["positions"], s["cos_sin"], EPS,
            value=s["v"], cache=s["cache"], slot_mapping=s["slots"],
            k_out=s["k_held"] if held else None, v_out=s["v_held"] if held else None)
        return (q, s["k_held"], s["v_held"]) if held else (q, *s["cache"])
    more = dict(window=s["window"] or None, sink_tokens=s["sinks"], output_gate=s["gate"],
                max_query_len=max(s["new"]), max_seq_len=max(s["total"]))
    if s["kind"] == "window":
        return ops.qsa_window_paged_attention(s["q"], s["k_cache"], s["v_cache"], s["table"],
                                              s["lens"], s["starts"], **more)
    return ops.qsa_int4_paged_attention(s["q"], s["cache"], s["table"], s["lens"], s["starts"], **more)


# ---------------------------------------------------------------------------
# Work and exact results
# ---------------------------------------------------------------------------

def work(case):
    ctx, new = _lengths(case)
    heads, kv_heads, dim, rows = case["heads"], case["kv_heads"], case["dim"], sum(new)
    if case["kind"] == "rope":
        held = dim // 2 + dim // 16 + 2 * dim if case["bits"] == 4 else 2 * dim
        size = rows * (heads * 4 * dim + 2 * kv_heads * (2 * dim + held) + 16)
        size += rows * 4 * case["rotary"]
        return {"bytes": size, "flops": 8 * rows * (heads + kv_heads) * dim}
    window, sinks = case["window"], case["sinks"]
    tokens = pairs = 0
    for c, n in zip(ctx, new):
        pos = torch.arange(c, c + n, dtype=torch.float64)
        seen = torch.clamp(pos + 1, max=window) if window else pos + 1
        first = pos + 1 - seen
        pairs += int((seen + torch.clamp(first, max=sinks)).sum())
        tokens += c + n if not window else min(c + n, window + n - 1)
        tokens += min(sinks, max(0, c + n - (window + n - 1))) if window else 0
    row = dim // 2 + dim // 16 if case["kind"] == "kv4" else 2 * dim
    size = tokens * kv_heads * 2 * row + rows * heads * dim * 2 * (3 if case["gate"] else 2)
    return {"bytes": size, "flops": 4 * pairs * heads * dim}


def _exact_norm_rope(x, weight, positions, rotary):
    """Complex numbers of 64 bits, the angles from their definition."""
    y = x.double()
    if weight is not None:
        y = y / torch.sqrt((y * y).sum(-1, keepdim=True) / y.shape[-1] + EPS) * weight.double()
    half = rotary // 2
    if half:
        i = torch.arange(half, device=x.device, dtype=torch.float64)
        angle = positions.double()[:, None, None] * torch.exp(-math.log(THETA) * 2 * i / rotary)
        z = torch.complex(y[..., :half], y[..., half:rotary]) * torch.polar(torch.ones_like(angle), angle)
        y[..., :half], y[..., half:rotary] = z.real, z.imag
    return y


def _exact_rope(s, case):
    q = _exact_norm_rope(s["q"], s["q_weight"], s["positions"], case["rotary"])
    k = _exact_norm_rope(s["k"], s["k_weight"], s["positions"], case["rotary"])
    if case["bits"] == 4:
        # (What a rounding to 4 bits leaves jumps with the last bit before it: no
        # value of K's or V's codes is nearer than another.)
        return q, None, None
    kc, vc = (torch.zeros(x.shape, dtype=torch.float64, device=DEV) for x in s["cache"])
    kc.view(-1, *kc.shape[2:]).index_copy_(0, s["slots"], k)
    vc.view(-1, *vc.shape[2:]).index_copy_(0, s["slots"], s["v"].double())
    return q, kc, vc


def _exact_cache4(s):
    """Both halves of a 4-bit cache as 64-bit [blocks, page, kv_heads, dim]."""
    data, page, dim = s["data"], s["page"], s["dim"]
    out = []
    words = 2 * page * dim // 2
    for which in (0, 1):
        raw = data[:, :, which * page * dim // 2:(which + 1) * page * dim // 2].contiguous()
        w = raw.view(torch.int32).unflatten(2, (page, dim // 8)).long()
        x = torch.empty(*w.shape[:3], dim, dtype=torch.float64, device=data.device)
        for d in range(dim):
            if which == 0:
                word = (d % 32 // 8) * (dim // 32) + d // 32
                shift = 4 * (d % 8 // 2) + 16 * (d % 2)
            else:
                word, shift = d // 8, 4 * (d % 8)
            x[..., d] = (w[..., word] >> shift) & 15
        first = words + which * _pad16(page * dim // 16)
        meta = data[:, :, first:first + page * dim // 16].contiguous().view(torch.int16).int()
        meta = meta.unflatten(2, (page, dim // 32))
        scale = (meta & 0xFFF0).to(torch.int16).view(torch.bfloat16).double()
        for a in range(dim // 32):
            x[..., 32 * a:32 * a + 32] -= (meta[..., a:a + 1] & 15).double()
            x[..., 32 * a:32 * a + 32] *= scale[..., a:a + 1]
        out.append(x.transpose(1, 2))
    return out


def _exact_attn(s):
    """Request by request and kv head by kv head, 256 rows of it at a time, over
    every position up to the last one that they see."""
    kc, vc = _exact_cache4(s) if s["kind"] == "kv4" else (s["k_cache"], s["v_cache"])
    q = s["q"].double()
    out = torch.zeros_like(q)
    kv_heads, dim = kc.shape[2], s["dim"]
    group = q.shape[1] // kv_heads
    row = 0
    for b, (rows, length) in enumerate(zip(s["new"], s["total"])):
        j = torch.arange(length, device=q.device)
        block = s["table"][b].long()[j // s["page"]]
        k, v = kc[block, j % s["page"]].double(), vc[block, j % s["page"]].double()
        for i in range(0, rows, 256):
            n = min(256, rows - i)
            pos = length - rows + i + torch.arange(n, device=q.device)[:, None]
            last = length - rows + i + n
            hidden = j[:last] > pos
            if s["window"]:
                hidden |= (pos - j[:last] >= s["window"]) & (j[:last] >= s["sinks"])
            for h in range(kv_heads):
                kt, vh = k[:last, h].t().contiguous(), v[:last, h].contiguous()
                for m in range(h * group, (h + 1) * group):
                    score = q[row + i:row + i + n, m] @ kt / math.sqrt(dim)
                    score.masked_fill_(hidden, -math.inf)
                    out[row + i:row + i + n, m] = torch.softmax(score, 1) @ vh
        row += rows
    return out if s["gate"] is None else out * torch.sigmoid(s["gate"].double())


def exact(case, seed):
    state = prepare(case, seed)
    return _exact_rope(state, case) if case["kind"] == "rope" else _exact_attn(state)
