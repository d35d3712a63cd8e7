"""Tree attention on the GPU against a 64-bit statement of it, row by row.

Tolerance. Each weight is rounded to bf16, p (1 + e) with |e| <= 2^-8, before it
meets V, and the rounded weights are what is summed: the weighted mean o moves by
sum p e (v - o) / sum p (1 + e), at most 2^-8 (1 + 2^-7) sum p |v - o|; a score's fp32 sum of D products
passes at most 36 roundings of 2^-24 on sum |q k|, scaled by D^-0.5, which moves
a weight by as much (numerator and sum: twice); the fp32 exponentials and sums
stay under 2^-19 of a weight. The gate's factor is at most 1 and off by 2^-20.
Then one rounding to bf16, 2^-8 of the value."""

import math

import pytest
import torch

from qsa_vllm_amd.ops import qsa_sparse_paged_attention, qsa_tree_paged_attention, tree_ancestors

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


class Case:
    """Random requests: committed lengths, node counts, random trees, a shuffled
    paged cache whose unused slots (and pages) hold NaN."""

    def __init__(self, ctx, nodes, heads=4, kv_heads=2, dim=128, page=16, gate=False, seed=0,
                 layout="token_major", chain=False, scale=1.0, words=None):
        gen = torch.Generator().manual_seed(seed)
        self.gen, self.ctx, self.nodes, self.page, self.dim = gen, ctx, nodes, page, dim
        self.heads, self.kv_heads = heads, kv_heads
        rows = sum(nodes)
        self.starts = [0]
        for t in nodes:
            self.starts.append(self.starts[-1] + t)
        self.parents = [j - 1 if chain else (int(torch.randint(-1, j, (1,), generator=gen)) if j else -1)
                        for t in nodes for j in range(t)]
        pages = [-(-(c + t) // page) for c, t in zip(ctx, nodes)]
        order = torch.randperm(sum(pages) + 2, generator=gen).to(torch.int32)
        self.table = torch.full((len(ctx), max(max(pages), 1)), -1, dtype=torch.int32)
        kv = torch.full((len(order), page, kv_heads, 2 * dim), float("nan"), dtype=torch.bfloat16)
        at = 0
        for b, p in enumerate(pages):
            self.table[b, :p] = order[at:at + p]
            at += p
            for pos in range(ctx[b] + nodes[b]):
                kv[self.table[b, pos // page], pos % page] = (
                    torch.randn(kv_heads, 2 * dim, generator=gen) * scale).bfloat16()
        self.q = (torch.randn(rows, heads, dim, generator=gen) * scale).bfloat16()
        self.gate = torch.randn(rows, heads, dim, generator=gen).bfloat16() if gate else None
        self.kv, self.layout = kv, layout
        self.qsl = torch.tensor(self.starts, dtype=torch.int32)
        most = max(max(nodes), 1)
        self.anc = tree_ancestors(torch.tensor(self.parents, dtype=torch.int64), self.qsl, most)
        if words is not None:
            self.anc = torch.nn.functional.pad(self.anc, (0, words - self.anc.shape[1]))

    def device_cache(self):
        if self.layout == "head_major":   # [blocks, kv_heads, page, 2 D] storage
            kv = self.kv.permute(0, 2, 1, 3).contiguous().to(DEV).permute(0, 2, 1, 3)
        else:
            kv = self.kv.to(DEV)
        return kv[..., :self.dim], kv[..., self.dim:]

    def run(self, out=None, q=None, max_query_len=None, max_context_len=None, anc=None, table=None):
        k, v = self.device_cache()
        return qsa_tree_paged_attention(
            self.q.to(DEV) if q is None else q, k, v,
            (self.table if table is None else table).to(DEV),
            torch.tensor(self.ctx, dtype=torch.int32, device=DEV), self.qsl.to(DEV),
            (self.anc if anc is None else anc).to(DEV), out,
            output_gate=self.gate.to(DEV) if self.gate is not None else None,
            max_query_len=max(self.nodes) if max_query_len is None else max_query_len,
            max_context_len=max(self.ctx) if max_context_len is None else max_context_len)

    def want(self, anc=None, table=None):
        """(result, tolerance), 64 bits: each row over its own list of slots."""
        anc = self.anc if anc is None else anc
        table = self.table if table is None else table
        out = torch.zeros(self.q.shape, dtype=torch.float64)
        tol = torch.zeros_like(out)
        group = self.heads // self.kv_heads
        blocks = self.kv.shape[0]
        for b, (c, t) in enumerate(zip(self.ctx, self.nodes)):
            for r in range(self.starts[b], self.starts[b + 1]):
                seen = list(range(c)) + [c + j for j in range(min(t, 32 * anc.shape[1]))
                                         if (int(anc[r, j // 32]) >> (j % 32)) & 1]
                slots = [(int(table[b, p // self.page]), p % self.page) for p in seen
                         if p // self.page < table.shape[1]]
                slots = [s for s in slots if 0 <= s[0] < blocks]
                if not slots:
                    continue
                kv = self.kv[[s[0] for s in slots], [s[1] for s in slots]].double()
                for h in range(self.heads):
                    k, v = kv[:, h // group, :self.dim], kv[:, h // group, self.dim:]
                    q = self.q[r, h].double()
                    score = k @ q / math.sqrt(self.dim)
                    p = torch.softmax(score, 0)
                    spread = (k.abs() @ q.abs()).max().item() / math.sqrt(self.dim)
                    o = p @ v
                    off = (2 ** -8 * (1 + 2 ** -7) * (p @ (v - o).abs()) +
                           (2 * 36 * 2 ** -24 * spread + 2 ** -18) * (p @ v.abs()))
                    if self.gate is not None:
                        s = torch.sigmoid(self.gate[r, h].double())
                        off = off * s + 2 ** -20 * (o * s).abs()
                        o = o * s
                    out[r, h] = o
                    tol[r, h] = off + 2 ** -8 * (o.abs() + off) + 2 ** -100
        return out, tol

    def check(self, got, **kw):
        want, tol = self.want(**kw)
        off = (got.cpu().double() - want).abs()
        assert torch.isfinite(got).all()
        assert (off <= tol).all(), f"{(off / tol).max().item():.2f} times the tolerance"


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("ctx,nodes,heads,kv_heads,page", [
    ([0], [1], 1, 1, 16),                      # the node itself is all there is
    ([1], [1], 8, 1, 16),
    ([37], [5], 4, 2, 16),                     # under one stage
    ([128, 127, 129], [1, 1, 1], 16, 2, 16),   # single tokens about a stage's end
    ([300], [3], 16, 2, 272),
    ([64, 0, 63, 200], [2, 4, 1, 7], 8, 4, 48),
    ([500, 20], [8, 8], 16, 2, 16),            # 64 rows a kv head
    ([130, 700], [17, 33], 4, 1, 16),          # 132 rows: two tiles
    ([90], [64], 8, 1, 1),                     # pages of one token
    ([0, 5, 2], [40, 0, 70], 6, 2, 16),        # no context, an empty request, three words
    ([33], [100], 3, 3, 16),                   # no sharing of kv heads
])
def test_matches_64_bits(ctx, nodes, heads, kv_heads, page, dim):
    c = Case(ctx, nodes, heads, kv_heads, dim, page, gate=len(ctx) % 2 == 1, seed=sum(ctx) + dim)
    c.check(c.run())


@pytest.mark.parametrize("max_context_len", [3000, 0, 100000])
@pytest.mark.parametrize("nodes", [[1, 3, 2], [9, 2, 20], [12, 64, 1]])
def test_long_contexts_split(nodes, max_context_len):
    """Several chunks a request, of ragged lengths; the bound on the context only
    shapes the launch."""
    c = Case([3000, 1, 1111], nodes, heads=4, kv_heads=1, gate=True, seed=7)
    c.check(c.run(max_context_len=max_context_len))


@pytest.mark.parametrize("requests,most,longest,heads,kv_heads,dim", [
    (150, 3, 200, 4, 2, 64),        # more requests than a wave has lanes
    (70, 40, 130, 8, 1, 64),        # row tiles of their own number in each request
    (65, 1, 700, 2, 1, 128), (3, 64, 1500, 16, 1, 64), (130, 2, 1, 2, 2, 64)])
def test_ragged_batches(requests, most, longest, heads, kv_heads, dim):
    """Stretches of the work that start and end anywhere: in requests without
    nodes or context, between kv heads, in the middle of a request."""
    gen = torch.Generator().manual_seed(requests)
    ctx = torch.randint(0, longest + 1, (requests,), generator=gen).tolist()
    nodes = torch.randint(0, most + 1, (requests,), generator=gen).tolist()
    nodes[0], nodes[-1], nodes[1] = 0, 0, most
    c = Case(ctx, nodes, heads, kv_heads, dim, seed=requests)
    c.check(c.run())


@pytest.mark.parametrize("ctx,nodes", [
    ([2000], [150]),           # one request of 19 row tiles: lines of one length
    ([300], [530]),            # of 67: more lines than workgroups in blocks of 8 hold
    ([700, 1500, 90], [90, 20, 130]),   # lines of 17 lengths
])
def test_many_row_tiles(ctx, nodes):
    c = Case(ctx, nodes, heads=16, kv_heads=1, dim=64, seed=sum(nodes))
    c.check(c.run())


def test_layouts_and_strides():
    c = Case([50, 200], [6, 3], heads=8, kv_heads=2, dim=64, layout="head_major", seed=8)
    c.check(c.run())
    big = torch.full((9, 8, 3 * 64), 3.0, dtype=torch.bfloat16, device=DEV)
    out = big[:, :, 64:128]
    q = torch.zeros(9, 8, 128, dtype=torch.bfloat16, device=DEV)
    q[..., 64:] = c.q.to(DEV)
    assert c.run(out=out, q=q[..., 64:]) is out
    c.check(out)
    assert (big[:, :, :64] == 3).all() and (big[:, :, 128:] == 3).all()
    wide = torch.zeros(9, 5, dtype=torch.int32)
    wide[:, 1:2] = c.anc
    c.check(c.run(anc=wide[:, 1:2]))
    c.check(c.run(anc=torch.nn.functional.pad(c.anc, (0, 3))))     # more words than nodes


def test_rows_that_see_nothing_are_zero():
    c = Case([0, 30], [4, 3], seed=9)
    anc = c.anc.clone()
    anc[:3] = 0
    anc[5] = 0                        # sees the context alone
    got = c.run(anc=anc)
    assert (got[:3] == 0).all()
    c.check(got, anc=anc)
    # no words at all: nothing drafted is seen
    none = torch.zeros(7, 0, dtype=torch.int32)
    got = c.run(anc=none)
    assert (got[:4] == 0).all()
    c.check(got, anc=none)


def test_any_mask_is_taken():
    """Not only trees: later nodes, arbitrary subsets, bits past the nodes."""
    c = Case([20, 7], [40, 33], heads=2, kv_heads=1, seed=10)
    anc = torch.randint(-2**31, 2**31, (73, 2), generator=c.gen).to(torch.int32)
    c.check(c.run(anc=anc), anc=anc)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("ctx", [100, 0, 61])
@pytest.mark.parametrize("nodes", [6, 60])
def test_unseen_nodes_may_hold_anything(bad, ctx, nodes):
    """A node whose K/V are not finite is seen by its descendants only; every
    other row has the bits that it has without it."""
    c = Case([ctx], [nodes], heads=8, kv_heads=2, seed=11)
    clean = c.run()
    node = 1
    pos = ctx + node
    c.kv[c.table[0, pos // 16], pos % 16] = bad
    got = c.run()
    sees = (c.anc[:, 0] >> node) & 1 != 0
    assert sees.any() and not sees.all()
    off = (got.float() - clean.float())[~sees.to(DEV)].abs()
    c_want, tol = c.want()
    assert torch.isfinite(got[~sees.to(DEV)]).all()
    assert ((got.cpu().double() - c_want).abs() <= tol)[~sees].all()
    assert got[sees.to(DEV)].isnan().all()
    assert off.max() <= 2 * tol[~sees].max()


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("at", [0, 63, 64, 69])
@pytest.mark.parametrize("ctx,nodes,heads", [([70], [5], 16), ([70, 130], [1, 20], 4),
                                             ([128, 70], [2, 2], 8), ([700, 70], [1, 3], 4)])
def test_committed_values_that_are_not_finite_reach_every_row(bad, ctx, nodes, heads, at):
    """Wherever the committed token lies: in a stage of its own kind or in one
    that the drafted tokens share. Only its dimension is lost."""
    case = Case(ctx, nodes, heads=heads, kv_heads=2, seed=at)
    b = len(ctx) - 1
    case.kv[case.table[b, at // 16], at % 16, 0, case.dim + 3] = bad
    got = case.run().cpu()
    hit = torch.zeros(got.shape, dtype=torch.bool)
    if at < ctx[b]:
        hit[case.starts[b]:case.starts[b + 1], :heads // 2, 3] = True
    assert torch.equal(~torch.isfinite(got), hit)
    case.kv[case.table[b, at // 16], at % 16, 0, case.dim + 3] = 0.0
    want, tol = case.want()
    assert ((got.double() - want).abs() <= tol)[~hit].all()


def test_positions_without_a_page_are_not_seen():
    c = Case([100, 70], [3, 2], heads=4, kv_heads=1, seed=12)
    table = c.table.clone()
    table[0, 2] = -1
    table[1, 0] = c.kv.shape[0]          # past the cache
    table[0, 4] = -2**31
    table[1, 3] = 2**31 - 1
    c.check(c.run(table=table), table=table)
    short = c.table[:, :5]               # a table that ends inside the first context
    c.check(c.run(table=short), table=short)
    empty = c.table[:, :0]
    assert (c.run(table=empty) == 0).all()


def test_lengths_on_the_device_stay_within_the_tensors():
    """Starts outside the rows, falling starts, negative and huge contexts: no
    access outside the tensors, and the requests that are sound are right."""
    c = Case([40, 25], [4, 4], heads=4, kv_heads=1, seed=13)
    want = c.run()
    k, v = c.device_cache()

    def call(ctx, qsl):
        out = torch.full((8, 4, 128), 5.0, dtype=torch.bfloat16, device=DEV)
        return qsa_tree_paged_attention(
            c.q.to(DEV), k, v, c.table.to(DEV), torch.tensor(ctx, dtype=torch.int32, device=DEV),
            torch.tensor(qsl, dtype=torch.int32, device=DEV), c.anc.to(DEV), out,
            max_query_len=4, max_context_len=40)

    got = call([40, 25], [0, 4, 4])
    assert torch.equal(got[:4], want[:4]) and (got[4:] == 5).all()   # rows of no request
    got = call([40, -3], [0, 4, 2])
    assert torch.equal(got[:4], want[:4]) and (got[4:] == 5).all()
    got = call([40, 2**31 - 1], [0, 4, 8])
    assert torch.equal(got[:4], want[:4])
    got = call([-2**31, 25], [-5, 4, 1 << 30])
    assert torch.equal(got[4:], want[4:])


def test_more_nodes_than_said_are_left():
    c = Case([30], [20], heads=2, kv_heads=1, seed=14)
    out = torch.full((20, 2, 128), 5.0, dtype=torch.bfloat16, device=DEV)
    c.run(out=out, max_query_len=8)
    want, tol = c.want()
    assert ((out.cpu().double() - want).abs() <= tol)[:8].all()


def test_a_chain_equals_the_sparse_attention_over_every_slot():
    """Single tokens: the sparse op with every slot of the context selected does
    the same sum (its own tolerance: two bf16 roundings of the weights)."""
    c = Case([90, 33], [1, 1], heads=16, kv_heads=2, seed=15)
    k, v = c.device_cache()
    idx = torch.full((2, 91), -1, dtype=torch.int32)
    for b, n in enumerate((91, 34)):
        for p in range(n):
            idx[b, p] = int(c.table[b, p // 16]) * 16 + p % 16
    other = qsa_sparse_paged_attention(
        c.q.to(DEV), k, v, idx.to(DEV), c.table.to(DEV),
        torch.arange(2, dtype=torch.int32, device=DEV), use_decode_kernel=True,
        indices_are_physical=True, valid_counts=torch.tensor([91, 34], dtype=torch.int32, device=DEV))
    got = c.run()
    _, tol = c.want()
    assert ((got.cpu().double() - other.cpu().double()).abs() <= 2 * tol).all()


def test_large_scores():
    """Scores of hundreds: one weight takes all, nothing overflows."""
    c = Case([200, 50], [4, 9], heads=4, kv_heads=2, scale=6.0, seed=16)
    c.check(c.run())


def test_offsets_past_32_bits():
    """Pages whose byte offsets pass 4 GiB."""
    blocks, page, heads, dim = 300000, 16, 2, 128
    if torch.cuda.mem_get_info()[0] < (12 << 30):
        pytest.skip("needs 12 GiB of free GPU memory")
    c = Case([40, 70], [3, 5], heads=4, kv_heads=heads, seed=17)
    kv = torch.empty(blocks, page, heads, 2 * dim, dtype=torch.bfloat16, device=DEV)
    far = c.table.clone()
    for b in range(2):
        for i in range(c.table.shape[1]):
            if c.table[b, i] >= 0:
                far[b, i] = blocks - 1 - int(c.table[b, i]) * 7
                kv[far[b, i]] = c.kv[c.table[b, i]].to(DEV)
    got = qsa_tree_paged_attention(
        c.q.to(DEV), kv[..., :dim], kv[..., dim:], far.to(DEV),
        torch.tensor(c.ctx, dtype=torch.int32, device=DEV), c.qsl.to(DEV), c.anc.to(DEV),
        max_query_len=5, max_context_len=70)
    assert torch.equal(got, c.run())


def test_streams_and_graphs():
    """The same bits on another stream and in every replay of a graph, whose
    lengths, tables and ancestors are read anew each time."""
    c = Case([900, 60], [7, 12], heads=8, kv_heads=2, seed=18)
    k, v = c.device_cache()
    q, table, qsl, anc = (t.to(DEV) for t in (c.q, c.table, c.qsl, c.anc))
    ctx = torch.tensor(c.ctx, dtype=torch.int32, device=DEV)
    out = torch.zeros_like(q)

    def step():
        return qsa_tree_paged_attention(q, k, v, table, ctx, qsl, anc, out, max_query_len=12,
                                        max_context_len=900)
    first = step().clone()
    c.check(first)
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    outs = [torch.zeros_like(q) for _ in range(2)]
    for s, o in zip((a, b), outs):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            for _ in range(5):
                qsa_tree_paged_attention(q, k, v, table, ctx, qsl, anc, o, max_query_len=12,
                                         max_context_len=900)
    torch.cuda.synchronize()
    assert torch.equal(outs[0], first) and torch.equal(outs[1], first)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for shorter in (0, 100, 333, 0):
        ctx.copy_(torch.tensor([900 - shorter, 60 - shorter // 10], dtype=torch.int32))
        graph.replay()
        got = out.clone()
        out.zero_()
        want = step().clone()
        torch.cuda.synchronize()
        assert torch.equal(got, want)


def test_refusals():
    c = Case([20], [3], seed=19)
    k, v = c.device_cache()
    i32 = dict(dtype=torch.int32, device=DEV)
    args = [c.q.to(DEV), k, v, c.table.to(DEV), torch.tensor([20], **i32), c.qsl.to(DEV),
            c.anc.to(DEV)]

    def call(**over):
        a = list(args)
        kw = dict(max_query_len=3, max_context_len=20)
        for key, value in over.items():
            if key.startswith("a"):
                a[int(key[1:])] = value
            else:
                kw[key] = value
        return qsa_tree_paged_attention(*a, **kw)

    call()
    for over, match in ((dict(a0=args[0].half()), "q must be"), (dict(a1=k.half()), "k_cache"),
                        (dict(a0=args[0][..., :64]), "cache head dim"),
                        (dict(a2=v[:, :8]), "one shape"), (dict(a3=args[3].long()), "block_table"),
                        (dict(a4=args[4].long()), "context_lens"), (dict(a4=args[4][:0]), "entries"),
                        (dict(a5=args[5][:1]), "entries"), (dict(a6=args[6][:2]), "each query row"),
                        (dict(a6=args[6].long()), "ancestors"), (dict(max_query_len=-1), "max_query"),
                        (dict(max_context_len=1 << 40), "max_context"),
                        (dict(out=torch.empty(2, 4, 128, dtype=torch.bfloat16, device=DEV)), "out"),
                        (dict(output_gate=args[0][:2]), "output_gate"),
                        (dict(a0=args[0][:, :3]), "multiple of kv heads"),
                        (dict(a6=args[6].cpu()), "GPU")):
        with pytest.raises(RuntimeError, match=match):
            call(**over)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("scale", [1.0, 5.0])
@pytest.mark.parametrize("longest", [None, 0])
@pytest.mark.parametrize("ctx,nodes,heads", [([100], [6], 8), ([0], [60], 8), ([61, 300], [9, 30], 16),
                                             ([1500], [20], 4)])
def test_a_row_has_its_own_bits(bad, ctx, nodes, heads, longest, scale):
    """Neither nodes that it does not see nor the other rows' queries reach a
    row's result: the same bits whatever those hold. A stage for each workgroup and
    (no context announced) all stages in one, with maxima that keep rising."""
    c = Case(ctx, nodes, heads=heads, kv_heads=2, seed=21, scale=scale)
    clean = c.run(max_context_len=longest)
    b, node = len(ctx) - 1, 1
    first, pos = c.starts[b], ctx[b] + node
    sees = torch.zeros(clean.shape[0], dtype=torch.bool)
    sees[first:] = (c.anc[first:, 0] >> node) & 1 != 0
    assert sees.any() and not sees.all()
    keep = c.kv[c.table[b, pos // 16], pos % 16].clone()
    for what in (slice(None), slice(0, c.dim), slice(c.dim, None)):      # K and V, K, V
        c.kv[c.table[b, pos // 16], pos % 16, :, what] = bad
        got = c.run(max_context_len=longest)
        assert torch.equal(got[~sees], clean[~sees])
        assert not torch.isfinite(got[sees]).any()
        c.kv[c.table[b, pos // 16], pos % 16] = keep
    one = torch.arange(clean.shape[0]) % 3 == 0
    q = torch.where(one[:, None, None], c.q, (c.q.float() * 9).bfloat16()).to(DEV)
    assert torch.equal(c.run(q=q, max_context_len=longest)[one], clean[one])
    q[~one.to(DEV)] = bad
    assert torch.equal(c.run(q=q, max_context_len=longest)[one], clean[one])


def _softmax(case, row, head, b):
    """A row's result in 64 bits by IEEE arithmetic, but for a score of -inf, whose
    weight is 0: zeros if there is no other."""
    h = head // (case.heads // case.kv_heads)
    seen = list(range(case.ctx[b])) + [case.ctx[b] + j for j in range(case.nodes[b])
                                       if (int(case.anc[row, j // 32]) >> (j % 32)) & 1]
    kv = torch.stack([case.kv[case.table[b, p // case.page], p % case.page, h] for p in seen]).double()
    s = kv[:, :case.dim] @ case.q[row, head].double() / math.sqrt(case.dim)
    live = s != -math.inf
    if not live.any():
        return torch.zeros(case.dim, dtype=torch.float64)
    p = torch.exp(s[live] - s[live].max())
    return (p / p.sum()) @ kv[live, case.dim:]


@pytest.mark.parametrize("ctx,at", [(100, 101), (100, 60), (64, 65), (700, 702), (700, 3)])
@pytest.mark.parametrize("heads", [2, 16])
def test_infinite_values_give_what_their_sum_gives(ctx, at, heads):
    """One infinity in a dimension: an infinity of its sign. Two of unlike signs, or
    a NaN: NaN. The same for committed tokens and drafted ones."""
    inf, nan = math.inf, math.nan
    c = Case([ctx], [8], heads=heads, kv_heads=2, seed=22, chain=True)
    near = at + 1 if at + 1 != ctx else at - 1
    for pos, dim, value in ((at, 0, inf), (at, 17, -inf), (at, 40, nan), (at, 63, inf),
                            (near, 63, -inf), (near, 100, -inf), (at, 100, -inf)):
        c.kv[c.table[0, pos // 16], pos % 16, :, c.dim + dim] = value
    for longest in (None, 0):
        got = c.run(max_context_len=longest).cpu().double()
        for row in (0, 1, 2, 4, 7):
            want = _softmax(c, row, 0, 0)
            fine = torch.isfinite(want)
            assert torch.equal(torch.nan_to_num(got[row, 0, ~fine], nan=7.0),
                               torch.nan_to_num(want[~fine], nan=7.0)), (row, longest)
            assert torch.isfinite(got[row, 0, fine]).all()


@pytest.mark.parametrize("ctx,at", [(100, 20), (100, 102), (3, 0), (900, 640)])
def test_infinite_keys_follow_their_scores(ctx, at):
    """One infinite element of K: the score is an infinity of its product's sign.
    Infinity gives NaN, minus infinity no weight; a row that has no other score
    gets zeros like one that sees nothing."""
    c = Case([ctx], [5], heads=4, kv_heads=2, seed=23, chain=True)
    for sign in (1.0, -1.0):
        c.kv[c.table[0, at // 16], at % 16, :, 5] = sign * math.inf
        for longest in (None, 0):
            got = c.run(max_context_len=longest).cpu().double()
            for row in range(5):
                for head in range(4):
                    want = _softmax(c, row, head, 0)
                    assert torch.equal(want.isnan(), got[row, head].isnan())
                    if not want.isnan().any():       # values of about 1, weights off by 2^-8
                        assert (got[row, head] - want).abs().max() < 0.1
    c = Case([40], [3], heads=2, kv_heads=1, seed=24, chain=True)
    for pos in range(43):
        c.kv[c.table[0, pos // 16], pos % 16, :, 5] = math.inf
    c.q[:, :, 5] = -c.q[:, :, 5].abs() - 1
    assert (c.run() == 0).all() and (c.run(max_context_len=0) == 0).all()


@pytest.mark.parametrize("ctx,nodes,heads,longest", [([30], [20], 2, None), ([700, 90], [20, 13], 16, None),
                                                     ([90, 2500, 64], [9, 40, 8], 8, None),
                                                     ([700, 90], [20, 13], 16, 0)])
def test_rows_past_the_announced_nodes_are_not_written(ctx, nodes, heads, longest):
    """Requests of more nodes than ``max_query_len``, in one stage and over several
    workgroups and the joining launch: the first ones are right, the rest left."""
    c = Case(ctx, nodes, heads=heads, kv_heads=2 if heads > 2 else 1, seed=25)
    out = torch.full((sum(nodes), heads, 128), 5.0, dtype=torch.bfloat16, device=DEV)
    c.run(out=out, max_query_len=8, max_context_len=longest)
    want, tol = c.want()
    done = torch.zeros(sum(nodes), dtype=torch.bool)
    for start, n in zip(c.starts, nodes):
        done[start:start + min(n, 8)] = True
    got = out.cpu().double()
    assert ((got - want).abs() <= tol)[done].all()
    assert (got[~done] == 5).all()


@pytest.mark.parametrize("ctx,nodes,heads,kv_heads,dim,page", [
    ([131072], [1], 16, 2, 128, 16), ([131072], [64], 16, 2, 128, 16), ([65537], [33], 8, 1, 64, 272),
    ([32768, 4096, 20000, 1, 9999], [24, 5, 1, 16, 17], 16, 2, 128, 16)])
def test_served_lengths(ctx, nodes, heads, kv_heads, dim, page):
    """Contexts as long as they are served, against 64 bits on the GPU. The
    tolerance is the 64-bit statement's of the other tests, one row at a time."""
    gen = torch.Generator(device=DEV).manual_seed(sum(ctx))
    cpu = torch.Generator().manual_seed(sum(ctx))
    pages = [-(-(c + t) // page) for c, t in zip(ctx, nodes)]
    order = torch.randperm(sum(pages), generator=cpu).to(torch.int32)
    table = torch.full((len(ctx), max(pages)), -1, dtype=torch.int32)
    at = 0
    for b, p in enumerate(pages):
        table[b, :p] = order[at:at + p]
        at += p
    table = table.to(DEV)
    kv = torch.randn(len(order), page, kv_heads, 2 * dim, generator=gen, device=DEV).bfloat16()
    rows, group = sum(nodes), heads // kv_heads
    q = torch.randn(rows, heads, dim, generator=gen, device=DEV).bfloat16()
    starts = torch.tensor([0] + nodes).cumsum(0)
    parents = torch.cat([torch.arange(t) - 1 - torch.randint(0, 4, (t,), generator=cpu) for t in nodes])
    anc = tree_ancestors(parents, starts, max(nodes))
    got = qsa_tree_paged_attention(
        q, kv[..., :dim], kv[..., dim:], table, torch.tensor(ctx, dtype=torch.int32, device=DEV),
        starts.to(torch.int32).to(DEV), anc.to(DEV), max_query_len=max(nodes),
        max_context_len=max(ctx)).double()
    for b, (c, t) in enumerate(zip(ctx, nodes)):
        pos = torch.arange(c + t, device=DEV)
        of = kv[table[b].long()[pos // page], pos % page].double()
        for j in {0, t // 2, t - 1}:
            row = int(starts[b]) + j
            seen = torch.ones(c + t, dtype=torch.bool)
            seen[c:] = torch.tensor([(int(anc[row, i // 32]) >> (i % 32)) & 1 != 0 for i in range(t)])
            mine = of[seen.to(DEV)]
            for h in range(heads):
                k, v = mine[:, h // group, :dim], mine[:, h // group, dim:]
                x = q[row, h].double()
                p = torch.softmax((k * x).sum(1) / math.sqrt(dim), 0)
                o = (p[:, None] * v).sum(0)
                spread = (k * x).abs().sum(1).max() / math.sqrt(dim)
                off = (2 ** -8 * (1 + 2 ** -7) * (p[:, None] * (v - o).abs()).sum(0)
                       + (2 * 36 * 2 ** -24 * spread + 2 ** -18) * (p[:, None] * v.abs()).sum(0))
                tol = off + 2 ** -8 * (o.abs() + off)
                assert ((got[row, h] - o).abs() <= tol).all(), (b, j, h)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("longest", [None, 0])
def test_keys_and_values_in_caches_of_their_own(dim, longest):
    """K and V of unlike strides: tokens before heads in one, heads before tokens
    with a margin around each row in the other; a gate of any strides."""
    c = Case([333, 64, 5], [7, 20, 1], heads=8, kv_heads=2, dim=dim, gate=True, seed=27)
    k = c.kv[..., :dim].contiguous().to(DEV)
    blocks, page = c.kv.shape[:2]
    wide = torch.full((blocks, 2, page, dim + 24), float("nan"), dtype=torch.bfloat16, device=DEV)
    v = wide.permute(0, 2, 1, 3)[..., 8:8 + dim]
    v.copy_(c.kv[..., dim:])
    gate = c.gate.permute(2, 0, 1).contiguous().to(DEV).permute(1, 2, 0)
    got = qsa_tree_paged_attention(
        c.q.to(DEV), k, v, c.table.to(DEV), torch.tensor(c.ctx, dtype=torch.int32, device=DEV),
        c.qsl.to(DEV), c.anc.to(DEV), output_gate=gate, max_query_len=20,
        max_context_len=max(c.ctx) if longest is None else longest)
    c.check(got)


def test_a_padded_batch():
    """Requests behind the last one (no rows, whatever their lengths and pages) and
    rows behind the last request: the others are right, those rows left."""
    c = Case([500, 90], [9, 4], heads=8, kv_heads=2, seed=28)
    k, v = c.device_cache()
    i32 = dict(dtype=torch.int32, device=DEV)
    table = torch.cat([c.table, torch.full((3, c.table.shape[1]), 2**31 - 1, dtype=torch.int32)]).to(DEV)
    ctx = torch.tensor(c.ctx + [2**31 - 1, -5, 7], **i32)
    qsl = torch.tensor([0, 9, 13, 13, 13, 13], **i32)
    q = torch.cat([c.q, torch.full((6, 8, 128), float("nan"), dtype=torch.bfloat16)]).to(DEV)
    anc = torch.nn.functional.pad(c.anc, (0, 0, 0, 6), value=-1).to(DEV)
    out = torch.full_like(q, 5.0)
    for longest in (500, 0):
        qsa_tree_paged_attention(q, k, v, table, ctx, qsl, anc, out, max_query_len=9,
                                 max_context_len=longest)
        c.check(out[:13])
        assert (out[13:] == 5).all()
