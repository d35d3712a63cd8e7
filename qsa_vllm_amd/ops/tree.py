"""Attention of drafted token trees over the paged cache (``csrc/tree_attn.hip``).

A speculative step verifies a tree of drafted tokens per request: every node
attends over the request's committed tokens and over its ancestors in the tree.
The nodes' K/V lie in the request's cache at the positions after the committed
ones (written by ``qsa_prepare`` or ``qsa_store_cache_rows`` before), in node
order. Which nodes a row sees is a bit row (``ancestors``), made from parent
indices by ``tree_ancestors``; a chain of drafted tokens, or a single token, is
a tree too. Unlike ``qsa_sparse_paged_attention`` nothing is selected: rows
attend over the whole committed context, whose K/V are read once for all nodes.
So past the number of tokens that a sparse layer selects, the result is not that
layer's.
"""

from __future__ import annotations

import torch

from . import _torch_ops  # noqa: F401  (registers torch.ops.yulan_qsa_kernels)
from ._torch_ops import _require

__all__ = ["qsa_tree_paged_attention", "tree_ancestors"]


def tree_ancestors(parents: torch.Tensor, query_start_loc: torch.Tensor,
                   max_query_len: int) -> torch.Tensor:
    """int32 ``[rows, ceil(max_query_len / 32)]``: bit ``j % 32`` of word
    ``j // 32`` is set where node ``j`` of the row's request is the row itself
    or one of its ancestors. ``parents`` (``[rows]``): each node's parent as a
    node index of its own request, an earlier node; any other value is the
    committed context. ``query_start_loc``: int32 ``[requests + 1]``. Runs on the
    tensors' device without a synchronisation."""
    _require(parents.dim() == 1 and not parents.is_floating_point(),
             "parents must be a vector of node indices")
    _require(max_query_len > 0, "max_query_len must be positive")
    rows, dev = parents.numel(), parents.device
    words = -(-int(max_query_len) // 32)
    row = torch.arange(rows, device=dev)
    starts = query_start_loc.long()
    request = (torch.searchsorted(starts, row, right=True) - 1).clamp_(0, max(0, starts.numel() - 2))
    first = starts[request]
    node = row - first
    word = torch.arange(words, device=dev)
    own = (torch.ones_like(node) << (node & 31))[:, None] * (word == (node >> 5)[:, None])
    # 32 bits as a signed word; one more row, of no bits, is every root's parent.
    bits = torch.zeros(rows + 1, words, dtype=torch.int32, device=dev)
    bits[:rows] = (own - ((own >> 31) << 32)).to(torch.int32)
    parent = parents.long()
    up = torch.full((rows + 1,), rows, dtype=torch.int64, device=dev)
    up[:rows] = torch.where((parent >= 0) & (parent < node), first + parent,
                            torch.full_like(parent, rows))
    # Doubling: after step s a row holds its ancestors up to 2^s levels up.
    for _ in range(int(max_query_len).bit_length()):
        bits |= bits[up]
        up = up[up]
    return bits[:rows]


def qsa_tree_paged_attention(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    block_table: torch.Tensor,
    context_lens: torch.Tensor,
    query_start_loc: torch.Tensor,
    ancestors: torch.Tensor,
    out: torch.Tensor | None = None,
    *,
    output_gate: torch.Tensor | None = None,
    max_query_len: int,
    max_context_len: int,
) -> torch.Tensor:
    """BF16 paged GQA of drafted nodes ``q`` (``[rows, heads, dim]``, request b's
    at rows ``query_start_loc[b] ..``) over ``context_lens[b]`` committed tokens
    and the nodes that ``ancestors`` shows each row. Row order, caches, table and
    gate as in ``qsa_sparse_paged_attention``; the gated result is rounded once.
    A row that sees nothing gets zeros. Infinities and NaN in K or V reach the rows
    that see them, as arithmetic has it, and no others; a score of minus infinity
    weighs nothing, and a row that has no other gets zeros. Rows of no request
    (past ``query_start_loc[-1]``) are not written. The caches must span less than
    64 GiB each. ``max_query_len`` must be at least every request's node count
    (further nodes are not computed); ``max_context_len`` should be at least every
    context length: it shapes the launch, not the result. Captured into a graph,
    both hold for its replays."""
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    torch.ops.yulan_qsa_kernels.tree_attention(
        q, k_cache, v_cache, block_table, context_lens, query_start_loc, ancestors, out,
        output_gate, int(max_query_len), int(max_context_len))
    return out
