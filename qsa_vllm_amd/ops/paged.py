"""Causal attention over the paged cache: a sliding window with a few first tokens
that stay visible, or the whole context, from a bf16 cache or one of 4 bits
(``csrc/paged_attn.hip``).

Unlike ``qsa_sparse_paged_attention`` nothing is selected, and unlike
``qsa_tree_paged_attention`` the rows are the last tokens of their requests in order:
single tokens, prompt chunks, or both in one call.
"""

from __future__ import annotations

import torch

from . import _torch_ops  # noqa: F401  (registers torch.ops.yulan_qsa_kernels)
from ._torch_ops import _require
from .kv_cache import Int4KVCache

__all__ = ["qsa_int4_paged_attention", "qsa_window_paged_attention"]

# (looked up once: 1 us of a call)
_window_attention = torch.ops.yulan_qsa_kernels.window_attention.default
_int4_kv_attention = torch.ops.yulan_qsa_kernels.int4_kv_attention.default


def _window(window: int | None) -> int:
    _require(window is None or window > 0, f"window must be positive or None, got {window}")
    return 0 if window is None else int(window)


def qsa_window_paged_attention(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    block_table: torch.Tensor,
    seq_lens: torch.Tensor,
    query_start_loc: torch.Tensor,
    out: torch.Tensor | None = None,
    *,
    window: int | None = None,
    sink_tokens: int = 0,
    output_gate: torch.Tensor | None = None,
    max_query_len: int,
    max_seq_len: int,
) -> torch.Tensor:
    """BF16 paged GQA of ``q`` (``[rows, heads, dim]``): request b's rows
    ``query_start_loc[b] ..`` are the last tokens of its ``seq_lens[b]`` (int32, on the
    device), whose K/V are in the cache. A row at position p sees the positions j <= p
    with j > p - ``window`` (itself and the ``window`` - 1 before it; None: all) or j <
    ``sink_tokens``. Caches ``[blocks, page, kv_heads, dim]``, table and gate as in
    ``qsa_sparse_paged_attention``; the gated result is rounded once.

    Positions without a page (an entry of ``block_table`` that is no block, such as -1
    for pages that left every window and were freed) are not seen, and a row that sees
    nothing gets zeros. Infinities and NaN in K or V reach the rows that see them, as
    arithmetic has it, and no others; a score of minus infinity weighs nothing. Scores and
    weighted sums are held in fp32: V's largest magnitude times the tokens that a row sees
    must be under 2^117, the sum of a query's magnitudes times K's largest under 2^125
    (past that finite values may give infinities or NaN). Rows of no request (past ``query_start_loc[-1]``) are not written. The caches must span less
    than 64 GiB each. ``max_query_len`` must be at least every request's row count
    (further rows are not computed); ``max_seq_len`` should be at least every length: it
    shapes the launch, not the result. Captured into a graph, both hold for its replays."""
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    _window_attention(
        q, k_cache, v_cache, block_table, seq_lens, query_start_loc, out, output_gate,
        _window(window), int(sink_tokens), int(max_query_len), int(max_seq_len))
    return out


def qsa_int4_paged_attention(
    q: torch.Tensor,
    cache: Int4KVCache,
    block_table: torch.Tensor,
    seq_lens: torch.Tensor,
    query_start_loc: torch.Tensor,
    out: torch.Tensor | None = None,
    *,
    window: int | None = None,
    sink_tokens: int = 0,
    output_gate: torch.Tensor | None = None,
    max_query_len: int,
    max_seq_len: int,
) -> torch.Tensor:
    """``qsa_window_paged_attention`` over a cache held in 4 bits (written by
    ``qk_norm_rope``): the attention of the values that its codes stand for."""
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    _require(q.dim() == 3 and q.shape[2] == cache.head_dim, "the cache's head dim must match q")
    _int4_kv_attention(
        q, cache.data, cache.page_size, block_table, seq_lens, query_start_loc, out, output_gate,
        _window(window), int(sink_tokens), int(max_query_len), int(max_seq_len))
    return out
