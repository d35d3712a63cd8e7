"""What an attention layer does to its heads before it attends, and a KV cache
held in 4 bits (``csrc/head_rope.hip``, ``csrc/kv4.h``).

``qk_norm_rope`` norms the queries and keys of each head, rotates them by their
position and writes keys and values into the paged cache, in one launch. The cache
is the bf16 one of the other layers or an :class:`Int4KVCache`, whose values take
4.5 bits: codes with one scale and zero point for each token, head and 32 dims.
``qsa_window_paged_attention`` and ``qsa_int4_paged_attention`` read them.
"""

from __future__ import annotations

from dataclasses import dataclass

import torch

from .. import _lib
from . import _torch_ops  # noqa: F401  (registers torch.ops.yulan_qsa_kernels)
from ._torch_ops import _require

__all__ = ["Int4KVCache", "qk_norm_rope", "rotary_table"]

_GROUP = 32
# (looked up once: 1 us of a call)
_qk_norm_rope = torch.ops.yulan_qsa_kernels.qk_norm_rope.default


@dataclass(frozen=True)
class Int4KVCache:
    """K and V of ``data.shape[0]`` pages of ``page_size`` tokens in 4 bits. ``data``
    (uint8 ``[blocks, kv_heads, page bytes]``) has the C ABI's layout
    (``qsa_qk_norm_rope``); :meth:`allocate` makes an empty one."""

    data: torch.Tensor
    page_size: int
    head_dim: int

    @staticmethod
    def page_bytes(page_size: int, head_dim: int) -> int:
        """Bytes of one kv head's page."""
        _require(page_size > 0 and head_dim in (64, 128),
                 "a 4-bit cache needs a positive page size and a head dim of 64 or 128")
        return _lib.load().qsa_kv4_page_bytes(int(page_size), int(head_dim))

    @classmethod
    def allocate(cls, num_blocks: int, page_size: int, kv_heads: int, head_dim: int,
                 device=None) -> "Int4KVCache":
        data = torch.zeros(num_blocks, kv_heads, cls.page_bytes(page_size, head_dim),
                           dtype=torch.uint8, device=device)
        return cls(data, page_size, head_dim)

    @property
    def kv_heads(self) -> int:
        return self.data.shape[1]

    def dequantize(self) -> tuple[torch.Tensor, torch.Tensor]:
        """K and V ``[blocks, page, kv_heads, dim]`` as the bf16 values that they stand
        for (for checks)."""
        page, dim = self.page_size, self.head_dim
        blocks, heads = self.data.shape[:2]
        codes, words = page * dim // 2, page * dim // 16
        out = []
        for which in (0, 1):
            c = self.data[:, :, which * codes:(which + 1) * codes].reshape(blocks, heads, page, -1)
            c = torch.stack((c & 15, c >> 4), -1).flatten(-2)
            if which == 0:
                # Rows of words [8 dims' place b][group a]; nibble i is dim 2 i, then 2 i + 1.
                c = c.unflatten(-1, (4, dim // _GROUP, 2, 4)).transpose(-1, -2)
                c = c.flatten(-2).transpose(-3, -2).flatten(-3)
            first = 2 * codes + which * (-(-words // 16) * 16)
            w = self.data[:, :, first:first + words].reshape(blocks, heads, page, -1, 2).to(torch.int32)
            w = w[..., 0] | (w[..., 1] << 8)
            scale = ((w & 0xFFF0) << 16).view(torch.float32)
            scale = torch.where(scale.isfinite(), scale, torch.nan)  # as the attention reads it
            x = (c.unflatten(-1, (-1, _GROUP)) - (w & 15).float()[..., None]) * scale[..., None]
            out.append(x.flatten(-2).to(torch.bfloat16).transpose(1, 2))
        return out[0], out[1]


def rotary_table(max_position: int, rotary_dim: int, theta: float, device=None) -> torch.Tensor:
    """fp32 ``[max_position, rotary_dim]``: cosines, then sines, of the angles position
    * theta^(-2 c / rotary_dim), which are formed in 64 bits (in 32 a position of 10^5
    would be off by 2^-8 of a turn)."""
    even = torch.arange(0, rotary_dim, 2, dtype=torch.float64, device=device)
    positions = torch.arange(max_position, dtype=torch.float64, device=device)
    angles = torch.outer(positions, float(theta) ** (-even / max(rotary_dim, 1)))
    return torch.cat((angles.cos(), angles.sin()), dim=-1).float()


def qk_norm_rope(
    query: torch.Tensor | None,
    key: torch.Tensor,
    q_weight: torch.Tensor | None,
    k_weight: torch.Tensor | None,
    positions: torch.Tensor | None,
    cos_sin: torch.Tensor | None,
    eps: float,
    *,
    value: torch.Tensor | None = None,
    cache: Int4KVCache | tuple[torch.Tensor, torch.Tensor] | None = None,
    slot_mapping: torch.Tensor | None = None,
    q_out: torch.Tensor | None = None,
    k_out: torch.Tensor | None = None,
    v_out: torch.Tensor | None = None,
) -> tuple[torch.Tensor | None, torch.Tensor | None]:
    """RMSNorm of every ``query`` and ``key`` head (bf16 ``[tokens, heads, dim]``, any
    token and head strides) times its weight (``[dim]``; None: no norm), then the
    rotate-half rotation of the first ``cos_sin.shape[1]`` dims at each token's position
    (``cos_sin`` fp32 or bf16, ``rotary_table`` or ``rotary_cache``; None: none). All in
    fp32, rounded once. Positions outside the table give zeros in those dims, as in
    ``indexer_norm_rope``.

    With a ``cache`` - the bf16 pair (k_cache, v_cache) ``[blocks, page, kv_heads, dim]``
    or an :class:`Int4KVCache` - keys (so treated) and values go to ``slot_mapping``'s
    slots in the same launch (negative slots and those past the cache: nothing). Slots
    must differ. ``k_out`` and ``v_out`` receive the rows as the cache holds them: of a
    4-bit cache the values that its codes stand for. Groups of 32 dims with infinities,
    NaN or values from 2^126 on read as NaN from a 4-bit cache.

    Returns (q_out, k_out): made if not given, ``k_out`` only without a cache. An output
    may be its own input. ``query`` may be None."""
    if query is not None and q_out is None:
        q_out = torch.empty_like(query, memory_format=torch.contiguous_format)
    if cache is None and k_out is None:
        k_out = torch.empty_like(key, memory_format=torch.contiguous_format)
    page = 0
    if cache is None:
        _require(slot_mapping is None, "slot_mapping needs a cache")
        k_cache = v_cache = None
    elif isinstance(cache, Int4KVCache):
        _require(key.dim() == 3 and key.shape[2] == cache.head_dim,
                 "the cache's head dim must match key")
        k_cache, v_cache, page = cache.data, None, cache.page_size
    else:
        k_cache, v_cache = cache
    _qk_norm_rope(
        query, key, value, q_weight, k_weight, float(eps), positions, cos_sin, q_out, k_out, v_out,
        slot_mapping, k_cache, v_cache, int(page))
    return q_out, k_out
