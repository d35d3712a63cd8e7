"""Rules on logits before sampling (``csrc/logits.hip``): penalties for repeated
tokens, biases and grammar masks, on decode rows or drafted nodes."""

from __future__ import annotations

from dataclasses import dataclass

import torch

from . import _torch_ops  # noqa: F401  (registers torch.ops.yulan_qsa_kernels)

__all__ = ["LogitsRules", "process_logits"]


@dataclass
class LogitsRules:
    """What a step's requests ask of their logits; the arguments of
    :func:`process_logits` of the same names. The tensors may be persistent
    buffers that a captured step reads anew on every replay."""

    history: torch.Tensor | None = None
    history_lens: torch.Tensor | None = None
    prompt_lens: torch.Tensor | None = None
    repetition: torch.Tensor | None = None
    frequency: torch.Tensor | None = None
    presence: torch.Tensor | None = None
    bias_ids: torch.Tensor | None = None
    bias_values: torch.Tensor | None = None
    allowed: torch.Tensor | None = None
    vocab_start: int = 0


def process_logits(
    logits: torch.Tensor,
    out: torch.Tensor | None = None,
    *,
    token_to_req: torch.Tensor | None = None,
    history: torch.Tensor | None = None,
    history_lens: torch.Tensor | None = None,
    prompt_lens: torch.Tensor | None = None,
    repetition: torch.Tensor | None = None,
    frequency: torch.Tensor | None = None,
    presence: torch.Tensor | None = None,
    bias_ids: torch.Tensor | None = None,
    bias_values: torch.Tensor | None = None,
    allowed: torch.Tensor | None = None,
    vocab_start: int = 0,
    draft_tokens: torch.Tensor | None = None,
    ancestors: torch.Tensor | None = None,
    query_start_loc: torch.Tensor | None = None,
) -> torch.Tensor:
    """fp32 logits ``[rows, vocab]`` with each request's rules applied, from
    fp32, bf16 or fp16 ``logits``; ``out`` may be the logits themselves when they
    are fp32. Column v is token ``vocab_start + v`` (a vocabulary shard).

    Row r belongs to request ``token_to_req[r]`` (int32; without it, to request
    r); rows of no request (negative or too large) get their grammar mask alone.
    All of the requests' tensors must have as many entries (rows).
    In this order (penalties before biases: an engine that adds biases first gives
    other logits to tokens that have both), each rule left out where its tensors
    are None:

    * ``history`` int32 ``[requests, width]`` holds a request's tokens, the first
      ``history_lens`` of them valid and the first ``prompt_lens`` of those (0
      without) its prompt. Tokens seen there: ``x / repetition`` if positive, else
      ``x * repetition``. Of those past the prompt (count c): ``- frequency * c``,
      then ``- presence``. All four per request, fp32.
    * With ``ancestors`` (``tree_ancestors``), ``draft_tokens`` int32 ``[rows]`` and
      ``query_start_loc``, rows are drafted nodes, and the tokens of the nodes a
      row sees (itself among them) count as said.
    * ``bias_values[b, i]`` fp32 is added to token ``bias_ids[b, i]`` (int32; ids
      outside the shard, such as -1, are passed over; an id listed twice gets both,
      in list order).
    * ``allowed`` int32 ``[rows, ceil(vocab / 32)]``: columns whose bit ``v % 32`` of
      word ``v // 32`` is 0 become -inf, whatever they held.

    At most 1024 biases and 1024 nodes (32 ancestor words) a request."""
    if out is None:
        out = torch.empty(logits.shape, dtype=torch.float32, device=logits.device)
    torch.ops.yulan_qsa_kernels.process_logits(
        logits, out, token_to_req, history, history_lens, prompt_lens, repetition,
        frequency, presence, bias_ids, bias_values, allowed, int(vocab_start), draft_tokens,
        ancestors, query_start_loc)
    return out
