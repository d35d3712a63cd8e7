"""Cases of attention over the paged cache and their 64-bit results, for the tests of
``qsa_window_paged_attention``, ``qsa_int4_paged_attention`` and ``qk_norm_rope``.

Tolerance of the attention. Each weight is rounded to bf16, p (1 + e) with |e| <= 2^-8,
before it meets V, and the rounded weights are what is summed (a 4-bit cache's scale
may be rounded into the weight that meets V: as much again, and the sum then of the
others): the weighted mean o moves by at most 2^-8 (1 + 2^-7) (sum p |v| + |o|), twice
that from 4 bits. A score's fp32 sum of D products passes at most D + 8 roundings of
2^-24 on sum |q k| (from codes on sum |q| (|k| + 32 s): the kernel takes the zero points
off at the end), scaled by D^-0.5, which moves a weight by as much (numerator and sum:
twice); the fp32 exponentials and sums stay under 2^-16 of a weight. The gate's factor
is at most 1 and off by 2^-17. Then one rounding to bf16, 2^-8 of the value."""

import math

import numpy as np
import torch

from qsa_vllm_amd.ops import (Int4KVCache, qsa_int4_paged_attention, qsa_window_paged_attention)

DEV = "cuda:0"


def quantize4(x):
    """(codes, zero points, scales) of fp32 rows [..., dim] that hold bf16 values, step by
    step in numpy's fp32."""
    y = np.ascontiguousarray(x, dtype=np.float32).reshape(*x.shape[:-1], -1, 32)
    low = np.minimum(y.min(-1), np.float32(0))
    high = np.maximum(y.max(-1), np.float32(0))
    step = np.maximum((high - low) / np.float32(15), np.float32(2.0 ** -100))
    scale = ((step.view(np.uint32) + np.uint32(0xFFFFF)) & np.uint32(0xFFF00000)).view(np.float32)
    zero = np.minimum(np.rint(-low / scale), np.float32(15))
    codes = np.clip(np.rint(y / scale[..., None]) + zero[..., None], 0, 15)
    return codes.reshape(x.shape), zero, scale


def values4(codes, zero, scale):
    c = codes.reshape(*codes.shape[:-1], -1, 32)
    return ((c - zero[..., None]) * scale[..., None]).reshape(codes.shape)


def pack4(codes_k, words_k, codes_v, words_v):
    """A 4-bit cache's data from codes [blocks, page, heads, dim] and 16-bit words
    [blocks, page, heads, dim / 32], place by place."""
    blocks, page, heads, dim = codes_k.shape
    fill = -(-(page * dim // 16) // 16) * 16
    data = np.zeros((blocks, heads, page * dim + 2 * fill), dtype=np.uint8)
    for which, (codes, words) in enumerate(((codes_k, words_k), (codes_v, words_v))):
        packed = np.zeros((blocks, heads, page, dim // 8), dtype=np.uint32)
        for d in range(dim):
            if which == 0:
                word, shift = (d % 32 // 8) * (dim // 32) + d // 32, 4 * (d % 8 // 2) + 16 * (d % 2)
            else:
                word, shift = d // 8, 4 * (d % 8)
            packed[..., word] |= codes[..., d].transpose(0, 2, 1).astype(np.uint32) << np.uint32(shift)
        size = page * dim // 2
        data[:, :, which * size:(which + 1) * size] = packed.view(np.uint8).reshape(blocks, heads, -1)
        w = np.ascontiguousarray(words.transpose(0, 2, 1, 3).astype(np.uint16))
        first = 2 * size + which * fill
        data[:, :, first:first + page * dim // 16] = w.view(np.uint8).reshape(blocks, heads, -1)
    return torch.from_numpy(data)


class Case:
    """Requests of ``ctx`` cached and ``new`` own tokens over a shuffled paged cache whose
    unused slots (and pages) hold NaN."""

    def __init__(self, ctx, new, heads=4, kv_heads=2, dim=128, page=16, window=None, sinks=0,
                 gate=False, seed=0, bits=16, layout="token_major", scale=1.0):
        gen = torch.Generator().manual_seed(seed)
        self.gen, self.ctx, self.new, self.page, self.dim = gen, ctx, new, page, dim
        self.heads, self.kv_heads, self.window, self.sinks = heads, kv_heads, window, sinks
        self.bits, self.layout = bits, layout
        self.lens = [c + n for c, n in zip(ctx, new)]
        self.starts = [0]
        for n in new:
            self.starts.append(self.starts[-1] + n)
        pages = [-(-n // page) for n in self.lens]
        order = torch.randperm(sum(pages) + 2, generator=gen).to(torch.int32)
        self.table = torch.full((len(ctx), max(max(pages), 1)), -1, dtype=torch.int32)
        blocks = len(order)
        used = torch.zeros(blocks, page, dtype=torch.bool)
        at = 0
        for b, p in enumerate(pages):
            self.table[b, :p] = order[at:at + p]
            at += p
            pos = torch.arange(self.lens[b])
            used[self.table[b][pos // page].long(), pos % page] = True
        kv = (torch.randn(blocks, page, kv_heads, 2 * dim, generator=gen) * scale).bfloat16()
        if bits == 4:
            self.parts = [list(quantize4(kv[..., i * dim:(i + 1) * dim].float().numpy()))
                          for i in (0, 1)]
            self.words = [(s.view(np.uint32) >> 16).astype(np.uint16) | z.astype(np.uint16)
                          for _, z, s in self.parts]
            for w in self.words:
                w[~used.numpy()] = 0x7FC0
            held = [torch.from_numpy(values4(*p)) for p in self.parts]
            kv = torch.cat(held, -1)
        kv = kv.clone()
        kv[~used] = float("nan")
        self.kv = kv
        rows = self.starts[-1]
        self.q = (torch.randn(rows, heads, dim, generator=gen) * scale).bfloat16()
        self.gate = torch.randn(rows, heads, dim, generator=gen).bfloat16() if gate else None
        self.qsl = torch.tensor(self.starts, dtype=torch.int32)

    def device_cache(self):
        if self.bits == 4:
            (ck, _, _), (cv, _, _) = self.parts
            data = pack4(ck, self.words[0], cv, self.words[1]).to(DEV)
            if self.layout == "strided":     # pages inside larger blocks
                wide = torch.zeros(data.shape[0], data.shape[1], data.shape[2] + 48, dtype=torch.uint8,
                                   device=DEV)
                wide[:, :, :data.shape[2]] = data
                data = wide[:, :, :data.shape[2]]
            return Int4KVCache(data, self.page, self.dim)
        if self.layout == "head_major":   # [blocks, kv_heads, page, 2 D] storage
            kv = self.kv.permute(0, 2, 1, 3).contiguous().to(DEV).permute(0, 2, 1, 3)
        else:
            kv = self.kv.to(DEV)
        if self.layout == "separate":
            return kv[..., :self.dim].contiguous(), kv[..., self.dim:].contiguous()
        return kv[..., :self.dim], kv[..., self.dim:]

    def run(self, out=None, q=None, table=None, lens=None, qsl=None, max_query_len=None,
            max_seq_len=None, cache=None):
        cache = self.device_cache() if cache is None else cache
        call = qsa_int4_paged_attention if self.bits == 4 else qsa_window_paged_attention
        args = (cache,) if self.bits == 4 else cache
        return call(
            self.q.to(DEV) if q is None else q, *args,
            (self.table if table is None else table).to(DEV),
            torch.tensor(self.lens, dtype=torch.int32, device=DEV) if lens is None else lens,
            self.qsl.to(DEV) if qsl is None else qsl, out, window=self.window,
            sink_tokens=self.sinks,
            output_gate=self.gate.to(DEV) if self.gate is not None else None,
            max_query_len=max(self.new) if max_query_len is None else max_query_len,
            max_seq_len=max(self.lens) if max_seq_len is None else max_seq_len)

    def seen(self, b, i, table=None):
        """Positions that row i of request b sees."""
        table = self.table if table is None else table
        p = self.lens[b] - self.new[b] + i
        j = torch.arange(max(0, min(p + 1, table.shape[1] * self.page)))
        if self.window is not None:
            j = j[(j > p - self.window) | (j < self.sinks)]
        block = table[b][j // self.page]
        return j[(block >= 0) & (block < self.kv.shape[0])]

    def want(self, table=None):
        """(result, tolerance) in 64 bits, each row over its own list of positions."""
        table = self.table if table is None else table
        out = torch.zeros(self.q.shape, dtype=torch.float64)
        tol = torch.zeros_like(out)
        group = self.heads // self.kv_heads
        weight = 2 ** -8 * (1 + 2 ** -7) * (2 if self.bits == 4 else 1)
        for b in range(len(self.ctx)):
            for i in range(self.new[b]):
                r, j = self.starts[b] + i, self.seen(b, i, table)
                if not len(j):
                    continue
                kv = self.kv[table[b][j // self.page].long(), j % self.page].double()
                k = kv[..., :self.dim].permute(1, 2, 0)      # [kv, dim, n]
                v = kv[..., self.dim:].permute(1, 0, 2)      # [kv, n, dim]
                q = self.q[r].double().view(self.kv_heads, group, self.dim)
                score = q @ k / math.sqrt(self.dim)
                p = torch.softmax(score, -1)
                extra = 0.0
                if self.bits == 4:
                    s = torch.from_numpy(self.parts[0][2]).double()
                    s = s[table[b][j // self.page].long(), j % self.page].repeat_interleave(32, -1)
                    extra = 32 * s.permute(1, 2, 0)
                spread = (q.abs() @ (k.abs() + extra)).amax(-1, keepdim=True) / math.sqrt(self.dim)
                o, size = p @ v, p @ v.abs()
                off = weight * (size + o.abs())
                off = off + (2 * (self.dim + 8) * 2 ** -24 * spread + 2 ** -16) * size
                if self.gate is not None:
                    g = torch.sigmoid(self.gate[r].double()).view(self.kv_heads, group, self.dim)
                    off = off * g + 2 ** -17 * (o * g).abs()
                    o = o * g
                out[r] = o.reshape(self.heads, self.dim)
                tol[r] = (off + 2 ** -8 * (o.abs() + off) + 2 ** -100).reshape(self.heads, self.dim)
        return out, tol

    def check(self, got, **kw):
        want, tol = self.want(**kw)
        assert torch.isfinite(got).all()
        off = (got.cpu().double() - want).abs()
        worst = (off / tol.clamp(min=2 ** -100)).max().item()
        assert (off <= tol).all(), f"{worst:.2f} times the tolerance"
