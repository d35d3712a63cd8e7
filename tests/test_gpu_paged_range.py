"""How large K, V and queries may be: attention up to the ends of the stated range
(tolerance: ``paged_cases``, all of it relative)."""

import numpy as np
import pytest
import torch

from .paged_cases import Case, quantize4, values4

pytestmark = pytest.mark.gpu


def _hold(c, kv):
    """Makes ``kv`` [blocks, page, heads, 2 dim] what the case's cache holds (unused slots
    keep their NaN)."""
    live = ~torch.isnan(c.kv).all(-1, keepdim=True)
    kv = kv.bfloat16()
    if c.bits == 4:
        for i in (0, 1):
            part = list(quantize4(kv[..., i * c.dim:(i + 1) * c.dim].float().numpy()))
            word = (part[2].view(np.uint32) >> 16).astype(np.uint16) | part[1].astype(np.uint16)
            c.words[i] = np.where(live.numpy(), word, np.uint16(0x7FC0))
            c.parts[i] = part
        kv = torch.cat([torch.from_numpy(values4(*p)) for p in c.parts], -1)
    c.kv = torch.where(live, kv, torch.tensor(float("nan"), dtype=kv.dtype))


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("new", [[1], [3], [40], [1, 40]])
@pytest.mark.parametrize("dim", [128, 64])
def test_values_times_tokens_up_to_2_to_the_117(bits, new, dim):
    """V of both signs at the end of the range under the largest weights that the kernels
    hold: every later token's score lies just under 2^8 above the first ones', whose maximum
    the exponents are then still taken from."""
    tokens = 900
    c = Case([tokens - n for n in new], new, heads=4, kv_heads=1, dim=dim, bits=bits)
    kv = torch.zeros_like(c.kv, dtype=torch.float32)
    size = 1.99 * 2.0 ** 116 / tokens
    sign = 1 - 2 * (torch.arange(dim) % 2)
    for b in range(len(new)):
        for j in range(tokens):
            row = kv[int(c.table[b, j // 16]), j % 16, 0]
            row[:dim] = float(j >= 512)
            row[dim:] = size * sign * (1 if j % 3 else 0.75)
    _hold(c, kv)
    held = c.kv[int(c.table[0, 40]), 0, 0, :dim].double()
    assert (held == held[0]).all()
    c.q[:] = 7.75 / (dim ** 0.5 * 1.4427 * held[0].item())
    assert c.kv.nan_to_num(0.0)[..., dim:].double().abs().max() * tokens <= 2.0 ** 117
    c.check(c.run())


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("new", [[1], [40], [1, 40]])
@pytest.mark.parametrize("power", [100, -60])
def test_large_and_small_keys(bits, new, power):
    """Keys scaled by a power of two and queries by its inverse: the scores are the same."""
    c = Case([700] * len(new), new, heads=8, kv_heads=2, bits=bits, window=500, sinks=3, seed=power)
    kv = c.kv.nan_to_num(0.0).float()
    kv[..., :128] *= 2.0 ** power
    _hold(c, kv)
    c.q = (c.q.float() * 2.0 ** -power).bfloat16()
    c.check(c.run())
