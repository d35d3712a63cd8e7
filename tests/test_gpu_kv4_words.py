"""Words of a 4-bit cache that its own writer does not make: scales of either sign and
scales that are not finite, in data of the documented layout from elsewhere
(tolerance: ``paged_cases``)."""

import numpy as np
import pytest
import torch

from .paged_cases import Case

pytestmark = pytest.mark.gpu


def _negate(c, which, groups):
    """Gives ``groups`` (a mask [blocks, page, heads, dim / 32]) of K (0) or V (1) the
    negative of their scale: their values change sign, exactly."""
    c.words[which][groups] |= 0x8000
    kv = c.kv.unflatten(-1, (2, -1, 32))[..., which, :, :]
    kv[torch.from_numpy(groups)] *= -1


@pytest.mark.parametrize("dim", [128, 64])
@pytest.mark.parametrize("ctx,new,heads,kv_heads,window,sinks", [
    ([37], [1], 8, 1, None, 0),                    # one block, seen in part
    ([100, 700, 63], [1, 2, 1], 8, 2, 90, 4),      # blocks at windows' ends, sinks
    ([3000], [1], 16, 2, None, 0),                 # whole blocks in pieces, a last one in part
    ([130, 20], [60, 33], 4, 2, 70, 3),            # tiles
    ([500, 90, 300], [1, 100, 1], 8, 2, 200, 1),   # tiles beside single tokens
])
def test_negative_scales(ctx, new, heads, kv_heads, window, sinks, dim):
    c = Case(ctx, new, heads, kv_heads, dim, window=window, sinks=sinks, bits=4, seed=sum(ctx) + dim)
    pick = np.random.default_rng(dim)
    for which in (0, 1):
        live = c.words[which] != 0x7FC0
        _negate(c, which, live & (pick.random(live.shape) < 0.5))
    c.check(c.run())
    # Every group of V: nothing else is left of them.
    _negate(c, 1, (c.words[1] & 0x8000 == 0) & (c.words[1] != 0x7FC0))
    c.check(c.run())


@pytest.mark.parametrize("word", [0x7F80, 0x7F87, 0xFF80, 0xFF8F, 0x7FC0, 0xFFF5])
@pytest.mark.parametrize("ctx,new,window", [([300], [1], None), ([300, 40], [2, 50], 100)])
def test_scales_that_are_not_finite_read_as_nan(ctx, new, window, word):
    """Infinities of either sign as NaN, whatever the zero point: the group's dims of the
    rows that see V's, all dims of those that see K's, and nothing else."""
    c = Case(ctx, new, heads=4, kv_heads=2, window=window, bits=4, seed=word)
    clean = c.run()
    for which, pos in ((w, p) for w in (1, 0) for p in (130, 210, 290, c.lens[0] - 1)):
        block, place = int(c.table[0, pos // 16]), pos % 16
        saved = c.words[which].copy()
        c.words[which][block, place, 1, 2] = word
        held = c.device_cache()
        got = c.run(cache=held)
        c.words[which] = saved
        for r in range(c.starts[-1]):
            want = torch.zeros(4, 128, dtype=torch.bool)
            if r < c.starts[1] and pos in c.seen(0, r).tolist():
                want[2:, 64:96] = True
                if which == 0:
                    want[2:] = True
            want = want.to(got.device)
            assert torch.isnan(got[r][want]).all(), (which, pos, r)
            assert torch.equal(got[r][~want], clean[r][~want]), (which, pos, r)
        value = held.dequantize()[which][block, place, 1]
        assert torch.isnan(value[64:96]).all() and torch.isfinite(value[:64]).all()
