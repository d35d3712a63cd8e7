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
