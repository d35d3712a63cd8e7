"""What a 4-bit cache's words stand for, on the CPU."""

import numpy as np
import pytest
import torch

from qsa_vllm_amd.ops import Int4KVCache

from .paged_cases import pack4


@pytest.mark.parametrize("which", [0, 1])
def test_dequantize_of_scales_of_any_kind(which):
    """Negative scales count as they are; a scale that is not finite, of either sign and
    with any zero point, reads as NaN as a whole group, as in the attention."""
    gen = np.random.default_rng(which)
    codes = gen.integers(0, 16, (2, 1, 16, 1, 64)).astype(np.float32)
    words = np.full((1, 16, 1, 2), 0x3F80, dtype=np.uint16)
    special = [0x7F80, 0x7F81, 0x7F8F, 0xFF80, 0xFF83, 0x7FC0, 0xFFC7, 0x7FF0]
    words[0, :8, 0, 1] = special
    words[0, 8:, 0, 0] = [0xBF80 | z for z in range(8)]
    plain = np.full_like(words, 0x3F80)
    parts = [(codes[i], words if i == which else plain) for i in (0, 1)]
    held = Int4KVCache(pack4(*parts[0], *parts[1]), 16, 64).dequantize()
    got = held[which][0, :, 0].float()
    assert torch.isnan(got[:8, 32:]).all()
    want = torch.from_numpy(codes[which][0, :, 0])
    want[8:, :32] = -(want[8:, :32] - torch.arange(8)[:, None])
    assert torch.equal(got[8:], want[8:]) and torch.equal(got[:8, :32], want[:8, :32])
    assert torch.equal(held[1 - which][0, :, 0].float(), torch.from_numpy(codes[1 - which][0, :, 0]))
