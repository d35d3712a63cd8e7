"""Layers of windowed attention in the hybrid decoder, as they are built (no GPU)."""

import torch

from qsa_vllm_amd.hybrid import HybridConfig, HybridDecoder


def test_layers_share_one_table_of_angles():
    cfg = HybridConfig(num_layers=4, hidden_size=128, vocab_size=64, num_heads=4, num_kv_heads=2,
                       head_dim=128, intermediate_size=64, linear_num_key_heads=2,
                       linear_num_value_heads=4, indexer_heads=2, rope_dim=64,
                       window_layers=(0, 2, 3))
    model = HybridDecoder(cfg, num_blocks=2, comp_blocks=2, ring_blocks=2, state_slots=2,
                          max_tokens=8, max_position=96, device="cpu")
    tables = [layer.mixer.cos_sin for layer in model.layers if layer.kind == "sliding_attention"]
    assert len(tables) == 3 and tables[0].shape == (96, 64) and tables[0].dtype == torch.float32
    assert all(t.data_ptr() == tables[0].data_ptr() for t in tables)
