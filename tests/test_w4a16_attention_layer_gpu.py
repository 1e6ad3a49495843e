"""W4A16Attention: what it refuses before anything is launched or stored, and other types and heads than the chain's test has."""
import pytest
import torch

import intent_b200 as ib
from intent_b200.attention import AttentionWeights, PagedKVCache, W4A16Attention, rotary_table

pytestmark = pytest.mark.gpu

HIDDEN, HEADS, KV_HEADS, DIM = 256, 4, 2, 64


def make_weights(device, dtype=torch.bfloat16, hidden=HIDDEN, heads=HEADS, kv_heads=KV_HEADS, dim=DIM, seed=0):
    g = torch.Generator().manual_seed(seed)

    def packed(K, N):
        p = torch.randint(-2 ** 31, 2 ** 31, (K // 8, N), generator=g, dtype=torch.int64).to(torch.int32)
        return p.to(device), (0.01 + 0.01 * torch.rand((K // 128, N), generator=g)).to(dtype).to(device)

    return AttentionWeights(*packed(hidden, (heads + 2 * kv_heads) * dim), *packed(heads * dim, hidden),
                            *((1 + 0.1 * torch.randn(dim, generator=g)).to(dtype).to(device) for _ in range(2)))


def test_positions_beyond_the_rotary_table(cuda_device):
    """Their keys would be stored as NaN, for the rest of the sequence."""
    cache = PagedKVCache(layers=1, pages=8, kv_heads=KV_HEADS, head_dim=DIM, page_size=16, device=cuda_device)
    cache.k.zero_(), cache.v.zero_()
    layer, w = W4A16Attention(hidden=HIDDEN, heads=HEADS, kv_heads=KV_HEADS, head_dim=DIM), make_weights(cuda_device)
    table = rotary_table(32, DIM, device=cuda_device)
    x = torch.randn((40, HIDDEN), device=cuda_device).bfloat16()
    step = cache.step({"a": 32})
    assert layer.forward(x[:32], w, table, *cache.layer(0), step).isfinite().all()
    before = cache.k.clone()
    step = cache.step({"a": 1, "b": 2})
    with pytest.raises(ValueError, match="rotary"):
        layer.forward(x[:3], w, table, *cache.layer(0), step)
    assert torch.equal(cache.k, before)


def test_sizes_other_than_the_layers(cuda_device):
    """Refused before the keys are stored, not by the last projection."""
    cache = PagedKVCache(layers=1, pages=8, kv_heads=KV_HEADS, head_dim=DIM, page_size=16, device=cuda_device)
    cache.k.zero_(), cache.v.zero_()
    layer, w = W4A16Attention(hidden=HIDDEN, heads=HEADS, kv_heads=KV_HEADS, head_dim=DIM), make_weights(cuda_device)
    table = rotary_table(32, DIM, device=cuda_device)
    wide = make_weights(cuda_device, hidden=384)
    more = make_weights(cuda_device, heads=8)
    mixed = AttentionWeights(w.qkv_packed, w.qkv_scales, more.out_packed, more.out_scales, w.q_norm, w.k_norm)
    broad = AttentionWeights(w.qkv_packed, w.qkv_scales, wide.out_packed, wide.out_scales, w.q_norm, w.k_norm)
    step = cache.step({"a": 3})
    for hidden, weights in ((384, wide), (HIDDEN, mixed), (HIDDEN, broad)):
        with pytest.raises(ValueError):
            layer.forward(torch.randn((3, hidden), device=cuda_device).bfloat16(), weights, table, *cache.layer(0), step)
    assert not cache.k.any() and not cache.v.any()
