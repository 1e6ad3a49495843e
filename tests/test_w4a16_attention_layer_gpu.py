"""W4A16Attention: what it refuses before anything is launched or stored, and other types and heads than the chain's test has."""
import pytest
import torch

import oracle
from intent_b200.attention import AttentionWeights, PagedKVCache, W4A16Attention, rotary_table
from oracle import attention

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


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("dim,pairs", [(128, "halves"), (64, "neighbours")])
def test_prompts_and_tokens(cuda_device, dtype, dim, pairs):
    """Two sequences, a prompt and tokens after it, in types and heads that the chain's own test leaves out."""
    torch_dtype = torch.float16 if dtype == "f16" else torch.bfloat16
    heads, total = 6, {"a": 150, "b": 35}
    w = make_weights(cuda_device, torch_dtype, heads=heads, dim=dim, seed=dim)
    rotary = rotary_table(160, dim)
    g = torch.Generator().manual_seed(dim)
    inputs = {name: torch.randn((n, HIDDEN), generator=g).to(torch_dtype) for name, n in total.items()}
    cache = PagedKVCache(layers=1, pages=16, kv_heads=KV_HEADS, head_dim=dim, page_size=32, act_dtype=dtype, device=cuda_device)
    layer = W4A16Attention(hidden=HIDDEN, heads=heads, kv_heads=KV_HEADS, head_dim=dim, act_dtype=dtype, pairs=pairs)
    table, done, got = rotary.to(cuda_device), dict.fromkeys(total, 0), {name: [] for name in total}
    for new in ({"a": 130, "b": 33}, {"a": 1, "b": 1}, {"a": 18}, {"b": 1, "a": 1}):
        x = torch.cat([inputs[name][done[name]:done[name] + n] for name, n in new.items()]).to(cuda_device)
        rows = layer.forward(x, w, table, *cache.layer(0), cache.step(new)).split(list(new.values()))
        for (name, n), part in zip(new.items(), rows):
            got[name].append(part)
            done[name] += n
    layer.check()
    assert done == total

    def dense(packed, scales):
        return oracle.dequantize_int4(packed.cpu(), scales.cpu().double(), group_size=128, zero_point=8).double()

    for name, n in total.items():                  # the whole sequence in 64 bits, nothing rounded between the steps
        q, k, v = (inputs[name].double() @ dense(w.qkv_packed, w.qkv_scales)).view(n, -1, dim).split([heads, KV_HEADS, KV_HEADS], 1)
        q, k = (attention.rotate(t, torch.arange(n), rotary, s.cpu(), pairs=pairs) for t, s in ((q, w.q_norm), (k, w.k_norm)))
        out, _ = attention.paged_attention(q, k.transpose(0, 1)[None], v.transpose(0, 1)[None],
                                           torch.zeros((1, 1), dtype=torch.int32), torch.tensor([0, n]), torch.tensor([n]))
        expected = out.reshape(n, heads * dim) @ dense(w.out_packed, w.out_scales)
        actual = torch.cat(got[name]).cpu().double()
        # the projections' own tolerance, for the whole chain
        assert (actual - expected).abs().max() <= 2e-2 * expected.abs().max()
