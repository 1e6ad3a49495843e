"""The chain of a layer's attention half: int4 projections, append and attention over the pages."""
import pytest
import torch

import intent_b200 as ib
import oracle
from intent_b200.attention import AttentionWeights, PagedKVCache, W4A16Attention, rotary_table
from oracle import attention

pytestmark = pytest.mark.gpu

HIDDEN, HEADS, KV_HEADS, DIM, DTYPE = 512, 8, 2, 64, torch.bfloat16


def make_weights(seed):
    g = torch.Generator().manual_seed(seed)

    def packed(K, N):
        _, p, _ = ib.workloads.w4a16_inputs(1, K, N, dtype=DTYPE, seed=seed + N)
        return p, (0.01 + 0.01 * torch.rand((K // 128, N), generator=g)).to(DTYPE)

    return AttentionWeights(*packed(HIDDEN, (HEADS + 2 * KV_HEADS) * DIM), *packed(HEADS * DIM, HIDDEN),
                            *((1 + 0.1 * torch.randn(DIM, generator=g)).to(DTYPE) for _ in range(2)))


def dense(packed, scales):
    return oracle.dequantize_int4(packed, scales.double(), group_size=128, zero_point=8).double()


def reference(x, w, rotary, norm, window):
    """One whole sequence [n, hidden] in 64 bits, nothing rounded between the steps."""
    n = x.shape[0]
    qkv = (x.double() @ dense(w.qkv_packed, w.qkv_scales)).view(n, HEADS + 2 * KV_HEADS, DIM)
    q, k, v = qkv.split([HEADS, KV_HEADS, KV_HEADS], 1)
    place = torch.arange(n)
    q, k = (attention.rotate(t, place, rotary, s if norm else None) for t, s in ((q, w.q_norm), (k, w.k_norm)))
    out, _ = attention.paged_attention(q, k.transpose(0, 1)[None], v.transpose(0, 1)[None], torch.zeros((1, 1), dtype=torch.int32),
                                       torch.tensor([0, n]), torch.tensor([n]), window=window)
    return out.reshape(n, HEADS * DIM) @ dense(w.out_packed, w.out_scales)


@pytest.mark.parametrize("norm,window", [(True, 0), (False, 24)])
def test_prompts_chunks_and_tokens(cuda_device, norm, window):
    """Three sequences that begin at different steps, in chunks and token by token, two layers over one cache; their rows are
    those of the whole sequence worked out at once."""
    g = torch.Generator().manual_seed(5)
    total = {"a": 75, "b": 40, "c": 21}
    inputs = {name: torch.randn((n, HIDDEN), generator=g).to(DTYPE) for name, n in total.items()}
    weights = [make_weights(s) for s in (1, 2)]
    if not norm:
        for w in weights:                                  # scores of a few units without the norm
            w.qkv_scales.mul_(0.05)
    rotary = rotary_table(128, DIM)
    expected = [{name: reference(x, w, rotary, norm, window) for name, x in inputs.items()} for w in weights]

    cache = PagedKVCache(layers=2, pages=16, kv_heads=KV_HEADS, head_dim=DIM, page_size=16, device=cuda_device)
    layer = W4A16Attention(hidden=HIDDEN, heads=HEADS, kv_heads=KV_HEADS, head_dim=DIM, norm=norm, window=window)
    on_device = [AttentionWeights(*(getattr(w, f).to(cuda_device) for f in w.__dataclass_fields__)) for w in weights]
    table, done = rotary.to(cuda_device), dict.fromkeys(total, 0)
    got = [{name: [] for name in total} for _ in weights]
    steps = [{"a": 30}, {"a": 20, "b": 33}, {"b": 1, "a": 1}, {"c": 18, "a": 1, "b": 1}, {"a": 20, "c": 1, "b": 3}]
    steps += [{"a": 1, "b": 1, "c": 1}] * 2 + [{"a": 1}]
    for new in steps:
        step = cache.step(new)
        x = torch.cat([inputs[name][done[name]:done[name] + n] for name, n in new.items()]).to(cuda_device)
        for index, w in enumerate(on_device):
            rows = layer.forward(x, w, table, *cache.layer(index), step).split(list(new.values()))
            for name, part in zip(new, rows):
                got[index][name].append(part)
        for name, n in new.items():
            done[name] += n
    assert done == total
    layer.check()
    for index in range(2):
        for name in total:
            actual = torch.cat(got[index][name]).cpu().double()
            # the projections' own tolerance, for the whole chain
            assert (actual - expected[index][name]).abs().max() <= 2e-2 * expected[index][name].abs().max()
    cache.release("a")
    assert cache.free_pages == 16 - 3 - 2


def test_refusals(cuda_device):
    cache = PagedKVCache(layers=1, pages=4, kv_heads=KV_HEADS, head_dim=DIM, page_size=16, device=cuda_device)
    layer = W4A16Attention(hidden=HIDDEN, heads=HEADS, kv_heads=KV_HEADS, head_dim=DIM)
    w = make_weights(1)
    w = AttentionWeights(*(getattr(w, f).to(cuda_device) for f in w.__dataclass_fields__))
    x, table = torch.zeros((3, HIDDEN), dtype=DTYPE, device=cuda_device), rotary_table(64, DIM, device=cuda_device)
    step = cache.step({"a": 2})
    with pytest.raises(ValueError):
        layer.forward(x, w, table, *cache.layer(0), step)
    with pytest.raises(TypeError):
        layer.forward(x[:2].half(), w, table, *cache.layer(0), step)
    wrong = AttentionWeights(w.out_packed, w.out_scales, w.out_packed, w.out_scales, w.q_norm, w.k_norm)
    with pytest.raises(ValueError):
        layer.forward(x[:2], wrong, table, *cache.layer(0), step)
