"""W4A16Attention on a cache in 4 bits: prompts and tokens as they would be served, what is stored read back, and refusals."""
import pytest
import torch

import oracle
from intent_b200.attention import PagedKVCache, W4A16Attention, rotary_table
from oracle import attention
from test_w4a16_attention_layer_gpu import DIM, HEADS, HIDDEN, KV_HEADS, make_weights

pytestmark = pytest.mark.gpu


def dense(packed, scales):
    return oracle.dequantize_int4(packed.cpu(), scales.cpu().double(), group_size=128, zero_point=8).double()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("dim,group,pairs", [(128, 64, "halves"), (64, 32, "neighbours"), (128, 128, "halves")])
def test_prompts_and_tokens(cuda_device, dtype, dim, group, pairs):
    """Two sequences, a prompt and tokens after it.  What the cache holds is within half a step of the keys and values in 64 bits, and
    the attention is that of the definition over what it holds."""
    torch_dtype = torch.float16 if dtype == "f16" else torch.bfloat16
    heads, total = 6, {"a": 150, "b": 35}
    w = make_weights(cuda_device, torch_dtype, heads=heads, dim=dim, seed=dim)
    rotary = rotary_table(160, dim)
    g = torch.Generator().manual_seed(dim)
    inputs = {name: torch.randn((n, HIDDEN), generator=g).to(torch_dtype) for name, n in total.items()}
    cache = PagedKVCache(layers=2, pages=16, kv_heads=KV_HEADS, head_dim=dim, page_size=32, act_dtype=dtype, device=cuda_device,
                         bits=4, group_size=group)
    layer = W4A16Attention(hidden=HIDDEN, heads=heads, kv_heads=KV_HEADS, head_dim=dim, act_dtype=dtype, pairs=pairs,
                           cache_bits=4, cache_group=group)
    table, done, got = rotary.to(cuda_device), dict.fromkeys(total, 0), {name: [] for name in total}
    for new in ({"a": 130, "b": 33}, {"a": 1, "b": 1}, {"a": 18}, {"b": 1, "a": 1}):
        x = torch.cat([inputs[name][done[name]:done[name] + n] for name, n in new.items()]).to(cuda_device)
        rows = layer.forward(x, w, table, *cache.layer(1), cache.step(new)).split(list(new.values()))
        for (name, n), part in zip(new.items(), rows):
            got[name].append(part)
            done[name] += n
    layer.check()
    assert done == total
    half = torch.finfo(torch_dtype).eps / 2
    for name, n in total.items():
        q, k, v = (inputs[name].double() @ dense(w.qkv_packed, w.qkv_scales)).view(n, -1, dim).split([heads, KV_HEADS, KV_HEADS], 1)
        q, k = (attention.rotate(t, torch.arange(n), rotary, s.cpu(), pairs=pairs) for t, s in ((q, w.q_norm), (k, w.k_norm)))
        held = [t.cpu() for t in cache.read(1, name)]
        part = [t.cpu() for t in cache.read(1, name, 7, n - 2)]
        assert all(torch.equal(a[7:n - 2], b) for a, b in zip(held, part))
        for x, y in ((k, held[0]), (v, held[1])):
            # half a step, the rounding of the projection's results (up to the largest of a row) and of the group's numbers, and
            # of what is read
            least, most = x.unflatten(-1, (-1, group)).aminmax(dim=-1, keepdim=True)
            step = (most - least) / 15
            size = x.abs().amax(-1, keepdim=True)[..., None]
            bound = (step / 2 * (1 + half) + 8 * half * size + 15 * step * half).expand(-1, -1, -1, group).flatten(-2)
            assert ((x - y.double()).abs() <= bound).all()
        out, _ = attention.paged_attention(q, held[0].double().transpose(0, 1)[None], held[1].double().transpose(0, 1)[None],
                                           torch.zeros((1, 1), dtype=torch.int32), torch.tensor([0, n]), torch.tensor([n]))
        expected = out.reshape(n, heads * dim) @ dense(w.out_packed, w.out_scales)
        actual = torch.cat(got[name]).cpu().double()
        # the projections' own tolerance, for the whole chain
        assert (actual - expected).abs().max() <= 2e-2 * expected.abs().max()


def test_what_is_refused(cuda_device):
    layer = W4A16Attention(hidden=HIDDEN, heads=HEADS, kv_heads=KV_HEADS, head_dim=DIM, cache_bits=4)
    plain = W4A16Attention(hidden=HIDDEN, heads=HEADS, kv_heads=KV_HEADS, head_dim=DIM)
    w, table = make_weights(cuda_device), rotary_table(32, DIM, device=cuda_device)
    sizes = {"layers": 1, "pages": 8, "kv_heads": KV_HEADS, "head_dim": DIM, "page_size": 16, "device": cuda_device}
    small, wide = PagedKVCache(bits=4, **sizes), PagedKVCache(**sizes)
    fine = PagedKVCache(bits=4, group_size=32, **sizes)
    x = torch.randn((3, HIDDEN), device=cuda_device).bfloat16()
    for c in (small.k, wide.k, fine.k):
        c.zero_()
    for some, cache, error in ((layer, wide, TypeError), (plain, small, TypeError), (layer, fine, ValueError)):
        with pytest.raises(error):
            some.forward(x, w, table, *cache.layer(0), cache.step({"a": 3}))
    assert not small.k.any() and not wide.k.any() and not fine.k.any()
    assert layer.forward(x, w, table, *small.layer(0), small.step({"b": 3})).isfinite().all()


@pytest.mark.parametrize("bits", [4, 16])
def test_reading_no_tokens(cuda_device, bits):
    cache = PagedKVCache(layers=1, pages=2, kv_heads=2, head_dim=64, page_size=16, device=cuda_device, bits=bits)
    cache.step({"a": 20})
    for start, stop in ((20, None), (3, 3), (0, 0)):
        assert [tuple(t.shape) for t in cache.read(0, "a", start, stop)] == [(0, 2, 64)] * 2
    with pytest.raises(ValueError):
        cache.read(0, "a", 21)


def test_a_step_in_a_graph(cuda_device):
    """A decode step of a layer, captured and replayed, is the step itself."""
    layer = W4A16Attention(hidden=HIDDEN, heads=HEADS, kv_heads=KV_HEADS, head_dim=DIM, cache_bits=4)
    w, table = make_weights(cuda_device), rotary_table(64, DIM, device=cuda_device)
    cache = PagedKVCache(layers=1, pages=8, kv_heads=KV_HEADS, head_dim=DIM, page_size=16, device=cuda_device, bits=4)
    x = torch.randn((42, HIDDEN), device=cuda_device).bfloat16()
    layer.forward(x[:40], w, table, *cache.layer(0), cache.step({"a": 30, "b": 10}))
    step = cache.step({"a": 1, "b": 1})
    expected = layer.forward(x[40:], w, table, *cache.layer(0), step)
    stored = cache.read(0, "a")
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        layer.forward(x[40:], w, table, *cache.layer(0), step)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out = layer.forward(x[40:], w, table, *cache.layer(0), step)
    for _ in range(2):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, expected)
    assert all(torch.equal(a, b) for a, b in zip(cache.read(0, "a"), stored))
