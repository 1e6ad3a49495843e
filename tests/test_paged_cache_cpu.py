"""Host side of the attention programs: bookkeeping of pages, the step's tensors, declarations and refusals."""
import math

import pytest
import torch

import intent_b200 as ib
from intent_b200.attention import PagedKVCache, W4A16Attention, rotary_table


def cache(pages=8, page_size=16):
    return PagedKVCache(layers=2, pages=pages, kv_heads=2, head_dim=64, page_size=page_size, device="cpu")


def check(store, step, new, before):
    """The step's tensors against the definition."""
    size, at = store.page_size, 0
    assert step.query_offsets.tolist() == [sum(list(new.values())[:i]) for i in range(len(new) + 1)]
    for row, (name, count) in enumerate(new.items()):
        length = before.get(name, 0) + count
        assert step.kv_lengths[row] == length == store.length(name)
        pages = step.page_table[row].tolist()
        used = -(-length // size)
        assert len(set(pages[:used])) == used and all(0 <= p < store.k.shape[1] for p in pages[:used])
        assert all(p == -1 for p in pages[used:])
        for i in range(count):
            place = length - count + i
            assert step.positions[at] == place
            assert step.slots[at] == pages[place // size] * size + place % size
            at += 1
    assert step.positions.shape == step.slots.shape == (at,)
    assert step.positions.dtype == step.page_table.dtype == step.kv_lengths.dtype == step.query_offsets.dtype == torch.int32
    assert step.slots.dtype == torch.int64 and step.page_table.is_contiguous()


def test_steps_and_release():
    store, lengths = cache(), {}
    for new in ({"a": 20, "b": 1}, {"b": 1, "a": 1}, {"a": 12, "c": 16}, {"b": 0, "c": 1}):
        step = store.step(new)
        check(store, step, new, lengths)
        assert step.single == all(n == 1 for n in new.values())
        for name, n in new.items():
            lengths[name] = lengths.get(name, 0) + n
    assert store.free_pages == 8 - 3 - 1 - 2
    held = set(store.step({"a": 1, "c": 1}).page_table.flatten().tolist()) - {-1}
    store.release("b")
    assert store.free_pages == 3 and store.length("b") == 0
    fresh = set(store.step({"d": 48}).page_table.flatten().tolist())
    assert not fresh & held and len(fresh) == 3          # no page belongs to two sequences
    with pytest.raises(KeyError):
        store.release("b")


def test_no_room_changes_nothing():
    store = cache(pages=3)
    store.step({"a": 30})
    with pytest.raises(MemoryError):
        store.step({"a": 1, "b": 33})
    assert store.free_pages == 1 and store.length("a") == 30 and store.length("b") == 0
    check(store, store.step({"a": 18}), {"a": 18}, {"a": 30})
    assert store.free_pages == 0


def test_layers_are_views():
    store = cache()
    k, v = store.layer(1)
    k[0, 0, 0, 0] = 3
    assert store.k[1, 0, 0, 0, 0] == 3 and k.is_contiguous() and v.shape == (8, 2, 16, 64)


def test_refusals():
    for wrong in ({"pages": 0}, {"head_dim": 96}, {"page_size": 8}, {"page_size": 48}, {"page_size": 512}, {"kv_heads": 0}):
        with pytest.raises(ValueError):
            PagedKVCache(**{**dict(layers=1, pages=4, kv_heads=2, head_dim=64, page_size=16, device="cpu"), **wrong})
    with pytest.raises(ValueError):
        cache().step({})
    with pytest.raises(ValueError):
        cache().step({"a": -1})
    with pytest.raises(ValueError):
        W4A16Attention(hidden=256, heads=6, kv_heads=4, head_dim=64)
    for wrong in ((0, 64), (4, 0), (4, 24)):
        with pytest.raises(ValueError):
            rotary_table(*wrong)


def test_rotary_table():
    table = rotary_table(5, 32, base=100.0)
    assert table.shape == (5, 32) and table.dtype == torch.float32
    for p in (0, 4):
        for i in (0, 7, 15):
            angle = p * 100.0 ** (-2 * i / 32)
            assert float(table[p, i]) == pytest.approx(math.cos(angle), abs=1e-7)
            assert float(table[p, 16 + i]) == pytest.approx(math.sin(angle), abs=1e-7)


@pytest.mark.parametrize("name", ["qk_norm_rope", "paged_kv_append", "paged_attention", "paged_decode_attention"])
def test_declarations(name):
    artifact = ib.compile(getattr(ib.programs, name), resolve_target=False)
    names = [p.name for p in artifact.interface.parameters]
    outputs = [p.name for p in artifact.interface.outputs]
    assert outputs == {"qk_norm_rope": ["q_out", "k_out"], "paged_kv_append": ["q_out"]}.get(name, ["output"])
    assert names[0] == "q" and all(p.layout in ("contiguous", "rows") for p in artifact.interface.parameters)
    assert [p.name for p in artifact.interface.mutable_inputs] == (["k_cache", "v_cache"] if name == "paged_kv_append" else [])


def test_shapes_are_inferred_without_a_device():
    """What fake tensors go through."""
    artifact = ib.compile(ib.programs.paged_attention, resolve_target=False, constexprs={"ACT_DTYPE": "f16"})
    device = torch.device("meta")
    q = torch.empty((5, 8, 64), dtype=torch.float16, device=device)
    cache_ = torch.empty((7, 2, 16, 64), dtype=torch.float16, device=device)
    ints = [torch.empty(s, dtype=torch.int32, device=device) for s in ((3, 4), (4,), (3,))]
    assert artifact.runtime.infer_outputs((q, cache_, cache_.clone(), *ints)).shape == (5, 8, 64)
