"""Arguments of the attention programs that have to be refused, and what a refusal leaves behind."""
import math

import pytest
import torch

import intent_b200 as ib
from intent_b200.attention import PagedKVCache


@pytest.mark.parametrize("program", ["paged_attention", "paged_decode_attention"])
@pytest.mark.parametrize("scale", [1e-46, 1e-300, 1e39, 0, -0.0, -1e-3, math.inf, math.nan, "a"])
def test_scales_that_are_no_positive_f32(program, scale):
    """One that is zero as f32 is not the default of 1 / sqrt(D)."""
    with pytest.raises(ib.CompilationStageError):
        ib.compile(getattr(ib.programs, program), constexprs={"SCALE": scale}, resolve_target=False)


@pytest.mark.parametrize("scale", [None, 1e-45, 0.125, 1, 3e38])
def test_scales_that_are_one(scale):
    artifact = ib.compile(ib.programs.paged_attention, constexprs={"SCALE": scale}, resolve_target=False)
    assert (artifact.runtime.constants[0] == 0) == (scale is None)


@pytest.mark.parametrize("failing", ["from_numpy", "split"])
def test_a_step_that_fails_changes_nothing(monkeypatch, failing):
    """Memory for its tensors, say, may run out after the pages were found."""
    store = PagedKVCache(layers=1, pages=8, kv_heads=2, head_dim=64, page_size=16, device="cpu")
    store.step({"a": 20})
    with monkeypatch.context() as patch:
        def fail(*_):
            raise RuntimeError("out of memory")

        patch.setattr(torch, failing, fail)
        with pytest.raises(RuntimeError):
            store.step({"a": 30, "b": 5})
    assert store.free_pages == 6 and store.length("a") == 20 and store.length("b") == 0
    with pytest.raises(KeyError):
        store.release("b")
    step = store.step({"b": 5, "a": 30})
    assert step.kv_lengths.tolist() == [5, 50] and step.positions.tolist() == [*range(5), *range(20, 50)]
    used = step.page_table[0, :1].tolist() + step.page_table[1, :4].tolist()
    assert sorted(used) == sorted(set(used)) and store.free_pages == 3


def test_where_the_positions_of_a_step_end():
    store = PagedKVCache(layers=1, pages=8, kv_heads=2, head_dim=64, page_size=16, device="cpu")
    assert store.step({"a": 20, "b": 3}).longest == 20
    assert store.step({"b": 1}).longest == 4
    assert store.step({"a": 0, "b": 2}).longest == 6 and store.step({"a": 0}).longest == 0


def test_workspace_of_a_call():
    """The parts of chunks, 40 MB with heads of 128, are asked for by calls that may have chunks only."""
    query = ib.compile(ib.programs.paged_attention, resolve_target=False).runtime._workspace_spec
    single = ib.compile(ib.programs.paged_decode_attention, resolve_target=False).runtime._workspace_spec
    sizes = {"HQ": 32, "HK": 8, "D": 128, "PAGE": 64, "W": 512}
    few = single({**sizes, "B": 64})
    assert few < 4 << 20
    for T, B in ((1, 1), (64, 64), (4, 1), (96, 89)):
        assert query({**sizes, "T": T, "B": B}) == few
    for T, B in ((33, 1), (64, 16), (800, 64), (1023, 256), (4096, 1), (1 << 20, 1)):
        assert query({**sizes, "T": T, "B": B}) > 40 << 20
    assert query({**sizes, "T": 64, "B": 16, "W": 64}) == few                    # (histories that are short)
    assert query({**sizes, "HQ": 130, "HK": 1, "T": 4096, "B": 1}) == few        # (heads that the chunk kernel does not take)
    narrow = ib.compile(ib.programs.paged_attention, constexprs={"WINDOW": 100}, resolve_target=False).runtime._workspace_spec
    assert narrow({**sizes, "T": 64, "B": 16}) == few
