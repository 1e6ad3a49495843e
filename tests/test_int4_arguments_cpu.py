"""What the programs of a cache in 4 bits refuse, in the compiler and at the C entries, without a GPU."""
import ctypes
import math

import pytest

import intent_b200 as ib
from intent_b200.runtime import native

PROGRAMS = ["paged_kv_append_int4", "paged_kv_read_int4", "paged_attention_int4", "paged_decode_attention_int4"]


@pytest.mark.parametrize("name", PROGRAMS)
@pytest.mark.parametrize("constexprs", [{"GROUP_SIZE": 16}, {"GROUP_SIZE": 48}, {"GROUP_SIZE": 256}, {"GROUP_SIZE": "64"},
                                        {"GROUP_SIZE": None}, {"ACT_DTYPE": "f32"}, {"BITS": 4}])
def test_constants(name, constexprs):
    with pytest.raises(ib.CompilationStageError):
        ib.compile(getattr(ib.programs, name), constexprs=constexprs, resolve_target=False)


@pytest.mark.parametrize("name", PROGRAMS[2:])
@pytest.mark.parametrize("scale", [0, -1.0, 1e-46, math.inf, math.nan, 2.0 ** 51, 3e38])
def test_scales_of_scores(name, scale):
    with pytest.raises(ib.CompilationStageError):
        ib.compile(getattr(ib.programs, name), constexprs={"SCALE": scale}, resolve_target=False)


@pytest.mark.parametrize("name", PROGRAMS)
def test_saved_and_loaded(name, tmp_path):
    artifact = ib.compile(getattr(ib.programs, name), constexprs={"GROUP_SIZE": 32}, resolve_target=False)
    again = ib.load(artifact.save(tmp_path / "program"), resolve_target=False)
    assert again.runtime.constants == artifact.runtime.constants and again.runtime.entry_name == artifact.runtime.entry_name


def view(shape, pointer=0x10000, strides=None):
    if strides is None:
        strides = [math.prod(shape[i + 1:]) for i in range(len(shape))]
    return [pointer, *shape, *strides]


def status(name, views, *rest):
    slots = [s for v in views for s in v]
    carriers = ["ptr" if i == 0 else "i64" for v in views for i in range(len(v))]
    return native.entry(f"intent_b200_{name}_bf16", (*carriers, *("i32" if r is not None else "ptr" for r in rest)))(*slots, *rest, None)


OK, SHAPE, LAYOUT, UNSUPPORTED, WORKSPACE, NULL = 0, 1, 2, 3, 5, 6


def cache(pages=4, heads=2, page=16, dim=128, group=64):
    return [view([pages, heads, page, dim // 2]), view([pages, heads, page, 2 * dim // group])] * 2


def read(slots=5, parts=None, heads=2, dim=128, group=64, **changes):
    views = [view([slots]), *(parts or cache(heads=heads, dim=dim, group=group)), view([slots, heads, dim]), view([slots, heads, dim])]
    for place, v in changes.items():
        views[int(place[1:])] = v
    return status("paged_kv_read_int4", views, group)


def test_entry_of_reads():
    assert read(slots=0) == OK
    assert read(group=48) == read(dim=64, group=128) == read(dim=96, group=32) == UNSUPPORTED
    assert read(parts=cache(page=24)) == read(parts=cache(page=8)) == UNSUPPORTED
    assert read(parts=cache(heads=3)) == read(parts=cache(dim=64)) == read(parts=cache(group=32)) == SHAPE
    assert read(_3=view([3, 2, 16, 64])) == read(_6=view([5, 2, 64])) == read(_5=view([4, 2, 128])) == SHAPE
    assert read(_1=view([4, 2, 16, 64], 0x10008)) == read(_2=view([4, 2, 16, 4], strides=[128, 4, 8, 1])) == LAYOUT
    assert read(_5=view([5, 2, 128], 0x10002)) == LAYOUT
    assert read(_1=view([4, 2, 16, 64], 0)) == read(_0=view([5], 0)) == read(_4=view([4, 2, 16, 4], 0)) == NULL


def attend(parts=None, group=64, scale=0, window=0, workspace=None, tokens=3, q=None, heads=4):
    views = [q or view([tokens, heads, 128]), *(parts or cache()), view([tokens, 2]), view([tokens]), view([tokens, heads, 128])]
    slots = [s for v in views for s in v]
    carriers = ["ptr" if i == 0 else "i64" for v in views for i in range(len(v))]
    entry = native.entry("intent_b200_paged_decode_attention_int4_bf16", (*carriers, "i32", "i32", "i32", "ptr", "i64"))
    return entry(*slots, group, scale, window, workspace, 0, None)


def test_entry_of_attention():
    assert attend(tokens=0) == OK
    assert attend() == WORKSPACE
    assert attend(group=48) == attend(window=-1) == attend(parts=cache(page=512)) == UNSUPPORTED
    assert attend(scale=0x59000000) == UNSUPPORTED          # 2^51
    assert attend(scale=0x58800000) == WORKSPACE            # 2^50
    assert attend(parts=cache(group=32)) == attend(parts=cache(heads=3)) == attend(parts=cache(dim=64)) == SHAPE
    assert attend(parts=[*cache()[:3], view([4, 2, 16, 4], 0x10004)]) == LAYOUT
    assert attend(parts=[*cache()[:3], view([4, 2, 16, 4], 0)]) == attend(q=view([3, 4, 128], 0)) == NULL
    assert ctypes.sizeof(ctypes.c_void_p) == 8


def test_pages_in_4_bits():
    from intent_b200.attention import PagedKVCache, QuantisedPages, W4A16Attention

    sizes = {"layers": 2, "pages": 8, "kv_heads": 2, "head_dim": 128, "page_size": 16, "device": "cpu"}
    store = PagedKVCache(bits=4, group_size=32, **sizes)
    for part in store.layer(1):
        assert isinstance(part, QuantisedPages)
        assert part.codes.shape == (8, 2, 16, 64) and part.scales.shape == (8, 2, 16, 8)
    step = store.step({"a": 20, "b": 3})
    assert step.kv_lengths.tolist() == [20, 3] and store.free_pages == 5
    for name, start, stop, error in (("c", 0, None, KeyError), ("a", 0, 21, ValueError), ("a", 5, 4, ValueError), ("a", -1, 4, ValueError)):
        with pytest.raises(error):
            store.read(0, name, start, stop)
    for wrong in ({"bits": 8}, {"bits": 4, "group_size": 16}, {"bits": 4, "group_size": 256}):
        with pytest.raises(ValueError):
            PagedKVCache(**{**sizes, **wrong})
    with pytest.raises(ValueError):
        PagedKVCache(**{**sizes, "head_dim": 64}, bits=4, group_size=128)
    with pytest.raises(ValueError):
        W4A16Attention(hidden=256, heads=4, kv_heads=2, head_dim=64, cache_bits=8)


def test_reading_pages_of_16_bits():
    import torch

    from intent_b200.attention import PagedKVCache

    store = PagedKVCache(layers=2, pages=8, kv_heads=2, head_dim=64, page_size=16, device="cpu")
    store.k.copy_(torch.randn(store.k.shape)), store.v.copy_(torch.randn(store.v.shape))
    store.step({"x": 20})
    step = store.step({"a": 40})
    for got, whole in zip(store.read(1, "a", 3, 39), (store.k[1], store.v[1])):
        flat = whole.transpose(1, 2).flatten(0, 1)
        assert torch.equal(got, flat[step.slots[3:39]])
    assert store.read(0, "a", 40)[0].shape == (0, 2, 64)


def test_shapes_are_inferred_without_a_device():
    """What fake tensors go through."""
    import torch

    def empty(*shape, dtype=torch.bfloat16):
        return torch.empty(shape, dtype=dtype, device="meta")

    caches = [empty(7, 2, 16, 64, dtype=torch.uint8), empty(7, 2, 16, 4)] * 2
    caches = [c.clone() for c in caches]
    program = {name: ib.compile(getattr(ib.programs, name), resolve_target=False).runtime for name in PROGRAMS}
    ints = [empty(n, dtype=torch.int32) for n in (5, 4, 3)]
    slots = empty(5, dtype=torch.int64)
    keys, values = program["paged_kv_read_int4"].infer_outputs((slots, *caches))
    assert keys.shape == values.shape == (5, 2, 128) and keys.dtype == torch.bfloat16
    q, k = empty(5, 8, 128), empty(5, 2, 128)
    out = program["paged_kv_append_int4"].infer_outputs((q, k, k.clone(), ints[0], slots, empty(9, 64, dtype=torch.float32), empty(128),
                                                         empty(128), *caches))
    assert out.shape == (5, 8, 128)
    pages = empty(3, 4, dtype=torch.int32)
    assert program["paged_attention_int4"].infer_outputs((q, *caches, pages, ints[1], ints[2])).shape == (5, 8, 128)
    assert program["paged_decode_attention_int4"].infer_outputs((q[:3], *caches, pages, ints[2])).shape == (3, 8, 128)


def test_workspace_of_a_call():
    """As of a cache of 16 bits: the parts of chunks are asked for by calls that may have chunks only."""
    query = ib.compile(ib.programs.paged_attention_int4, resolve_target=False).runtime._workspace_spec
    single = ib.compile(ib.programs.paged_decode_attention_int4, resolve_target=False).runtime._workspace_spec
    sizes = {"HQ": 32, "HK": 8, "D": 128, "PAGE": 64, "W": 512}
    few = single({**sizes, "B": 64})
    assert few < 4 << 20
    for T, B in ((1, 1), (64, 64), (8, 1), (75, 64)):
        assert query({**sizes, "T": T, "B": B}) == few
    for T, B in ((33, 1), (1000, 64), (4096, 1), (1 << 20, 1)):
        assert query({**sizes, "T": T, "B": B}) > 40 << 20
