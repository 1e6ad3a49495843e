"""paged_kv_append_int4 and paged_kv_read_int4 against their definitions in 64 bits."""
import math

import pytest
import torch

import intent_b200 as ib
from oracle import attention as oracle
from test_rope_append_gpu import DTYPES, F32, HALF_UNIT, assert_rounded, inputs, move, scale_of, table

pytestmark = pytest.mark.gpu


def empty_cache(pages, HK, page, D, group, dtype, device, seed=0):
    """Four tensors of arbitrary contents: keys' codes and scales, values' codes and scales."""
    g = torch.Generator().manual_seed(seed)
    parts = []
    for _ in range(2):
        parts.append(torch.randint(0, 256, (pages, HK, page, D // 2), generator=g, dtype=torch.uint8).to(device))
        parts.append(torch.randn((pages, HK, page, 2 * D // group), generator=g).to(DTYPES[dtype]).to(device))
    return parts


def rows(cache, slots):
    """[T, HK, ...] of the tokens at slots that are inside."""
    page = cache.shape[2]
    return cache.cpu()[slots // page, :, slots % page]


def assert_held(codes, scales, x, size, group, dtype):
    """x [T, HK, D] in f64, off by F32 * size: a value is at most half a scale from it, and what the roundings of the group's minimum
    and scale (15 of them at its upper end) leave."""
    held, _ = oracle.values(codes, scales, group)
    s, m = scales.double().unflatten(-1, (-1, 2)).unbind(-1)
    assert (s >= 0).all()
    least, most = x.unflatten(-1, (-1, group)).aminmax(dim=-1)
    tiny = 2.0 ** -24
    assert ((m - least).abs() <= HALF_UNIT[dtype] * least.abs() + F32 * size + tiny).all()
    assert ((s - (most - least) / 15).abs() <= HALF_UNIT[dtype] * s + F32 * size + tiny).all()
    bound = s / 2 * (1 + 2.0 ** -16) + HALF_UNIT[dtype] * (15 * s + m.abs()) + 2 * F32 * size + 16 * tiny
    assert ((held - x).abs().unflatten(-1, (-1, group)) <= bound[..., None]).all()


def assert_codes(codes, scales, x, group):
    """The codes of 16-bit values x, given the scales: the nearest, halves to the even one.  Where the difference to the minimum has
    more than 24 bits, its rounding may decide next to a half: 2^-20 of 16 around it."""
    n = torch.stack([codes % 16, codes // 16], -1).flatten(-2).double().unflatten(-1, (-1, group))
    s, m = scales.double().unflatten(-1, (-1, 2)).split(1, -1)
    exact = torch.where(s > 0, (x.double().unflatten(-1, (-1, group)) - m) / torch.where(s > 0, s, 1), 0)
    nearest = exact.round().clamp(0, 15)
    half = ((exact % 1) - 0.5).abs()
    assert ((n == nearest) | ((half > 0) & (half < 2.0 ** -16))).all()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("norm", [True, False])
@pytest.mark.parametrize("pairs", ["halves", "neighbours"])
@pytest.mark.parametrize("T,HQ,HK,D,R,page,group,packed", [
    (1, 8, 2, 128, 128, 64, 64, True), (40, 4, 4, 64, 64, 16, 32, False), (77, 6, 2, 128, 64, 256, 128, True),
    (19, 7, 1, 64, 32, 32, 64, True), (21, 3, 3, 128, 96, 16, 32, False), (600, 32, 8, 128, 128, 64, 64, True),
    (1100, 16, 5, 64, 48, 32, 32, False),
])
def test_append(cuda_device, dtype, norm, pairs, T, HQ, HK, D, R, page, group, packed):
    (q, k, v), weights = inputs(T, HQ, HK, D, dtype, packed, seed=T)
    g = torch.Generator().manual_seed(3)
    pages = -(-T // page) + 3
    rotary, positions = table(64, R), torch.arange(T, dtype=torch.int32) % 64
    slots = torch.randperm(pages * page, generator=g)[:T]
    if T > 4:
        slots[1], slots[2], slots[3] = -1, pages * page, -(1 << 40)       # padding
    inside = (slots >= 0) & (slots < pages * page)
    cache = empty_cache(pages, HK, page, D, group, dtype, cuda_device)
    before = [c.cpu() for c in cache]
    artifact = ib.compile(ib.programs.paged_kv_append_int4,
                          constexprs={"ACT_DTYPE": dtype, "NORM": norm, "PAIRS": pairs, "GROUP_SIZE": group})
    moved = move((q, k, v), cuda_device, packed)
    extra = [w.to(cuda_device) for w in weights] if norm else []
    w = weights if norm else (None, None)
    keys = oracle.rotate(k, positions, rotary, w[1], pairs=pairs)
    for _ in range(2):                       # bound in Python, then natively
        out = artifact.run(*moved, positions.to(cuda_device), slots.to(cuda_device), rotary.to(cuda_device), *extra, *cache)
        assert_rounded(out, oracle.rotate(q, positions, rotary, w[0], pairs=pairs), scale_of(q, w[0]), dtype)
        held = [rows(c, slots[inside]) for c in cache]
        assert_held(held[0], held[1], keys[inside], scale_of(k, w[1])[inside], group, dtype)
        assert_held(held[2], held[3], v[inside].double(), 0, group, dtype)
        assert_codes(held[2], held[3], v[inside], group)
        written = torch.zeros((pages, page), dtype=torch.bool)
        written[slots[inside] // page, slots[inside] % page] = True
        for now, then in zip(cache, before):                              # what is there already stays
            assert torch.equal(now.cpu().transpose(1, 2)[~written], then.transpose(1, 2)[~written])
    assert artifact.runtime.binder.last() is not None


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("T,HK,D,page,group", [(1, 1, 64, 16, 64), (33, 3, 128, 64, 32), (130, 8, 128, 256, 128), (7, 2, 64, 32, 32),
                                               (2000, 5, 128, 16, 64)])
def test_read(cuda_device, dtype, T, HK, D, page, group):
    pages = -(-T // page) + 2
    cache = empty_cache(pages, HK, page, D, group, dtype, cuda_device)
    slots = torch.randint(0, pages * page, (T,), generator=torch.Generator().manual_seed(1))
    if T > 4:
        slots[1], slots[2], slots[3] = -1, pages * page, 1 << 60
    inside = (slots >= 0) & (slots < pages * page)
    artifact = ib.compile(ib.programs.paged_kv_read_int4, constexprs={"ACT_DTYPE": dtype, "GROUP_SIZE": group})
    for _ in range(2):
        out = artifact.run(slots.to(cuda_device), *cache)
        for i, actual in enumerate(out):
            assert actual.shape == (T, HK, D) and actual.dtype == DTYPES[dtype]
            expected, _ = oracle.values(rows(cache[2 * i], slots[inside]), rows(cache[2 * i + 1], slots[inside]), group)
            # a sum in f32 (its terms: a minimum and 15 scales), rounded once
            bound = HALF_UNIT[dtype] * expected.abs() + 2.0 ** -24 * (expected.abs() + 2.0 ** -1)
            actual = actual.cpu()
            assert ((actual[inside].double() - expected).abs() <= bound).all()
            assert not actual[~inside].any()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("D,group", [(64, 32), (128, 64), (128, 128)])
def test_groups_of_every_kind(cuda_device, dtype, D, group):
    """All equal, whole numbers that are held as they are, halves between codes, the ends of the type, infinities and NaN."""
    top = torch.finfo(DTYPES[dtype]).max
    small = torch.finfo(DTYPES[dtype]).smallest_normal
    g = torch.Generator().manual_seed(0)
    v = torch.zeros((12, 1, D))
    v[1] = -3.25
    v[2] = torch.randint(0, 16, (D,), generator=g).float() - 7
    v[2, 0, ::group], v[2, 0, 1::group] = -7, 8
    v[3] = torch.randint(0, 31, (D,), generator=g).float()                # steps of two: odd numbers are halves
    v[3, 0, ::group], v[3, 0, 1::group] = 0, 30
    v[4] = torch.randn(D, generator=g) * top
    v[4, 0, ::group], v[4, 0, 1::group] = -top, top
    v[5] = torch.randn(D, generator=g) * small
    v[6, 0, 3], v[7, 0, 3], v[8, 0, 3] = math.inf, -math.inf, math.nan
    v[9] = 1000 + torch.randn(D, generator=g)                             # a range that is small beside the numbers
    v[10] = torch.randn(D, generator=g)
    v[10, 0, 5] = 3000.0
    v[11] = -torch.rand(D, generator=g)
    v = v.clamp(-top, top).where(v.isfinite(), v).to(DTYPES[dtype])
    T = len(v)
    cache = empty_cache(2, 1, 16, D, group, dtype, cuda_device)
    slots, positions = torch.arange(T), torch.zeros(T, dtype=torch.int32)
    append = ib.compile(ib.programs.paged_kv_append_int4, constexprs={"ACT_DTYPE": dtype, "NORM": False, "GROUP_SIZE": group})
    append.run(*(t.to(cuda_device) for t in (v, v, v, positions, slots, table(1, 16))), *cache)
    held = [rows(c, slots) for c in cache]
    finite = v.double().unflatten(-1, (-1, group)).isfinite().all(-1)     # [T, 1, groups]
    for codes, scales in (held[:2], held[2:]):                            # (position 0 turns keys by nothing)
        pairs = scales.unflatten(-1, (-1, 2))
        assert torch.equal(pairs.isnan().all(-1), ~finite) and torch.equal(pairs.isnan().any(-1), ~finite)
        n = torch.stack([codes % 16, codes // 16], -1).flatten(-2).unflatten(-1, (-1, group))
        assert not n[~finite].any()
        kept = finite.all(-1)[:, 0]
        assert_codes(codes[kept], scales[kept], v[kept], group)
        same = (pairs[..., 0] == 0) & finite
        assert not n[same].any()
    value, _ = oracle.values(held[2], held[3], group)
    for exact in (0, 1, 2):
        assert torch.equal(value[exact], v[exact].double())
    # a code in the middle between two numbers goes to the even one
    odd = (v[3, 0].double() % 2) == 1
    n = torch.stack([held[2] % 16, held[2] // 16], -1).flatten(-2)[3, 0]
    assert odd.any() and not (n[odd] % 2).any()
    out = ib.compile(ib.programs.paged_kv_read_int4, constexprs={"ACT_DTYPE": dtype, "GROUP_SIZE": group}).run(
        slots.to(cuda_device), *cache)[1].cpu()
    wide = finite.repeat_interleave(group, -1)
    assert torch.equal(out.isnan(), ~wide)
    s = held[3].double().unflatten(-1, (-1, 2))[..., 0].repeat_interleave(group, -1)
    m = held[3].double().unflatten(-1, (-1, 2))[..., 1].abs().repeat_interleave(group, -1)
    bound = s / 2 * (1 + 2.0 ** -16) + HALF_UNIT[dtype] * (15 * s + m + v.double().abs()) + 16 * torch.finfo(DTYPES[dtype]).tiny
    assert ((out.double() - v.double()).abs() <= bound)[wide].all()


def test_positions_outside_the_table(cuda_device):
    """Keys of such a token are NaN; its values and the other tokens are as they are."""
    (q, k, v), _ = inputs(4, 2, 1, 64, "bf16", False)
    positions = torch.tensor([-1, 0, 9, 10], dtype=torch.int32)
    cache = empty_cache(1, 1, 16, 64, 64, "bf16", cuda_device)
    slots = torch.arange(4)
    ib.compile(ib.programs.paged_kv_append_int4, constexprs={"NORM": False}).run(
        *(t.to(cuda_device) for t in (q, k, v, positions, slots, table(10, 64))), *cache)
    keys, found = ib.compile(ib.programs.paged_kv_read_int4).run(slots.to(cuda_device), *cache)
    assert keys.isnan().flatten(1).all(1).tolist() == keys.isnan().flatten(1).any(1).tolist() == [True, False, False, True]
    assert found.isfinite().all()


def test_a_cache_of_more_than_32_bits(cuda_device):
    """Slots whose bytes lie past 2^32."""
    HK, page, D, group = 8, 256, 128, 64
    pages = (1 << 32) // (HK * page * D // 2) + 2
    sizes = ((D // 2, torch.uint8), (2 * D // group, torch.bfloat16))
    cache = [torch.empty((pages, HK, page, n), dtype=t, device=cuda_device) for n, t in sizes * 2]
    for c in cache:
        c[0].fill_(1), c[-1].fill_(1)
    (q, k, v), _ = inputs(2, 8, HK, D, "bf16", False)
    slots, positions = torch.tensor([pages * page - 1, 5]), torch.zeros(2, dtype=torch.int32)
    moved = [t.to(cuda_device) for t in (q, k, v, positions, slots, table(4, 128))]
    ib.compile(ib.programs.paged_kv_append_int4, constexprs={"NORM": False}).run(*moved, *cache)
    for i, x in ((0, k), (2, v)):
        codes, scales = oracle.quantise(x, group, torch.bfloat16)
        for token, place in ((0, (-1, -1)), (1, (0, 5))):
            assert torch.equal(cache[i + 1][place[0], :, place[1]].cpu(), scales[token])
            assert (cache[i][place[0], :, place[1]].cpu() != codes[token]).float().mean() < 0.01
        assert (cache[i][0, :, 4] == 1).all() and (cache[i][0, :, 6] == 1).all() and (cache[i][-1, :, :-1] == 1).all()
    out = ib.compile(ib.programs.paged_kv_read_int4).run(slots.to(cuda_device), *cache)
    assert all(((a.cpu().float() - x.float()).abs() < 0.5).all() for a, x in zip(out, (k, v)))


def test_no_tokens_and_no_pages(cuda_device):
    (q, k, v), weights = inputs(0, 4, 2, 64, "bf16", False)
    cache = empty_cache(2, 2, 16, 64, 64, "bf16", cuda_device)
    none = torch.zeros(0, dtype=torch.int64)
    append, read = ib.compile(ib.programs.paged_kv_append_int4), ib.compile(ib.programs.paged_kv_read_int4)
    args = [t.to(cuda_device) for t in (q, k, v, none.int(), none, table(4, 64), *weights)]
    assert append.run(*args, *cache).shape == (0, 4, 64)
    assert [tuple(t.shape) for t in read.run(none.to(cuda_device), *cache)] == [(0, 2, 64)] * 2
    (q, k, v), weights = inputs(3, 4, 2, 64, "bf16", False)
    nowhere = [c[:0] for c in cache]
    args = [t.to(cuda_device) for t in (q, k, v, torch.arange(3).int(), torch.arange(3), table(4, 64), *weights)]
    assert append.run(*args, *nowhere).isfinite().all()
    assert not any(t.any() for t in read.run(args[4], *nowhere))


def test_graphs_and_streams(cuda_device):
    (q, k, v), weights = inputs(50, 8, 2, 128, "bf16", True)
    slots = torch.randperm(64)[:50].to(cuda_device)
    moved = move((q, k, v), cuda_device, True)
    rest = [t.to(cuda_device) for t in (torch.arange(50).int(), slots, table(64, 128), *weights)]
    append, read = ib.compile(ib.programs.paged_kv_append_int4), ib.compile(ib.programs.paged_kv_read_int4)
    cache = empty_cache(4, 2, 16, 128, 64, "bf16", cuda_device)
    expected = append.run(*moved, *rest, *cache), *read.run(slots, *cache)
    calls = append.prepare(*moved, *rest, *(c.clone() for c in cache)), None
    other = calls[0].invocation.arguments
    held = other[-5:-1]
    calls = calls[0], read.prepare(slots, *held)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        for call in calls:
            call.launch()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for call in calls:
            call.launch()
    for t in (*held, *calls[1].outputs):
        t.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(calls[0].result(), expected[0])
    assert all(torch.equal(a, b) for a, b in zip(calls[1].result(), expected[1:]))
    assert all(torch.equal(rows(a, slots.cpu()), rows(b, slots.cpu())) for a, b in zip(held, cache))


def test_refusals(cuda_device):
    (q, k, v), weights = inputs(4, 4, 2, 128, "bf16", False)
    args = [t.to(cuda_device) for t in (q, k, v, torch.zeros(4).int(), torch.arange(4), table(4, 128), *weights)]
    cache = empty_cache(2, 2, 16, 128, 64, "bf16", cuda_device)
    append, read = ib.compile(ib.programs.paged_kv_append_int4), ib.compile(ib.programs.paged_kv_read_int4)
    append.run(*args, *cache)
    read.run(args[4], *cache)
    wrong = {
        "groups": empty_cache(2, 2, 16, 128, 32, "bf16", cuda_device), "heads": empty_cache(2, 3, 16, 128, 64, "bf16", cuda_device),
        "pages": empty_cache(2, 2, 24, 128, 64, "bf16", cuda_device), "rows": empty_cache(2, 2, 16, 64, 32, "bf16", cuda_device),
        "one page fewer": [cache[0], cache[1][:1], *cache[2:]],
    }
    for name, parts in wrong.items():
        with pytest.raises(ValueError):
            append.run(*args, *parts)
        if name not in ("heads",):
            with pytest.raises(ValueError):
                read.run(args[4], *parts)
    for parts in ([cache[0], cache[1].half(), *cache[2:]], [cache[0].to(torch.int8), *cache[1:]]):
        with pytest.raises(TypeError):
            append.run(*args, *parts)
        with pytest.raises(TypeError):
            read.run(args[4], *parts)
    with pytest.raises(NotImplementedError):           # keys and values in one memory
        append.run(*args, cache[0], cache[1], cache[0], cache[3])
    with pytest.raises(NotImplementedError):           # tokens ahead of heads
        read.run(args[4], *(c.transpose(1, 2).contiguous().transpose(1, 2) for c in cache))
    with pytest.raises(TypeError):
        read.run(args[4].int(), *cache)


@pytest.mark.parametrize("norm", [True, False])
@pytest.mark.parametrize("dtype,D,R,group,pairs", [("bf16", 128, 128, 64, "halves"), ("f16", 128, 128, 32, "halves"), ("bf16", 128, 64, 128, "neighbours"),
                                                   ("f16", 64, 32, 64, "halves"), ("bf16", 64, 64, 32, "neighbours")])
def test_codes_of_keys_are_the_definitions(cuda_device, norm, dtype, D, R, group, pairs):
    """Also next to a border: of half a million elements none may be off by a step.  What decides is then at least 2^-40 away from
    equal (64 bits: a dozen operations of 2^-53 on numbers up to 2^4 of a step)."""
    T, HK = 1000, 4
    (q, k, v), weights = inputs(T, 2, HK, D, dtype, False, seed=5)
    rotary, positions = table(2000, R), torch.arange(T, dtype=torch.int32) * 2
    cache = empty_cache(-(-T // 64), HK, 64, D, group, dtype, cuda_device)
    slots = torch.arange(T)
    append = ib.compile(ib.programs.paged_kv_append_int4,
                        constexprs={"ACT_DTYPE": dtype, "NORM": norm, "PAIRS": pairs, "GROUP_SIZE": group})
    append.run(*(t.to(cuda_device) for t in (q, k, v, positions, slots, rotary, *(weights if norm else ()))), *cache)
    keys = oracle.rotate(k, positions, rotary, weights[1] if norm else None, pairs=pairs, eps=float(torch.tensor(1e-6)))
    codes, scales = oracle.quantise(keys, group, DTYPES[dtype])
    held = [rows(c, slots) for c in cache[:2]]
    assert torch.equal(held[1], scales)
    n, m = (torch.stack([c % 16, c // 16], -1).flatten(-2).int() for c in (held[0], codes))
    if norm:
        assert torch.equal(n, m)
    else:       # (halves of whole steps, where 64 bits round the quotient before it is rounded to a whole number)
        by, least = scales.double().unflatten(-1, (-1, 2)).split(1, -1)
        exact = ((keys.unflatten(-1, (-1, group)) - least) / by).flatten(-2)
        assert ((n == m) | (((exact % 1) - 0.5).abs() < 2.0 ** -40)).all()


def test_keys_that_are_nearly_equal(cuda_device):
    """A group whose range is far below the rounding of its minimum: codes are cut, whichever way."""
    k = torch.full((4, 1, 64), 1000.0, dtype=torch.bfloat16)
    rotary = torch.zeros((4, 32))
    rotary[:, :16] = torch.tensor([1.0, 1.003, 1 + 2.0 ** -20, 1 + 2.0 ** -23])[:, None]
    rotary[:, 0] += 2.0 ** -22
    cache = empty_cache(1, 1, 16, 64, 64, "bf16", cuda_device)
    slots = torch.arange(4)
    ib.compile(ib.programs.paged_kv_append_int4, constexprs={"NORM": False}).run(
        *(t.to(cuda_device) for t in (k, k, k, slots.int(), slots, rotary)), *cache)
    keys = oracle.rotate(k, slots, rotary)
    codes, scales = oracle.quantise(keys, 64, torch.bfloat16)
    held = [rows(c, slots) for c in cache[:2]]
    assert torch.equal(held[0], codes) and torch.equal(held[1], scales)
