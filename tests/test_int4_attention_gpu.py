"""paged_attention_int4 and paged_decode_attention_int4 against the definition in 64 bits."""
import math

import pytest
import torch

import intent_b200 as ib
from oracle import attention as oracle
from test_paged_attention_gpu import DTYPES, HALF_UNIT, LENGTHS

pytestmark = pytest.mark.gpu


def make(lengths, counts, HQ, HK, D, page, group, dtype, seed=0, spare=2):
    """Queries and a cache in which every place that no sequence uses has arbitrary codes and NaN for scales."""
    g = torch.Generator().manual_seed(seed)
    used = [-(-n // page) for n in lengths]
    pages, width = sum(used) + spare, max(max(used), 1)
    cache = []
    order = torch.randperm(pages, generator=g).to(torch.int32)
    table = torch.full((len(lengths), width), -1, dtype=torch.int32)
    at = 0
    held = torch.zeros((pages, page), dtype=torch.bool)
    for b, n in enumerate(lengths):
        table[b, :used[b]] = order[at:at + used[b]]
        at += used[b]
        for i in range(used[b]):
            held[int(table[b, i]), :min(page, n - i * page)] = True
    for offset in (0.5, 0.0):
        x = torch.randn((pages, HK, page, D), generator=g) + offset * torch.randn((HK, 1, D), generator=g)
        codes, scales = oracle.quantise(x, group, DTYPES[dtype])
        scales.masked_fill_(~held[:, None, :, None], math.nan)
        cache += [codes, scales]
    offsets = torch.tensor([0] + counts).cumsum(0).to(torch.int32)
    q = torch.randn((sum(counts), HQ, D), generator=g).to(DTYPES[dtype])
    return q, cache, table, offsets, torch.tensor(lengths, dtype=torch.int32)


def reference(data, group, scale=None, window=0):
    """(out, bound): the rounding of a weight (relative to its row's largest) is worth half a unit of what it is multiplied with, the
    distance from the group's middle; scores and sums are in f32 and of numbers as large as the middle and eight scales (2e-4: 128
    products, the exponential, thousands of additions); the result is rounded once."""
    q, (k_codes, k_scales, v_codes, v_scales), *rest = data
    keys, _ = oracle.values(k_codes, k_scales, group)
    values, middle = oracle.values(v_codes, v_scales, group)
    half = HALF_UNIT["bf16" if q.dtype == torch.bfloat16 else "f16"]
    out, _ = oracle.paged_attention(q, keys, values, *rest, scale=scale, window=window)
    _, away = oracle.paged_attention(q, keys, values - middle, *rest, scale=scale, window=window)
    size = v_scales.double().unflatten(-1, (-1, 2))[..., :1].mul(8).expand(*v_scales.shape[:-1], -1, group).flatten(-2)
    _, large = oracle.paged_attention(q, keys, middle.abs() + size, *rest, scale=scale, window=window)
    return out, half * away + 2e-4 * large + half * out.abs() + 2.0 ** -24


def of_rounded(data, group, scale=None, window=0):
    """The same where keys and values become numbers of the type first."""
    q, (k_codes, k_scales, v_codes, v_scales), *rest = data
    half = HALF_UNIT["bf16" if q.dtype == torch.bfloat16 else "f16"]
    keys, values = (oracle.values(c, s, group)[0].to(q.dtype) for c, s in ((k_codes, k_scales), (v_codes, v_scales)))
    out, weight = oracle.paged_attention(q, keys, values, *rest, scale=scale, window=window)
    return out, (half + 2e-4) * weight + half * out.abs() + 2.0 ** -24


def assert_close(actual, *expected):
    """Every token's rows are within the bound of one of the (out, bound)."""
    actual = actual.cpu().double()
    assert not actual.isnan().any()
    fine = [((actual - out).abs() <= bound).flatten(1).all(1) for out, bound in expected]
    bad = ~torch.stack(fine).any(0)
    assert not bad.any(), (bad.nonzero().flatten()[:8].tolist(), float((actual - expected[0][0]).abs()[bad].max()))


def run(artifact, device, data, single):
    q, cache, table, offsets, lengths = data
    return artifact.run(*(t.to(device) for t in (q, *cache, table, *(() if single else (offsets,)), lengths)))


def both(device, lengths, counts, HQ, HK, D, page, group, dtype, window=0, scale=None, seed=0):
    data = make(lengths, counts, HQ, HK, D, page, group, dtype, seed)
    expected = [reference(data, group, scale, window)]
    constants = {"ACT_DTYPE": dtype, "WINDOW": window, "SCALE": scale, "GROUP_SIZE": group}
    if all(c == 1 for c in counts):
        artifact = ib.compile(ib.programs.paged_decode_attention_int4, constexprs=constants)
        for _ in range(2):
            assert_close(run(artifact, device, data, True), *expected)
        artifact.check()
    expected.append(of_rounded(data, group, scale, window))
    artifact = ib.compile(ib.programs.paged_attention_int4, constexprs=constants)
    for _ in range(2):
        assert_close(run(artifact, device, data, False), *expected)
    artifact.check()
    return data, expected


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("HQ,HK,D,page,group", [
    (8, 2, 128, 64, 64), (4, 4, 64, 16, 32), (5, 1, 128, 32, 128), (12, 1, 64, 128, 64), (40, 2, 128, 256, 32), (16, 1, 128, 16, 128),
    (16, 1, 128, 16, 64), (16, 1, 64, 32, 32),
])
def test_single_tokens(cuda_device, dtype, HQ, HK, D, page, group):
    both(cuda_device, LENGTHS, [1] * len(LENGTHS), HQ, HK, D, page, group, dtype)


@pytest.mark.parametrize("window", [1, 16, 100, 128, 1000])
@pytest.mark.parametrize("D,page,group", [(64, 32, 64), (128, 16, 32)])
def test_single_tokens_with_a_window(cuda_device, window, D, page, group):
    both(cuda_device, LENGTHS, [1] * len(LENGTHS), 4, 2, D, page, group, "bf16", window=window)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("HQ,HK,D,page,group", [(8, 2, 128, 64, 64), (4, 4, 64, 16, 32), (7, 1, 64, 32, 64), (3, 1, 128, 256, 128),
                                                (24, 1, 128, 16, 32)])
def test_chunks(cuda_device, dtype, HQ, HK, D, page, group):
    # whole prompts, chunks at the end of a history, single tokens, a sequence without new tokens, one without any
    both(cuda_device, [1, 5, 64, 130, 300, 200, 77, 0, 257], [1, 5, 64, 130, 3, 40, 0, 0, 129], HQ, HK, D, page, group, dtype)


@pytest.mark.parametrize("window", [1, 20, 128, 300])
@pytest.mark.parametrize("D,page,group", [(64, 16, 32), (128, 64, 128)])
def test_chunks_with_a_window(cuda_device, window, D, page, group):
    both(cuda_device, [1, 64, 300, 450, 77], [1, 64, 200, 17, 77], 4, 2, D, page, group, "f16", window=window)


def test_more_new_tokens_than_the_cache_holds(cuda_device):
    """Queries ahead of the first token see nothing: rows of zeros."""
    _, (expected, _) = both(cuda_device, [3, 0, 10], [5, 4, 10], 4, 2, 64, 16, 32, "bf16")
    out = expected[0]
    assert not out[:2].any() and not out[5:9].any() and out[2].any()


@pytest.mark.parametrize("scale", [0.01, 1.0, 3.0])
def test_scale(cuda_device, scale):
    both(cuda_device, [300, 40], [1, 1], 4, 2, 64, 16, 64, "f16", scale=scale)


@pytest.mark.parametrize("single", [True, False])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_long_sequences_are_shared(cuda_device, single, dtype):
    """One sequence over all multiprocessors, beside very short ones."""
    both(cuda_device, [20011, 3, 1, 5000], [1] * 4 if single else [9, 1, 1, 30], 4, 1, 128, 64, 64, dtype)


def test_many_sequences(cuda_device):
    g = torch.Generator().manual_seed(1)
    lengths = torch.randint(0, 90, (300,), generator=g).tolist()
    both(cuda_device, lengths, [1] * 300, 4, 2, 64, 16, 32, "f16")
    counts = [min(n, 1 + i % 5) for i, n in enumerate(lengths)]
    both(cuda_device, lengths, counts, 4, 2, 64, 16, 64, "bf16")


@pytest.mark.parametrize("batch", [37, 75, 150])
@pytest.mark.parametrize("single", [True, False])
@pytest.mark.parametrize("D", [64, 128])
def test_tiles_of_few_steps(cuda_device, batch, single, D):
    """Shares of the multiprocessors that begin and end anywhere in tiles of one to three steps, and between tiles."""
    g = torch.Generator().manual_seed(batch)
    counts = [1] * batch if single else torch.randint(9, 40, (batch,), generator=g).tolist()
    lengths = [n + int(torch.randint(0, 1500 if single else 300, (1,), generator=g)) for n in counts]
    both(cuda_device, lengths, counts, 4, 2, D, 32, 64, "bf16", seed=batch)


def test_few_and_many_rows_in_one_call(cuda_device):
    """Sequences on both sides of the choice between the kernels, with empty ones between them."""
    counts = [1, 4, 5, 0, 17, 64, 65, 1, 2, 130, 3, 0]
    lengths = [200, 4, 90, 60, 17, 300, 65, 1, 129, 140, 40, 0]
    both(cuda_device, lengths, counts, 8, 2, 128, 16, 64, "bf16")
    both(cuda_device, lengths, counts, 7, 1, 64, 32, 32, "f16", window=50)


def test_heads_that_no_tile_holds(cuda_device):
    """More query heads per key head than half a tile has rows."""
    both(cuda_device, [40, 70], [9, 30], 130, 1, 64, 16, 64, "bf16")


@pytest.mark.parametrize("single", [True, False])
@pytest.mark.parametrize("page", [16, 32, 64])
def test_pages_outside_the_cache_are_not_seen(cuda_device, single, page):
    lengths, counts = [400, 700], [1, 1] if single else [30, 2]
    data = make(lengths, counts, 4, 2, 128, page, 64, "bf16", spare=0)
    table = data[2]
    table[0, 2], table[1, 0], table[1, 3] = -5, data[1][0].shape[0], 1 << 30
    expected = [reference(data, 64)] + ([] if single else [of_rounded(data, 64)])
    program = ib.programs.paged_decode_attention_int4 if single else ib.programs.paged_attention_int4
    assert_close(run(ib.compile(program), cuda_device, data, single), *expected)


@pytest.mark.parametrize("single", [True, False])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_groups_that_are_no_numbers_reach_only_the_rows_that_see_them(cuda_device, single, dtype):
    data = make([64, 80, 70], [1, 1, 1] if single else [40, 8, 40], 4, 2, 64, 16, 32, dtype)
    q, (k_codes, k_scales, v_codes, v_scales), table, offsets, n = data
    for b, token, part, at in ((0, 50, v_scales, 2), (1, 76, v_scales, 1), (2, 60, k_scales, 0)):
        part[int(table[b, token // 16]), 1, token % 16, at:at + 1] = math.nan if part is k_scales or at == 2 else math.inf
    program = ib.programs.paged_decode_attention_int4 if single else ib.programs.paged_attention_int4
    out = run(ib.compile(program, constexprs={"ACT_DTYPE": dtype, "GROUP_SIZE": 32}), cuda_device, data, single).cpu()
    expected, _ = reference(data, 32)
    fine = expected.isfinite()
    assert 0 < int((~fine).sum()) < fine.numel() / 2
    assert torch.equal(out.isfinite(), fine)
    q, _, *rest = data
    clean = make([64, 80, 70], [1, 1, 1] if single else [40, 8, 40], 4, 2, 64, 16, 32, dtype)
    bounds = [reference(clean, 32), of_rounded(clean, 32)]
    seen = torch.stack([((out.double() - e).abs() <= b) for e, b in bounds]).any(0)
    assert (seen | ~fine).all()


def test_scales_of_nothing_and_of_much(cuda_device):
    """Groups whose elements are all one number, small numbers, and values of 10^9 beside them (bf16)."""
    data = make([200, 50], [1, 1], 4, 2, 64, 16, 32, "bf16")
    q, cache, table, offsets, n = data
    for codes, scales in (cache[:2], cache[2:]):
        scales[:, :, ::3, 0] *= 0
        codes[:, :, ::3, :16] = 0
    cache[1][:, :, 1::3] *= 1e-6
    cache[3][:, 0] *= 1e-12
    cache[3][:, 1] *= 1e9
    artifact = ib.compile(ib.programs.paged_decode_attention_int4, constexprs={"GROUP_SIZE": 32})
    assert_close(run(artifact, cuda_device, data, True), reference(data, 32))


@pytest.mark.parametrize("single", [True, False])
@pytest.mark.parametrize("power", [-30, 40])
def test_powers_of_two(cuda_device, single, power):
    """Values 2^power times as large give a result as many times as large; keys so many times as large and queries as many times as
    small the same one.  All roundings are alike; what is too small for f32 is a product's 2^-57 at most (of values at 2^-30: 200
    tokens' 2^-27 each, below 2^-19)."""
    data = make([200, 50], [1, 1] if single else [3, 2], 4, 2, 64, 16, 32, "bf16")
    q, cache, table, offsets, n = data
    artifact = ib.compile(ib.programs.paged_decode_attention_int4 if single else ib.programs.paged_attention_int4,
                          constexprs={"GROUP_SIZE": 32})
    expected = run(artifact, cuda_device, data, single).cpu().double()
    by = 2.0 ** power
    values = run(artifact, cuda_device, (q, [*cache[:3], cache[3] * by], table, offsets, n), single).cpu().double() / by
    keys = run(artifact, cuda_device, (q / by, [cache[0], cache[1] * by, *cache[2:]], table, offsets, n), single).cpu().double()
    for actual in (values, keys):
        assert ((actual - expected).abs() <= 2.0 ** -7 * expected.abs() + 2.0 ** -19).all()


def test_f16_values_of_every_size(cuda_device):
    """Scales from the smallest f16 to thousands: weights times scales do not run out of range."""
    data = make([300, 120, 40], [1, 1, 1], 4, 1, 128, 32, 64, "f16")
    q, cache, table, offsets, n = data
    for b, factor in enumerate((1e-6, 4000.0, 30.0)):
        for page in table[b].tolist():
            if page >= 0:
                cache[3][page] *= factor
    out = run(ib.compile(ib.programs.paged_decode_attention_int4, constexprs={"ACT_DTYPE": "f16"}), cuda_device, data, True)
    assert_close(out, reference(data, 64))


def test_strided_queries(cuda_device):
    data = make([70, 200], [7, 1], 6, 2, 64, 16, 64, "bf16")
    q, cache, table, offsets, n = data
    expected = [reference(data, 64), of_rounded(data, 64)]
    wide = torch.full((8, 10, 72), math.nan, dtype=torch.bfloat16, device=cuda_device)
    wide[:, 2:8, :64] = q.to(cuda_device)
    artifact = ib.compile(ib.programs.paged_attention_int4)
    rest = [t.to(cuda_device) for t in (*cache, table, offsets, n)]
    for _ in range(2):
        assert_close(artifact.run(wide[:, 2:8, :64], *rest), *expected)
    turned = q.to(cuda_device).transpose(0, 1).contiguous().transpose(0, 1)     # heads ahead of tokens
    assert_close(artifact.run(turned, *rest), *expected)


@pytest.mark.parametrize("single", [True, False])
def test_lengths_and_offsets_beyond_what_there_is(cuda_device, single):
    """A length that the table cannot name counts as what it can name; rows that no sequence has are left alone."""
    data = make([48, 33], [1, 1] if single else [3, 20], 2, 1, 64, 16, 64, "f16")
    q, cache, table, offsets, n = data
    table[1, 2:] = -1
    program = ib.programs.paged_decode_attention_int4 if single else ib.programs.paged_attention_int4
    artifact = ib.compile(program, constexprs={"ACT_DTYPE": "f16"})
    expected = [reference(data, 64), of_rounded(data, 64)]
    for length in (49, (1 << 31) - 1):
        n[0] = length
        assert_close(run(artifact, cuda_device, data, single), *expected)
    if not single:
        out = torch.full((23, 2, 64), 7.0, dtype=torch.float16, device=cuda_device)
        artifact.launch(*(t.to(cuda_device) for t in (q, *cache, table, torch.tensor([-9, 3, 3], dtype=torch.int32), n)), out)
        assert (out[3:] == 7).all() and (out[:3] != 7).all()


def test_nothing_to_see_or_to_do(cuda_device):
    artifact = ib.compile(ib.programs.paged_decode_attention_int4)
    q = torch.randn((2, 4, 64), device=cuda_device).bfloat16()
    n = torch.tensor([5, 0], dtype=torch.int32, device=cuda_device)

    def cache(pages):
        return [torch.zeros((pages, 2, 16, 32), dtype=torch.uint8, device=cuda_device) if i % 2 == 0 else
                torch.full((pages, 2, 16, 2), math.nan, dtype=torch.bfloat16, device=cuda_device) for i in range(4)]

    assert not artifact.run(q, *cache(0), torch.zeros((2, 1), dtype=torch.int32, device=cuda_device), n).any()
    assert not artifact.run(q, *cache(1), torch.full((2, 1), -1, dtype=torch.int32, device=cuda_device), n).any()
    assert artifact.run(q[:0], *cache(1), torch.zeros((0, 1), dtype=torch.int32, device=cuda_device), n[:0]).shape == (0, 4, 64)


@pytest.mark.parametrize("single", [True, False])
def test_a_cache_of_more_than_32_bits(cuda_device, single):
    """Pages whose bytes lie past 2^32."""
    HK, page, D, group = 8, 256, 128, 64
    pages = (1 << 32) // (HK * page * D // 2) + 2
    data = make([300], [1] if single else [40], 16, HK, D, page, group, "bf16", spare=0)
    expected = [reference(data, group), of_rounded(data, group)]
    q, cache, table, offsets, n = data
    large = [torch.empty((pages, *c.shape[1:]), dtype=c.dtype, device=cuda_device) for c in cache]
    for whole, part in zip(large, cache):
        whole[-2:] = part.to(cuda_device)
    program = ib.programs.paged_decode_attention_int4 if single else ib.programs.paged_attention_int4
    assert_close(run(ib.compile(program), cuda_device, (q, large, table + pages - 2, offsets, n), single), *expected)


@pytest.mark.parametrize("single", [True, False])
def test_same_bits_streams_and_graphs(cuda_device, single):
    data = make([3000, 100, 700], [1, 1, 1] if single else [300, 1, 50], 8, 2, 128, 32, 64, "bf16")
    q, cache, table, offsets, n = data
    artifact = ib.compile(ib.programs.paged_decode_attention_int4 if single else ib.programs.paged_attention_int4)
    arguments = [t.to(cuda_device) for t in (q, *cache, table, *(() if single else (offsets,)), n)]
    expected = artifact.run(*arguments)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    outs = []
    for stream in streams * 3:
        with torch.cuda.stream(stream):
            outs.append(artifact.run(*arguments))
    torch.cuda.synchronize()
    assert all(torch.equal(o, expected) for o in outs)
    call = artifact.prepare(*arguments)
    call.launch()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call.launch()
        call.launch()
    call.result().zero_()
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(call.result(), expected)
    call.check()
    assert artifact.observation.kernel and "int4" in artifact.observation.kernel


def test_as_torch_op(cuda_device):
    data = make([90, 20], [1, 1], 4, 2, 64, 16, 64, "bf16")
    op = ib.compile(ib.programs.paged_decode_attention_int4).as_torch_op("intent_b200_test::paged_decode_int4")
    q, cache, table, _, n = data
    assert_close(op(*(t.to(cuda_device) for t in (q, *cache, table, n))), reference(data, 64))


def test_a_status_word_raises(cuda_device):
    """What a bounded wait that gave up leaves in the workspace is reported by ``check`` and cleared."""
    q, cache, table, _, n = make([40], [1], 4, 2, 64, 16, 64, "bf16")
    call = ib.compile(ib.programs.paged_decode_attention_int4).prepare(*(t.to(cuda_device) for t in (q, *cache, table, n)))
    call.launch()
    call.check()
    call._workspace[0][:4].view(torch.int32)[0] = 4
    with pytest.raises(ib.CompilationStageError):
        call.check()
    call.check()


def test_refusals(cuda_device):
    q, cache, table, offsets, n = make([40, 9], [2, 1], 4, 2, 128, 16, 64, "bf16")
    q, table, offsets, n, *cache = (t.to(cuda_device) for t in (q, table, offsets, n, *cache))
    artifact = ib.compile(ib.programs.paged_attention_int4)
    artifact.run(q, *cache, table, offsets, n)
    with pytest.raises(TypeError):                     # a cache of 16-bit elements
        artifact.run(q, *(torch.zeros((5, 2, 16, 128), dtype=torch.bfloat16, device=cuda_device) for _ in range(4)), table, offsets, n)
    with pytest.raises(TypeError):
        artifact.run(q, cache[0], cache[1].half(), *cache[2:], table, offsets, n)
    with pytest.raises(ValueError):                    # groups of another size
        ib.compile(ib.programs.paged_attention_int4, constexprs={"GROUP_SIZE": 32}).run(q, *cache, table, offsets, n)
    with pytest.raises(ValueError):
        artifact.run(q, *cache[:3], cache[3][:-1], table, offsets, n)
    with pytest.raises(ValueError):
        artifact.run(q[:, :3].contiguous(), *cache, table, offsets, n)
    with pytest.raises(ValueError):
        artifact.run(q[..., :64].contiguous(), *cache, table, offsets, n)
    with pytest.raises(ValueError):
        artifact.run(q, *cache, table, offsets[:-1], n)
    with pytest.raises(ValueError):                    # one token per sequence
        ib.compile(ib.programs.paged_decode_attention_int4).run(q, *cache, table, n)
    with pytest.raises(ValueError):                    # a group wider than a head
        ib.compile(ib.programs.paged_attention_int4, constexprs={"GROUP_SIZE": 128}).run(
            q[..., :64].contiguous(), *(c[..., :c.shape[-1] // 2].contiguous() for c in cache), table, offsets, n)
