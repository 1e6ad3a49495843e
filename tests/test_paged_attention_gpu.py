"""paged_attention and paged_decode_attention against the definition in 64 bits."""
import math

import pytest
import torch

import intent_b200 as ib
from oracle import attention as oracle

pytestmark = pytest.mark.gpu

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
HALF_UNIT = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8}


def make(lengths, counts, HQ, HK, D, page, dtype, seed=0, poison=True, spare=2):
    """Queries and a cache in which every place that no sequence uses holds NaN."""
    g = torch.Generator().manual_seed(seed)
    used = [-(-n // page) for n in lengths]
    pages, width = sum(used) + spare, max(max(used), 1)
    shape = (pages, HK, page, D)
    k, v = (torch.full(shape, math.nan if poison else 0.0, dtype=DTYPES[dtype]) for _ in range(2))
    order = torch.randperm(pages, generator=g).to(torch.int32)
    table = torch.full((len(lengths), width), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(lengths):
        table[b, :used[b]] = order[at:at + used[b]]
        at += used[b]
        for i in range(used[b]):
            rows = min(page, n - i * page)
            for cache in (k, v):
                cache[int(table[b, i]), :, :rows] = torch.randn((HK, rows, D), generator=g).to(DTYPES[dtype])
    offsets = torch.tensor([0] + counts).cumsum(0).to(torch.int32)
    q = torch.randn((sum(counts), HQ, D), generator=g).to(DTYPES[dtype])
    return q, k, v, table, offsets, torch.tensor(lengths, dtype=torch.int32)


def assert_close(actual, expected, weight, dtype):
    """A weight is rounded to the type for the product with V (relative to its row's largest: half a unit of all that is added
    up), scores and sums are in f32 (2e-4: 128 products of normal numbers, the exponential, thousands of additions), and the
    result is rounded once."""
    actual = actual.cpu().double()
    assert not actual.isnan().any()
    bound = (HALF_UNIT[dtype] + 2e-4) * weight + HALF_UNIT[dtype] * expected.abs() + 2.0 ** -24
    excess = (actual - expected).abs() - bound
    assert excess.numel() == 0 or excess.max() <= 0, float(excess.max())


def run(artifact, device, q, k, v, table, offsets, lengths, single):
    moved = [t.to(device) for t in (q, k, v, table)]
    return artifact.run(*moved, *([] if single else [offsets.to(device)]), lengths.to(device))


def both(device, lengths, counts, HQ, HK, D, page, dtype, window=0, scale=None, seed=0):
    data = make(lengths, counts, HQ, HK, D, page, dtype, seed)
    expected, weight = oracle.paged_attention(*data, scale=scale, window=window)
    constants = {"ACT_DTYPE": dtype, "WINDOW": window, "SCALE": scale}
    programs = [(ib.programs.paged_attention, False)]
    if all(c == 1 for c in counts):
        programs.append((ib.programs.paged_decode_attention, True))
    for program, single in programs:
        artifact = ib.compile(program, constexprs=constants)
        for _ in range(2):
            assert_close(run(artifact, device, *data, single), expected, weight, dtype)
        artifact.check()
    return data, expected, weight


LENGTHS = [1, 2, 15, 16, 17, 31, 33, 64, 100, 127, 128, 129, 200, 255, 257, 0, 400]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("HQ,HK,D,page", [(8, 2, 128, 64), (4, 4, 64, 16), (5, 1, 128, 32), (12, 1, 64, 128), (40, 2, 128, 256),
                                          (16, 1, 128, 16)])
def test_single_tokens(cuda_device, dtype, HQ, HK, D, page):
    both(cuda_device, LENGTHS, [1] * len(LENGTHS), HQ, HK, D, page, dtype)


@pytest.mark.parametrize("window", [1, 16, 100, 128, 1000])
@pytest.mark.parametrize("D,page", [(64, 32), (128, 16)])
def test_single_tokens_with_a_window(cuda_device, window, D, page):
    both(cuda_device, LENGTHS, [1] * len(LENGTHS), 4, 2, D, page, "bf16", window=window)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("HQ,HK,D,page", [(8, 2, 128, 64), (4, 4, 64, 16), (7, 1, 64, 32), (3, 1, 128, 256), (24, 1, 128, 16)])
def test_chunks(cuda_device, dtype, HQ, HK, D, page):
    # whole prompts, chunks at the end of a history, single tokens, a sequence without new tokens, one without any
    both(cuda_device, [1, 5, 64, 130, 300, 200, 77, 0, 257], [1, 5, 64, 130, 3, 40, 0, 0, 129], HQ, HK, D, page, dtype)


@pytest.mark.parametrize("window", [1, 20, 128, 300])
@pytest.mark.parametrize("D,page", [(64, 16), (128, 64)])
def test_chunks_with_a_window(cuda_device, window, D, page):
    both(cuda_device, [1, 64, 300, 450, 77], [1, 64, 200, 17, 77], 4, 2, D, page, "f16", window=window)


def test_more_new_tokens_than_the_cache_holds(cuda_device):
    """Queries ahead of the first token see nothing: rows of zeros."""
    data, expected, _ = both(cuda_device, [3, 0, 10], [5, 4, 10], 4, 2, 64, 16, "bf16")
    assert not expected[:2].any() and not expected[5:9].any() and expected[2].any()


@pytest.mark.parametrize("scale", [0.01, 1.0, 3.0])
def test_scale(cuda_device, scale):
    lengths = [300, 40]
    data = make(lengths, [20, 1], 4, 2, 64, 16, "f16")
    data = (data[0] * 0.5, *data[1:])
    expected, weight = oracle.paged_attention(*data, scale=scale)
    artifact = ib.compile(ib.programs.paged_attention, constexprs={"ACT_DTYPE": "f16", "SCALE": scale})
    assert_close(run(artifact, cuda_device, *data, False), expected, weight, "f16")


@pytest.mark.parametrize("single", [True, False])
def test_long_sequences_are_shared(cuda_device, single):
    """One sequence over all multiprocessors, beside very short ones."""
    lengths = [20011, 3, 1, 5000]
    counts = [1] * 4 if single else [9, 1, 1, 30]
    both(cuda_device, lengths, counts, 4, 1, 128, 64, "bf16")


def test_many_sequences(cuda_device):
    g = torch.Generator().manual_seed(1)
    lengths = torch.randint(0, 90, (300,), generator=g).tolist()
    both(cuda_device, lengths, [1] * 300, 4, 2, 64, 16, "f16")
    counts = [min(n, 1 + i % 5) for i, n in enumerate(lengths)]
    both(cuda_device, lengths, counts, 4, 2, 64, 16, "bf16")


@pytest.mark.parametrize("single", [True, False])
def test_pages_outside_the_cache_are_not_seen(cuda_device, single):
    lengths, counts = [100, 300], [1, 1] if single else [30, 2]
    q, k, v, table, offsets, n = make(lengths, counts, 4, 2, 128, 16, "bf16", spare=0)
    table[0, 2], table[1, 0], table[1, 18] = -5, k.shape[0], 1 << 30
    expected, weight = oracle.paged_attention(q, k, v, table, offsets, n)
    program = ib.programs.paged_decode_attention if single else ib.programs.paged_attention
    assert_close(run(ib.compile(program), cuda_device, q, k, v, table, offsets, n, single), expected, weight, "bf16")


@pytest.mark.parametrize("single", [True, False])
def test_scores_of_both_infinities(cuda_device, single):
    """A key of -inf takes its token out of a row, as its weight is zero; one that makes a score +inf gives NaN, and only to
    the rows that see it."""
    q, k, v, table, offsets, n = make([40, 40], [1, 1] if single else [4, 2], 2, 1, 64, 16, "f16", poison=False)
    q[:] = q.abs() + 0.1
    k[int(table[0, 1]), 0, 3] = -math.inf
    k[int(table[1, 0]), 0, 0] = math.inf
    expected, weight = oracle.paged_attention(q, k, v, table, offsets, n)
    program = ib.programs.paged_decode_attention if single else ib.programs.paged_attention
    out = run(ib.compile(program, constexprs={"ACT_DTYPE": "f16"}), cuda_device, q, k, v, table, offsets, n, single)
    first = int(offsets[1])
    assert_close(out[:first], expected[:first], weight[:first], "f16")
    assert out[first:].isnan().all() and expected[first:].isnan().all()


def test_values_that_are_no_numbers_reach_only_the_rows_that_see_them(cuda_device):
    q, k, v, table, offsets, n = make([64, 64], [40, 8], 4, 2, 64, 16, "bf16")
    for b, (token, value) in enumerate(((50, math.nan), (60, math.inf))):
        v[int(table[b, token // 16]), 1, token % 16, 7] = value
    expected, weight = oracle.paged_attention(q, k, v, table, offsets, n)
    out = run(ib.compile(ib.programs.paged_attention), cuda_device, q, k, v, table, offsets, n, False).cpu()
    fine = expected.isfinite()
    assert 0 < int((~fine).sum()) < 200
    assert torch.equal(out.isfinite(), fine) and torch.equal(out.isnan(), expected.isnan())
    bound = (HALF_UNIT["bf16"] + 2e-4) * weight + HALF_UNIT["bf16"] * expected.abs() + 2.0 ** -24
    assert ((out.double() - expected).abs() <= bound)[fine].all()


def test_strided_queries(cuda_device):
    lengths, counts = [70, 200], [7, 1]
    q, k, v, table, offsets, n = make(lengths, counts, 6, 2, 64, 16, "bf16")
    expected, weight = oracle.paged_attention(q, k, v, table, offsets, n)
    wide = torch.full((8, 10, 72), math.nan, dtype=torch.bfloat16, device=cuda_device)
    wide[:, 2:8, :64] = q.to(cuda_device)
    view = wide[:, 2:8, :64]
    artifact = ib.compile(ib.programs.paged_attention)
    rest = [t.to(cuda_device) for t in (k, v, table, offsets, n)]
    for _ in range(2):
        assert_close(artifact.run(view, *rest), expected, weight, "bf16")
    turned = q.to(cuda_device).transpose(0, 1).contiguous().transpose(0, 1)     # heads ahead of tokens
    assert_close(artifact.run(turned, *rest), expected, weight, "bf16")


@pytest.mark.parametrize("single", [True, False])
def test_lengths_beyond_the_table(cuda_device, single):
    """A length that the table cannot name counts as what it can name."""
    counts = [1] if single else [3]
    q, k, v, table, offsets, n = make([48], counts, 2, 1, 64, 16, "f16")
    expected, weight = oracle.paged_attention(q, k, v, table, offsets, n)
    program = ib.programs.paged_decode_attention if single else ib.programs.paged_attention
    for length in (49, (1 << 31) - 1):
        out = run(ib.compile(program, constexprs={"ACT_DTYPE": "f16"}), cuda_device, q, k, v, table, offsets,
                  torch.tensor([length], dtype=torch.int32), single)
        assert_close(out, expected, weight, "f16")


def test_offsets_beyond_the_queries(cuda_device):
    """Offsets are cut to the rows there are; rows that no sequence has are left alone."""
    q, k, v, table, offsets, n = make([48, 30], [3, 2], 2, 1, 64, 16, "f16")
    expected, weight = oracle.paged_attention(q, k, v, table, offsets, n)
    out = torch.full((5, 2, 64), 7.0, dtype=torch.float16, device=cuda_device)
    artifact = ib.compile(ib.programs.paged_attention, constexprs={"ACT_DTYPE": "f16"})
    moved = [t.to(cuda_device) for t in (q, k, v, table)]
    artifact.launch(*moved, torch.tensor([0, 3, 1 << 30], dtype=torch.int32, device=cuda_device), n.to(cuda_device), out)
    assert_close(out, expected, weight, "f16")
    out.fill_(7.0)
    artifact.launch(*moved, torch.tensor([-9, 3, 3], dtype=torch.int32, device=cuda_device), n.to(cuda_device), out)
    assert_close(out[:3], expected[:3], weight[:3], "f16")
    assert (out[3:] == 7).all()


def test_nothing_to_see_or_to_do(cuda_device):
    artifact = ib.compile(ib.programs.paged_decode_attention)
    q = torch.randn((2, 4, 64), device=cuda_device).bfloat16()
    n = torch.tensor([5, 0], dtype=torch.int32, device=cuda_device)
    cache = torch.empty((0, 2, 16, 64), dtype=torch.bfloat16, device=cuda_device)
    assert not artifact.run(q, cache, cache.clone(), torch.zeros((2, 1), dtype=torch.int32, device=cuda_device), n).any()
    cache = torch.full((1, 2, 16, 64), math.nan, dtype=torch.bfloat16, device=cuda_device)
    assert not artifact.run(q, cache, cache.clone(), torch.full((2, 1), -1, dtype=torch.int32, device=cuda_device), n).any()
    assert artifact.run(q[:0], cache, cache.clone(), torch.zeros((0, 1), dtype=torch.int32, device=cuda_device), n[:0]).shape == (0, 4, 64)


@pytest.mark.parametrize("single", [True, False])
def test_a_cache_of_more_than_32_bits(cuda_device, single):
    """Pages whose elements lie past 2^31."""
    HK, page, D = 8, 256, 128
    pages = (1 << 31) // (HK * page * D) + 2
    counts = [1] if single else [40]
    q, k, v, table, offsets, n = make([300], counts, 16, HK, D, page, "bf16", spare=0)
    expected, weight = oracle.paged_attention(q, k, v, table, offsets, n)
    caches = [torch.empty((pages, HK, page, D), dtype=torch.bfloat16, device=cuda_device) for _ in range(2)]
    for cache, part in zip(caches, (k, v)):
        cache[-2:] = part.to(cuda_device)
    program = ib.programs.paged_decode_attention if single else ib.programs.paged_attention
    out = run(ib.compile(program), cuda_device, q, *caches, table + pages - 2, offsets, n, single)
    assert_close(out, expected, weight, "bf16")


@pytest.mark.parametrize("single", [True, False])
def test_same_bits_streams_and_graphs(cuda_device, single):
    lengths, counts = [3000, 100, 700], [1, 1, 1] if single else [300, 1, 50]
    q, k, v, table, offsets, n = (t.to(cuda_device) for t in make(lengths, counts, 8, 2, 128, 32, "bf16"))
    artifact = ib.compile(ib.programs.paged_decode_attention if single else ib.programs.paged_attention)
    arguments = (q, k, v, table, n) if single else (q, k, v, table, offsets, n)
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
    assert artifact.observation.kernel and artifact.observation.spill_bytes == 0


def test_as_torch_op(cuda_device):
    data = make([90, 20], [1, 1], 4, 2, 64, 16, "bf16")
    expected, weight = oracle.paged_attention(*data)
    op = ib.compile(ib.programs.paged_decode_attention).as_torch_op("intent_b200_test::paged_decode")
    assert_close(op(*(t.to(cuda_device) for t in (*data[:4], data[5]))), expected, weight, "bf16")


def test_refusals(cuda_device):
    q, k, v, table, offsets, n = (t.to(cuda_device) for t in make([40, 9], [2, 1], 4, 2, 64, 16, "bf16"))
    artifact = ib.compile(ib.programs.paged_attention)
    artifact.run(q, k, v, table, offsets, n)
    with pytest.raises(TypeError):
        artifact.run(q, k, v, table.long(), offsets, n)
    with pytest.raises(TypeError):
        artifact.run(q, k.half(), v, table, offsets, n)
    with pytest.raises(ValueError):
        artifact.run(q, k, v, table, offsets[:-1], n)
    with pytest.raises(ValueError):
        artifact.run(q, k, v[:-1], table, offsets, n)
    with pytest.raises(ValueError):                    # heads that do not share evenly
        artifact.run(q[:, :3].contiguous(), k, v, table, offsets, n)
    with pytest.raises(ValueError):
        artifact.run(q, *(torch.zeros((2, 2, 8, 64), dtype=torch.bfloat16, device=cuda_device) for _ in range(2)), table, offsets, n)
    with pytest.raises(ValueError):
        artifact.run(*(t[..., :32].contiguous() for t in (q, k, v)), table, offsets, n)
    with pytest.raises(NotImplementedError):
        artifact.run(q, k.transpose(1, 2).contiguous().transpose(1, 2), v, table, offsets, n)
    with pytest.raises(NotImplementedError):
        artifact.run(q.transpose(1, 2).contiguous().transpose(1, 2), k, v, table, offsets, n)
    with pytest.raises(ValueError):                    # one token per sequence
        ib.compile(ib.programs.paged_decode_attention).run(q, k, v, table, n)
    for constexprs in ({"SCALE": 0.0}, {"SCALE": -1.0}, {"WINDOW": -1}, {"WINDOW": 1.5}, {"ACT_DTYPE": "f32"}, {"CAUSAL": 1}):
        with pytest.raises(ib.CompilationStageError):
            ib.compile(ib.programs.paged_attention, constexprs=constexprs)


@pytest.mark.parametrize("single", [True, False])
def test_a_window_of_any_size(cuda_device, single):
    """One that is wider than any history is none."""
    data = make([70, 300], [1, 1] if single else [90, 40], 2, 1, 64, 16, "bf16")
    expected, weight = oracle.paged_attention(*data)
    program = ib.programs.paged_decode_attention if single else ib.programs.paged_attention
    for window in (304, 305, (1 << 31) - 1):
        assert_close(run(ib.compile(program, constexprs={"WINDOW": window}), cuda_device, *data, single), expected, weight, "bf16")


@pytest.mark.parametrize("batch", [37, 75, 150, 223])
@pytest.mark.parametrize("single", [True, False])
@pytest.mark.parametrize("D", [64, 128])
def test_tiles_of_few_steps(cuda_device, batch, single, D):
    """Shares of the multiprocessors that begin and end anywhere in tiles of one to three steps, and between tiles."""
    g = torch.Generator().manual_seed(batch)
    counts = [1] * batch if single else torch.randint(9, 40, (batch,), generator=g).tolist()
    lengths = [n + int(torch.randint(0, 600 if single else 300, (1,), generator=g)) for n in counts]
    both(cuda_device, lengths, counts, 4, 2, D, 32, "bf16", seed=batch)


def test_few_and_many_rows_in_one_call(cuda_device):
    """Sequences on both sides of the choice between the kernels, with empty ones between them."""
    counts = [1, 4, 5, 0, 17, 64, 65, 1, 2, 130, 3, 0]
    lengths = [200, 4, 90, 60, 17, 300, 65, 1, 129, 140, 40, 0]
    both(cuda_device, lengths, counts, 8, 2, 128, 16, "bf16")
    both(cuda_device, lengths, counts, 7, 1, 64, 32, "f16", window=50)


def test_values_that_are_no_numbers_beside_few_rows(cuda_device):
    """The same as above for rows that are taken sixteen at a time."""
    q, k, v, table, offsets, n = make([64, 33, 50], [2, 4, 1], 4, 2, 64, 16, "bf16")
    for b, (token, value) in enumerate(((63, math.nan), (30, math.inf))):
        v[int(table[b, token // 16]), 1, token % 16, 7] = value
    expected, weight = oracle.paged_attention(q, k, v, table, offsets, n)
    out = run(ib.compile(ib.programs.paged_attention), cuda_device, q, k, v, table, offsets, n, False).cpu()
    fine = expected.isfinite()
    assert 0 < int((~fine).sum()) < 20
    assert torch.equal(out.isfinite(), fine) and torch.equal(out.isnan(), expected.isnan())
    bound = (HALF_UNIT["bf16"] + 2e-4) * weight + HALF_UNIT["bf16"] * expected.abs() + 2.0 ** -24
    assert ((out.double() - expected).abs() <= bound)[fine].all()


def test_heads_that_no_tile_holds(cuda_device):
    """More query heads per key head than half a tile has rows."""
    both(cuda_device, [40, 70], [9, 30], 130, 1, 64, 16, "bf16")


def test_a_status_word_raises(cuda_device):
    """What a bounded wait that gave up leaves in the workspace is reported by ``check`` and cleared."""
    q, k, v, table, _, n = (t.to(cuda_device) for t in make([40], [1], 4, 2, 64, 16, "bf16"))
    call = ib.compile(ib.programs.paged_decode_attention).prepare(q, k, v, table, n)
    call.launch()
    call.check()
    call._workspace[0][:4].view(torch.int32)[0] = 4
    with pytest.raises(ib.CompilationStageError):
        call.check()
    call.check()
