"""Corner cases of attention over pages on each of its kernels."""
import math

import pytest
import torch

import intent_b200 as ib
from intent_b200.runtime import native
from oracle import attention as oracle
from test_paged_attention_gpu import HALF_UNIT, assert_close, make, run

pytestmark = pytest.mark.gpu

ROWS, CHUNK = "paged_rows_kernel", "paged_chunk_kernel"


def attend(device, data, dtype="bf16", single=False, kernel=None, **constants):
    artifact = ib.compile(ib.programs.paged_decode_attention if single else ib.programs.paged_attention,
                          constexprs={"ACT_DTYPE": dtype, **constants})
    out = run(artifact, device, *data, single)
    artifact.check()
    if kernel:
        assert artifact.observation.kernel.startswith(kernel)
    return out.cpu()


def assert_numbers(out, expected, weight, dtype):
    """The same rows are no numbers, the others are close."""
    assert torch.equal(out.isnan(), expected.isnan())
    fine = ~expected.isnan()
    bound = (HALF_UNIT[dtype] + 2e-4) * weight + HALF_UNIT[dtype] * expected.abs() + 2.0 ** -24
    assert ((out.double() - expected).abs() <= bound)[fine].all()


@pytest.mark.parametrize("window", [0, 24])
@pytest.mark.parametrize("lengths,counts,kernel", [
    ([40, 9000, 300, 0], [1, 1, 1, 1], ROWS), ([40, 5000, 300, 0], [3, 2, 1, 2], ROWS), ([40, 3000, 300, 0], [40, 200, 130, 3], CHUNK)])
def test_rows_whose_scores_are_all_minus_infinity(cuda_device, lengths, counts, kernel, window):
    """Their softmax is no number; only a row without a token is zero.  (The second sequence is shared by many CTAs.)"""
    q, k, v, table, offsets, n = make(lengths, counts, 4, 2, 64, 16, "bf16", poison=False)
    q[:] = q.abs() + 0.1
    for b, tokens in ((0, range(30)), (1, range(lengths[1])), (2, range(280, 300))):
        for t in tokens:
            k[int(table[b, t // 16]), 1, t % 16] = -math.inf
    table[0, 0] = -1
    expected, weight = oracle.paged_attention(q, k, v, table, offsets, n, window=window)
    nan = expected.isnan().all(-1)
    assert torch.equal(nan, expected.isnan().any(-1)) and nan[offsets[1]:offsets[2], 2:].all()
    single = all(c == 1 for c in counts)
    assert_numbers(attend(cuda_device, (q, k, v, table, offsets, n), kernel=kernel, WINDOW=window), expected, weight, "bf16")
    if single:
        assert_numbers(attend(cuda_device, (q, k, v, table, offsets, n), single=True, kernel=kernel, WINDOW=window), expected,
                       weight, "bf16")


def lengths_of(counts, seed, most=150):
    g = torch.Generator().manual_seed(seed)
    return [n + int(torch.randint(0, most, (1,), generator=g)) if n else 0 for n in counts]


@pytest.mark.parametrize("counts,HQ,HK,D,launches", [
    ([150] + [1] * 59, 8, 2, 128, 3),                              # in tiles of sixteen rows, and the chunk by itself
    ([1] * 50 + [90] + [1] * 49, 8, 2, 128, 3),                    # in tiles of eight
    ([8, 9, 70, 0, 1, 3, 33] + [1] * 80, 8, 2, 64, 3),             # sequences of up to four tiles, more than that, none
    ([300] + [1] * 40, 16, 1, 64, 3),
    ([31] + [1] * 30, 4, 4, 64, 2),                                # so few that one kernel takes all
    ([60] + [1] * 30, 4, 4, 64, 3),
    ([3] * 12, 4, 4, 128, 2),
    ([1] * 70, 32, 1, 64, 2),
    ([0] * 90 + [75] + [0] * 9, 8, 2, 64, 3),                      # (a step of a fixed number of places, most of them empty)
])
def test_a_chunk_beside_many_single_tokens(cuda_device, counts, HQ, HK, D, launches):
    """What takes a sequence goes by its own new tokens, whatever the others have on average, where its history may be long: that
    is what the page table has room for."""
    data = make(lengths_of(counts, len(counts)), counts, HQ, HK, D, 16, "bf16")
    expected, weight = oracle.paged_attention(*data)
    table = torch.cat([data[3], torch.full((len(counts), 2048), -1, dtype=torch.int32)], 1)
    data = (*data[:3], table, *data[4:])
    artifact = ib.compile(ib.programs.paged_attention)
    assert_close(run(artifact, cuda_device, *data, False), expected, weight, "bf16")
    before = native.launch_count()
    assert_close(run(artifact, cuda_device, *data, False), expected, weight, "bf16")
    assert native.launch_count() - before == launches
    artifact.check()


def test_chunks_of_short_histories(cuda_device):
    """One kernel takes a call whose page table has room for little, or whose window leaves little of it."""
    counts = [150] + [1] * 59
    q, k, v, table, offsets, n = make(lengths_of(counts, 3), counts, 8, 2, 128, 16, "bf16")
    wide = torch.cat([table, torch.full((60, 2048), -1, dtype=torch.int32)], 1)
    for pages, window, launches in ((table, 0, 2), (wide, 0, 3), (wide, 100, 2)):
        expected, weight = oracle.paged_attention(q, k, v, table, offsets, n, window=window)
        before = native.launch_count()
        out = attend(cuda_device, (q, k, v, pages, offsets, n), kernel=ROWS, WINDOW=window)
        assert native.launch_count() - before == launches
        assert_close(out, expected, weight, "bf16")


def test_heads_too_many_for_the_rows_kernel(cuda_device):
    """With more query heads per key head than it takes rows of a sequence, a call launches the chunk kernel alone."""
    counts = [50] + [1] * 9
    data = make(lengths_of(counts, 1), counts, 40, 1, 128, 16, "bf16")
    expected, weight = oracle.paged_attention(*data)
    assert_close(attend(cuda_device, data, kernel=CHUNK), expected, weight, "bf16")


def test_queries_that_are_no_numbers_stay_among_themselves(cuda_device):
    """Rows of a tile that belong to the next sequence, or to none, do not reach the tile's own."""
    counts, lengths = [40, 70, 3], [200, 300, 90]
    q, k, v, table, offsets, n = make(lengths, counts, 10, 2, 64, 16, "bf16")
    q[40:110] = math.nan
    expected, weight = oracle.paged_attention(q, k, v, table, offsets, n)
    out = attend(cuda_device, (q, k, v, table, offsets, n), kernel=CHUNK)
    assert expected[40:110].isnan().all() and not expected[:40].isnan().any()
    assert_numbers(out, expected, weight, "bf16")


@pytest.mark.parametrize("D,HQ", [(64, 6), (128, 14)])
def test_strided_queries_of_chunks(cuda_device, D, HQ):
    counts, lengths = [70, 200], [90, 200]
    q, k, v, table, offsets, n = make(lengths, counts, HQ, 2, D, 16, "bf16")
    expected, weight = oracle.paged_attention(q, k, v, table, offsets, n)
    wide = torch.full((270, HQ + 4, D + 8), math.nan, dtype=torch.bfloat16, device=cuda_device)
    wide[:, 3:3 + HQ, :D] = q.to(cuda_device)
    turned = q.to(cuda_device).transpose(0, 1).contiguous().transpose(0, 1)     # heads ahead of tokens
    artifact = ib.compile(ib.programs.paged_attention)
    rest = [t.to(cuda_device) for t in (k, v, table, offsets, n)]
    for view in (wide[:, 3:3 + HQ, :D], turned):
        assert not view.is_contiguous()
        for _ in range(2):
            assert_close(artifact.run(view, *rest), expected, weight, "bf16")
        assert artifact.observation.kernel.startswith(CHUNK)
    artifact.check()


@pytest.mark.parametrize("scale", [0.01, 1.0, 3.0])
def test_scales_of_chunks(cuda_device, scale):
    data = make([300, 140], [200, 90], 4, 2, 64, 16, "f16")
    data = (data[0] * 0.5, *data[1:])
    expected, weight = oracle.paged_attention(*data, scale=scale)
    assert_close(attend(cuda_device, data, "f16", kernel=CHUNK, SCALE=scale), expected, weight, "f16")


def test_scores_of_both_infinities_in_chunks(cuda_device):
    """Rows ahead of the key that makes a score +inf are close, those that see it are no numbers; a key of -inf counts nothing."""
    lengths, counts = [200, 240], [100, 150]
    q, k, v, table, offsets, n = make(lengths, counts, 4, 2, 64, 16, "f16", poison=False)
    q[:] = q.abs() + 0.1
    for b, t, value in ((0, 19, -math.inf), (0, 150, -math.inf), (1, 130, math.inf)):
        k[int(table[b, t // 16]), 1, t % 16] = value
    expected, weight = oracle.paged_attention(q, k, v, table, offsets, n)
    out = attend(cuda_device, (q, k, v, table, offsets, n), "f16", kernel=CHUNK)
    assert expected[100 + 40:, 2:].isnan().all() and not expected[:100 + 40].isnan().any()
    assert_numbers(out, expected, weight, "f16")


def test_lengths_of_chunks_beyond_the_table(cuda_device):
    """A length that the table cannot name counts as what it can name."""
    data = make([144], [100], 2, 1, 64, 16, "f16")
    expected, weight = oracle.paged_attention(*data)
    for length in (145, (1 << 31) - 1):
        longer = (*data[:5], torch.tensor([length], dtype=torch.int32))
        assert_close(attend(cuda_device, longer, "f16", kernel=CHUNK), expected, weight, "f16")


def test_offsets_of_chunks_beyond_the_queries(cuda_device):
    """Offsets are cut to the rows there are; rows that no sequence has are left alone."""
    data = make([148, 90], [80, 60], 2, 1, 64, 16, "f16")
    expected, weight = oracle.paged_attention(*data)
    artifact = ib.compile(ib.programs.paged_attention, constexprs={"ACT_DTYPE": "f16"})
    moved = [t.to(cuda_device) for t in data]
    out = torch.full((140, 2, 64), 7.0, dtype=torch.float16, device=cuda_device)
    for offsets, rows in (([0, 80, 1 << 30], 140), ([-9, 80, 80], 80)):
        out.fill_(7.0)
        artifact.launch(*moved[:4], torch.tensor(offsets, dtype=torch.int32, device=cuda_device), moved[5], out)
        assert_close(out[:rows], expected[:rows], weight[:rows], "f16")
        assert (out[rows:] == 7).all() and artifact.observation.kernel.startswith(CHUNK)


@pytest.mark.parametrize("window", [0, 1, 20, 128])
@pytest.mark.parametrize("D", [64, 128])
def test_chunks_of_more_tokens_than_the_cache_holds(cuda_device, window, D):
    """Queries ahead of the first token see nothing: rows of zeros, also where whole tiles are ahead of it."""
    counts, lengths = [150, 700, 60, 300], [30, 40, 0, 300]
    data = make(lengths, counts, 4, 2, D, 16, "bf16")
    expected, weight = oracle.paged_attention(*data, window=window)
    assert not expected[:120].any() and not expected[150:810].any() and expected[:150].any()
    assert_close(attend(cuda_device, data, kernel=CHUNK, WINDOW=window), expected, weight, "bf16")


@pytest.mark.parametrize("HQ,HK", [(28, 4), (40, 8), (9, 3), (64, 1), (128, 1)])
@pytest.mark.parametrize("window", [0, 70])
def test_groups_of_chunks(cuda_device, HQ, HK, window):
    """Tiles that hold 2 x floor(128 / group) tokens, from 1 to 128 of them."""
    data = make([210, 150], [60, 130], HQ, HK, 64, 32, "bf16")
    expected, weight = oracle.paged_attention(*data, window=window)
    assert_close(attend(cuda_device, data, kernel=CHUNK, WINDOW=window), expected, weight, "bf16")


def test_chunks_as_torch_op(cuda_device):
    data = make([90, 220], [60, 150], 4, 2, 64, 16, "bf16")
    expected, weight = oracle.paged_attention(*data)
    op = ib.compile(ib.programs.paged_attention).as_torch_op("intent_b200_test::paged_chunks")
    assert_close(op(*(t.to(cuda_device) for t in data)), expected, weight, "bf16")
