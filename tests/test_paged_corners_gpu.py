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
    ([60] + [1] * 30, 4, 4, 64, 2),                                # so few that one kernel takes all
    ([4] * 12, 4, 2, 128, 2),
    ([1] * 70, 32, 1, 64, 2),
    ([0] * 90 + [75] + [0] * 9, 8, 2, 64, 3),                      # (a step of a fixed number of places, most of them empty)
])
def test_a_chunk_beside_many_single_tokens(cuda_device, counts, HQ, HK, D, launches):
    """What takes a sequence goes by its own new tokens, whatever the others have on average."""
    data = make(lengths_of(counts, len(counts)), counts, HQ, HK, D, 16, "bf16")
    expected, weight = oracle.paged_attention(*data)
    artifact = ib.compile(ib.programs.paged_attention)
    assert_close(run(artifact, cuda_device, *data, False), expected, weight, "bf16")
    before = native.launch_count()
    assert_close(run(artifact, cuda_device, *data, False), expected, weight, "bf16")
    assert native.launch_count() - before == launches
    artifact.check()


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
