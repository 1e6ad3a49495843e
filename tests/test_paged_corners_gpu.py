"""Corner cases of attention over pages on each of its kernels."""
import math

import pytest
import torch

import intent_b200 as ib
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
