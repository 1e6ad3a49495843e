"""Attention over pages near the limits of what a call may ask for."""
import pytest
import torch

import intent_b200 as ib
from oracle import attention as oracle
from test_paged_attention_gpu import assert_close

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D", [64, 128])
def test_more_than_two_to_the_thirtieth_steps(cuda_device, D):
    """Sequences of 2^30 tokens, all of them in pages that are not there but for the first and the last page."""
    B, HQ, HK, page = (40 if D == 64 else 20), 16, 8, 256           # a step of the kernel is 256 or 128 tokens
    width, length = (1 << 30) // page, (1 << 30) - 5
    g = torch.Generator().manual_seed(D)
    k, v = (torch.randn((2 * B, HK, page, D), generator=g).bfloat16() for _ in range(2))
    q = torch.randn((B, HQ, D), generator=g).bfloat16()
    ends = torch.randperm(2 * B, generator=g).to(torch.int32).view(B, 2)
    table = torch.full((B, width), -1, dtype=torch.int32, device=cuda_device)
    table[:, 0], table[:, -1] = ends[:, 0].to(cuda_device), ends[:, 1].to(cuda_device)
    expected, weight = oracle.paged_attention(q, k, v, ends, torch.arange(B + 1), torch.full((B,), 2 * page - 5))
    artifact = ib.compile(ib.programs.paged_decode_attention)
    lengths = torch.full((B,), length, dtype=torch.int32, device=cuda_device)
    out = artifact.run(*(t.to(cuda_device) for t in (q, k, v)), table, lengths)
    assert_close(out, expected, weight, "bf16")
    artifact.check()
