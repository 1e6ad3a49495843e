"""Attention over a cache in 4 bits where sums of queries, minima or scales are large, or a history is long."""
import math

import pytest
import torch

import intent_b200 as ib
from oracle import attention as oracle
from test_int4_attention_gpu import DTYPES, HALF_UNIT, assert_close, make, of_rounded, reference, run

pytestmark = pytest.mark.gpu


def opposite_minima(seed):
    """Single tokens of two sequences, heads of 128 in two groups whose minima are a and -a, thousands, and queries whose sums over both
    groups are nearly the same and take 20 bits: what a score is comes from the last of them."""
    q, cache, table, offsets, n = make([24, 9], [1, 1], 4, 2, 128, 16, 64, "bf16", seed=seed)
    g = torch.Generator().manual_seed(seed)
    a = (4000 * torch.randn(cache[1].shape[:-1], generator=g)).bfloat16()
    unused = cache[1][..., 1].isnan()
    cache[1][..., 1], cache[1][..., 3] = torch.where(unused, math.nan, a), torch.where(unused, math.nan, -a)
    x = torch.where(torch.rand((2, 4, 64), generator=g) < 0.5, 3 + torch.randn((2, 4, 64), generator=g), 0)
    x += (x == 0) * torch.randint(1, 128, x.shape, generator=g) * 2.0 ** -14
    x = (x.bfloat16() * 2.0 ** 14).round() * 2.0 ** -14            # (sums of such numbers are exact in f32)
    other = x.clone()
    other[..., 0] = 5 * 2.0 ** -8 + torch.randint(0, 32, x.shape[:2], generator=g) * 2.0 ** -14
    x[..., 0] = 2.0 ** -6
    return torch.cat([x, other], -1).bfloat16(), cache, table, offsets, n


@pytest.mark.parametrize("seed", range(6))
def test_sums_of_queries_beside_large_minima(cuda_device, seed):
    """A score is the difference of two products of a minimum and a sum, each of which may be rounded sixteen times as an f32 sum is: that
    changes a row by its weights' share of what they are off by, times their values' distance from the row."""
    data = opposite_minima(seed)
    q, (k_codes, k_scales, v_codes, v_scales), table, offsets, n = data
    out, bound = reference(data, 64)
    sums = q.double().unflatten(-1, (2, 64)).sum(-1)
    values, _ = oracle.values(v_codes, v_scales, 64)
    keys, _ = oracle.values(k_codes, k_scales, 64)
    for b in range(2):
        j = torch.arange(int(n[b]))
        at = table[b, j // 16].long(), j % 16
        for h in range(4):
            head = h // 2
            w = torch.softmax((keys[at[0], head, at[1]] @ q[b, h].double()) / 128 ** 0.5, 0)
            minima = k_scales[at[0], head, at[1]].double()[:, 1::2].abs()
            off = 16 * 2.0 ** -24 * (minima @ sums[b, h].abs()) / 128 ** 0.5
            bound[b, h] += ((w * off.expm1())[:, None] * (values[at[0], head, at[1]] - out[b, h]).abs()).sum(0)
    artifact = ib.compile(ib.programs.paged_decode_attention_int4, constexprs={"ACT_DTYPE": "bf16", "GROUP_SIZE": 64})
    assert_close(run(artifact, cuda_device, data, True), (out, bound))


@pytest.mark.parametrize("single", [True, False])
@pytest.mark.parametrize("power", [-100, 60, 64, 100])
@pytest.mark.parametrize("HQ,D,group", [(4, 128, 64), (16, 64, 32), (32, 128, 128)])
def test_values_of_every_size(cuda_device, single, power, HQ, D, group):
    """Groups of equal numbers (their scale is 0): thousands of them as large as the type allows beside a weight, or very small."""
    data = make([2500, 3], [1, 1] if single else [2, 3], HQ, 2, D, 32, group, "bf16")
    q, cache, table, offsets, n = data
    cache[3] = cache[3].unflatten(-1, (-1, 2)).mul(torch.tensor([0.0, 1.0])).flatten(-2).bfloat16()
    cache[3].masked_fill_(cache[1].isnan(), math.nan)
    expected = reference(data, group), of_rounded(data, group)
    program = ib.programs.paged_decode_attention_int4 if single else ib.programs.paged_attention_int4
    artifact = ib.compile(program, constexprs={"GROUP_SIZE": group})
    out = run(artifact, cuda_device, (q, [*cache[:3], cache[3] * 2.0 ** power], table, offsets, n), single)
    assert_close(out.double() * 2.0 ** -power, *expected)


@pytest.mark.parametrize("HQ,D,group", [(4, 128, 64), (8, 64, 32), (16, 128, 128)])
def test_values_with_large_scales(cuda_device, HQ, D, group):
    """Scales up to 2^55, thousands of them with weights alike, in so many sequences that one warp has a whole one."""
    L, B = 3000, 2400
    q, cache, table, _, n = make([L], [1], HQ, 1, D, 64, group, "bf16")
    cache[3] = cache[3] * 2.0 ** 54 / cache[3][..., ::2].nan_to_num().max()
    q = 0.01 * q.repeat(4, 1, 1) * torch.tensor([1.0, -1.0, 2.0, 0.0])[:, None, None].bfloat16()
    artifact = ib.compile(ib.programs.paged_decode_attention_int4, constexprs={"GROUP_SIZE": group})
    out = artifact.run(*(t.to(cuda_device) for t in (q.repeat(B // 4, 1, 1), *cache, table.repeat(B, 1), n.repeat(B))))
    expected = reference((q, cache, table.repeat(4, 1), torch.arange(5, dtype=torch.int32), n.repeat(4)), group)
    for part in out.split(4)[::50]:
        assert_close(part, expected)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("skew", [False, True])
@pytest.mark.parametrize("HQ,D,group", [(4, 128, 64), (8, 64, 32), (16, 128, 128)])
def test_sums_over_long_histories(cuda_device, dtype, skew, HQ, D, group):
    """So many sequences that one warp has a whole one of 65536 tokens, of which its sums must not lose what is below their last bits.
    For a step of 64 tokens four products (f16: eight) are added to a sum of codes, and as many to what is taken off it for the
    middle of the codes.  An addition may cut the sum, by 2^-23 of it, which is at most what sixteen steps leave between them (7.5
    scales a weight) and one puts on top (15); f16's sum is of four steps (15 each) and has less.  Whatever else is rounded goes
    either way: the mean of the results is four of its deviations from that at most."""
    L, B = 65536, 2400
    q, cache, table, _, n = make([L], [1], HQ, 1, D, 64, group, dtype)
    g = torch.Generator().manual_seed(1)
    q = torch.randn((4, HQ, D), generator=g).to(DTYPES[dtype])
    if skew:                             # (most codes are low ones)
        unused = cache[3].isnan()
        x = torch.empty((*cache[2].shape[:-1], D)).exponential_(generator=g) - 1
        cache[2], cache[3] = oracle.quantise(x, group, DTYPES[dtype])
        cache[3].masked_fill_(unused, math.nan)
    artifact = ib.compile(ib.programs.paged_decode_attention_int4, constexprs={"ACT_DTYPE": dtype, "GROUP_SIZE": group})
    out = artifact.run(*(t.to(cuda_device) for t in (q.repeat(B // 4, 1, 1), *cache, table.repeat(B, 1), n.repeat(B)))).cpu()
    once = q, cache, table.repeat(4, 1), torch.arange(5, dtype=torch.int32), n.repeat(4)
    expected, bound = reference(once, group)
    for part in out.split(4)[::50]:
        assert_close(part, (expected, bound))
    cut = 8 * (16 * 7.5 + 15) * 2.0 ** -23 * float(cache[3][..., ::2].double().nanmean())
    # (deviation of an element: half a unit of the result, and of 5 scales' weights over the root of their number)
    half, size = HALF_UNIT[dtype], float(expected.square().mean().sqrt()) + 5 * 2.0 ** -8
    off = float((out[:4].double() - expected).mean())
    print("off by %.2g, %.2g of the result" % (off, off / float(expected.square().mean().sqrt())))
    assert abs(off) <= cut + 4 * half * size / expected.numel() ** 0.5, (off, cut)
