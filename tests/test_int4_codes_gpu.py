"""paged_kv_append_int4: codes next to a border between two are those of the definition in 64 bits."""
import pytest
import torch

import intent_b200 as ib
from oracle import attention as oracle
from test_int4_cache_gpu import empty_cache, rows
from test_rope_append_gpu import DTYPES, table

pytestmark = pytest.mark.gpu


def append(device, k, v, group, dtype, weight=None, pairs="halves", rotary=None):
    """(codes, scales) of keys and of values, [T, HK, ...]; every token at position 0."""
    T, HK, D = k.shape
    cache = empty_cache(-(-T // 64), HK, 64, D, group, dtype, device)
    slots, positions = torch.arange(T), torch.zeros(T, dtype=torch.int32)
    norms = [] if weight is None else [weight.to(device)] * 2
    ib.compile(ib.programs.paged_kv_append_int4,
               constexprs={"ACT_DTYPE": dtype, "NORM": weight is not None, "PAIRS": pairs, "GROUP_SIZE": group}).run(
        *(t.to(device) for t in (k, k, v, positions, slots, table(1, 16) if rotary is None else rotary)), *norms, *cache)
    return [rows(c, slots) for c in cache]


# Multiples k + 1/2 of a scale s that are 16-bit numbers, as s is, and whose product with the rounded 1 / s in 64 bits lies on the
# other side of the half.
TIES = {"f16": [(1288, 3), (1456, 6), (1568, 7), (1576, 1), (1648, 5), (1680, 2), (1712, 7), (1816, 2), (1872, 4), (1896, 3), (1916, 1),
                (1968, 6), (2024, 3)],
        "bf16": [(196, 1)]}


@pytest.mark.parametrize("pairs", ["halves", "neighbours"])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_zeros_of_normalised_keys(cuda_device, dtype, pairs):
    """A key's element that is zero stays zero, and -m / s of the 16-bit m and s may lie in the middle between two codes.  Each row has
    two numbers whose weights make them such a minimum and maximum, and a third, of weight zero, that sets the norm."""
    D, eps = 128, float(torch.tensor(1e-6))
    ties = TIES[dtype] * 8 if dtype == "bf16" else TIES[dtype]
    k, weight = torch.zeros((len(ties), 1, D), dtype=DTYPES[dtype]), torch.zeros(D, dtype=DTYPES[dtype])
    for i, (s, multiple) in enumerate(ties):
        s = s * 2.0 ** (-10 - i // len(TIES[dtype]))
        minimum = (multiple + 0.5) * s
        low, high = 16 + 2 * i, 17 + 2 * i                    # (rotated are elements 0 to 15)
        norm = torch.linspace(0.5, 1.0, 20001).to(DTYPES[dtype]).unique()
        row = torch.zeros((len(norm), D), dtype=torch.float64)
        row[:, low], row[:, high], row[:, -1] = -1, 1, norm.double()
        factor = float((128 / 2.56) ** 0.5)
        weight[low], weight[high] = minimum / factor, (15 * s - minimum) / factor
        y = row / torch.sqrt((row * row).mean(-1, keepdim=True) + eps) * weight.double()
        _, scales = oracle.quantise(y, D, DTYPES[dtype])
        fits = ((scales[:, 0].double() == s) & (scales[:, 1].double() == -minimum)).nonzero().flatten()
        assert len(fits), (s, multiple)
        k[i, 0] = row[fits[0]].to(DTYPES[dtype])
    codes, scales, _, _ = append(cuda_device, k, k, D, dtype, weight, pairs)
    keys = oracle.rotate(k, torch.zeros(len(k), dtype=torch.int64), table(1, 16), weight, pairs=pairs, eps=eps)
    expected, expected_scales = oracle.quantise(keys, D, DTYPES[dtype])
    assert torch.equal(scales, expected_scales)
    assert torch.equal(codes, expected)


def next_to_halves(dtype, group):
    """Rows of a group whose quotients are a half and a little more or less, and rows of numbers of every size."""
    little = [2.0 ** -24, 2.0 ** -20] if dtype == "f16" else [2.0 ** -40, 2.0 ** -30, 2.0 ** -24, 2.0 ** -20]
    out = []
    for e in little:
        for sign in (1, -1):
            row = torch.arange(group).remainder(15) + 0.5     # multiples k + 1/2 of 1, less than nothing or more below them
            row[0], row[1] = sign * e, 15
            out.append(row)
            for multiple in range(0, 15, 2):                  # and of 2 from a minimum that is one
                row = torch.zeros(group)
                row[0], row[1], row[2::2] = -(2 * multiple + 1), 29 - 2 * multiple, sign * e
                out.append(row)
    g = torch.Generator().manual_seed(group)
    sizes = 2.0 ** torch.randint(-20, 1, (400, group), generator=g)
    out += list(torch.randn((400, group), generator=g) * sizes)
    return torch.stack(out).to(DTYPES[dtype])


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("D,group", [(64, 32), (128, 64), (128, 128)])
def test_values_next_to_halves(cuda_device, dtype, D, group):
    """Their difference to the minimum can have more bits than f32 has: it is 64 bits' (in which all of these are exact)."""
    x = next_to_halves(dtype, group).repeat(1, D // group)[:, None]
    held = append(cuda_device, x, x, group, dtype)
    expected, scales = oracle.quantise(x, group, DTYPES[dtype])
    for i in (0, 2):                                          # keys, which position 0 turns by nothing, and values
        assert torch.equal(held[i + 1], scales)
        assert torch.equal(held[i], expected)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("D,group", [(64, 32), (128, 128)])
def test_equal_numbers_of_every_size(cuda_device, dtype, D, group):
    """A group of equal numbers has the scale 0 and codes 0."""
    top = torch.finfo(DTYPES[dtype]).max
    x = torch.tensor([1.0, 2.0 ** -24, 60000.0] + ([2.0 ** 63, 2.0 ** 64, 2.0 ** 100, 2.0 ** -120] if dtype == "bf16" else []) + [top])
    x = torch.cat([x, -x]).to(DTYPES[dtype])[:, None, None].expand(-1, 1, D).contiguous()
    held = append(cuda_device, x, x, group, dtype)
    for codes, scales in (held[:2], held[2:]):
        assert not codes.any()
        assert not scales[..., ::2].any() and torch.equal(scales[..., 1::2], x[..., ::group])


def test_keys_beyond_the_type(cuda_device):
    """A key that the rotation takes beyond f16 is held as long as its group's minimum and scale are numbers; what it stands for is
    infinite when read in f16, as such a key is in a 16-bit cache."""
    g = torch.Generator().manual_seed(0)
    k = (20000 * torch.randn((5, 1, 64), generator=g)).clamp(-40000, 40000).half()
    k[:, 0, 0], k[:, 0, 1] = 60000, -50000
    k[4, 0, 2] = -60000                                     # (its minimum is beyond the type, too)
    rotary = torch.zeros((1, 64))
    rotary[:, :32] = 1.2
    held = append(cuda_device, k, k, 64, "f16", rotary=rotary)
    keys = oracle.rotate(k, torch.zeros(5, dtype=torch.int64), rotary)
    codes, scales = oracle.quantise(keys, 64, torch.float16)
    assert torch.equal(held[0], codes) and torch.equal(held[1].nan_to_num(-1.0), scales.nan_to_num(-1.0))
    assert scales[:4].isfinite().all() and scales[4].isnan().all()
    value, _ = oracle.values(codes[:4], scales[:4], 64)
    cache = empty_cache(1, 1, 16, 64, 64, "f16", cuda_device)
    slots = torch.arange(5)
    for to, part in zip(cache, held):
        to[0, :, :5] = part.transpose(0, 1).to(cuda_device)
    out = ib.compile(ib.programs.paged_kv_read_int4, constexprs={"ACT_DTYPE": "f16", "GROUP_SIZE": 64}).run(slots.to(cuda_device), *cache)
    read = out[0].cpu()
    assert torch.equal(read[:4], value.half()) and read[4].isnan().all()
    assert (read[:4, 0, 0] == torch.inf).all() and read[:4].isfinite().float().mean() > 0.9
