"""qk_norm_rope and paged_kv_append against their definitions in 64 bits."""
import pytest
import torch

import intent_b200 as ib
from oracle import attention as oracle

pytestmark = pytest.mark.gpu

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
# One rounding to the type (half a unit of its last place, relative; of f16's smallest numbers, absolute) after a chain of
# at most a dozen f32 operations: 16 * 2^-24 of the two products that meet in an element.
HALF_UNIT = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8}
F32 = 16 * 2.0 ** -24


def table(rows, R):
    angle = torch.arange(rows, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, R, 2, dtype=torch.float64) / max(R, 1))
    return torch.cat([angle.cos(), angle.sin()], 1).float()


def inputs(T, HQ, HK, D, dtype, packed, seed=0):
    g = torch.Generator().manual_seed(seed)
    qkv = torch.randn((T, HQ + 2 * HK, D), generator=g).to(DTYPES[dtype])
    q, k, v = qkv[:, :HQ], qkv[:, HQ:HQ + HK], qkv[:, HQ + HK:]
    weights = tuple((1 + 0.2 * torch.randn(D, generator=g)).to(DTYPES[dtype]) for _ in range(2))
    return (q, k, v) if packed else tuple(x.contiguous() for x in (q, k, v)), weights


def move(tensors, device, packed):
    """To the device, as slices of one tensor where they were such."""
    if not packed:
        return [t.to(device) for t in tensors]
    whole = torch.cat([t for t in tensors], 1).to(device)
    return list(whole.split([t.shape[1] for t in tensors], 1))


def assert_rounded(actual, expected, size, dtype):
    """``size``: the scale of what is added up in an element."""
    actual = actual.cpu().double()
    assert torch.equal(actual.isnan(), expected.isnan())
    bound = HALF_UNIT[dtype] * expected.abs() + F32 * size + 2.0 ** -24
    fine = ~expected.isnan()
    excess = ((actual - expected).abs() - bound)[fine]
    assert excess.numel() == 0 or excess.max() <= 0, excess.max()


def scale_of(x, weight, eps=1e-6):
    y = x.double()
    if weight is not None:
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + eps) * weight.double()
    return y.abs().amax(-1, keepdim=True) * 2


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("norm", [True, False])
@pytest.mark.parametrize("pairs", ["halves", "neighbours"])
@pytest.mark.parametrize("T,HQ,HK,D,R,packed", [
    (1, 1, 1, 64, 64, False), (1, 32, 8, 128, 128, True), (7, 5, 1, 64, 32, True), (33, 3, 3, 128, 96, False),
    (130, 12, 2, 128, 16, True), (3, 2, 1, 64, 48, False),
])
def test_norm_and_rotation(cuda_device, dtype, norm, pairs, T, HQ, HK, D, R, packed):
    (q, k, v), weights = inputs(T, HQ, HK, D, dtype, packed, seed=T)
    rotary, positions = table(300, R), torch.randint(0, 300, (T,), dtype=torch.int32)
    artifact = ib.compile(ib.programs.qk_norm_rope, constexprs={"ACT_DTYPE": dtype, "NORM": norm, "PAIRS": pairs})
    qd, kd, _ = move((q, k, v), cuda_device, packed)
    extra = [w.to(cuda_device) for w in weights] if norm else []
    for _ in range(2):                       # bound in Python, then natively
        out = artifact.run(qd, kd, positions.to(cuda_device), rotary.to(cuda_device), *extra)
        for x, y, w in zip((q, k), out, weights):
            w = w if norm else None
            assert_rounded(y, oracle.rotate(x, positions, rotary, w, pairs=pairs), scale_of(x, w), dtype)
    assert artifact.runtime.binder.last() is not None


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("norm", [True, False])
@pytest.mark.parametrize("T,HQ,HK,D,R,page,packed", [
    (1, 8, 2, 128, 128, 64, True), (40, 4, 4, 64, 64, 16, False), (77, 6, 2, 128, 64, 256, True), (19, 7, 1, 64, 32, 32, True),
])
def test_append(cuda_device, dtype, norm, T, HQ, HK, D, R, page, packed):
    (q, k, v), weights = inputs(T, HQ, HK, D, dtype, packed, seed=T)
    g = torch.Generator().manual_seed(3)
    pages = -(-T // page) + 3
    rotary, positions = table(64, R), torch.arange(T, dtype=torch.int32) % 64
    slots = torch.randperm(pages * page, generator=g)[:T]
    if T > 4:
        slots[1], slots[2], slots[3] = -1, pages * page, -(1 << 40)       # padding
    caches = [torch.randn((pages, HK, page, D), generator=g).to(DTYPES[dtype]) for _ in range(2)]
    artifact = ib.compile(ib.programs.paged_kv_append, constexprs={"ACT_DTYPE": dtype, "NORM": norm})
    moved = move((q, k, v), cuda_device, packed)
    held = [c.to(cuda_device) for c in caches]
    extra = [w.to(cuda_device) for w in weights] if norm else []
    for _ in range(2):
        out = artifact.run(*moved, positions.to(cuda_device), slots.to(cuda_device), rotary.to(cuda_device), *extra, *held)
        w = weights if norm else (None, None)
        assert_rounded(out, oracle.rotate(q, positions, rotary, w[0]), scale_of(q, w[0]), dtype)
        expected = oracle.append(caches[0].double(), oracle.rotate(k, positions, rotary, w[1]), slots)
        assert_rounded(held[0], expected, float(scale_of(k, w[1]).max()), dtype)
        written = oracle.append(torch.zeros_like(caches[0]), torch.ones_like(k), slots) != 0
        assert torch.equal(held[0].cpu()[~written], caches[0][~written])          # what is there already stays
        assert torch.equal(held[1].cpu(), oracle.append(caches[1], v, slots))     # values are copied


def test_positions_outside_the_table(cuda_device):
    """NaN for queries and keys of such a token; its values and the other tokens are as they are."""
    (q, k, v), _ = inputs(4, 2, 1, 64, "bf16", False)
    positions, rotary = torch.tensor([-1, 0, 9, 10], dtype=torch.int32), table(10, 64)
    out = ib.compile(ib.programs.qk_norm_rope, constexprs={"NORM": False}).run(
        q.to(cuda_device), k.to(cuda_device), positions.to(cuda_device), rotary.to(cuda_device))
    for x, y in zip((q, k), out):
        assert_rounded(y, oracle.rotate(x, positions, rotary), scale_of(x, None), "bf16")
        assert y.isnan().flatten(1).all(1).tolist() == [True, False, False, True]


def test_rows_of_zeros_and_of_large_numbers(cuda_device):
    """The norm's eps keeps a row of zeros zero; squares of f16's largest numbers do not overflow."""
    q = torch.zeros((3, 1, 64), dtype=torch.float16)
    q[1] = 65504
    q[2, 0, 5] = 6e-8
    one, positions = torch.ones(64, dtype=torch.float16), torch.tensor([3, 3, 3], dtype=torch.int32)
    artifact = ib.compile(ib.programs.qk_norm_rope, constexprs={"ACT_DTYPE": "f16", "EPS": 1e-5})
    out, _ = artifact.run(*(t.to(cuda_device) for t in (q, q, positions, table(8, 64), one, one)))
    assert_rounded(out, oracle.rotate(q, positions, table(8, 64), one, eps=1e-5), scale_of(q, one, 1e-5), "f16")
    assert not out[0].any()


def test_a_cache_of_more_than_32_bits(cuda_device):
    """Slots whose elements lie past 2^31."""
    HK, page, D = 8, 256, 128
    pages = (1 << 31) // (HK * page * D) + 2
    caches = [torch.empty((pages, HK, page, D), dtype=torch.bfloat16, device=cuda_device) for _ in range(2)]
    (q, k, v), _ = inputs(2, 8, HK, D, "bf16", False)
    slots, positions = torch.tensor([pages * page - 1, 5]), torch.zeros(2, dtype=torch.int32)
    caches[0][0, :, 4:7] = 1
    caches[0][-1] = 1
    ib.compile(ib.programs.paged_kv_append, constexprs={"NORM": False}).run(
        *(t.to(cuda_device) for t in (q, k, v, positions, slots, table(4, 128))), *caches)
    assert torch.equal(caches[0][-1, :, -1].cpu(), k[0]) and torch.equal(caches[1][-1, :, -1].cpu(), v[0])
    assert torch.equal(caches[0][0, :, 5].cpu(), k[1]) and torch.equal(caches[1][0, :, 5].cpu(), v[1])
    assert (caches[0][0, :, 4] == 1).all() and (caches[0][0, :, 6] == 1).all() and (caches[0][-1, :, :-1] == 1).all()


def test_no_tokens(cuda_device):
    (q, k, _), weights = inputs(0, 4, 2, 64, "bf16", False)
    out = ib.compile(ib.programs.qk_norm_rope).run(*(t.to(cuda_device) for t in (
        q, k, torch.zeros(0, dtype=torch.int32), table(4, 64), *weights)))
    assert [tuple(o.shape) for o in out] == [(0, 4, 64), (0, 2, 64)]


def test_refusals(cuda_device):
    (q, k, v), weights = inputs(4, 4, 2, 64, "bf16", False)
    (q, k, v), weights = [t.to(cuda_device) for t in (q, k, v)], [w.to(cuda_device) for w in weights]
    positions, rotary = torch.zeros(4, dtype=torch.int32, device=cuda_device), table(4, 64).to(cuda_device)
    slots = torch.arange(4, device=cuda_device)
    caches = [torch.zeros((2, 2, 16, 64), dtype=torch.bfloat16, device=cuda_device) for _ in range(2)]
    rope, append = ib.compile(ib.programs.qk_norm_rope), ib.compile(ib.programs.paged_kv_append)
    rope.run(q, k, positions, rotary, *weights)
    append.run(q, k, v, positions, slots, rotary, *weights, *caches)
    with pytest.raises(TypeError):
        rope.run(q.half(), k, positions, rotary, *weights)
    with pytest.raises(TypeError):
        append.run(q, k, v, positions, slots.int(), rotary, *weights, *caches)
    with pytest.raises(ValueError):
        rope.run(q, k[:3], positions, rotary, *weights)
    with pytest.raises(ValueError):
        rope.run(q, k, positions, rotary[:, :24].contiguous(), *weights)
    with pytest.raises((ValueError, NotImplementedError)):
        rope.run(q, k, positions, rotary[:, :0], *weights)
    with pytest.raises(ValueError):
        rope.run(q, k, positions, torch.zeros((4, 80), device=cuda_device), *weights)
    with pytest.raises(ValueError):
        rope.run(q[..., :32].contiguous(), k[..., :32].contiguous(), positions, rotary[:, :32].contiguous(),
                 *(w[:32] for w in weights))
    with pytest.raises(ValueError):
        append.run(q, k, v, positions, slots, rotary, *weights,
                   *(torch.zeros((2, 2, 24, 64), dtype=torch.bfloat16, device=cuda_device) for _ in range(2)))
    with pytest.raises(NotImplementedError):           # the last axis is not contiguous
        rope.run(q.transpose(1, 2).contiguous().transpose(1, 2), k, positions, rotary, *weights)
    with pytest.raises(NotImplementedError):           # rows off their boundary
        rope.run(torch.zeros((4, 4, 68), dtype=torch.bfloat16, device=cuda_device)[..., :64], k, positions, rotary, *weights)
    with pytest.raises(NotImplementedError):           # both caches in one memory
        append.run(q, k, v, positions, slots, rotary, *weights, caches[0], caches[0])
    for constexprs in ({"PAIRS": "odd"}, {"ACT_DTYPE": "f32"}, {"EPS": "x"}, {"EPS": -1.0}, {"BASE": 1}):
        with pytest.raises(ib.CompilationStageError):
            ib.compile(ib.programs.qk_norm_rope, constexprs=constexprs)
