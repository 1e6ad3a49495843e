"""qk_norm_rope and paged_kv_append in calls of many rows, where a group of lanes takes several of them, and as torch operators."""
import pytest
import torch

import intent_b200 as ib
from oracle import attention as oracle
from test_rope_append_gpu import DTYPES, assert_rounded, inputs, move, scale_of, table

pytestmark = pytest.mark.gpu

SEVERAL = "rotate_kernel several rows per group"


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("norm,pairs", [(True, "halves"), (True, "neighbours"), (False, "halves"), (False, "neighbours")])
@pytest.mark.parametrize("T,HQ,HK,D,R,packed", [
    (2501, 5, 3, 64, 64, True), (1999, 7, 4, 128, 96, False), (2223, 8, 1, 128, 128, True), (10001, 1, 1, 64, 32, True)])
def test_norm_and_rotation_of_many_rows(cuda_device, dtype, norm, pairs, T, HQ, HK, D, R, packed):
    """Numbers of heads that fill a group of four, leave one over, or do not fill one."""
    (q, k, v), weights = inputs(T, HQ, HK, D, dtype, packed, seed=T)
    g = torch.Generator().manual_seed(T)
    rotary, positions = table(300, R), torch.randint(0, 300, (T,), generator=g, dtype=torch.int32)
    positions[[3, T - 1]] = torch.tensor([-1, 300], dtype=torch.int32)
    artifact = ib.compile(ib.programs.qk_norm_rope, constexprs={"ACT_DTYPE": dtype, "NORM": norm, "PAIRS": pairs})
    qd, kd, _ = move((q, k, v), cuda_device, packed)
    extra = [w.to(cuda_device) for w in weights] if norm else []
    out = artifact.run(qd, kd, positions.to(cuda_device), rotary.to(cuda_device), *extra)
    assert artifact.observation.kernel == SEVERAL
    for x, y, w in zip((q, k), out, weights):
        w = w if norm else None
        assert_rounded(y, oracle.rotate(x, positions, rotary, w, pairs=pairs), scale_of(x, w), dtype)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("norm,pairs", [(True, "neighbours"), (False, "halves")])
@pytest.mark.parametrize("T,HQ,HK,D,R,page,packed", [
    (2001, 6, 3, 64, 48, 16, True), (1667, 3, 5, 128, 128, 64, False), (2877, 5, 1, 128, 64, 256, True)])
def test_append_of_many_rows(cuda_device, dtype, norm, pairs, T, HQ, HK, D, R, page, packed):
    (q, k, v), weights = inputs(T, HQ, HK, D, dtype, packed, seed=T)
    g = torch.Generator().manual_seed(3)
    pages = -(-T // page) + 3
    rotary, positions = table(64, R), torch.arange(T, dtype=torch.int32) % 64
    slots = torch.randperm(pages * page, generator=g)[:T]
    slots[1], slots[2], slots[1000], slots[T - 1] = -1, pages * page, -(1 << 40), 1 << 40      # padding
    caches = [torch.randn((pages, HK, page, D), generator=g).to(DTYPES[dtype]) for _ in range(2)]
    artifact = ib.compile(ib.programs.paged_kv_append, constexprs={"ACT_DTYPE": dtype, "NORM": norm, "PAIRS": pairs})
    held = [c.to(cuda_device) for c in caches]
    extra = [w.to(cuda_device) for w in weights] if norm else []
    out = artifact.run(*move((q, k, v), cuda_device, packed), positions.to(cuda_device), slots.to(cuda_device),
                       rotary.to(cuda_device), *extra, *held)
    assert artifact.observation.kernel == SEVERAL
    w = weights if norm else (None, None)
    assert_rounded(out, oracle.rotate(q, positions, rotary, w[0], pairs=pairs), scale_of(q, w[0]), dtype)
    expected = oracle.append(caches[0].double(), oracle.rotate(k, positions, rotary, w[1], pairs=pairs), slots)
    assert_rounded(held[0], expected, float(scale_of(k, w[1]).max()), dtype)
    written = oracle.append(torch.zeros_like(caches[0]), torch.ones_like(k), slots) != 0
    assert torch.equal(held[0].cpu()[~written], caches[0][~written])          # what is there already stays
    assert torch.equal(held[1].cpu(), oracle.append(caches[1], v, slots))     # values are copied


def test_rotation_as_torch_op(cuda_device):
    """Two outputs."""
    (q, k, _), weights = inputs(9, 4, 2, 64, "bf16", False)
    rotary, positions = table(20, 64), torch.arange(9, dtype=torch.int32)
    op = ib.compile(ib.programs.qk_norm_rope).as_torch_op("intent_b200_test::norm_rope")
    out = op(*(t.to(cuda_device) for t in (q, k, positions, rotary, *weights)))
    assert len(out) == 2
    for x, y, w in zip((q, k), out, weights):
        assert_rounded(y, oracle.rotate(x, positions, rotary, w), scale_of(x, w), "bf16")


def test_append_as_torch_op(cuda_device):
    """Two mutated arguments."""
    (q, k, v), weights = inputs(9, 4, 2, 64, "bf16", True)
    rotary, positions, slots = table(20, 64), torch.arange(9, dtype=torch.int32), torch.arange(9) * 3
    caches = [torch.zeros((2, 2, 16, 64), dtype=torch.bfloat16) for _ in range(2)]
    held = [c.to(cuda_device) for c in caches]
    op = ib.compile(ib.programs.paged_kv_append).as_torch_op("intent_b200_test::kv_append")
    versions = [h._version for h in held]
    out = op(*move((q, k, v), cuda_device, True), *(t.to(cuda_device) for t in (positions, slots, rotary, *weights)), *held)
    assert all(h._version > before for h, before in zip(held, versions))
    assert_rounded(out, oracle.rotate(q, positions, rotary, weights[0]), scale_of(q, weights[0]), "bf16")
    assert_rounded(held[0], oracle.append(caches[0].double(), oracle.rotate(k, positions, rotary, weights[1]), slots),
                   float(scale_of(k, weights[1]).max()), "bf16")
    assert torch.equal(held[1].cpu(), oracle.append(caches[1], v, slots))
    with pytest.raises(NotImplementedError):           # both caches in one memory
        op(*move((q, k, v), cuda_device, True), *(t.to(cuda_device) for t in (positions, slots, rotary, *weights)), held[0], held[0])
