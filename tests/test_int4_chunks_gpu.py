"""paged_attention_int4 where it takes the kernel for chunks, and what may go on beside a call: pages that are not there, groups that
are no numbers, pages of several sequences, threads on one stream, torch operators."""
import math
import threading

import pytest
import torch

import intent_b200 as ib
from oracle import attention as oracle
from test_int4_attention_gpu import assert_close, make, of_rounded, reference, run
from test_int4_cache_gpu import empty_cache
from test_rope_append_gpu import inputs, table

pytestmark = pytest.mark.gpu


def is_chunk_kernel(artifact):
    return artifact.observation.kernel.startswith("paged_chunk_kernel int4")


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("D,group", [(64, 32), (64, 64), (128, 32), (128, 64), (128, 128)])
@pytest.mark.parametrize("page", [16, 64, 256])
def test_pages_outside_the_cache(cuda_device, dtype, D, group, page):
    """Missing in the middle of a history, ahead of it and among the new tokens."""
    data = make([900, 530], [280, 200], 4, 2, D, page, group, dtype, spare=0)
    pages = data[2]
    pages[0, 1], pages[1, 0] = -5, data[1][0].shape[0]
    if page < 256:
        pages[0, 700 // page], pages[1, 500 // page] = 1 << 30, -1
    artifact = ib.compile(ib.programs.paged_attention_int4, constexprs={"ACT_DTYPE": dtype, "GROUP_SIZE": group})
    assert_close(run(artifact, cuda_device, data, False), reference(data, group), of_rounded(data, group))
    assert is_chunk_kernel(artifact)
    artifact.check()


@pytest.mark.parametrize("window", [0, 70])
@pytest.mark.parametrize("dtype,D,group", [("bf16", 128, 64), ("f16", 64, 32)])
def test_groups_that_are_no_numbers(cuda_device, window, dtype, D, group):
    """They reach the rows that see them, and no others of the tile."""
    sizes = [400, 333], [300, 200], 4, 2, D, 16, group, dtype
    data, clean = make(*sizes), make(*sizes)
    _, (_, k_scales, _, v_scales), pages, _, _ = data
    for b, token, part, value in ((0, 350, v_scales, math.nan), (0, 40, v_scales, math.inf), (1, 300, v_scales, math.inf),
                                  (1, 320, k_scales, math.nan)):
        part[int(pages[b, token // 16]), 1, token % 16, 2:4] = value
    artifact = ib.compile(ib.programs.paged_attention_int4, constexprs={"ACT_DTYPE": dtype, "GROUP_SIZE": group, "WINDOW": window})
    out = run(artifact, cuda_device, data, False).cpu()
    assert is_chunk_kernel(artifact)
    expected, _ = reference(data, group, window=window)
    fine = expected.isfinite()
    assert 0 < int((~fine).sum()) < 0.7 * fine.numel()
    assert torch.equal(out.isfinite(), fine)
    bounds = [reference(clean, group, window=window), of_rounded(clean, group, window=window)]
    near = torch.stack([(out.double() - e).abs() <= b for e, b in bounds]).any(0)
    assert (near | ~fine).all()


@pytest.mark.parametrize("single", [True, False])
def test_pages_of_several_sequences(cuda_device, single):
    """A common prefix is there once; and one sequence has a page twice."""
    data = make([200, 230, 96], [1, 1, 1] if single else [40, 60, 30], 4, 2, 128, 32, 64, "bf16")
    pages = data[2]
    pages[1, :4] = pages[0, :4]
    pages[2, 1] = pages[2, 0]
    program = ib.programs.paged_decode_attention_int4 if single else ib.programs.paged_attention_int4
    assert_close(run(ib.compile(program), cuda_device, data, single), reference(data, 64), of_rounded(data, 64))


@pytest.mark.parametrize("single", [True, False])
def test_threads_on_one_stream(cuda_device, single):
    """They share the stream's workspace: what one call's launches hand over does not meet those of another."""
    cases = [make([1500, 700, 20], [1, 1, 1] if single else [200, 1, 20], 8, 2, 64, 16, 32, "bf16", seed=seed) for seed in range(3)]
    program = ib.programs.paged_decode_attention_int4 if single else ib.programs.paged_attention_int4
    artifact = ib.compile(program, constexprs={"GROUP_SIZE": 32})
    moved = [[t.to(cuda_device) for t in (q, *cache, pages, *(() if single else (offsets,)), n)] for q, cache, pages, offsets, n in cases]
    expected = [artifact.run(*arguments) for arguments in moved]
    torch.cuda.synchronize()
    outs, start = [[] for _ in cases], threading.Barrier(len(cases))

    def work(index):
        start.wait()
        for _ in range(40):
            outs[index].append(artifact.run(*moved[index]))

    threads = [threading.Thread(target=work, args=(index,)) for index in range(len(cases))]
    for thread in threads:
        thread.start()
    for thread in threads:
        thread.join()
    torch.cuda.synchronize()
    for index, results in enumerate(outs):
        assert len(results) == 40 and all(torch.equal(result, expected[index]) for result in results)


def test_as_torch_ops(cuda_device):
    """The append, which writes into the caches, and the read of them."""
    (q, k, v), weights = inputs(20, 4, 2, 128, "bf16", False)
    cache = empty_cache(3, 2, 16, 128, 64, "bf16", cuda_device)
    slots = torch.randperm(48)[:20]
    rest = [t.to(cuda_device) for t in (q, k, v, torch.arange(20).int(), slots, table(32, 128), *weights)]
    append, read = ib.compile(ib.programs.paged_kv_append_int4), ib.compile(ib.programs.paged_kv_read_int4)
    other = [c.clone() for c in cache]
    expected = append.run(*rest, *other)
    assert append.observation.kernel.startswith("append_int4_kernel")
    op = append.as_torch_op("intent_b200_test::append_int4")
    assert torch.equal(op(*rest, *cache), expected)
    for a, b in zip(cache, other):
        assert torch.equal(a, b)
    found = read.run(rest[4], *cache)
    assert read.observation.kernel.startswith("read_kernel") and read.observation.spill_bytes == 0
    op = read.as_torch_op("intent_b200_test::read_int4")
    assert all(torch.equal(a, b) for a, b in zip(op(rest[4], *cache), found))


def test_rows_of_zeros(cuda_device):
    """Keys that are all zero are held as zeros, with and without a norm; a norm's eps keeps them numbers."""
    (q, k, v), weights = inputs(6, 2, 1, 64, "f16", False)
    k[2], v[3] = 0, 0
    cache = empty_cache(1, 1, 16, 64, 64, "f16", cuda_device)
    slots = torch.arange(6)
    for norm in (True, False):
        append = ib.compile(ib.programs.paged_kv_append_int4, constexprs={"ACT_DTYPE": "f16", "NORM": norm})
        append.run(*(t.to(cuda_device) for t in (q, k, v, slots.int(), slots, table(8, 64), *(weights if norm else ()))), *cache)
        keys, values = ib.compile(ib.programs.paged_kv_read_int4, constexprs={"ACT_DTYPE": "f16"}).run(slots.to(cuda_device), *cache)
        assert not keys[2].any() and not values[3].any() and keys[[0, 1, 3, 4, 5]].flatten(1).any(1).all()
        assert keys.isfinite().all() and values.isfinite().all()
    exact, _ = oracle.values(*(c.cpu() for c in cache[2:]), 64)
    assert torch.equal(values.cpu().double(), exact[0, :, :6].transpose(0, 1).to(torch.float16).double())
