"""Host threads on one stream share that stream's workspace: what one call's launches hand to each other must not meet the
launches of another call."""
import threading

import pytest
import torch

import intent_b200 as ib

pytestmark = pytest.mark.gpu


def _attention(g, device, counts, length):
    HQ, HK, D, page = 8, 2, 64, 16
    B, used = len(counts), -(-length // page)
    cache = [torch.randn((B * used, HK, page, D), generator=g).bfloat16().to(device) for _ in range(2)]
    table = torch.randperm(B * used, generator=g).to(torch.int32).view(B, used).to(device)
    q = torch.randn((sum(counts), HQ, D), generator=g).bfloat16().to(device)
    offsets = torch.tensor([0] + counts).cumsum(0).to(torch.int32).to(device)
    return q, *cache, table, offsets, torch.full((B,), length, dtype=torch.int32, device=device)


def _case(name, seed, device):
    g = torch.Generator().manual_seed(seed)

    def numbers(low, high, shape, dtype):
        return torch.randint(low, high, shape, generator=g, dtype=dtype).to(device)

    if name == "paged_attention":
        return {}, _attention(g, device, [200, 1, 70], 1500)
    if name == "paged_decode_attention":
        arguments = _attention(g, device, [1] * 5, 3000)
        return {}, arguments[:4] + arguments[5:]
    if name == "w4a8_packed_matmul":
        return {}, (numbers(-128, 128, (64, 512), torch.int8), numbers(0, 256, (256, 256), torch.uint8))
    if name == "bitnet_int2_matmul":
        return {}, (numbers(-128, 128, (64, 512), torch.int8), numbers(0, 256, (256, 128), torch.uint8))
    if name == "dequant_bf16_fp4_matmul":
        return {}, (torch.randn((64, 512), generator=g).bfloat16().to(device), numbers(0, 256, (256, 256), torch.uint8))
    if name == "quantized_projection":
        records = torch.randint(0, 256, (256, 4, 144), generator=g, dtype=torch.uint8)
        records[..., :4] = torch.tensor([0, 0x20, 0, 0x20], dtype=torch.uint8)     # scales that are numbers
        return {}, (records.to(device), torch.randn((4, 256), generator=g).to(device))
    members = torch.randperm(128, generator=g).to(torch.int32).to(device)
    offsets = torch.tensor([0, 40, 40, 100, 128], dtype=torch.int32, device=device)
    return {"TOP_K": 2}, (torch.randn((64, 256), generator=g).bfloat16().to(device), offsets, members,
                          torch.randn((4, 128, 256), generator=g).bfloat16().to(device))


@pytest.mark.parametrize("name", ["paged_attention", "paged_decode_attention", "w4a8_packed_matmul", "bitnet_int2_matmul",
                                  "dequant_bf16_fp4_matmul", "quantized_projection", "routed_expert_projection_bf16"])
def test_threads_on_one_stream(cuda_device, name):
    cases = [_case(name, seed, cuda_device) for seed in range(3)]
    artifact = ib.compile(getattr(ib.programs, name), target=ib.B200Target(0), constexprs=cases[0][0])
    expected = [artifact.run(*arguments) for _, arguments in cases]
    torch.cuda.synchronize()
    assert not torch.equal(expected[0], expected[1])
    outs, start = [[] for _ in cases], threading.Barrier(len(cases))

    def work(index):
        torch.cuda.set_device(cuda_device)
        start.wait()
        for _ in range(150):
            outs[index].append(artifact.run(*cases[index][1]))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(cases))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for wanted, got in zip(expected, outs):
        assert len(got) == 150 and all(torch.equal(wanted, o) for o in got)
    artifact.check()
