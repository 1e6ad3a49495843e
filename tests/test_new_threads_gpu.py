"""A thread's first call may be one that has to describe its operands to TMA, before anything has given the thread a context."""
import threading

import pytest
import torch

import intent_b200 as ib

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("name", ["gemm", "paged_attention", "paged_decode_attention"])
def test_first_call_of_a_thread(cuda_device, name):
    artifact = ib.compile(getattr(ib.programs, name), constexprs={} if name == "gemm" else {"ACT_DTYPE": "f16"})
    if name == "gemm":
        arguments = [torch.randn((64, 64), device=cuda_device).half() for _ in range(2)]
    else:
        tokens = 2 if name == "paged_decode_attention" else 400
        cache = [torch.randn((30, 1, 16, 64), device=cuda_device).half() for _ in range(2)]
        pages = torch.arange(30, dtype=torch.int32, device=cuda_device)[None].repeat(2, 1)
        offsets = torch.tensor([0, 200, 400], dtype=torch.int32, device=cuda_device)
        lengths = torch.full((2,), 450, dtype=torch.int32, device=cuda_device)
        arguments = [torch.randn((tokens, 2, 64), device=cuda_device).half(), *cache, pages, *([offsets] if tokens > 2 else []), lengths]
    expected = artifact.run(*arguments)
    call = artifact.prepare(*arguments)          # (nothing of the thread's own asks for memory, which would give it a context)
    call.result().zero_()
    torch.cuda.synchronize()
    failures = []

    def work():
        try:
            call.launch()
        except Exception as error:
            failures.append(error)

    thread = threading.Thread(target=work)
    thread.start()
    thread.join()
    torch.cuda.synchronize()
    assert not failures and torch.equal(call.result(), expected)
