"""How a thread that describes operands to TMA comes by a context, with the CUDA calls replaced."""
import subprocess
from pathlib import Path

from intent_b200.build import CSRC, _nvcc

PROGRAM = r"""
#include <cstdio>
#include <cstring>
#include "tma.cuh"

static bool lookups = true, devices = true;
static CUcontext context = nullptr;
static int set = 0, errors = 0;
static CUresult get_current(CUcontext* c) { *c = context; return CUDA_SUCCESS; }
static int encode_here;

extern "C" {
cudaError_t cudaGetDriverEntryPoint(const char* name, void** p, unsigned long long, cudaDriverEntryPointQueryResult* query) {
  *query = cudaDriverEntryPointSuccess;
  *p = std::strcmp(name, "cuCtxGetCurrent") == 0 ? reinterpret_cast<void*>(get_current) : static_cast<void*>(&encode_here);
  return lookups ? cudaSuccess : (++errors, cudaErrorInitializationError);
}
cudaError_t cudaGetDevice(int* device) { *device = 3; return cudaSuccess; }
cudaError_t cudaSetDevice(int device) {
  if (!devices) return ++errors, cudaErrorMemoryAllocation;
  ++set;
  context = reinterpret_cast<CUcontext>(&set);
  return device == 3 ? cudaSuccess : cudaErrorInvalidDevice;
}
cudaError_t cudaGetLastError() { errors = 0; return cudaSuccess; }
}

static void call(const char* name) {
  const bool found = ib200::encode_tiled_fn() != nullptr;
  std::printf("%s %d %d %d\n", name, found, set, errors);
}
int main() {
  devices = false;
  call("no_memory");
  devices = true;
  lookups = false;
  call("no_driver");
  lookups = true;
  call("first");
  context = reinterpret_cast<CUcontext>(&errors);
  call("own_context");
  std::printf("kept %d", context == reinterpret_cast<CUcontext>(&errors));
}
"""


def test_a_failure_is_not_kept_and_a_context_is(tmp_path):
    """A call that could not make a context, or not ask the driver, leaves no error behind and does not decide for the next; a thread
    that has a context keeps it, whichever it is."""
    source, binary = tmp_path / "context.cpp", tmp_path / "context"
    source.write_text(PROGRAM)
    include = Path(_nvcc()).resolve().parent.parent / "include"
    subprocess.run(["g++", "-std=c++17", f"-I{CSRC}", f"-I{include}", str(source), "-o", str(binary)], check=True, capture_output=True)
    lines = subprocess.run([str(binary)], check=True, capture_output=True, text=True).stdout.split("\n")
    (no_memory, no_driver, first, own), kept = ([list(map(int, line.split()[1:])) for line in lines[:4]], lines[4])
    assert no_memory == [0, 0, 0]                      # no function, no device set, no error left
    assert no_driver[0] == 0 and no_driver[2] == 0
    assert first[0] == 1 and first[1] >= 1 and first[2] == 0
    assert own == [1, first[1], 0] and kept == "kept 1"
