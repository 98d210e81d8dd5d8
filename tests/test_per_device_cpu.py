"""What the serving kernels' launches set up holds for each device of a process, shown against a stand-in for the CUDA runtime."""
import re
import shutil
import subprocess
from pathlib import Path

import pytest

from oa_b200.ops import paged as P

KERNELS = Path(__file__).resolve().parents[1] / "oa_b200" / "csrc" / "kernels"
CUDA = Path("/usr/local/cuda/include")

PROGRAM = r"""
#include <cstdio>
#include "per_device.h"
static int current = 0, failing = -1, asked[128], counted[128];
extern "C" cudaError_t cudaGetDevice(int* d) { *d = current; return cudaSuccess; }
extern "C" cudaError_t cudaFuncSetAttribute(const void*, cudaFuncAttribute, int) {
  if (current == failing) return cudaErrorInvalidValue;
  ++asked[current];
  return cudaSuccess;
}
extern "C" cudaError_t cudaDeviceGetAttribute(int* v, cudaDeviceAttr, int d) { ++counted[d]; *v = 100 + d; return cudaSuccess; }
#define CHECK(x) if (!(x)) { std::printf("line %d: %s\n", __LINE__, #x); return 1; }
int main() {
  std::atomic<unsigned long long> one{0}, two{0};
  for (int round = 0; round < 3; ++round)
    for (current = 0; current < 4; ++current) CHECK(oa::allow_smem(one, nullptr, 1000) == cudaSuccess);
  for (int d = 0; d < 4; ++d) CHECK(asked[d] == 1);              // once on each
  current = 1;
  CHECK(oa::allow_smem(two, nullptr, 1000) == cudaSuccess && asked[1] == 2);       // another kernel asks for itself
  current = failing = 5;
  CHECK(oa::allow_smem(one, nullptr, 1000) != cudaSuccess);      // a refusal is told, and asked again
  failing = -1;
  CHECK(oa::allow_smem(one, nullptr, 1000) == cudaSuccess && asked[5] == 1);
  current = 100;                                                  // beyond those that are remembered
  for (int i = 0; i < 2; ++i) CHECK(oa::allow_smem(one, nullptr, 1000) == cudaSuccess);
  CHECK(asked[100] == 2);
  for (int round = 0; round < 3; ++round)
    for (current = 0; current < 4; ++current) CHECK(oa::sm_count() == 100 + current);
  for (int d = 0; d < 4; ++d) CHECK(counted[d] == 1);
  current = 100;
  CHECK(oa::sm_count() == 200);
  std::printf("all ok\n");
  return 0;
}
"""


def test_each_device_is_asked_once(tmp_path):
    if shutil.which("g++") is None or not (CUDA / "cuda_runtime_api.h").exists():
        pytest.skip("no g++ or no CUDA headers")
    (tmp_path / "main.cpp").write_text(PROGRAM)
    r = subprocess.run(["g++", "-std=c++17", "-I", str(KERNELS), "-I", str(CUDA), "-o", str(tmp_path / "main"), str(tmp_path / "main.cpp")], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    r = subprocess.run([str(tmp_path / "main")], capture_output=True, text=True)
    assert r.returncode == 0 and "all ok" in r.stdout, r.stdout


@pytest.mark.parametrize("name", ["paged.cu", "paged_attn.cu", "sampling.cu"])
def test_launches_keep_nothing_of_one_device_for_all(name):
    source = (KERNELS / name).read_text()
    assert not re.search(r"static (bool|int) \w+ = ", source)
    assert not re.search(r"\b148\b", re.sub(r"//[^\n]*", "", source))


def test_layouts_are_kept_for_each_device(monkeypatch):
    """The bytes of scratch follow from the device's SMs: a layout of one device is not another's."""
    class Lib:
        calls = 0

        def oa_paged_attn_scratch_bytes(self, *_):
            Lib.calls += 1
            return 1000 * Lib.calls

    monkeypatch.setattr(P.N, "require", lambda: Lib())
    import torch
    P._attention_layout.cache_clear()
    try:
        args = (torch.Size((3, 256)), torch.bfloat16, torch.Size((4, 2, 16, 64)), (2048, 1024, 64, 1), torch.Size((4, 2, 16, 64)), (2048, 1024, 64, 1),
                torch.bfloat16, torch.bfloat16, torch.Size((3, 2)), (2, 1), torch.int32, 3, 4, 1, None, 0, None)
        assert [P._attention_layout(*args, device)[-1] for device in (0, 1, 0, 1, -1)] == [1000, 2000, 1000, 2000, 0]
    finally:
        P._attention_layout.cache_clear()
