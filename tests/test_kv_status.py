"""CPU test of how the status of the cache's kernels is read (csrc/kv_status.h), compiled against a fake CUDA runtime: a wait that gave up is told, and the attention's
counters are emptied, whatever else the kernels have to tell."""
import shutil
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "dinoml_v2_b200" / "csrc"
HARNESS = r"""
#include "kv_status.h"
#include <cassert>
#include <cstdio>
#include <cstring>
using namespace b200gguf::kv;

static bool fail_copy = false;
extern "C" {
cudaError_t cudaMemcpy(void* d, const void* s, size_t n, cudaMemcpyKind) {
  if (fail_copy) return cudaErrorUnknown;
  std::memcpy(d, s, n);
  return cudaSuccess;
}
cudaError_t cudaMemset(void* p, int v, size_t n) { std::memset(p, v, n); return cudaSuccess; }
}

int main() {
  int words[2] = {}, resets = 0;
  auto take = [&] { return take_status(words, [&] { ++resets; }); };
  assert(take() == 0 && resets == 0);
  words[0] = ST_KV_RANGE;
  assert(take() == 10 && resets == 0 && words[0] == 0 && take() == 0);
  words[1] = ST_KV_TIMEOUT;
  assert(take() == 16 && resets == 1 && words[1] == 0 && take() == 0 && resets == 1);
  words[0] = ST_KV_RANGE;                              // a range that came first, or last, hides nothing
  words[1] = ST_KV_TIMEOUT;
  assert(take() == 16 && resets == 2 && words[0] == 0 && words[1] == 0 && take() == 0);
  words[0] = ST_KV_RANGE;                              // what cannot be read is no success, and is there still
  fail_copy = true;
  assert(take() == -1 && words[0] == 10);
  fail_copy = false;
  assert(take() == 10 && take_status(nullptr, [&] { ++resets; }) == -1 && resets == 2);
  std::puts("ok");
}
"""


def test_status_of_the_cache(tmp_path):
    from dinoml_v2_b200 import build
    if shutil.which("g++") is None:
        pytest.skip("no g++")
    try:
        include = Path(build.nvcc()).resolve().parents[1] / "include"
    except RuntimeError:
        pytest.skip("no CUDA headers")
    (tmp_path / "harness.cpp").write_text(HARNESS)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", f"-I{CSRC}", f"-I{include}", str(tmp_path / "harness.cpp"), "-o", str(tmp_path / "harness")], check=True)
    assert subprocess.run([str(tmp_path / "harness")], check=True, capture_output=True, text=True).stdout == "ok\n"


def test_each_kind_of_trouble_has_a_word_of_its_own():
    """No kernel writes a word that another kind of trouble may have taken first."""
    for path in CSRC.glob("kv_*"):
        assert "atomicCAS" not in path.read_text(), path.name
