"""CPU tests of the attention's workspaces (csrc/scratch_sets.h), compiled against a fake CUDA runtime whose stream work is carried out when the stream is
waited for."""
import shutil
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "dinoml_v2_b200" / "csrc"
FAKE = r"""
#include <cassert>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <functional>
#include <map>
#include <set>
#include <vector>
#include <cuda_runtime_api.h>

static std::map<cudaStream_t, std::vector<std::function<void()>>> queued;
static std::set<void*> live;
extern "C" {
cudaError_t cudaMalloc(void** p, size_t n) { *p = std::malloc(n); std::memset(*p, 0xEE, n); live.insert(*p); return cudaSuccess; }
cudaError_t cudaFree(void* p) { assert(live.erase(p) == 1); std::free(p); return cudaSuccess; }
cudaError_t cudaMemsetAsync(void* p, int v, size_t n, cudaStream_t s) { queued[s].push_back([=] { std::memset(p, v, n); }); return cudaSuccess; }
cudaError_t cudaStreamSynchronize(cudaStream_t s) {
  auto work = std::move(queued[s]);
  queued[s].clear();
  for (auto& f : work) f();
  return cudaSuccess;
}
}
static cudaStream_t stream(int i) { return reinterpret_cast<cudaStream_t>(size_t(i)); }
"""
EMPTIED = FAKE + r"""
#include "scratch_sets.h"
using namespace b200gguf;

int main() {
  ScratchSets<AttnScratch> sets;
  std::vector<int*> counters;
  for (int i = 1; i < 4; ++i) {
    AttnScratch& set = sets.at(i == 3 ? 1 : 0, stream(i));
    cudaMalloc(reinterpret_cast<void**>(&set.arrived), sizeof(int) * AttnScratch::kMaxWorkers);
    std::memset(set.arrived, 0, sizeof(int) * AttnScratch::kMaxWorkers);
    set.arrived[i] = 5;                                  // a launch that gave up left it behind
    counters.push_back(set.arrived);
  }
  assert(sets.empty_all(0));
  // a launch on any stream finds the counters at zero without waiting for anything
  for (int i = 0; i < AttnScratch::kMaxWorkers; ++i) assert(counters[0][i] == 0 && counters[1][i] == 0);
  assert(counters[2][3] == 5);                           // (another device's)
  std::puts("ok");
}
"""


def _run(source, tmp_path):
    from dinoml_v2_b200 import build
    if shutil.which("g++") is None:
        pytest.skip("no g++")
    try:
        include = Path(build.nvcc()).resolve().parents[1] / "include"
    except RuntimeError:
        pytest.skip("no CUDA headers")
    (tmp_path / "harness.cpp").write_text(source)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", f"-I{CSRC}", f"-I{include}", str(tmp_path / "harness.cpp"), "-o", str(tmp_path / "harness")], check=True)
    assert subprocess.run([str(tmp_path / "harness")], check=True, capture_output=True, text=True).stdout == "ok\n"


def test_counters_are_empty_when_the_status_has_been_read(tmp_path):
    _run(EMPTIED, tmp_path)
