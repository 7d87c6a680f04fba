"""CPU tests of how many CTAs have a row of the sampling together (csrc/sample_clusters.h), for devices of which less is there: where clusters of one size do not run a smaller one is taken, and only
where none that holds a row does is there no answer."""
import shutil
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "dinoml_v2_b200" / "csrc"
HARNESS = r"""
#include "sample_clusters.h"
#include <cassert>
#include <cstdio>
#include <map>
using namespace b200gguf;

int main() {
  constexpr int kPart16 = 65528, kPart32 = 32768;
  using Device = std::map<int, int>;                     // clusters of each size that run at once
  const Device whole{{1, 148}, {2, 74}, {4, 35}, {8, 17}}, few{{1, 6}, {2, 3}, {4, 1}, {8, 0}}, single{{1, 3}, {2, 0}, {4, 0}, {8, 0}}, none{{1, 0}, {2, 0}, {4, 0}, {8, 0}};
  auto of16 = [](const Device& d, int vocabulary, int64_t rows) {
    const SampleClusters c = sample_clusters_16(vocabulary, rows, 65528, [&](int n) { return d.at(n); });
    assert(c.ctas == 0 ? c.at_once == 0 : c.at_once == d.at(c.ctas) && c.at_once > 0);
    return c.ctas;
  };
  auto of32 = [](const Device& d, int vocabulary, int64_t rows) {
    const SampleClusters c = sample_clusters_32(vocabulary, rows, 32768, [&](int n) { return d.at(n); });
    assert(c.ctas == 0 || (c.at_once > 0 && int64_t(c.ctas) * 32768 >= vocabulary));
    return c.ctas;
  };
  // the whole device, as before
  assert(of16(whole, 128256, 1) == 8 && of16(whole, 128256, 17) == 8 && of16(whole, 128256, 18) == 4 && of16(whole, 128256, 36) == 2 && of16(whole, 128256, 75) == 1);
  assert(of16(whole, 28672, 1) == 1 && of16(whole, 28680, 1) == 8 && of16(whole, 49152, 74) == 1 && of16(whole, 50257, 74) == 2 && of16(whole, 131056, 74) == 2 && of16(whole, 131072, 74) == 1);
  assert(of16(whole, 12000, 1) == 1 && of16(whole, 262144, 18) == 1 && of16(whole, 262112, 18) == 4);
  assert(of32(whole, 50001, 7) == 8 && of32(whole, 50001, 18) == 4 && of32(whole, 50001, 256) == 2 && of32(whole, 300, 1) == 1 && of32(whole, 262144, 500) == 8);
  // a part of one
  assert(of16(few, 128256, 1) == 4 && of16(few, 128256, 2) == 2 && of16(few, 128256, 9) == 1 && of16(few, 262144, 1) == 1);
  assert(of32(few, 20000, 1) == 4 && of32(few, 50001, 1) == 4 && of32(few, 50001, 9) == 2 && of32(few, 262144, 1) == 0 && of32(few, 131072, 9) == 4);
  assert(of16(single, 262144, 1) == 1 && of16(single, 100, 7) == 1 && of32(single, 32768, 2) == 1 && of32(single, 32769, 2) == 0);
  assert(of16(none, 128256, 1) == 0 && of32(none, 100, 1) == 0);
  // what cannot be found out is an error
  for (int size : {1, 2, 4, 8}) {
    Device broken = few;
    broken[size] = -1;
    if (size > 1) broken[8] = size == 8 ? -1 : 0;
    assert(sample_clusters_16(128256, 50, kPart16, [&](int n) { return broken.at(n); }).ctas == 0);
    assert(sample_clusters_32(20000, 50, kPart32, [&](int n) { return broken.at(n); }).ctas == 0);
  }
  std::puts("ok");
}
"""


def test_sizes_of_clusters(tmp_path):
    compiler = shutil.which("g++")
    if compiler is None:
        pytest.skip("no compiler")
    (tmp_path / "harness.cpp").write_text(HARNESS)
    subprocess.run([compiler, "-std=c++17", "-Wall", "-Wextra", "-Werror", f"-I{CSRC}", str(tmp_path / "harness.cpp"), "-o", str(tmp_path / "harness")], check=True, capture_output=True, text=True)
    assert subprocess.run([str(tmp_path / "harness")], check=True, capture_output=True, text=True).stdout == "ok\n"
