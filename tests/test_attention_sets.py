"""CPU tests of the attention's workspaces (csrc/scratch_sets.h, csrc/captured_sets.h), compiled against a fake CUDA runtime whose stream work is carried out when the stream is
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
CAPTURED = FAKE + r"""
#include "captured_sets.h"
using namespace b200gguf;

struct Object { cudaHostFn_t destroy; void* data; int references; };
struct Graph { std::vector<Object*> owned; };
static std::map<cudaStream_t, std::pair<unsigned long long, Graph*>> capturing;
static cudaStreamCaptureMode mode = cudaStreamCaptureModeGlobal;
static bool fail_retain = false, fail_malloc = false;
static void drop(Object* o, unsigned n) { if ((o->references -= int(n)) == 0) { o->destroy(o->data); delete o; } }
extern "C" {
cudaError_t cudaStreamGetCaptureInfo_v2(cudaStream_t s, cudaStreamCaptureStatus* status, unsigned long long* id, cudaGraph_t* graph, const cudaGraphNode_t**, size_t*) {
  const auto it = capturing.find(s);
  *status = it == capturing.end() ? cudaStreamCaptureStatusNone : cudaStreamCaptureStatusActive;
  if (it != capturing.end()) { *id = it->second.first; *graph = reinterpret_cast<cudaGraph_t>(it->second.second); }
  return cudaSuccess;
}
cudaError_t cudaThreadExchangeStreamCaptureMode(cudaStreamCaptureMode* m) { std::swap(*m, mode); return cudaSuccess; }
cudaError_t cudaStreamCreateWithFlags(cudaStream_t* s, unsigned) { *s = reinterpret_cast<cudaStream_t>(size_t(999)); return cudaSuccess; }
cudaError_t cudaStreamDestroy(cudaStream_t s) { assert(queued[s].empty()); return cudaSuccess; }
cudaError_t cudaUserObjectCreate(cudaUserObject_t* o, void* p, cudaHostFn_t f, unsigned n, unsigned) {
  *o = reinterpret_cast<cudaUserObject_t>(new Object{f, p, int(n)});
  return cudaSuccess;
}
cudaError_t cudaUserObjectRelease(cudaUserObject_t o, unsigned n) { drop(reinterpret_cast<Object*>(o), n); return cudaSuccess; }
cudaError_t cudaGraphRetainUserObject(cudaGraph_t g, cudaUserObject_t o, unsigned n, unsigned flags) {
  assert(n == 1 && flags == cudaGraphUserObjectMove);
  if (fail_retain) return cudaErrorUnknown;
  reinterpret_cast<Graph*>(g)->owned.push_back(reinterpret_cast<Object*>(o));
  return cudaSuccess;
}
}
static void destroy(Graph& g) { for (Object* o : g.owned) drop(o, 1); g.owned.clear(); }

struct Got { float* room; int* counters; };
static Got get(AttnWorkspaces& all, cudaStream_t s, size_t floats = 100) {
  const cudaStreamCaptureMode before = mode;
  Got got{nullptr, nullptr};
  got.room = all.get(0, s, floats, &got.counters);
  assert(mode == before);
  if (got.room != nullptr && capturing.count(s) == 0) cudaStreamSynchronize(s);      // (the launch behind it would wait)
  if (got.room != nullptr) for (int i = 0; i < AttnScratch::kMaxWorkers; ++i) assert(got.counters[i] == 0);
  return got;
}

int main() {
  AttnWorkspaces all;
  Graph one, two, three;
  const Got eager = get(all, stream(1));
  capturing[stream(1)] = {11, &one};
  const Got a = get(all, stream(1)), again = get(all, stream(1), 50);
  assert(a.room != eager.room && a.counters != eager.counters);                          // not the stream's own
  assert(again.room == a.room && again.counters == a.counters);                          // ordered within a capture
  const Got more = get(all, stream(1), 1000);
  assert(more.room != a.room && more.counters == a.counters && live.count(a.room) == 1); // the smaller room stays: nodes have its address
  capturing[stream(2)] = {11, &one};
  const Got fork = get(all, stream(2));
  assert(fork.room != more.room && fork.counters != a.counters);                         // a branch of the same capture
  capturing.clear();
  capturing[stream(1)] = {12, &two};
  const Got b = get(all, stream(1));
  assert(b.counters != a.counters && b.counters != eager.counters && b.counters != fork.counters);     // another graph of the same stream
  capturing.clear();
  assert(get(all, stream(1)).counters == eager.counters);
  // A status read empties all of them.
  a.counters[3] = fork.counters[4] = b.counters[5] = eager.counters[6] = 1;
  all.reset(0);
  assert(a.counters[3] == 0 && fork.counters[4] == 0 && b.counters[5] == 0 && eager.counters[6] == 0);
  // Sets of graphs that are gone are used again, empty; nothing is allocated.
  b.counters[7] = 9;
  destroy(two);
  const size_t before = live.size();
  capturing[stream(3)] = {13, &three};
  assert(get(all, stream(3)).counters == b.counters && live.size() == before);
  // What can't be had leaves nothing behind.
  capturing[stream(3)] = {14, &three};
  fail_retain = true;
  assert(get(all, stream(3)).room == nullptr);
  fail_retain = false;
  capturing.clear();
  destroy(one);
  destroy(three);
  // A stream that is released leaves its set, empty, to the next one.
  const Got own = get(all, stream(5));
  own.counters[2] = 1;
  all.release(stream(5));
  const Got next = get(all, stream(6));
  assert(next.counters == own.counters && next.room == own.room);
  all.release(stream(6));
  all.release(stream(6));                                                                // (nothing left)
  // A bounded number is kept.
  std::vector<Graph> many(20);
  for (int i = 0; i < 20; ++i) {
    capturing[stream(4)] = {100ull + unsigned(i), &many[i]};
    assert(get(all, stream(4)).room != nullptr);
  }
  for (Graph& g : many) destroy(g);
  all.reset(0);
  assert(live.size() <= 2 + 2 + 4 * 3);                                                  // a stream's, a spare one, and four sets of up to three
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


def test_captures_have_workspaces_of_their_own(tmp_path):
    _run(CAPTURED, tmp_path)
