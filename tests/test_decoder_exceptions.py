"""CPU test: no C++ exception leaves a C entry of the decoder operators (csrc/decoder_abi.cu), which is compiled here against operators that throw."""
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "dinoml_v2_b200" / "csrc"
HARNESS = r"""
#include "decoder_abi.cu"
#include <cassert>
#include <cstdio>
#include <new>
#include <stdexcept>

static int messages_left = 0;
namespace b200gguf {
int set_error(int rc, const char*) {
  if (messages_left-- <= 0) throw std::bad_alloc();
  return rc;
}
void stream_release_scratch(cudaStream_t) { throw std::runtime_error("lock"); }
void umma_release_scratch(cudaStream_t) {}
void attention_release_scratch(cudaStream_t) {}
namespace kv {
int cache_write(const DinoB200KvCache*, const DinoB200KvBatch*, const void*, const void*, int, int64_t, int64_t, int64_t, int64_t, cudaStream_t) { throw std::bad_alloc(); }
int cache_read(const DinoB200KvCache*, const DinoB200KvBatch*, const int*, void*, void*, int, cudaStream_t) { throw std::bad_alloc(); }
int cache_attention(const DinoB200KvCache*, const DinoB200KvBatch*, const void*, void*, int, int, int64_t, int64_t, float, int, cudaStream_t) { throw std::length_error("x"); }
}  // namespace kv
namespace norm {
int rms_norm(const void*, const void*, const void*, void*, void*, int, int, int, int, float, int, cudaStream_t) { throw 1; }
}  // namespace norm
}  // namespace b200gguf

int main() {
  for (int messages = 0; messages < 2; ++messages) {      // (without and with room for a message)
    auto ready = [&] { messages_left = messages; };
    ready(); assert(dinoml_b200_kv_cache_write(nullptr, nullptr, nullptr, nullptr, 0, 0, 0, 0, 0, nullptr) == RC_LAUNCH);
    ready(); assert(dinoml_b200_kv_cache_read(nullptr, nullptr, nullptr, nullptr, nullptr, 0, nullptr) == RC_LAUNCH);
    ready(); assert(dinoml_b200_kv_cache_attention(nullptr, nullptr, nullptr, nullptr, 0, 0, 0, 0, 0.f, 0, nullptr) == RC_LAUNCH);
    ready(); assert(dinoml_b200_rms_norm(nullptr, nullptr, nullptr, nullptr, nullptr, 0, 0, 0, 0, 0.f, 0, nullptr) == RC_LAUNCH);
    ready(); assert(dinoml_b200_release_stream(nullptr) == RC_LAUNCH);
  }
  std::puts("ok");
}
"""


def test_exceptions_become_codes(tmp_path):
    from dinoml_v2_b200 import build
    try:
        nvcc = build.nvcc()
    except RuntimeError:
        pytest.skip("no nvcc")
    (tmp_path / "harness.cu").write_text(HARNESS)
    subprocess.run([nvcc, "-std=c++17", "-gencode", "arch=compute_100a,code=sm_100a", f"-I{CSRC}", str(tmp_path / "harness.cu"), "-o", str(tmp_path / "harness")],
                   check=True, capture_output=True)
    assert subprocess.run([str(tmp_path / "harness")], check=True, capture_output=True, text=True).stdout == "ok\n"
