"""CPU tests of the C entries of the embedding, the rotation, the pool of blocks and the choice of tokens (include/dinoml_b200_decoder.h): what they refuse before anything is launched, that no
exception leaves them, and that their kernels do not spill.  Nothing is launched here."""
import ctypes
import re
import subprocess
from pathlib import Path

import pytest

from dinoml_v2_b200 import _native

ROOT = Path(__file__).resolve().parents[1]
CSRC, BUILD = ROOT / "dinoml_v2_b200" / "csrc", ROOT / "dinoml_v2_b200" / "build"
AT = 1 << 20                          # an aligned address that is never used
NULL, DIMS, KBLOCK, QTYPE, DTYPE, ALIGN, RANGE = 1, 2, 3, 5, 6, 7, 8
F16, BF16, F32 = (_native.DINO_DTYPE[n] for n in ("float16", "bfloat16", "float32"))


@pytest.fixture(scope="module")
def lib():
    if not _native.LIB_PATH.exists():
        pytest.skip("the library is not built in this tree")
    return _native.lib()


def _struct(kind, fields):
    return kind(*(fields[n] for n, _ in kind._fields_))


def test_embedding(lib):
    def call(tokens=AT, token_bytes=4, table=AT, vocabulary=100, out=AT, qtype=12, dtype=BF16, count=3, width=512):
        return lib.dinoml_b200_embedding(tokens, token_bytes, table, vocabulary, out, qtype, dtype, count, width, 1.0, None)

    assert call(tokens=None) == call(table=None) == call(out=None) == NULL
    assert call(vocabulary=0) == call(count=0) == call(width=-256) == DIMS
    assert call(qtype=99) == QTYPE and call(width=300) == KBLOCK and call(qtype=8, width=48) == KBLOCK
    assert call(token_bytes=2) == call(dtype=77) == DTYPE
    assert call(tokens=AT + 2) == call(tokens=AT + 4, token_bytes=8) == call(out=AT + 8) == call(table=AT + 2) == call(table=AT + 1, qtype=8, width=512) == ALIGN
    assert call(width=1 << 32) == call(count=1 << 60) == call(vocabulary=1 << 60) == RANGE
    assert _native.last_error()


def test_rotary(lib):
    def call(rows=4, positions=AT, frequencies=AT, pairs=32, dtype=BF16, weight_dtype=F32, head_dim=64, k=True, **other):
        sides = []
        for heads in (4, 2):
            fields = dict(x=AT, out=AT, weight=None, row_stride=512, head_stride=64, out_row_stride=512, out_head_stride=64, heads=heads) | other
            sides.append(ctypes.byref(_struct(_native.Heads, fields)))
        return lib.dinoml_b200_rotary(sides[0], sides[1] if k else None, positions, frequencies, pairs, dtype, weight_dtype, rows, head_dim, 1e-5, 1.0, 0, None)

    assert lib.dinoml_b200_rotary(None, None, AT, AT, 32, BF16, F32, 4, 64, 1e-5, 1.0, 0, None) == NULL
    assert call(positions=None) == call(frequencies=None) == call(x=None) == call(out=None, k=False) == NULL
    assert call(rows=0) == call(head_dim=0) == call(heads=0) == DIMS
    assert call(head_dim=63) == call(head_dim=514) == call(pairs=33) == call(pairs=-1) == call(heads=1 << 20) == RANGE
    assert call(dtype=77) == call(weight_dtype=F16) == DTYPE
    assert call(x=AT + 1) == call(out=AT + 2, dtype=F32) == call(weight=AT + 2) == call(positions=AT + 2) == call(frequencies=AT + 4) == ALIGN
    assert _native.last_error()


def test_pool(lib):
    def call(new=AT, drop=None, rows=3, lengths=AT, starts=None, positions=AT, slots=AT, pool=True, **other):
        fields = dict(block_table=AT, table_stride=4, free_blocks=AT, free_count=AT, table_blocks=4, sequences=3, blocks=10, block_size=16, of=AT) | other
        struct = _struct(_native.KvPool, {**fields, "lengths": fields["of"]})
        return lib.dinoml_b200_kv_pool_step(ctypes.byref(struct) if pool else None, new, drop, rows, lengths, starts, positions, slots, None)

    assert call(pool=False) == call(new=None) == call(lengths=None) == call(positions=None) == call(slots=None) == call(block_table=None) == call(of=None) == NULL
    assert call(free_blocks=None) == call(free_count=None) == NULL
    assert call(sequences=0) == call(blocks=0) == call(table_blocks=-1) == call(rows=-1, starts=AT) == DIMS
    assert call(block_size=24) == call(block_size=256) == call(sequences=8193, rows=8193) == call(table_stride=3) == call(rows=4) == call(blocks=1 << 27) == RANGE
    assert _native.last_error()


def test_sample(lib):
    def call(logits=AT, stride=1000, dtype=BF16, rows=2, vocabulary=1000, uniforms=AT, settings=True, tokens=AT):
        struct = _native.SampleSettings(None, None, None, None, 1.0, 0, 1.0, 0.0)
        return lib.dinoml_b200_sample(logits, stride, dtype, rows, vocabulary, uniforms, ctypes.byref(struct) if settings else None, tokens, None, None)

    assert call(logits=None) == call(uniforms=None) == call(settings=False) == call(tokens=None) == NULL
    assert call(rows=0) == call(vocabulary=0) == DIMS
    assert call(vocabulary=262145, stride=262145) == call(stride=999) == call(rows=1 << 30) == RANGE
    assert call(dtype=77) == DTYPE and call(logits=AT + 1) == call(logits=AT + 2, dtype=F32) == ALIGN
    assert _native.last_error()


HARNESS = r"""
#include "decoder_ends_abi.cu"
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
int embedding(const void*, int, const void*, int64_t, void*, int, int, int64_t, int64_t, float, cudaStream_t) { throw std::bad_alloc(); }
int rotary(const DinoB200Heads*, const DinoB200Heads*, const int*, const double*, int, int, int, int, int, float, float, int, cudaStream_t) { throw std::length_error("x"); }
int sample(const void*, int64_t, int, int, int, const float*, const DinoB200SampleSettings*, int*, float*, cudaStream_t) { throw 1; }
namespace kv {
int pool_step(const DinoB200KvPool*, const int*, const int*, int, int*, int*, int*, int*, cudaStream_t) { throw std::runtime_error("x"); }
}  // namespace kv
}  // namespace b200gguf

int main() {
  for (int messages = 0; messages < 2; ++messages) {      // (without and with room for a message)
    auto ready = [&] { messages_left = messages; };
    ready(); assert(dinoml_b200_embedding(nullptr, 0, nullptr, 0, nullptr, 0, 0, 0, 0, 0.f, nullptr) == RC_LAUNCH);
    ready(); assert(dinoml_b200_rotary(nullptr, nullptr, nullptr, nullptr, 0, 0, 0, 0, 0, 0.f, 0.f, 0, nullptr) == RC_LAUNCH);
    ready(); assert(dinoml_b200_kv_pool_step(nullptr, nullptr, nullptr, 0, nullptr, nullptr, nullptr, nullptr, nullptr) == RC_LAUNCH);
    ready(); assert(dinoml_b200_sample(nullptr, 0, 0, 0, 0, nullptr, nullptr, nullptr, nullptr, nullptr) == RC_LAUNCH);
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


@pytest.mark.parametrize("log", ["ptxas_embedding.log", "ptxas_rotary.log", "ptxas_kv_pool.log", "ptxas_sample.log"])
def test_kernels_do_not_spill(log):
    path = BUILD / log
    if not path.exists():
        pytest.skip("no ptxas log: the library was not built in this tree")
    spills = re.findall(r"(\d+) bytes spill stores, (\d+) bytes spill loads", path.read_text())
    assert spills and all(pair == ("0", "0") for pair in spills), spills
