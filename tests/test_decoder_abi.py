"""CPU tests of the decoder operators' C entries (include/dinoml_b200_decoder.h): what they refuse before anything is launched, and the registers of the
kernels that carry them.  Nothing is launched here: every call is refused for its arguments."""
import ctypes
import re
from pathlib import Path

import pytest

from dinoml_v2_b200 import _native

BUILD = Path(__file__).resolve().parents[1] / "dinoml_v2_b200" / "build"
AT = 1 << 20                          # an aligned address that is never used
NULL, DIMS, DTYPE, ALIGN, RANGE, KBLOCK = 1, 2, 6, 7, 8, 3
F16, BF16, F32 = (_native.DINO_DTYPE[n] for n in ("float16", "bfloat16", "float32"))


@pytest.fixture(scope="module")
def lib():
    if not _native.LIB_PATH.exists():
        pytest.skip("the library is not built in this tree")
    return _native.lib()


def _cache(**other):
    fields = dict(k=AT, v=AT, k_scale=AT, v_scale=AT, type=1, blocks=8, kv_heads=2, block_size=16, head_dim=64) | other
    return _native.KvCache(*(fields[n] for n, _ in _native.KvCache._fields_))


def _batch(**other):
    fields = dict(block_table=AT, table_stride=4, table_blocks=4, lengths=AT, starts=None, sequences=2, rows=2) | other
    return _native.KvBatch(*(fields[n] for n, _ in _native.KvBatch._fields_))


CACHES = [
    (dict(k=None), NULL), (dict(v_scale=None), NULL), (dict(blocks=0), DIMS), (dict(kv_heads=-1), DIMS), (dict(type=0), DTYPE), (dict(type=3), DTYPE),
    (dict(block_size=24), RANGE), (dict(block_size=8), RANGE), (dict(block_size=256), RANGE), (dict(head_dim=96), RANGE), (dict(head_dim=32), RANGE),
    (dict(k=AT + 8), ALIGN),
]
BATCHES = [
    (dict(block_table=None), NULL), (dict(lengths=None), NULL), (dict(sequences=0), DIMS), (dict(rows=-2), DIMS), (dict(table_blocks=0), DIMS),
    (dict(table_stride=3), RANGE), (dict(rows=3), RANGE),
]


@pytest.mark.parametrize("fields,code", CACHES)
def test_caches_that_are_refused(lib, fields, code):
    c, b = ctypes.byref(_cache(**fields)), ctypes.byref(_batch())
    assert lib.dinoml_b200_kv_cache_write(c, b, AT, AT, BF16, 128, 64, 128, 64, None) == code
    assert lib.dinoml_b200_kv_cache_read(c, b, None, AT, AT, BF16, None) == code
    assert lib.dinoml_b200_kv_cache_attention(c, b, AT, AT, BF16, 4, 256, 64, 0.125, 0, None) == code
    assert _native.last_error()


@pytest.mark.parametrize("fields,code", BATCHES)
def test_batches_that_are_refused(lib, fields, code):
    c, b = ctypes.byref(_cache()), ctypes.byref(_batch(**fields))
    assert lib.dinoml_b200_kv_cache_write(c, b, AT, AT, BF16, 128, 64, 128, 64, None) == code
    assert lib.dinoml_b200_kv_cache_attention(c, b, AT, AT, BF16, 4, 256, 64, 0.125, 0, None) == code
    if "lengths" not in fields:                                                           # (a read has none)
        assert lib.dinoml_b200_kv_cache_read(c, b, None, AT, AT, BF16, None) == code


def test_attention_arguments_that_are_refused(lib):
    def call(q=AT, out=AT, dtype=BF16, heads=4, window=0, **cache):
        return lib.dinoml_b200_kv_cache_attention(ctypes.byref(_cache(**cache)), ctypes.byref(_batch()), q, out, dtype, heads, 256, 64, 0.125, window, None)

    assert call(q=None) == NULL and call(out=None) == NULL
    assert call(heads=0) == DIMS
    assert call(heads=5) == RANGE and call(window=-1) == RANGE
    assert call(blocks=1 << 30) == RANGE                                                  # rows of the cache past 2^31
    assert call(dtype=77) == DTYPE
    assert call(q=AT + 1) == ALIGN and call(q=AT + 2, dtype=F32) == ALIGN and call(out=AT + 4) == ALIGN


def test_null_structs_are_refused(lib):
    assert lib.dinoml_b200_kv_cache_write(None, ctypes.byref(_batch()), AT, AT, BF16, 128, 64, 128, 64, None) == NULL
    assert lib.dinoml_b200_kv_cache_read(ctypes.byref(_cache()), None, None, AT, AT, BF16, None) == NULL
    assert lib.dinoml_b200_kv_cache_attention(ctypes.byref(_cache()), None, AT, AT, BF16, 4, 256, 64, 0.125, 0, None) == NULL


def test_norm_arguments_that_are_refused(lib):
    def call(x=AT, residual=None, weight=AT, y=AT, total=None, dtype=BF16, weight_dtype=F32, rows=2, width=64, q8_0=0):
        return lib.dinoml_b200_rms_norm(x, residual, weight, y, total, dtype, weight_dtype, rows, width, 1e-5, q8_0, None)

    assert call(x=None) == NULL and call(weight=None) == NULL and call(y=None) == NULL
    assert call(rows=0) == DIMS and call(width=-4) == DIMS
    assert call(width=48, q8_0=1) == KBLOCK
    assert call(weight_dtype=F16) == DTYPE and call(dtype=77, weight_dtype=F32) == DTYPE
    assert call(x=AT + 1) == ALIGN and call(residual=AT + 1) == ALIGN and call(weight=AT + 2) == ALIGN and call(y=AT + 1) == ALIGN


# Kernels whose loops were laid out for the registers that they have: without spills.  (log, part of the mangled name)
HOT = [
    ("ptxas_kv_attention_many.log", "attention_many_kernel"),
    ("ptxas_kv_cache.log", "kv_write_kernel"),
    ("ptxas_kv_cache.log", "kv_read_kernel"),
]


@pytest.mark.parametrize("log,fragment", HOT)
def test_hot_kernels_do_not_spill(log, fragment):
    path = BUILD / log
    if not path.exists():
        pytest.skip("no ptxas log: the library was not built in this tree")
    entries = re.findall(r"Compiling entry function '(\S+)'.*?\n.*?\n\s*(\d+) bytes stack frame, (\d+) bytes spill stores, (\d+) bytes spill loads", path.read_text())
    hits = [e for e in entries if fragment in e[0]]
    assert hits, f"{fragment} not found in {log}"
    assert all(stores == loads == "0" for _, _, stores, loads in hits), hits
