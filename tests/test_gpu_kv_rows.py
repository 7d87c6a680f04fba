"""Rows and positions that nobody has: what the calls leave there, and what they tell of it.

Bound of the rows that somebody has: one rounding, u |out|; the weights' own rounding (2^-11, float32 2^-21) and twice that of their scores, float32 sums of head_dim
products, relative to sum p |v| and once more through the sum of the weights."""
import pytest
import torch

from dinoml_v2_b200 import kernels
from oracle import decoder as D

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _cache(dim, kind="int8"):
    g = torch.Generator(device=DEV)
    g.manual_seed(dim)
    cache = kernels.kv_cache(8, 2, 16, dim, kind)
    for x, scale in zip(cache[:2], cache[2:]):
        x.copy_((torch.randn(x.shape, device=DEV, generator=g) * 40).round().clamp(-127, 127))
        scale.fill_(1 / 32)
    return cache, _ints([[0, 1, 2, 3], [4, 5, 6, 7]])


@pytest.mark.parametrize("dtype", ["float16", "bfloat16", "float32"])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_rows_of_nobody_are_zero(dim, dtype):
    """A batch padded to more rows than its sequences have, at either end, with single tokens and with prompts."""
    cache, table = _cache(dim)
    g = torch.Generator(device=DEV)
    g.manual_seed(1)
    q = torch.randn(120, 6, dim, device=DEV, generator=g).to(getattr(torch, dtype))
    for starts in ([0, 1, 3], [0, 1, 2], [5, 6, 41], [0, 50, 51], [3, 53, 110], [0, 0, 0], [120, 120, 120]):
        out = torch.full_like(q, 7)
        kernels.kv_cache_attention(q, cache, table, _ints([60, 64]), _ints(starts), out=out)
        assert kernels.device_status() == 0
        assert not out[:starts[0]].any() and not out[starts[2]:].any(), starts
        ref, spread, terms = D.attention(q, cache, table, _ints([60, 64]), _ints(starts), dim ** -0.5, 0)
        weights = (2.0 ** -21 if dtype == "float32" else 2.0 ** -11) + 2 * (dim + 8) * 2.0 ** -24 * terms[..., None]
        assert ((out.cpu().double() - ref).abs() <= D.UNIT[dtype] * ref.abs() + 2 * weights * spread + D.SMALLEST[dtype]).all(), starts


def test_rows_of_a_sequence_with_bad_starts_are_zero():
    cache, table = _cache(64)
    q = torch.ones(10, 2, 64, device=DEV, dtype=torch.float16)
    for starts, mine in (([0, 4, 11], 4), ([0, 4, 1 << 30], 4), ([0, -3, 10], 0), ([-1, 4, 10], None)):
        out = torch.full_like(q, 7)
        kernels.kv_cache_attention(q, cache, table, _ints([60, 64]), _ints(starts), out=out)
        assert kernels.device_status() == 10
        if mine is None:                                         # the second sequence is a good one
            assert not out[:4].any() and out[4:].any(-1).all()
        else:
            assert out[:mine].any(-1).all() and not out[mine:].any()


def test_no_sequences_at_all():
    cache, table = _cache(64)
    q = torch.ones(5, 2, 64, device=DEV, dtype=torch.float16)
    none = dict(block_table=table[:0], starts=_ints([0]))
    out = torch.full_like(q, 7)
    assert kernels.kv_cache_attention(q, cache, lengths=_ints([]), out=out, **none) is out and not out.any()
    k, v = (torch.full((5, 2, 64), 7.0, device=DEV) for _ in range(2))
    kernels.kv_cache_read(cache, rows=5, dtype="float32", out=(k, v), **none)
    assert not k.any() and not v.any() and kernels.device_status() == 0


def test_positions_before_the_first_token():
    """A range that begins before the first token: zeros, told by the status word."""
    cache, table = _cache(64)
    k, v = kernels.kv_cache_read(cache, table, _ints([0, 5, 8]), 8, "float32", begins=_ints([-2, 0]))
    assert kernels.device_status() == 10
    want, _ = kernels.kv_cache_read(cache, table, _ints([0, 3, 6]), 6, "float32")
    assert kernels.device_status() == 0
    assert not k[:2].any() and not v[:2].any() and torch.equal(k[2:], want)


def test_tensors_of_another_device_are_refused(monkeypatch):
    """(The current device stands in for the other one; the native path leaves such calls to the checks in Python.)"""
    cache, table = _cache(64)
    q = torch.ones(2, 2, 64, device=DEV, dtype=torch.float16)
    monkeypatch.setattr(kernels, "_native_call", lambda name: lambda *args: None)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 1)
    for call, args in ((kernels.kv_cache_attention, (q, cache, table, _ints([3, 3]))), (kernels.kv_cache_write, (cache, q, q, table, _ints([3, 3]))),
                       (kernels.kv_cache_read, (cache, table, None, 2)), (kernels.rms_norm, (q, torch.ones(64, device=DEV)))):
        with pytest.raises(ValueError, match="current device"):
            call(*args)
