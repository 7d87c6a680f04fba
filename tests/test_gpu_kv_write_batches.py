"""Writes of batches of every size: a unit of a write (a sequence's new tokens in a block, a head of K or V) is a warp's in large batches and a CTA's in small ones.  Both
against the formula in float64, and the same tokens in one call of a large batch and in calls of one sequence each, byte for byte.

Bounds, from the arithmetic: int8 half a step of the scale (2^-16 of a step more for the float32 quotient), e4m3 2^-4 of the value or half of the smallest step, 2^-10
of the scale."""
import pytest
import torch

from dinoml_v2_b200 import kernels
from oracle import decoder as D

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("kind", ["int8", "float8_e4m3fn"])
@pytest.mark.parametrize("block,dim,heads", [(16, 64, 8), (32, 128, 5), (64, 256, 4), (128, 128, 8)])
@pytest.mark.parametrize("most", [1, 5, 40])
def test_batches(most, block, dim, heads, kind, dtype):
    g = torch.Generator()
    g.manual_seed(block + most)
    sequences = 70
    lengths = [int(torch.randint(0, 3 * block, (1,), generator=g)) for _ in range(sequences)]
    counts = [1 if most == 1 else min(n, int(torch.randint(0, most + 1, (1,), generator=g))) for n in lengths]
    starts = [sum(counts[:i]) for i in range(sequences + 1)]
    table = torch.randperm(3 * sequences, generator=g).to(torch.int32).view(sequences, 3).to(DEV)
    k, v = (torch.randn(starts[-1], heads, dim, generator=g).to(DEV, getattr(torch, dtype)) for _ in range(2))
    cache = kernels.kv_cache(3 * sequences, heads, block, dim, kind)
    for x, scale in zip(cache[:2], cache[2:]):
        x.copy_((40 * torch.randn(x.shape, generator=g)).round().clamp(-127, 127))
        scale.copy_(torch.exp2(torch.randint(-7, -3, scale.shape, generator=g).float()))
    alone = kernels.KVCache(*(t.clone() for t in cache))
    before = [t.clone() for t in cache]
    some = None if most == 1 else _ints(starts)
    found = D.write(before, k, v, table, _ints(lengths), some)
    kernels.kv_cache_write(cache, k, v, table, _ints(lengths), some)
    for b, n in enumerate(lengths):
        rows = slice(starts[b], starts[b + 1])
        kernels.kv_cache_write(alone, k[rows], v[rows], table[b:b + 1], _ints([n]), _ints([0, counts[b]]))
    assert kernels.device_status() == 0
    assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(cache, alone))
    assert found
    host = [t.cpu() for t in cache]
    for (which, i, h), (scale, slot, old, new) in found.items():
        got, want = float(host[2 + which][i, h]), torch.cat([old, new])
        assert abs(got - scale) <= 2.0 ** -22 * scale
        value = host[which][i, h, :slot + len(new)].to(torch.float32).double() * got
        if kind == "int8":
            bound = torch.full_like(want, (0.5 + 2.0 ** -16) * got)
        else:
            bound = torch.maximum(want.abs() * 2.0 ** -4, torch.full_like(want, 2.0 ** -10 * got)) * (1 + 2.0 ** -20)
        assert ((value - want).abs() <= bound).all(), (which, i, h)
