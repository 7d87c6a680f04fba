"""The norm with the residual's addition against its formula in float64: widths around the kernels' tiles and no multiple of anything, single rows, the float32
and the 16-bit weights, results in place, Q8_0 blocks.

Bounds: y is rounded once, u |y|; the sum of squares, its root and the two products are float32, fewer than 40 roundings one after another (the sum is a
tree over partial sums of at most 32 values): 2^-18 |y|.  A Q8_0 value is within half a step of the block's scale, which is a float16 (2^-11 of the
largest value, times 127 of the steps that it is off by)."""
import pytest
import torch

import oracle
from dinoml_v2_b200 import kernels
from oracle import decoder as D

pytestmark = pytest.mark.gpu
DTYPES = ("bfloat16", "float16", "float32")
DEV = torch.device("cuda:0")


def _inputs(rows, width, dtype, weight, seed=1, scale=1.0):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    t = getattr(torch, dtype)
    x, r = ((scale * torch.randn(rows, width, device=DEV, generator=g)).to(t) for _ in range(2))
    return x, r, (1 + 0.3 * torch.randn(width, device=DEV, generator=g)).to(getattr(torch, weight))


def _check(y, total, x, weight, eps, residual, dtype):
    want, want_total = D.rms_norm(x, weight, eps, residual)
    assert ((y.cpu().double() - want).abs() <= (D.UNIT[dtype] + 2.0 ** -18) * want.abs() + D.SMALLEST[dtype]).all()
    if residual is None:
        assert total is None
    else:
        assert ((total.cpu().double() - want_total).abs() <= (D.UNIT[dtype] + 2.0 ** -24) * want_total.abs() + D.SMALLEST[dtype]).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("width", [1, 7, 32, 33, 255, 256, 1000, 2048, 4096, 4100, 8192, 14336, 28672, 40001])
def test_norm(width, dtype):
    for rows in (1, 2, 5, 300):
        for weight in {"float32", dtype}:
            x, r, w = _inputs(rows, width, dtype, weight, seed=width + rows)
            _check(*kernels.rms_norm(x, w), x, w, 1e-5, None, dtype)
            _check(*kernels.rms_norm(x, w, 1e-2, residual=r), x, w, 1e-2, r, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
def test_in_place_and_shapes(dtype):
    x, r, w = _inputs(6, 1032, dtype, "float32")
    y, total = kernels.rms_norm(x, w, residual=r)
    for given in ("residual", "x"):
        x2, r2 = x.clone(), r.clone()
        y2, total2 = kernels.rms_norm(x2, w, residual=r2, total=r2 if given == "residual" else x2)
        assert torch.equal(y, y2) and torch.equal(total, total2)
    out = torch.empty(2, 3, 1032, dtype=x.dtype, device=DEV)
    y3, total3 = kernels.rms_norm(x.view(2, 3, 1032), w, residual=r.view(2, 3, 1032), out=out)
    assert y3 is out and torch.equal(y3.view(6, -1), y) and total3.shape == out.shape
    odd = torch.empty(6 * 1032 + 1, dtype=x.dtype, device=DEV)[1:].view(6, 1032)          # not at a multiple of 16 bytes
    odd.copy_(x)
    assert torch.equal(kernels.rms_norm(odd, w)[0], kernels.rms_norm(x, w)[0])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("width", [32, 96, 2080, 4096, 8192, 28704])
def test_q8_0(width, dtype):
    for rows in (1, 3, 150):
        x, r, w = _inputs(rows, width, dtype, "float32", seed=rows)
        y8, total = kernels.rms_norm(x, w, residual=r, q8_0=True)
        want, want_total = D.rms_norm(x, w, 1e-5, r)
        assert y8.shape == (rows, width // 32 * 34) and torch.equal(total, kernels.rms_norm(x, w, residual=r)[1])
        largest = want.abs().view(rows, -1, 32).amax(-1, keepdim=True)
        got = torch.from_numpy(oracle.dequantize(y8.cpu().numpy(), "Q8_0", width)).double().view(rows, -1, 32)
        step = largest / 127 * (1 + 2.0 ** -11)
        # the largest value is 127 steps of a scale that is up to 2^-11 off, and is cut off there
        bound = 0.5 * step + 2.0 ** -18 * largest + 2.0 ** -11 * largest
        assert ((got - want.view(rows, -1, 32)).abs() <= bound).all()
        assert torch.equal(kernels.dequantize_rows(y8, "Q8_0", width).cpu().double().view(rows, -1, 32), got)


def test_range_of_values():
    for dtype, sizes in (("float32", (1e-30, 1e-15, 1e15)), ("bfloat16", (1e-30, 1e-15, 1e15)), ("float16", (1e-6, 1e-3, 1e4))):
        for scale in sizes:
            x, r, w = _inputs(2, 4096, dtype, "float32", scale=scale)
            _check(*kernels.rms_norm(x, w, 0.0 if scale > 1e-20 else 1e-5), x, w, 0.0 if scale > 1e-20 else 1e-5, None, dtype)
    zero = torch.zeros(2, 4096, device=DEV)
    assert not kernels.rms_norm(zero, w)[0].any()
    y8, _ = kernels.rms_norm(zero, w, q8_0=True)
    assert not kernels.dequantize_rows(y8, "Q8_0", 4096).any()
    zero[1, 5] = float("nan")
    y = kernels.rms_norm(zero, w)[0]
    assert not y[0].any() and torch.isnan(y[1]).all()


def test_refusals():
    x, r, w = _inputs(2, 100, "float16", "float32")
    for args, kwargs in (((x.cpu(), w), {}), ((x, w[:50]), {}), ((x, w.double()), {}), ((x.t(), w), {}), ((x, w), {"residual": r[:1]}), ((x, w), {"residual": r.float()}),
                         ((x, w), {"total": r}), ((x, w), {"q8_0": True}), ((x, w), {"out": r[:1]}), ((x.int(), w), {}), ((x, w.bfloat16()), {})):
        with pytest.raises(ValueError):
            kernels.rms_norm(*args, **kwargs)
    empty, total = kernels.rms_norm(x[:0], w, residual=r[:0])
    assert empty.shape == (0, 100) and total.shape == (0, 100)
