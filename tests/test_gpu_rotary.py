"""Rotation by position with the norms of heads against its formula in float64: head sizes whole and odd for the kernels' pieces, parts of a head, both pairings, far positions, strided
and misaligned heads, results in place, rows that are nobody's.

Bounds: one rounding at the end, u of the value.  Inside, float32: the norm's sum of squares, root and products are fewer than 40 roundings (2^-18 of the value, as for `rms_norm`;
nothing without a weight), sine and cosine (2 units of the last place and 2^-24 of the angle's rest), two products, a sum and the magnitude: 8 roundings of a pair's length, 2^-21."""
import pytest
import torch

from dinoml_v2_b200 import kernels
from oracle import decode_ends as E
from oracle import decoder as D

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
DTYPES = ("bfloat16", "float16", "float32")


def _inputs(rows, heads, kv_heads, dim, dtype, seed=1, pad=0, most=131072):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    x = torch.randn(rows, (heads + 2 * kv_heads) * dim + pad, device=DEV, generator=g).to(getattr(torch, dtype))
    q, k = x[:, pad:pad + heads * dim].unflatten(1, (heads, dim)), x[:, pad + heads * dim:pad + (heads + kv_heads) * dim].unflatten(1, (kv_heads, dim))
    positions = torch.randint(0, most, (rows,), device=DEV, generator=g, dtype=torch.int32)
    return q, k, positions, [(1 + 0.3 * torch.randn(dim, device=DEV, generator=g)) for _ in range(2)]


def _close(got, x, weight, positions, frequencies, eps, interleaved, magnitude):
    dtype = str(x.dtype)[6:]
    want, size = E.rotate(x, weight, positions, frequencies, eps, interleaved, magnitude)
    nobody = positions.cpu() < 0
    want[nobody], size[nobody] = 0, 0
    inside = 2.0 ** -21 + (2.0 ** -18 if weight is not None else 0)
    assert ((got.cpu().double() - want).abs() <= D.UNIT[dtype] * (want.abs() + inside * size) + inside * size + D.SMALLEST[dtype]).all()


def _check(q, k, positions, frequencies, weights=(None, None), eps=1e-5, interleaved=False, magnitude=1.0, **kwargs):
    got = kernels.rotary(q, k, positions, frequencies, q_weight=weights[0], k_weight=weights[1], eps=eps, interleaved=interleaved, magnitude=magnitude, **kwargs)
    for y, x, w in zip(got, (q, k), weights):
        if x is None:
            assert y is None
        else:
            assert y.shape == x.shape and y.dtype == x.dtype
            _close(y, x, w, positions, frequencies, eps, interleaved, magnitude)
    return got


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim,turned", [(128, 128), (64, 64), (256, 256), (512, 512), (80, 80), (96, 96), (128, 64), (256, 64), (64, 16), (80, 40), (96, 32), (2, 2), (6, 2), (34, 18),
                                        (130, 130), (288, 288), (320, 96)])
def test_heads(dim, turned, dtype):
    frequencies = kernels.rotary_frequencies(turned, 500000.0)
    for i, (rows, heads, kv_heads) in enumerate(((1, 8, 2), (5, 3, 1), (70, 7, 5), (3, 65, 1))):
        q, k, positions, weights = _inputs(rows, heads, kv_heads, dim, dtype, seed=dim + i)
        for interleaved in (False, True):
            _check(q, k, positions, frequencies, interleaved=interleaved)
            _check(q, k, positions, frequencies, weights, 1e-6, interleaved, magnitude=1.19)
            _check(q, k, positions, frequencies, [w.to(q.dtype) for w in weights], 1e-2, interleaved)


@pytest.mark.parametrize("dtype", DTYPES)
def test_one_side_and_one_weight(dtype):
    q, k, positions, (wq, wk) = _inputs(9, 4, 2, 128, dtype)
    f = kernels.rotary_frequencies(128)
    _check(q, None, positions, f)
    _check(q, None, positions, f, (wq, None))
    _check(q, k, positions, f, (wq, None))
    _check(q, k, positions, f, (None, wk))
    _check(q, k, positions, f[:0], (wq, wk))                                              # norms alone


@pytest.mark.parametrize("dtype", DTYPES)
def test_positions(dtype):
    """The first token, far ones, and the ends of int32; frequencies of order one, whose angles are then two billion radians."""
    q, k, _, weights = _inputs(8, 4, 2, 64, dtype)
    positions = torch.tensor([0, 1, 2, 131071, 1 << 20, (1 << 31) - 1, -1, -(1 << 31)], dtype=torch.int32, device=DEV)
    y, z = _check(q, k, positions, kernels.rotary_frequencies(64), weights)
    assert not y[6:].any() and not z[6:].any()
    y, _ = _check(q, k, positions[:1].expand(8).contiguous(), kernels.rotary_frequencies(64))
    assert torch.equal(y, q)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("pad", [1, 2, 3, 4, 8])
def test_addresses_and_strides(pad, dtype):
    f = kernels.rotary_frequencies(128)
    q, k, positions, weights = _inputs(6, 5, 3, 128, dtype, pad=pad)
    want = kernels.rotary(q.contiguous(), k.contiguous(), positions, f, q_weight=weights[0], k_weight=weights[1])
    got = _check(q, k, positions, f, weights)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    swapped = q.transpose(0, 1).contiguous().transpose(0, 1)                              # heads outside, rows inside
    assert torch.equal(kernels.rotary(swapped, k, positions, f, q_weight=weights[0], k_weight=weights[1])[0], want[0])
    odd = torch.empty(128 + pad, device=DEV)[pad:]                                        # weights at any address
    odd.copy_(weights[0])
    assert torch.equal(kernels.rotary(q, k, positions, f, q_weight=odd, k_weight=weights[1])[0], want[0])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
def test_in_place_and_given(interleaved, dtype):
    f = kernels.rotary_frequencies(96)
    q, k, positions, weights = _inputs(11, 6, 2, 96, dtype)
    positions[[3, 10]] = torch.tensor([-1, -7], dtype=torch.int32, device=DEV)
    args = dict(q_weight=weights[0], k_weight=weights[1], interleaved=interleaved)
    want = kernels.rotary(q, k, positions, f, **args)
    fresh = [torch.full_like(t.contiguous(), 5.0) for t in (q, k)]
    got = kernels.rotary(q, k, positions, f, out=fresh, **args)
    assert got[0] is fresh[0] and got[1] is fresh[1] and all(torch.equal(a, b) for a, b in zip(got, want)) and not got[0][3].any()
    before = q.clone(), k.clone()
    fused = q._base.clone() if q._base is not None else None
    got = kernels.rotary(q, k, positions, f, out=(q, k), **args)
    assert got[0] is q and got[1] is k
    for y, w, x in zip((q, k), want, before):
        live = positions >= 0
        assert torch.equal(y[live], w[live]) and torch.equal(y[~live], x[~live])          # nobody's rows are as they were
    if fused is not None:
        assert torch.equal(q._base[:, 8 * 96:], fused[:, 8 * 96:])                        # and so is v
    mixed = kernels.rotary(before[0], before[1], positions, f, out=(None, fresh[1]), **args)
    assert torch.equal(mixed[0], want[0]) and mixed[1] is fresh[1]


def test_many_rows():
    q, k, positions, weights = _inputs(3000, 9, 3, 64, "bfloat16")
    _check(q, k, positions, kernels.rotary_frequencies(64, factors=torch.linspace(1, 8, 32)), weights)


def test_values_that_are_not_finite():
    q, k, positions, weights = _inputs(3, 2, 1, 64, "float32")
    q[0, 0, 3], q[1, 1, 40] = float("nan"), float("inf")
    f = kernels.rotary_frequencies(64)
    y, _ = kernels.rotary(q, k, positions, f)
    assert torch.isnan(y[0, 0, [3, 35]]).all() and torch.isfinite(y[0, 0, :3]).all() and torch.isfinite(y[0, 1]).all() and not torch.isfinite(y[1, 1, [8, 40]]).any()
    y, _ = kernels.rotary(q, k, positions, f, q_weight=weights[0])
    assert torch.isnan(y[0, 0]).all() and torch.isfinite(y[0, 1]).all() and torch.isfinite(y[2]).all()
    zero = torch.zeros(2, 2, 64, device=DEV)
    assert not kernels.rotary(zero, None, positions[:2], f, q_weight=weights[0], eps=1e-6)[0].any()


def test_frequencies():
    f = kernels.rotary_frequencies(8, 100.0, scale=0.25, factors=[1, 2, 4, 8])
    want = [0.25 * 100.0 ** (-i / 4) / 2 ** i for i in range(4)]
    assert f.dtype == torch.float64 and all(abs(a - b) <= 1e-15 for a, b in zip(f.tolist(), want))
    for args, kwargs in (((7,), {}), ((0,), {}), ((8,), {"factors": [1, 2]})):
        with pytest.raises(ValueError):
            kernels.rotary_frequencies(*args, **kwargs)


def test_refusals():
    q, k, p, (wq, wk) = _inputs(4, 4, 2, 64, "float16")
    f = kernels.rotary_frequencies(64)
    wide = torch.empty(4, 8, 64, dtype=q.dtype, device=DEV)
    for args, kwargs in (((q.cpu(), k, p, f), {}), ((q, k.float(), p, f), {}), ((q, k[:3], p, f), {}), ((q, k, p.long(), f), {}), ((q, k, p[:3], f), {}), ((q, k, p, f.float()), {}),
                         ((q, k, p, f.cpu()), {}), ((q, k, p, kernels.rotary_frequencies(66)), {}), ((q[..., :63], k[..., :63], p, f[:8]), {}), ((q[..., ::2], None, p, f[:8]), {}),
                         ((q, k, p, f), {"q_weight": wq[:32]}), ((q, k, p, f), {"q_weight": wq.double()}), ((q, k, p, f), {"q_weight": wq, "k_weight": wk.half()}),
                         ((q, None, p, f), {"k_weight": wk}), ((q, k, p, f), {"out": (wide, None)}), ((q, k, p, f), {"out": (wide[:, ::2].expand(4, 4, 64)[:1].expand(4, 4, 64), None)}),
                         ((wide[:, :4], None, p, f), {"out": (wide[:, 1:5], None)}), ((q, k, p, f), {"out": (None,)}), ((q.int(), k.int(), p, f), {}),
                         ((torch.zeros(4, 1, 514, device=DEV), None, p, f), {})):
        with pytest.raises(ValueError):
            kernels.rotary(*args, **kwargs)
    y, z = kernels.rotary(q[:0], k[:0], p[:0], f)
    assert y.shape == (0, 4, 64) and z.shape == (0, 2, 64)


def test_results_that_would_overlap():
    """q and k are columns of one tensor, and so are their results; what one of them still reads is not written."""
    f = kernels.rotary_frequencies(64)
    q, k, p, _ = _inputs(5, 4, 4, 64, "bfloat16")
    want = kernels.rotary(q, k, p, f)
    for out in ((k, None), (None, q), (k, q)):
        with pytest.raises(ValueError):
            kernels.rotary(q, k, p, f, out=out)
    both = torch.empty(5, 12, 64, dtype=q.dtype, device=DEV)
    for out in ((both[:, :4], both[:, 2:6]), (both[:, 8:], both[:, 8:])):
        with pytest.raises(ValueError):
            kernels.rotary(q, k, p, f, out=out)
    for out in ((both[:, :4], both[:, 8:]), (both[:, 8:], both[:, 4:8]), (q, both[:, :4]), (q, k)):
        q2, k2 = q.clone(), k.clone()
        got = kernels.rotary(q2, k2, p, f, out=tuple(q2 if t is q else k2 if t is k else t for t in out))
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_other_streams_and_graphs():
    q, k, positions, weights = _inputs(17, 8, 2, 128, "bfloat16")
    f = kernels.rotary_frequencies(128)
    want = kernels.rotary(q, k, positions, f, q_weight=weights[0])
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    got = kernels.rotary(q, k, positions, f, q_weight=weights[0], stream=stream)
    stream.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = kernels.rotary(q, k, positions, f, q_weight=weights[0])
    positions += 1
    graph.replay()
    torch.cuda.synchronize()
    again = kernels.rotary(q, k, positions, f, q_weight=weights[0])
    assert torch.equal(got[0], again[0]) and torch.equal(got[1], again[1]) and not torch.equal(got[0], want[0])
