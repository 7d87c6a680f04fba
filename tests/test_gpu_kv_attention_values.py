"""Attention over the 8-bit cache at values that a kernel can lose: keys of small codes under a large scale,
infinite rows of q, keys that stand for NaN, values near the largest float32.
Every case but the last goes through the kernel of few rows and through the one of many (which holds the scale of a block of values in exponents).

Bounds, from the arithmetic: an output is rounded once, u |out|; weights carry a rounding of 2^-11 (16-bit activations) and twice that of their scores, which are float32 sums
of head_dim products of what q and the keys are - (head_dim + 8) 2^-24 of the sum of |q k|, whatever the block's scale is -, relative to sum p |v| and once more
through the sum of the weights."""
import pytest
import torch

from dinoml_v2_b200 import kernels
from oracle import decoder as D

pytestmark = pytest.mark.gpu
TYPES = ("int8", "float8_e4m3fn")
DEV = torch.device("cuda:0")


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _prompt(tokens, block, singles=1):
    """Table, lengths and starts of one prompt of `tokens` and of sequences of as many tokens with one new one each: the rows of the first take the kernel of
    many rows, those of the others the one of few."""
    need = -(-tokens // block)
    return _ints([list(range(need))] * (1 + singles)), _ints([tokens] * (1 + singles)), _ints([0, *range(tokens, tokens + singles + 1)])


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("dim,mean", [(64, 30.0), (128, 8.0), (128, 30.0), (256, 8.0), (256, 30.0)])
def test_small_codes_under_a_large_scale(dim, mean, dtype):
    """One outlier sets the scale of every block, the other keys are a step or none; all of q has one sign.  q is zero in the outlier's channel, so the
    scores are sums of small products.  All values are of one size: an output shows what its scores are off by."""
    g = torch.Generator()
    g.manual_seed(dim)
    tokens, block, group, singles = 48, 16, 4, 40
    cache = kernels.kv_cache(3, 1, block, dim, "int8")
    base = torch.randint(-1, 2, (dim,), generator=g)
    k = base.repeat(tokens, 1)
    for j in range(tokens):
        at = torch.randint(0, dim, (4,), generator=g)
        k[j, at] = torch.randint(-1, 2, (4,), generator=g)
    k[:, 5] = 0
    k[::block, 5] = 127
    cache.k.copy_(k.to(torch.int8).view(3, 1, block, dim))
    cache.v.copy_((254 * torch.randint(0, 2, (3, 1, block, dim), generator=g) - 127).to(torch.int8))
    cache.k_scale.fill_(100 / 127)
    cache.v_scale.fill_(1 / 127)
    q = (mean + torch.randn(tokens + singles, group, dim, generator=g)).to(getattr(torch, dtype))
    q[:, :, 5] = 0
    q = q.to(DEV)
    table, lengths, starts = _prompt(tokens, block, singles)
    out = kernels.kv_cache_attention(q, cache, table, lengths, starts)
    assert kernels.device_status() == 0
    ref, spread, terms = D.attention(q, cache, table, lengths, starts, dim ** -0.5, 0)
    weights = 2.0 ** -11 + 2 * (dim + 8) * 2.0 ** -24 * terms[..., None]
    bound = D.UNIT[dtype] * ref.abs() + 2 * weights * spread + D.SMALLEST[dtype]
    off = (out.cpu().double() - ref).abs() / bound
    assert (off <= 1).all(), (float(off[:tokens].max()), float(off[tokens:].max()))


def _cache_of_ones(blocks, heads, block, dim, kind, seed):
    """Random codes; keys and values of order one."""
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    cache = kernels.kv_cache(blocks, heads, block, dim, kind)
    for x, scale in zip(cache[:2], cache[2:]):
        r = torch.randn(x.shape, device=DEV, generator=g)
        x.copy_((r * 40).round().clamp(-127, 127) if kind == "int8" else (r * 100).clamp(-448, 448))
        scale.fill_(1 / 32 if kind == "int8" else 1 / 128)
    return cache


@pytest.mark.parametrize("dtype", ["float16", "bfloat16", "float32"])
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("tokens", [1, 33, 80])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_infinite_q_is_nan(sign, tokens, kind, dtype):
    """inf times keys is inf, -inf or NaN and its softmax is NaN, also where every score is -inf; other heads and rows are what they are without."""
    for dim in (64, 128, 256):
        cache = _cache_of_ones(5, 2, 16, dim, kind, 3)
        cache.k.view(torch.uint8)[..., 9] = 0x38                 # of one sign in this channel (56, or e4m3's 1.0)
        g = torch.Generator(device=DEV)
        g.manual_seed(4)
        q = torch.randn(tokens + 1, 4, dim, device=DEV, generator=g).to(getattr(torch, dtype))
        table, lengths, starts = _prompt(tokens, 16)
        clean = kernels.kv_cache_attention(q, cache, table, lengths, starts)
        rows = sorted({0, tokens // 2, tokens})
        bad = q.clone()
        bad[rows, 3, 9] = sign * float("inf")
        got = kernels.kv_cache_attention(bad, cache, table, lengths, starts)
        assert kernels.device_status() == 0 and torch.isfinite(clean).all()
        assert torch.isnan(got[rows, 3]).all()
        got[rows, 3] = clean[rows, 3]
        assert torch.equal(got, clean)


@pytest.mark.parametrize("dtype", ["float16", "float32"])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_keys_of_nan_codes_are_nan(dim, dtype):
    """An e4m3 NaN among the keys makes every row that sees it NaN, at every place of a tile."""
    tokens = 200
    cache = _cache_of_ones(13, 1, 16, dim, "float8_e4m3fn", 3)
    g = torch.Generator(device=DEV)
    g.manual_seed(4)
    q = torch.randn(tokens + 1, 2, dim, device=DEV, generator=g).to(getattr(torch, dtype))
    table, lengths, starts = _prompt(tokens, 16)
    clean = kernels.kv_cache_attention(q, cache, table, lengths, starts)
    position = torch.cat([torch.arange(tokens), torch.tensor([tokens - 1])]).to(DEV)
    for at in [*range(64, 80), 127, 128, 199]:
        spoilt = [t.clone() for t in cache]
        spoilt[0].view(torch.uint8)[at // 16, 0, at % 16, 21] = 0x7f
        got = kernels.kv_cache_attention(q, spoilt, table, lengths, starts)
        sees = position >= at
        assert torch.isnan(got[sees]).all(), at
        assert torch.equal(got[~sees], clean[~sees]), at


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_values_near_the_largest_float32(dtype, kind):
    """A sequence of one token answers with its value, whatever its size is."""
    for dim in (64, 128, 256):
        g = torch.Generator(device=DEV)
        g.manual_seed(dim)
        x = torch.randn(1, 2, dim, device=DEV, generator=g).clamp(-3, 3).to(getattr(torch, dtype))
        for size in (1e30, 3e36, 1e38):
            cache = kernels.kv_cache(1, 2, 16, dim, kind)
            v = x * size
            kernels.kv_cache_write(cache, x, v, _ints([[0]]), _ints([1]))
            held = kernels.kv_cache_read(cache, _ints([[0]]), None, 1, "float32")[1]
            got = kernels.kv_cache_attention(x, cache, _ints([[0]]), _ints([1])).float()
            assert kernels.device_status() == 0 and torch.isfinite(held).all()
            assert ((got - held).abs() <= (D.UNIT[dtype] + 2.0 ** -11) * held.abs()).all(), size
