"""The 8-bit cache: write, read and attention against the formulas in float64, at the sizes and masks where they can go wrong - one token and none, the first
and last slots of blocks, blocks that end inside a tile, scales that grow, heads shared by odd groups, rows far apart, garbage behind the last
token, table entries that are nobody's.

Bounds, from the arithmetic: a written int8 value is within half a step of its scale (2^-16 of a step more for the float32 quotient), an e4m3 value
within 2^-4 of itself or half of the smallest step, 2^-10 of the scale; a value read is one product in float32 and one rounding.  An attention output
is rounded once, u |out|; its weights carry their own rounding (the 16-bit kernels hold them in float16, u = 2^-11, float32 in two terms, 2^-21)
and that of their scores, (head_dim + 8) 2^-24 of the sum of |q k| at most, both relative to sum p |v|, and once more through the sum of the weights."""
import pytest
import torch

from dinoml_v2_b200 import kernels
from oracle import decoder as D

pytestmark = pytest.mark.gpu
TYPES = ("int8", "float8_e4m3fn")
DTYPES = ("bfloat16", "float16", "float32")
DEV = torch.device("cuda:0")


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _random_cache(blocks, heads, block, dim, kind, seed, garbage=True):
    """Values of order one; scales of different size."""
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    cache = kernels.kv_cache(blocks, heads, block, dim, kind)
    for q, scale in zip(cache[:2], cache[2:]):
        x = torch.randn(q.shape, device=DEV, generator=g)
        q.copy_((x * 40).round().clamp(-127, 127) if kind == "int8" else (x * 100).clamp(-448, 448))
        s = torch.exp(0.5 * torch.randn(scale.shape, device=DEV, generator=g)) / (40 if kind == "int8" else 100)
        scale.copy_(s if kind == "int8" else torch.exp2(torch.round(torch.log2(s))))
    return cache


def _table(lengths, block, blocks, seed, pad=-1, extra=0):
    """Blocks in random order; entries that no token uses are `pad`."""
    g = torch.Generator()
    g.manual_seed(seed)
    order = torch.randperm(blocks, generator=g).tolist()
    width = max(1, max(-(-n // block) for n in lengths)) + extra
    rows = []
    for n in lengths:
        need = -(-n // block)
        rows.append([order.pop() for _ in range(need)] + [pad] * (width - need))
    return _ints(rows)


def _spoil(cache, table, lengths, block):
    """Bytes behind a sequence's last token, and blocks and scales that no sequence has, become the worst there is."""
    used = set()
    for b, n in enumerate(lengths):
        for j in range(-(-n // block)):
            i = int(table[b, j])
            used.add(i)
            if n < (j + 1) * block:
                for q in cache[:2]:
                    q.view(torch.uint8)[i, :, n - j * block:] = 0x7f if q.dtype != torch.int8 else 0x80       # e4m3 NaN; -128
    free = [i for i in range(cache[0].shape[0]) if i not in used]
    if free:
        for q in cache[:2]:
            q.view(torch.uint8)[free] = 0xff
        for s in cache[2:]:
            s[free] = float("nan")


def _qkv(rows, heads, kv_heads, dim, dtype, seed, pad=0, scale=1.0):
    """q, k, v cut out of one tensor whose rows are `pad` values longer."""
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    x = (scale * torch.randn(rows, (heads + 2 * kv_heads) * dim + pad, device=DEV, generator=g)).to(getattr(torch, dtype))
    q = x[:, :heads * dim].view(rows, heads, dim) if not pad else x[:, pad:pad + heads * dim].unflatten(1, (heads, dim))
    at = pad + heads * dim
    return q, x[:, at:at + kv_heads * dim].unflatten(1, (kv_heads, dim)), x[:, at + kv_heads * dim:].unflatten(1, (kv_heads, dim))


def _check_attention(q, cache, table, lengths, starts=None, window=0, scale=None, dtype="bfloat16"):
    out = kernels.kv_cache_attention(q, cache, table, lengths, starts, window=window, scale=scale)
    assert kernels.device_status() == 0
    dim = q.shape[2]
    ref, spread, terms = D.attention(q, cache, table, lengths, starts, dim ** -0.5 if scale is None else scale, window)
    weights = (2.0 ** -21 if dtype == "float32" else 2.0 ** -11) + 2 * (dim + 8) * 2.0 ** -24 * terms[..., None]
    bound = D.UNIT[dtype] * ref.abs() + 2 * weights * spread + D.SMALLEST[dtype]
    off = (out.cpu().double() - ref).abs()
    assert torch.isfinite(out).all()
    assert (off <= bound).all(), (float((off / bound.clamp(min=1e-300)).max()), out.shape)
    return out


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("block,dim", [(16, 64), (32, 128), (64, 128), (128, 256)])
def test_attention_of_single_tokens(block, dim, kind, dtype):
    """Lengths around blocks and tiles, idle slots among them; one head per cached head and odd groups."""
    for kv_heads, group in ((2, 1), (1, 3), (2, 4), (1, 7), (1, 8), (1, 16), (1, 20)):
        lengths = [1, 0, 2, block - 1, block, block + 1, 0, 63, 64, 65, 127, 128, 129, 300, 1000]
        blocks = sum(-(-n // block) for n in lengths) + 3
        cache, table = _random_cache(blocks, kv_heads, block, dim, kind, group), _table(lengths, block, blocks, group, extra=2)
        _spoil(cache, table, lengths, block)
        q, _, _ = _qkv(len(lengths), kv_heads * group, kv_heads, dim, dtype, group)
        out = _check_attention(q, cache, table, _ints(lengths), dtype=dtype)
        assert not out[1].any() and not out[6].any()


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim,block", [(64, 32), (128, 16), (128, 64), (128, 128), (256, 16)])
def test_attention_of_chunks(dim, block, dtype, kind):
    """Ragged chunks beside single tokens, none and a whole prompt, over every row count around a tile."""
    for kv_heads, group in ((1, 1), (2, 4), (1, 3)):
        sizes = [(70, 70), (200, 1), (5, 5), (0, 0), (129, 2), (300, 131), (64, 64), (1, 1), (257, 33), (40, 17)]
        lengths, counts = [n for n, _ in sizes], [m for _, m in sizes]
        starts = [sum(counts[:i]) for i in range(len(counts) + 1)]
        blocks = sum(-(-n // block) for n in lengths) + 2
        cache, table = _random_cache(blocks, kv_heads, block, dim, kind, 5), _table(lengths, block, blocks, 6)
        _spoil(cache, table, lengths, block)
        q, _, _ = _qkv(starts[-1], kv_heads * group, kv_heads, dim, dtype, 7)
        _check_attention(q, cache, table, _ints(lengths), _ints(starts), dtype=dtype)
        if group == 4:
            _check_attention(q, cache, table, _ints(lengths), _ints(starts), window=37, dtype=dtype)
            _check_attention(q, cache, table, _ints(lengths), _ints(starts), window=1, scale=0.3, dtype=dtype)


@pytest.mark.parametrize("dim,dtype", [(64, "bfloat16"), (128, "float16"), (256, "bfloat16"), (64, "float32"), (128, "float32")])
def test_attention_of_short_prompts_one_after_the_other(dim, dtype):
    """More of them than there are CTAs: every one begins items while its warps still have results of the ones before to store."""
    sizes = [(64 + 7 * (i % 3), 64 + 5 * (i % 4) - 20) for i in range(120)]
    lengths, counts = [n for n, _ in sizes], [m for _, m in sizes]
    starts = [sum(counts[:i]) for i in range(len(counts) + 1)]
    blocks = sum(-(-n // 32) for n in lengths)
    cache, table = _random_cache(blocks, 4, 32, dim, "int8", 11), _table(lengths, 32, blocks, 12)
    q, _, _ = _qkv(starts[-1], 4, 4, dim, dtype, 13)
    first = kernels.kv_cache_attention(q, cache, table, _ints(lengths), _ints(starts))
    for _ in range(10):
        assert torch.equal(kernels.kv_cache_attention(q, cache, table, _ints(lengths), _ints(starts)), first)
    _check_attention(q, cache, table, _ints(lengths), _ints(starts), dtype=dtype)


@pytest.mark.parametrize("window", [1, 15, 16, 17, 64, 100, 129, 5000])
def test_attention_windows(window):
    lengths = [1, 16, 63, 128, 500, 1111]
    blocks = 200
    cache, table = _random_cache(blocks, 2, 16, 128, "int8", 3), _table(lengths, 16, blocks, 4)
    _spoil(cache, table, lengths, 16)
    # blocks that are out of the window altogether may be gone: their entries are anything
    gone = table.clone()
    for b, n in enumerate(lengths):
        gone[b, :max(0, n - window) // 16] = 1 << 30
    q, _, _ = _qkv(len(lengths), 8, 2, 128, "float16", 5)
    want = _check_attention(q, cache, table, _ints(lengths), window=window, dtype="float16")
    got = kernels.kv_cache_attention(q, cache, gone, _ints(lengths), window=window)
    assert kernels.device_status() == 0 and torch.equal(want, got)


def test_attention_of_a_long_cache_is_split_and_joined():
    """One sequence on all SMs, a second one behind it; the same answer every time."""
    for dtype in DTYPES:
        lengths = [20000, 3, 4097]
        cache, table = _random_cache(400, 2, 64, 128, "float8_e4m3fn", 3), _table(lengths, 64, 400, 4)
        q, _, _ = _qkv(3, 8, 2, 128, dtype, 5, scale=2.0)
        out = _check_attention(q, cache, table, _ints(lengths), dtype=dtype)
        for _ in range(5):
            assert torch.equal(out, kernels.kv_cache_attention(q, cache, table, _ints(lengths)))


def test_attention_past_32_bit_offsets():
    """A block whose bytes lie past 2^31 and one past 2^32."""
    block, heads, dim = 128, 8, 256
    blocks = (1 << 32) // (block * heads * dim) + 40
    cache = kernels.kv_cache(blocks, heads, block, dim, "int8")
    small = _random_cache(4, heads, block, dim, "int8", 1)
    ids = [blocks - 1, 3, (1 << 31) // (block * heads * dim) + 7, blocks - 30]
    for big, few in zip(cache, small):
        big.view(torch.uint8 if big.dtype == torch.int8 else torch.float32)[ids] = few.view(torch.uint8 if big.dtype == torch.int8 else torch.float32)
    q, k, v = _qkv(1, 16, heads, dim, "bfloat16", 2)
    lengths = _ints([500])
    few = kernels.kv_cache_attention(q, small, _ints([[0, 1, 2, 3]]), lengths)
    assert torch.equal(few, kernels.kv_cache_attention(q, cache, _ints([ids]), lengths))
    for c, t in ((cache, _ints([ids])), (small, _ints([[0, 1, 2, 3]]))):
        kernels.kv_cache_write(c, k, v, t, lengths)
    a = kernels.kv_cache_read(cache, _ints([ids]), _ints([0, 500]), 500)
    b = kernels.kv_cache_read(small, _ints([[0, 1, 2, 3]]), _ints([0, 500]), 500)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]) and kernels.device_status() == 0


@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_strides_and_alignment(dtype):
    """Rows cut out of wider ones at odd places, heads in another order."""
    lengths, starts = _ints([40, 90]), _ints([0, 3, 30])
    cache, table = _random_cache(20, 2, 16, 64, "int8", 3), _table([40, 90], 16, 20, 4)
    for pad in (0, 1, 3, 8):
        q, _, _ = _qkv(30, 8, 2, 64, dtype, 5, pad=pad)
        _check_attention(q, cache, table, lengths, starts, dtype=dtype)
        _check_attention(q.flip(1).transpose(0, 1).contiguous().transpose(0, 1), cache, table, lengths, starts, dtype=dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", TYPES)
def test_attention_range_of_values(kind, dtype):
    """Scores of hundreds, rows of q of very different size, scales from 2^-60 to 2^20 in one sequence, zeros."""
    lengths = [700]
    cache, table = _random_cache(12, 1, 64, 128, kind, 3), _table(lengths, 64, 12, 4)
    q, _, _ = _qkv(1, 8, 1, 128, dtype, 5)
    q = q * torch.tensor([0.0, 1e-4, 0.1, 1.0, 3.0, 10.0, 30.0, 60.0], device=DEV, dtype=q.dtype)[None, :, None]
    _check_attention(q, cache, table, _ints(lengths), dtype=dtype)
    cache.v_scale.copy_(torch.exp2(torch.tensor([-60, -30, -12, -4, 0, 3, 10, 6, -20, 0, 1, 2], device=DEV, dtype=torch.float32))[:, None] / 128)
    _check_attention(q, cache, table, _ints(lengths), dtype=dtype)
    cache.v_scale.zero_()
    assert not kernels.kv_cache_attention(q, cache, table, _ints(lengths)).any()


@pytest.mark.parametrize("rows", [1, 40, 200])
def test_attention_non_finite(rows):
    """A block that reads as NaN: rows that see it are NaN, rows that do not are what they are without it."""
    n, block = 400, 32
    cache, table = _random_cache(16, 2, block, 128, "int8", 3), _table([n, 50], block, 16, 4)
    q, _, _ = _qkv(rows + 1, 8, 2, 128, "bfloat16", 5)
    lengths, starts = _ints([n, 50]), _ints([0, rows, rows + 1])
    for which in (2, 3):
        for window in (0, 20):
            clean = kernels.kv_cache_attention(q, cache, table, lengths, starts, window=window)
            assert torch.isfinite(clean).all()
            spoilt = [t.clone() for t in cache]
            at = 9                                               # positions 288 .. 319, of kv head 1
            spoilt[which][int(table[0, at]), 1] = float("nan")
            got = kernels.kv_cache_attention(q, spoilt, table, lengths, starts, window=window)
            p = torch.arange(n - rows, n, device=DEV)
            sees = p >= at * block
            if window:
                sees &= p - window + 1 < (at + 1) * block
            assert torch.isnan(got[:rows][sees][:, 4:]).all()
            hidden = torch.cat([~sees, torch.ones(1, dtype=torch.bool, device=DEV)])
            assert torch.equal(got[hidden], clean[hidden]) and torch.equal(got[:, :4], clean[:, :4])
    q[:, 3] = float("nan")
    q[:, 6, 5] = float("inf")
    got = kernels.kv_cache_attention(q, cache, table, lengths, starts)
    assert not torch.isfinite(got[:, [3, 6]]).any() and torch.isfinite(got[:, [0, 1, 2, 4, 5, 7]]).all()


# ---------------------------------------------------------------------------------------------- write and read
def _check_written(before, cache, found):
    for (which, i, h), (scale, slot, old, new) in found.items():
        got = float(cache[2 + which][i, h])
        if cache[0].dtype == torch.int8:
            assert abs(got - scale) <= 2.0 ** -22 * scale, (got, scale)
        else:
            assert got == scale
        value = cache[which][i, h, :slot + len(new)].cpu().to(torch.float32).double() * got
        want = torch.cat([old, new])
        if cache[0].dtype == torch.int8:
            bound = torch.full_like(want, (0.5 + 2.0 ** -16) * got)
        else:
            bound = torch.maximum(want.abs() * 2.0 ** -4, torch.full_like(want, 2.0 ** -10 * got)) * (1 + 2.0 ** -20)
        if got == float(before[2 + which][i, h]):
            bound[:slot] = 0                                     # nothing has grown: as they were
        assert ((value - want).abs() <= bound).all(), (which, i, h)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("block,dim,heads", [(16, 64, 3), (32, 128, 2), (128, 256, 1), (64, 128, 8)])
def test_write(block, dim, heads, kind, dtype):
    """Single tokens at every kind of slot, then chunks over several blocks; what is not written stays."""
    one = [1, block, block + 1, 0, 2 * block - 1, 77]
    sizes = [(3 * block, 3 * block), (2 * block + 1, 1), (100, 37), (0, 0), (block, 1), (block + 5, block), (3, 2)]
    for lengths, counts in ((one, None), ([n for n, _ in sizes], [m for _, m in sizes])):
        rows = len(lengths) if counts is None else sum(counts)
        starts = None if counts is None else _ints([sum(counts[:i]) for i in range(len(counts) + 1)])
        blocks = sum(-(-n // block) for n in lengths) + 2
        for scale in (0.01, 1.0, 30.0):
            cache, table = _random_cache(blocks, heads, block, dim, kind, 3), _table(lengths, block, blocks, 4)
            _, k, v = _qkv(rows, heads, heads, dim, dtype, 5, scale=scale)
            before = [t.clone() for t in cache]
            found = D.write(before, k, v, table, _ints(lengths), starts)
            assert kernels.kv_cache_write(cache, k, v, table, _ints(lengths), starts) is cache
            assert kernels.device_status() == 0
            _check_written(before, cache, found)
            for which in (0, 1):
                same = torch.ones(cache[which].shape[:3], dtype=torch.bool, device=DEV)
                for (w, i, h), (_, slot, _, new) in found.items():
                    if w == which:
                        same[i, h, :slot + len(new)] = False
                assert torch.equal(cache[which].view(torch.uint8)[same], before[which].view(torch.uint8)[same])
                kept = torch.ones_like(cache[2 + which], dtype=torch.bool)
                for w, i, h in found:
                    if w == which:
                        kept[i, h] = False
                assert torch.equal(cache[2 + which][kept], before[2 + which][kept])
            again = [t.clone() for t in cache]
            kernels.kv_cache_write(cache, k, v, table, _ints(lengths), starts)             # the same tokens once more change nothing
            assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(again, cache))


@pytest.mark.parametrize("kind", TYPES)
def test_write_token_by_token(kind):
    """A block filled one token at a time: its scale ends where writing all at once puts it, values within a step for each time it grew."""
    block, dim = 64, 128
    _, k, v = _qkv(block, 1, 1, dim, "float32", 5)
    k, v = (t * torch.linspace(0.05, 2.0, block, device=DEV)[:, None, None] for t in (k, v))
    table = _ints([[1]])
    steps, whole = kernels.kv_cache(3, 1, block, dim, kind), kernels.kv_cache(3, 1, block, dim, kind)
    steps.k_scale.fill_(1e30)                                    # of a sequence that is gone
    growths = 0
    for n in range(1, block + 1):
        last = float(steps.k_scale[1, 0])
        kernels.kv_cache_write(steps, k[n - 1:n], v[n - 1:n], table, _ints([n]))
        growths += n > 1 and float(steps.k_scale[1, 0]) > last
    kernels.kv_cache_write(whole, k, v, table, _ints([block]), _ints([0, block]))
    assert torch.equal(steps.k_scale[1], whole.k_scale[1]) and torch.equal(steps.v_scale[1], whole.v_scale[1]) and growths > 3
    got, _ = kernels.kv_cache_read(steps, table, _ints([0, block]), block, "float32")
    scale = float(steps.k_scale[1, 0])
    bound = scale * (0.51 * (growths + 1)) if kind == "int8" else k.abs() * 2.0 ** -4 * 1.001 + 2.0 ** -10 * scale * (growths + 1)
    assert ((got - k).abs() <= bound).all()


def test_write_range_of_values():
    """Zeros, the smallest and largest numbers, ties, values that are not finite."""
    for kind in TYPES:
        cache = kernels.kv_cache(8, 1, 16, 64, kind)
        table = _ints([[i] for i in range(8)])
        x = torch.zeros(8, 1, 64, device=DEV)
        x[1] = 1e-44
        x[2] = 3e38
        x[3, 0, :4] = torch.tensor([127.0, 0.5, 1.5, -2.5], device=DEV)
        x[4, 0, 7] = float("inf")
        x[5, 0, 9] = float("nan")
        x[6, 0, ::2], x[6, 0, 1::2] = 1e30, -1e-30
        x[7] = 448.0
        kernels.kv_cache_write(cache, x, x, table, _ints([1] * 8))
        k, v = kernels.kv_cache_read(cache, table, None, 8, "float32")
        assert torch.equal(k.isnan(), v.isnan())
        assert not k[0].any() and torch.isnan(k[4]).all() and torch.isnan(k[5]).all()
        good = [2, 3, 6, 7]
        step = cache.k_scale[good].view(-1, 1, 1) if kind == "int8" else x[good].abs() * 2.0 ** -3 + 2.0 ** -9 * cache.k_scale[good].view(-1, 1, 1)
        assert ((k[good] - x[good]).abs() <= 0.5001 * step).all() and (k[1] - x[1]).abs().max() < 2e-38
        if kind == "int8":
            assert k[3, 0, :4].tolist() == [127.0, 0.0, 2.0, -2.0]
        else:
            assert torch.equal(k[7], x[7]) and float(cache.k_scale[7]) == 1.0
        kernels.kv_cache_write(cache, x[:6], x[:6], table[:6], _ints([2] * 6))             # a second token: NaN stays, the others take theirs
        k, _ = kernels.kv_cache_read(cache, table, None, 8, "float32", begins=_ints([1] * 8))
        assert torch.isnan(k[4]).all() and torch.isnan(k[5]).all() and torch.isfinite(k[:4]).all() and kernels.device_status() == 0


@pytest.mark.parametrize("dtype", DTYPES)
def test_write_strides_and_alignment(dtype):
    lengths, starts = _ints([20, 9]), _ints([0, 20, 27])
    want = None
    _, k0, v0 = _qkv(27, 1, 3, 64, dtype, 9)
    for pad in (0, 1, 8):
        wide = torch.empty(27, 2 * 3 * 64 + 2 * pad, dtype=k0.dtype, device=DEV)
        k, v = wide[:, pad:pad + 192].unflatten(1, (3, 64)), wide[:, pad + 192:2 * 192 + pad].unflatten(1, (3, 64))
        k.copy_(k0)
        v.copy_(v0)
        for kk, vv in ((k, v), (k.transpose(0, 1).contiguous().transpose(0, 1), v)):
            cache = kernels.kv_cache(6, 3, 16, 64)
            kernels.kv_cache_write(cache, kk, vv, _ints([[0, 1], [2, -1]]), lengths, starts)
            want = want or cache
            assert all(torch.equal(a, b) for a, b in zip(want, cache))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("block,dim,heads", [(16, 64, 3), (64, 128, 2), (128, 256, 1)])
def test_read(block, dim, heads, kind, dtype):
    lengths, first = [1, 0, block, 3 * block - 1, 200], [0, 0, 3, block, 199]
    cache, table = _random_cache(40, heads, block, dim, kind, 3), _table(lengths, block, 40, 4)
    counts = [n - f for n, f in zip(lengths, first)]
    starts = _ints([sum(counts[:i]) for i in range(len(counts) + 1)])
    k, v = kernels.kv_cache_read(cache, table, starts, sum(counts), dtype, begins=_ints(first))
    assert kernels.device_status() == 0
    for which, got in ((0, k), (1, v)):
        want = torch.cat([D.cached(cache, table, b, which, n)[f:] for b, (n, f) in enumerate(zip(lengths, first))])
        bound = (D.UNIT[dtype] + 2.0 ** -24) * want.abs() + D.SMALLEST[dtype]
        assert ((got.cpu().double() - want).abs() <= bound).all()
    out = tuple(torch.full_like(t, 7) for t in (k, v))
    assert kernels.kv_cache_read(cache, table, starts, sum(counts), dtype, begins=_ints(first), out=out)[0] is out[0]
    assert torch.equal(out[0], k) and torch.equal(out[1], v)


def test_entries_outside_of_the_cache():
    """Table entries, lengths and starts that point nowhere: left out, told by the status word, nothing else touched."""
    cache, table = _random_cache(12, 2, 16, 64, "int8", 3), _table([30, 30], 16, 12, 4)
    q, k, v = _qkv(2, 4, 2, 64, "float16", 5)
    good = kernels.kv_cache_attention(q, cache, table, _ints([30, 30]))
    assert kernels.device_status() == 0
    for entry in (-1, 12, 1 << 30, -(1 << 31)):
        bad = table.clone()
        bad[1, 1] = entry
        before = [t.clone() for t in cache]
        kernels.kv_cache_write(cache, k, v, bad, _ints([0, 30]))
        assert kernels.device_status() == 10 and all(torch.equal(a, b) for a, b in zip(before, cache))
        out = kernels.kv_cache_attention(q, cache, bad, _ints([30, 30]))
        assert kernels.device_status() == 10 and torch.equal(out[0], good[0]) and torch.isfinite(out).all()
        got, _ = kernels.kv_cache_read(cache, bad, _ints([0, 30, 60]), 60)
        assert kernels.device_status() == 10 and not got[46:].any() and got[:46].any(-1).all()
    for lengths, starts in (([30, 1000], None), ([30, 30], [0, 1, 7]), ([30, 30], [0, -3, 2]), ([30, 1 << 30], None)):
        before = [t.clone() for t in cache]
        out = kernels.kv_cache_attention(q, cache, table, _ints(lengths), None if starts is None else _ints(starts))
        assert kernels.device_status() == 10
        kernels.kv_cache_write(cache, k, v, table, _ints(lengths), None if starts is None else _ints(starts))
        assert kernels.device_status() == 10
        if starts is None:
            assert torch.equal(out[0], good[0])
        for t, s in zip(cache, before):
            t.copy_(s)
    assert kernels.device_status() == 0


def test_other_streams_and_graphs():
    """The calls run on the stream that they are given, side by side with others, and from a captured graph."""
    lengths = [5000, 70, 900]
    cache, table = _random_cache(150, 2, 64, 128, "int8", 3), _table(lengths, 64, 150, 4)
    q, k, v = _qkv(3, 8, 2, 128, "bfloat16", 5)
    n = _ints(lengths)
    kernels.kv_cache_write(cache, k, v, table, n)
    want = kernels.kv_cache_attention(q, cache, table, n)
    streams = [torch.cuda.Stream() for _ in range(4)]
    outs = [torch.empty_like(q) for _ in range(40)]
    torch.cuda.synchronize()
    for i, out in enumerate(outs):
        kernels.kv_cache_attention(q, cache, table, n, out=out, stream=streams[i % 4])
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
    side = torch.cuda.Stream()
    out, x = torch.empty_like(q), torch.empty_like(q)
    w = torch.ones(128, device=DEV)
    with torch.cuda.stream(side):
        kernels.kv_cache_attention(q, cache, table, n, out=out)
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            kernels.kv_cache_write(cache, k, v, table, n)
            kernels.kv_cache_attention(q, cache, table, n, out=out)
            kernels.rms_norm(out, w, out=x)
    for _ in range(3):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.isfinite(x).all()
    assert kernels.device_status() == 0


def test_refusals():
    cache, table = _random_cache(12, 2, 16, 64, "int8", 3), _table([30, 30], 16, 12, 4)
    q, k, v = _qkv(2, 4, 2, 64, "float16", 5)
    n = _ints([30, 30])

    def refused(call, *args, **kwargs):
        with pytest.raises(ValueError):
            call(*args, **kwargs)

    attention, write, read = kernels.kv_cache_attention, kernels.kv_cache_write, kernels.kv_cache_read
    refused(attention, q.cpu(), cache, table, n)
    refused(attention, q[:, :3], cache, table, n)                                        # no multiple of the cached heads
    refused(attention, q.double(), cache, table, n)
    refused(attention, q[..., :32], cache, table, n)
    refused(attention, q.transpose(1, 2).contiguous().transpose(1, 2), cache, table, n)  # head_dim apart
    refused(attention, q, cache, table.long(), n)
    refused(attention, q, cache, table, n.long())
    refused(attention, q, cache, table, n[:1])
    refused(attention, q, cache, table[:1], n[:1])                                       # two rows, one sequence, no starts
    refused(attention, q, cache, table, n, n)                                            # starts of another length
    refused(attention, q, cache, table, n, window=-1)
    refused(attention, q, cache, table, n, out=torch.empty_like(q)[:, :2])
    refused(attention, q, (cache.k, cache.v, cache.k_scale, cache.v_scale.half()), table, n)
    refused(attention, q, (cache.k, cache.v.view(torch.float8_e4m3fn), cache.k_scale, cache.v_scale), table, n)
    refused(attention, q, (cache.k[:, :, ::2], cache.v, cache.k_scale, cache.v_scale), table, n)
    refused(write, cache, k, v[:1], table, n)
    refused(write, cache, k, v.float(), table, n)
    refused(write, cache, k[:, :1], v[:, :1], table, n)
    refused(read, cache, table, _ints([0, 3, 5]), 5, "float64")
    refused(read, cache, table, _ints([0, 3, 5]), 5, begins=_ints([0]))
    refused(read, cache, table, _ints([0, 3, 5]), 5, out=(torch.empty(5, 2, 64, device=DEV),) * 2)
    refused(kernels.kv_cache, 4, 2, 24, 64)
    refused(kernels.kv_cache, 4, 2, 16, 96)
    refused(kernels.kv_cache, 4, 2, 16, 64, "int4")
    # nothing to do is no error
    none = torch.empty(0, 4, 64, device=DEV, dtype=torch.float16)
    assert attention(none, cache, table, n, _ints([0, 0, 0])).shape == none.shape
    assert read(cache, table, _ints([0, 0, 0]), 0)[0].shape == (0, 2, 64)
    write(cache, none[:, :2], none[:, :2], table, n, _ints([0, 0, 0]))
    assert kernels.device_status() == 0
