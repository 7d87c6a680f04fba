"""The choice of tokens against its definition in float64: vocabularies from one to 262144 and around the kernels' parts, every filter alone and together, ties, zeros of both signs,
infinities, rows that leave nothing, strided and misaligned rows, settings for a batch and for each row.

Tokens are equal unless a running sum comes nearer to a border than its rounding: 16-bit logits are summed in float64, less than 2^18 terms of 2^-52 (exponentials of 2^-51 and arguments
within 2^-46), 2^-33 at the very most; float32 logits in multiples of 2^-45 of the largest weight, half of one off for each of less than 2^18, 2^-28 of the whole at most.  Probabilities are one
quotient of such sums, rounded to float32: 2^-24 and these."""
import pytest
import torch

from dinoml_v2_b200 import kernels
from oracle import decode_ends as E

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
DTYPES = ("bfloat16", "float16", "float32")
BORDER = {"bfloat16": 2.0 ** -33, "float16": 2.0 ** -33, "float32": 2.0 ** -28}


def _logits(rows, vocabulary, dtype, seed, spread=2.0, peaks=10):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    x = spread * torch.randn(rows, vocabulary, device=DEV, generator=g)
    at = torch.randint(0, vocabulary, (rows, min(peaks, vocabulary)), device=DEV, generator=g)
    return x.scatter_add_(1, at, 4 + 6 * torch.rand(at.shape, device=DEV, generator=g)).to(getattr(torch, dtype)), torch.rand(rows, device=DEV, generator=g)


def _of(value, row, none):
    return none if value is None else value[row].item() if isinstance(value, torch.Tensor) else torch.tensor(float(value), dtype=torch.float32).item()


def _check(logits, u, rows=None, **settings):
    tokens, probabilities = kernels.sample(logits, u, **settings)
    assert tokens.dtype == torch.int32 and probabilities.dtype == torch.float32 and tokens.shape == probabilities.shape == u.shape
    near, border = 0, BORDER[str(logits.dtype)[6:]]
    x = logits.cpu()
    for r in range(len(x)) if rows is None else rows:
        want, share, margin = E.choose(x[r], u[r].item(), _of(settings.get("temperature", 1.0), r, 1.0), int(_of(settings.get("top_k"), r, 0)),
                                       _of(settings.get("top_p"), r, 1.0), _of(settings.get("min_p"), r, 0.0))
        if margin <= border:
            near += 1
            continue
        assert int(tokens[r]) == want, (r, int(tokens[r]), want, margin)
        assert abs(float(probabilities[r]) - share) <= share * (2.0 ** -24 + 2.0 ** -26) + 2.0 ** -149, r
    assert near <= 1 and kernels.device_status() == 0


FILTERS = [{}, {"top_k": 1}, {"top_k": 7}, {"top_k": 1000}, {"top_p": 0.3}, {"top_p": 0.9}, {"top_p": 0.999}, {"min_p": 0.02}, {"min_p": 0.5}, {"min_p": 1.0},
           {"top_k": 40, "top_p": 0.8, "min_p": 0.05}, {"top_k": 3, "top_p": 0.99}, {"top_p": 0.6, "min_p": 0.3}, {"temperature": 0.0}, {"temperature": 0.05, "top_k": 500},
           {"temperature": 8.0, "top_p": 0.95}, {"temperature": 1e-30}, {"temperature": 1e30, "top_k": 100}]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocabulary", [1, 2, 7, 31, 257, 1000, 4099, 32000, 50001])
def test_vocabularies(vocabulary, dtype):
    for i, settings in enumerate(FILTERS):
        x, u = _logits(3, vocabulary, dtype, vocabulary + i)
        _check(x, u, **settings)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocabulary", [65528, 65537, 128256, 131072, 200003, 262144])
def test_large_vocabularies(vocabulary, dtype):
    for i, settings in enumerate(({}, {"top_k": 50, "top_p": 0.95, "temperature": 0.8}, {"top_p": 0.99, "temperature": 1.3}, {"min_p": 0.01, "temperature": 1.5})):
        x, u = _logits(2, vocabulary, dtype, vocabulary + i)
        _check(x, u, **settings)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [1, 5, 33, 150, 300])
def test_settings_of_each_row(rows, dtype):
    x, u = _logits(rows, 2003, dtype, rows)
    g = torch.Generator(device=DEV)
    g.manual_seed(rows)
    one = lambda: torch.rand(rows, device=DEV, generator=g)                               # noqa: E731
    _check(x, u, temperature=torch.where(one() < 0.2, 0.0, 0.3 + one()), top_k=(one() * 60).to(torch.int32), top_p=torch.where(one() < 0.3, 1.0, 0.2 + 0.8 * one()),
           min_p=torch.where(one() < 0.5, 0.0, 0.1 * one()))
    _check(x, u, top_k=torch.full((rows,), -3, dtype=torch.int32, device=DEV), top_p=2.0)      # off


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocabulary", [5, 1000, 70001])
def test_equals_come_in_the_order_of_their_indices(vocabulary, dtype):
    x = torch.zeros(8, vocabulary, dtype=getattr(torch, dtype), device=DEV)
    x[:, ::2] = -0.0                                                                      # zero is zero
    u = torch.tensor([0.0, 0.2, 0.4, 0.5, 0.6, 0.8, 0.9, 1 - 2.0 ** -24], device=DEV)
    every = (u.double() * vocabulary).floor().int()                                       # exact: sums of ones
    tokens, probabilities = kernels.sample(x, u)
    assert torch.equal(tokens, every) and torch.allclose(probabilities, torch.tensor(1 / vocabulary, device=DEV), rtol=2.0 ** -23, atol=0)
    k = max(1, vocabulary // 3)
    assert torch.equal(kernels.sample(x, u, top_k=k)[0], (u.double() * k).floor().int())
    kept = torch.ceil(torch.tensor(0.75).double() * vocabulary)
    assert torch.equal(kernels.sample(x, u, top_p=0.75)[0], (u.double() * kept.to(DEV)).floor().int())
    assert torch.equal(kernels.sample(x, u, min_p=1.0)[0], every)
    assert not kernels.sample(x, u, min_p=1.5)[0].any() and not kernels.sample(x, u, top_p=0.0)[0].any()      # the first in any case
    x[:, 2:] = 3.0                                                                        # two lower ones before many equals
    assert torch.equal(kernels.sample(x, u, top_k=vocabulary - 2)[0], 2 + (u.double() * (vocabulary - 2)).floor().int())
    assert (kernels.sample(x, u, temperature=0.0)[0] == 2).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_values_at_the_ends(dtype):
    t = getattr(torch, dtype)
    inf, lowest, nan = float("inf"), torch.finfo(t).min, float("nan")
    rows = [[1.0, -inf, 2.0, -inf, 1.0], [-inf, -inf, -inf, 0.5, -inf], [-inf] * 5, [nan, 1.0, 2.0, 3.0, 4.0], [1.0, 2.0, 3.0, 4.0, -nan], [1.0, inf, 2.0, inf, 3.0],
            [lowest] * 5, [lowest, 0.0, lowest, 0.0, -inf], [inf, -inf, inf, -inf, inf], [torch.finfo(t).max, lowest, 0.0, torch.finfo(t).max, 1.0], [nan, nan, nan, nan, nan],
            [-inf, inf, nan, 0.0, 1.0], [torch.finfo(t).tiny, 0.0, -torch.finfo(t).tiny, -0.0, 0.0]]
    x = torch.tensor(rows, dtype=t, device=DEV)
    x[4, 4] = torch.tensor(nan, dtype=t).neg()
    for number in (0.0, 0.3, 0.7, 0.999):
        u = torch.full((len(rows),), number, device=DEV)
        for settings in FILTERS:
            _check(x, u, **settings)
    tokens, probabilities = kernels.sample(x, u)
    assert tokens[[2, 3, 4, 10, 11]].tolist() == [-1] * 5 and not probabilities[[2, 3, 4, 10, 11]].any()
    wide = torch.full((2, 40000), -inf, dtype=t, device=DEV)                              # one left among many
    wide[0, 39999] = wide[1, 20000] = lowest
    assert kernels.sample(wide, u[:2], top_k=5)[0].tolist() == [39999, 20000]


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_at_any_address(dtype):
    x, u = _logits(6, 3001, dtype, 3)
    want = kernels.sample(x, u, top_p=0.9)
    for pad in (1, 2, 5, 8, 13):
        wide = torch.full((6, 3001 + pad), float("nan"), dtype=x.dtype, device=DEV)       # what lies between the rows is not read
        for at in {0, pad}:
            view = wide[:, at:at + 3001]
            view.copy_(x)
            got = kernels.sample(view, u, top_p=0.9)
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
            wide.fill_(float("nan"))


@pytest.mark.parametrize("dtype", DTYPES)
def test_deep_cuts_and_dense_values(dtype):
    """top_k far down in the tail; logits so close together that float32 needs its last bits; 16-bit values that fill a few codes."""
    x, u = _logits(2, 30011, dtype, 9)
    _check(x, u, top_k=29000, temperature=0.2)
    _check(x, u, top_k=29000, temperature=5.0, top_p=0.7)
    near = (20 + 1e-4 * torch.randn(2, 30011, device=DEV)).to(x.dtype)
    _check(near, u)
    _check(near, u, top_k=15000, top_p=0.5)
    few = torch.randint(0, 3, (2, 30011), device=DEV).to(x.dtype)
    _check(few, u, top_k=11000)
    _check(few, u, top_p=0.9, min_p=0.2)
    _check(few * 1e-3, u, temperature=0.001)


@pytest.mark.parametrize("dtype", DTYPES)
def test_frequencies_are_the_probabilities(dtype):
    """A grid of numbers takes every kept token as often as its share says: the running sums' borders, whatever their order, off by one number at most."""
    x, _ = _logits(1, 500, dtype, 4)
    n = 4000
    u = (torch.arange(n, device=DEV) + 0.5) / n
    tokens, probabilities = kernels.sample(x.expand(n, 500).contiguous(), u, top_k=30, temperature=1.5)
    for token in tokens.unique().tolist():
        mine = tokens == token
        assert abs(int(mine.sum()) - float(probabilities[mine][0]) * n) <= 1 + n * 2.0 ** -22
    assert len(tokens.unique()) >= 10


def test_settings_that_are_none():
    x, u = _logits(4, 1000, "bfloat16", 1)
    nan = float("nan")
    per_row = lambda *v: torch.tensor(v, device=DEV)                                      # noqa: E731
    for settings in ({"temperature": per_row(1.0, nan, -1.0, 1.0)}, {"top_p": per_row(0.5, nan, nan, 0.5)}, {"min_p": per_row(0.5, nan, nan, 0.5)}):
        for t in (torch.bfloat16, torch.float32):
            tokens, probabilities = kernels.sample(x.to(t), u, **settings)
            assert (tokens[1:3] == -1).all() and (tokens[[0, 3]] >= 0).all() and not probabilities[1:3].any()
            assert kernels.device_status() == 10 and kernels.device_status() == 0
    tokens, _ = kernels.sample(x, per_row(nan, 0.5, 0.5, 0.5))
    assert int(tokens[0]) == -1 and (tokens[1:] >= 0).all() and kernels.device_status() == 10
    beside = kernels.sample(x, per_row(-1.0, 0.0, 1.0, 2.0), top_k=5)[0]                  # outside of [0, 1): its ends
    inside = kernels.sample(x, per_row(0.0, 0.0, 1 - 2.0 ** -24, 1 - 2.0 ** -24), top_k=5)[0]
    assert torch.equal(beside, inside) and kernels.device_status() == 0


def test_refusals():
    x, u = _logits(4, 100, "float16", 1)
    for args, kwargs in (((x.cpu(), u), {}), ((x, u.cpu()), {}), ((x, u[:3]), {}), ((x, u.double()), {}), ((x[0], u[:1]), {}), ((x.t(), u), {}), ((x.double(), u), {}), ((x.int(), u), {}),
                         ((x, u), {"temperature": None}), ((x, u), {"temperature": -0.1}), ((x, u), {"top_p": float("nan")}), ((x, u), {"min_p": -1.0}), ((x, u), {"top_k": 2.5}),
                         ((x, u), {"top_k": u}), ((x, u), {"top_p": u[:2]}), ((x, u), {"temperature": u.half()}), ((x, u.view(2, 2)), {}),
                         ((x[:1].expand(4, 100), u), {}), ((torch.zeros(1, 262145, dtype=torch.float16, device=DEV), u[:1]), {})):
        with pytest.raises(ValueError):
            kernels.sample(*args, **kwargs)
    tokens, probabilities = kernels.sample(x[:0], u[:0])
    assert tokens.shape == probabilities.shape == (0,)
    assert kernels.sample(x, u, temperature=1, top_p=1, min_p=0, top_k=1 << 40)[0].shape == (4,)      # whole numbers do


def test_other_streams_and_graphs():
    x, u = _logits(9, 40000, "bfloat16", 6)
    want = kernels.sample(x, u, top_p=0.9)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    got = kernels.sample(x, u, top_p=0.9, stream=stream)
    stream.synchronize()
    assert torch.equal(got[0], want[0])
    graphs = []
    for _ in range(2):                                                                    # nothing is shared: they may run side by side
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = kernels.sample(x, u, top_p=0.9), kernels.sample(x.float(), u, top_p=0.9)
        graphs.append((graph, out, torch.cuda.Stream()))
    torch.cuda.synchronize()
    for _ in range(5):
        for graph, _, s in graphs:
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for _, (a, b), _ in graphs:
        assert torch.equal(a[0], want[0]) and torch.equal(b[0], want[0])
    x.copy_(_logits(9, 40000, "bfloat16", 7)[0])                                          # a replay reads what is there now
    graphs[0][0].replay()
    torch.cuda.synchronize()
    assert torch.equal(graphs[0][1][0][0], kernels.sample(x, u, top_p=0.9)[0])


@pytest.mark.parametrize("dtype", DTYPES)
def test_many_rows_of_large_vocabularies(dtype):
    """More rows than run at once, parts that are counted in several turns, counts past 16 bits, the next row's parts beside each other."""
    rows, vocabulary = 160, 140001
    x, u = _logits(rows, vocabulary, dtype, 12)
    x[3] = 0.5                                                                            # one value for all
    x[5, 1000:] = torch.finfo(x.dtype).min                                                # a mask of the lowest value
    x[7, :70000], x[7, 70000:] = 1.0, -1.0                                                # two, both past 65535
    x[9, :] = -float("inf")
    x[9, 139999] = -3.0
    x[11, ::2], x[11, 1::2] = 0.0, -0.0
    x[13, 0] = float("nan")
    checked = [0, 1, 3, 5, 7, 9, 11, 13, 100, 147, 148, 149, 159]
    for settings in ({}, {"top_k": 100000, "top_p": 0.9}, {"temperature": 3.0, "top_p": 0.99, "min_p": 0.001}):
        _check(x, u, rows=checked, **settings)
    first = kernels.sample(x, u, top_p=0.99, temperature=2.0)
    for _ in range(3):
        again = kernels.sample(x, u, top_p=0.99, temperature=2.0)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [1, 20, 40])
def test_equals_of_several_parts(rows, dtype):
    """Counts past 16 bits only where the parts of a row meet; the chosen one in each of them."""
    x = torch.full((rows, 200003), 2.0, dtype=getattr(torch, dtype), device=DEV)
    x[:, 100000] = 3.0
    u = torch.linspace(0, 0.999, rows, device=DEV)
    for settings in ({}, {"top_k": 150000}, {"top_p": 0.6}, {"temperature": 0.5, "min_p": 0.1}):
        _check(x, u, **settings)
