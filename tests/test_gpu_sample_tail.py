"""The choice of tokens far down in the order: one confident logit and many that are each 2^-23 to 2^-41 of it, of which one number in some millions takes one.  Against the definition in
whole numbers: weights of extended precision in multiples of 2^-110, whose sums and borders are exact.

Bounds.  A weight is off by 2^-44 of itself at most (16-bit logits: float64, |x| <= 40, 2^-52 of it in the argument; float32: 2^-45 of rounding, an argument within 2^-47, a
polynomial of 2^-50), the largest not at all; a running sum has less than 32 float64 roundings of 2^-53 of the whole.  So a sum is within 2^-44 of what is not the largest, and 2^-48 of the whole; tokens
are equal unless twice that reaches a border.  Probabilities are a quotient of such numbers, rounded to float32: 2^-24 of themselves, and 2^-42."""
from bisect import bisect_left, bisect_right
from fractions import Fraction
from itertools import accumulate
from math import ceil, floor

import numpy as np
import pytest
import torch

from dinoml_v2_b200 import kernels

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
DTYPES = ("bfloat16", "float16", "float32")
BITS = 110


class Definition:
    def __init__(self, x, temperature):
        values = x.double().numpy()
        order = np.argsort(-values, kind="stable")
        values = values[order].astype(np.longdouble)
        exact = np.exp((values - values[0]) / np.longdouble(temperature))
        self.order, self.weights = order.tolist(), [int(w) for w in np.ldexp(exact, BITS)]
        self.total = sum(self.weights)
        ones = sum(w == 1 << BITS for w in self.weights) << BITS
        self.off = 2 * (Fraction(self.total - ones, 1 << 44) + Fraction(self.total, 1 << 48))      # how far two sums may be off together

    def choose(self, u, top_k=0, top_p=1.0, min_p=0.0):
        """(token, share of it), or None where a border is too near."""
        w, near = self.weights[:top_k] if top_k else self.weights, False
        run = list(accumulate(w))
        if top_p < 1:
            wanted = Fraction(top_p) * run[-1]
            n = bisect_left(run, ceil(wanted)) + 1
            near |= any(abs(run[i] - wanted) <= self.off for i in {max(0, n - 2), n - 1})
            w, run = w[:n], run[:n]
        if min_p > 0:
            border = Fraction(min_p) * (1 << BITS)
            n = max(1, bisect_right(w, -ceil(border), key=lambda v: -v))
            near |= any(abs(v - border) <= border / 2 ** 44 for v in w[max(0, n - 1):n + 1] if v != 1 << BITS)
            w, run = w[:n], run[:n]
        target = Fraction(u) * run[-1]
        at = bisect_right(run, floor(target))
        near |= any(abs(run[i] - target) <= self.off for i in {max(0, at - 1), at})
        return None if near else (self.order[at], float(Fraction(w[at], run[-1])))


def _check(x, u, most_near=1, temperature=1.0, **settings):
    """Rows of u with the same logits."""
    numbers = torch.tensor(u, device=DEV)
    u = numbers.tolist()
    tokens, probabilities = kernels.sample(x.expand(len(u), -1).contiguous(), numbers, temperature=temperature, **settings)
    definition = Definition(x[0].cpu(), torch.tensor(temperature).item())
    single = {name: v if name == "top_k" else torch.tensor(v).item() for name, v in settings.items()}
    near, tail = 0, 0
    for i, number in enumerate(u):
        want = definition.choose(number, **single)
        if want is None:
            near += 1
            continue
        assert int(tokens[i]) == want[0], (i, number, int(tokens[i]), want)
        assert abs(float(probabilities[i]) - want[1]) <= want[1] * (2.0 ** -24 + 2.0 ** -42) + 2.0 ** -149, (i, number, float(probabilities[i]), want)
        tail += want[1] < 2.0 ** -20
    assert near <= most_near and kernels.device_status() == 0
    return tail


LAST = [1 - k * 2.0 ** -24 for k in (1, 2, 3, 5, 8, 13)]


def _peak(vocabulary, height, spread, dtype, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    x = spread * torch.randn(1, vocabulary, device=DEV, generator=g)
    x[0, vocabulary // 3] = height
    return x.to(getattr(torch, dtype))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocabulary,depth", [(200003, 28.0), (262144, 26.0), (128256, 24.0), (50001, 22.0), (32000, 20.0), (5000, 18.0)])
def test_many_equals_below_one(vocabulary, depth, dtype):
    x = torch.zeros(1, vocabulary, device=DEV)
    x[0, vocabulary // 3] = depth
    assert _check(x.to(getattr(torch, dtype)), LAST) >= 1
    _check(x.to(getattr(torch, dtype)), LAST, top_k=3 * vocabulary // 4, top_p=1 - 2.0 ** -24, min_p=2.0 ** -45)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocabulary,height,spread", [(128256, 25.0, 3.0), (128256, 16.0, 1.0), (128256, 24.0, 0.1), (262144, 28.0, 1.0), (40000, 21.0, 1.5)])
def test_a_peak_and_its_tail(vocabulary, height, spread, dtype):
    x = _peak(vocabulary, height, spread, dtype, vocabulary)
    assert _check(x, LAST) >= 1
    _check(x, LAST, top_k=vocabulary // 3)
    _check(x, LAST, top_p=1 - 2.0 ** -22)
    _check(x, LAST, min_p=float(np.exp(-height)))                                         # about half of the tail
    _check(x, LAST, top_k=vocabulary // 2, top_p=1 - 2.0 ** -23, min_p=float(np.exp(-height - spread)))
    _check((x.float() * 2).to(x.dtype), LAST, temperature=2.0)


@pytest.mark.parametrize("dtype", DTYPES)
def test_tails_with_weights_in_every_range(dtype):
    """Logits from the largest down to 60 below it: sums of ranges whose weights are of very different sizes."""
    g = torch.Generator(device=DEV)
    g.manual_seed(8)
    for power in (1.0, 0.25):
        x = (-60 * torch.rand(1, 150001, device=DEV, generator=g) ** power).to(getattr(torch, dtype))
        u = [0.0, 0.1, 0.5, 0.9, 0.999, 1 - 2.0 ** -15, *LAST]
        _check(x, u, 2)
        _check(x, u, 2, top_k=100001, min_p=1e-9)
        _check(x, u, 2, top_p=1 - 2.0 ** -20, temperature=1.7)


@pytest.mark.parametrize("temperature,largest,others", [(1e38, 3e38, [-3e38, -1e38, 0.0, 1e38]), (3e38, 3.4e38, [-3.4e38, 1.0]), (1e-38, 2e-38, [0.0, 1e-38, -2e-38, 1.9e-38]),
                                                        (2e-45, 3e-45, [0.0, 1.4e-45, -7e-45]), (1e-40, 1e-39, [0.0, 9.9e-40, -5e-40])])
def test_temperatures_at_the_ends(temperature, largest, others):
    """Differences that pass float32, quotients that do not."""
    values = torch.tensor([largest] + others).repeat(401)
    values[0] = largest
    assert _check(values[None].to(DEV), [0.0, 0.2, 0.4, 0.6, 0.8, 0.97], 2, temperature=temperature) == 0
