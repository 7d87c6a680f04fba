"""TEST INFRASTRUCTURE ONLY - the operators between the quantized linears, from their formulas in float64 (tensors on the CPU)."""
from __future__ import annotations

import math

import torch

UNIT = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}          # unit roundoff
SMALLEST = {"float32": 2.0 ** -150, "float16": 2.0 ** -25, "bfloat16": 2.0 ** -134}   # half the spacing of the smallest numbers


def cached(cache, table, b, which, count):
    """Keys (0) or values (1) of the first `count` tokens of sequence b: float64 [count, kv_heads, head_dim]."""
    q, scale = cache[which].cpu(), cache[2 + which].cpu().double()
    block = q.shape[2]
    ids = table[b, :-(-count // block)].cpu().long()
    x = q.view(torch.uint8)[ids].view(q.dtype).to(torch.float32).double() * scale[ids][..., None, None]
    return x.permute(0, 2, 1, 3).reshape(-1, q.shape[1], q.shape[3])[:count]


def rows_of(lengths, starts):
    """(first packed row, rows, tokens) of every sequence."""
    lengths = lengths.tolist()
    starts = list(range(len(lengths) + 1)) if starts is None else starts.tolist()
    return [(starts[b], starts[b + 1] - starts[b], n) for b, n in enumerate(lengths)]


def attention(q, cache, table, lengths, starts, scale, window):
    """(out, sum of p |v|, largest |scores| by term) - float64 [rows, heads, head_dim], the same, [rows, heads]: what rounding errors of
    the weights and of the scores are relative to."""
    q = q.cpu().double()
    out, spread, terms = torch.zeros_like(q), torch.zeros_like(q), torch.zeros(q.shape[:2], dtype=torch.float64)
    group = q.shape[1] // cache[0].shape[1]
    for b, (row, count, n) in enumerate(rows_of(lengths, starts)):
        if n <= 0:
            continue
        k, v = cached(cache, table, b, 0, n), cached(cache, table, b, 1, n)
        for j in range(count):
            p = n - count + j
            if p < 0:
                continue
            low = max(0, p - window + 1) if window else 0
            for h in range(q.shape[1]):
                kh, vh = k[low:p + 1, h // group], v[low:p + 1, h // group]
                w = torch.softmax(kh @ q[row + j, h] * scale, 0)
                out[row + j, h], spread[row + j, h] = w @ vh, w @ vh.abs()
                terms[row + j, h] = (kh.abs() @ q[row + j, h].abs()).max() * scale
    return out, spread, terms


def write(cache, k, v, table, lengths, starts):
    """What a write leaves: for every (which, block, head) it comes into, (scale, first slot, [(old values it stood for)], [new values])."""
    block = cache[0].shape[2]
    found = {}
    for b, (row, count, n) in enumerate(rows_of(lengths, starts)):
        first = n - count
        for j in range(max(0, first) // block, -(-n // block)):
            low, high = max(0, first, j * block), min(n, (j + 1) * block)
            if low >= high:
                continue
            i = int(table[b, j])
            for which, x in enumerate((k, v)):
                new = x[row + low - first:row + high - first].cpu().double()
                old = cache[which][i, :, :low - j * block].cpu().to(torch.float32).double() * cache[2 + which][i].cpu().double()[:, None, None]
                for h in range(new.shape[1]):
                    largest = float(new[:, h].abs().max())
                    if cache[0].dtype == torch.int8:
                        wanted = largest / 127
                    else:
                        wanted = 2.0 ** max(-126, math.ceil(math.log2(largest / 448))) if largest else 0.0
                    before = float(cache[2 + which][i, h]) if low > j * block else 0.0
                    found[which, i, h] = (max(before, wanted), low - j * block, old[h], new[:, h])
    return found


def rms_norm(x, weight, eps, residual=None):
    total = x.cpu().double() + (residual.cpu().double() if residual is not None else 0)
    return total / torch.sqrt((total * total).mean(-1, keepdim=True) + eps) * weight.cpu().double(), total
