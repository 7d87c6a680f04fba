"""TEST INFRASTRUCTURE ONLY - the operators at a decode step's ends, from their definitions: float64 and whole numbers, on the CPU, one row or sequence at a time."""
from __future__ import annotations

import math

import torch


def choose(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(token, probability, margin) of one row: margin is how near a sum comes to the border that decides by it, relative to the sums (whole numbers decide exactly)."""
    x = logits.double() + 0.0                                                             # (-0 is 0)
    if bool(x.isnan().any()) or bool((x == -math.inf).all()):
        return -1, 0.0, math.inf
    x, order = torch.sort(x, descending=True, stable=True)
    order = order[x > -math.inf]
    x = x[x > -math.inf]
    if temperature == 0:
        return int(order[0]), 1.0, math.inf
    w = torch.where(x == x[0], 1.0, torch.zeros_like(x) if bool(x[0].isinf()) else torch.exp((x - x[0]) / temperature))
    margin = math.inf
    if top_k > 0:
        w = w[:top_k]
    if top_p < 1:
        run = w.cumsum(0)
        wanted = top_p * float(run[-1])
        keep = max(1, int((run - w < wanted).sum()))
        if wanted > 0 and not bool((w == 1).all()):
            margin = min(margin, float(((run - wanted).abs() / run[-1]).min()))
        w = w[:keep]
    if min_p > 0:
        margin = min([margin, *(w[w < 1] / min_p - 1).abs().tolist()])                     # (one is exact)
        w = w[:max(1, int((w >= min_p).sum()))]
    run = w.cumsum(0)
    target = u * float(run[-1])
    at = min(int((run <= target).sum()), len(w) - 1)
    if u > 0:
        margin = min(margin, float(((run - target).abs() / run[-1]).min()))
    if bool((w == 1).all()):
        margin = math.inf                                                                 # sums of less than 2^18 ones, and their products with 24 bits, are exact
    return int(order[at]), float(w[at] / run[-1]), margin


def rotate(x, weight, positions, frequencies, eps, interleaved, magnitude):
    """float64 [rows, heads, head_dim], and what its roundings are relative to: a pair's length, magnitude included, or a value that stays."""
    y = x.cpu().double()
    if weight is not None:
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + eps) * weight.cpu().double()
    n = frequencies.shape[0]
    angle = positions.cpu().double()[:, None, None] * frequencies.cpu()
    a, b = (y[..., 0:2 * n:2], y[..., 1:2 * n:2]) if interleaved else (y[..., :n], y[..., n:2 * n])
    turned = [magnitude * (a * torch.cos(angle) - b * torch.sin(angle)), magnitude * (b * torch.cos(angle) + a * torch.sin(angle))]
    size = abs(magnitude) * torch.sqrt(a * a + b * b)
    out, spread = y.clone(), y.abs()
    for which, t in enumerate(turned):
        where = slice(which, 2 * n, 2) if interleaved else slice(which * n, (which + 1) * n)
        out[..., where], spread[..., where] = t, size
    return out, spread


class Pool:
    """A pool of blocks as lists: tables, lengths, and the free blocks with the next one last."""

    def __init__(self, blocks, sequences, table_blocks, block_size):
        self.size, self.columns = block_size, table_blocks
        self.tables, self.lengths, self.free = [[] for _ in range(sequences)], [0] * sequences, list(range(blocks))[::-1]

    def _need(self, tokens):
        return -(-tokens // self.size)

    def step(self, new, rows=None, drop=None):
        """(lengths, starts, positions, slots)."""
        kept = [max(0, n - (drop[b] if drop else 0)) for b, n in enumerate(self.lengths)]
        for b in reversed(range(len(kept))):
            while len(self.tables[b]) > self._need(kept[b]):
                self.free.append(self.tables[b].pop())
        available, wanted, wanted_rows = len(self.free), 0, 0
        granted = []
        for b, n in enumerate(new):
            fits = n > 0 and kept[b] + n <= self.columns * self.size
            more = self._need(kept[b] + n) - self._need(kept[b]) if fits else 0
            wanted, wanted_rows = wanted + more, wanted_rows + (n if fits else 0)
            granted.append(n if fits and (more == 0 or wanted <= available) and wanted_rows <= (len(new) if rows is None else rows) else 0)
        out_lengths, starts, positions, slots = [], [0], [], []
        for b, n in enumerate(granted):
            self.lengths[b] = kept[b] + n
            while len(self.tables[b]) < self._need(self.lengths[b]):
                self.tables[b].append(self.free.pop())
            at = list(range(kept[b], kept[b] + n)) or ([-1] if rows is None else [])
            positions += at
            slots += [self.tables[b][p // self.size] * self.size + p % self.size if p >= 0 else -1 for p in at]
            starts.append(starts[-1] + n)
            out_lengths.append(self.lengths[b] if n else 0)
        pad = [-1] * ((len(new) if rows is None else rows) - len(positions))
        return out_lengths, None if rows is None else starts, positions + pad, slots + pad
