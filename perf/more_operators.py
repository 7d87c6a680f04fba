"""What a decode loop runs at its two ends and between its steps, as cases that can be timed and compared.

A program that serves a decoder from GGUF weights goes from tokens to tokens.  Around the quantized linears, the cache and the norm it calls

* ``embedding``: `kernels.embedding`, rows of a GGUF table for the step's tokens, times a scale: out = dequantized row * scale;
* ``rotary``: `kernels.rotary`, the root-mean-square norm of every head of q and k (where the model has one) and the rotation by position in the same
  pass: pairs (a, b) become (a cos - b sin, b cos + a sin) with the angle position * frequency;
* ``pool``: `kernels.kv_pool_step`, who has which blocks of the cache: takes tokens away from the ends of sequences (all of a finished request, the rejected ones of
  a speculative step), gives their blocks back, hands out blocks for the new ones, and tells every packed row its position and slot;
* ``sample``: `kernels.sample`, the next token of every row of logits from one given random number, with temperature, top-k, top-p and min-p, and the
  probability that it had.

Tokens are ordered by value, the lowest index first among equals.  Their weights are w = exp((x - largest) / temperature).  top_k keeps the first k, top_p the fewest of
those whose weights are at least p of these, min_p those with w >= min_p; the token is the first whose running sum is above u times the sum of the kept,
its probability its share of that sum (1 where the temperature is zero, which takes the first).
Free blocks are a stack; blocks are given back in the order in which the next step takes them."""
from __future__ import annotations

import math
import random

import torch

own = False

ELEMENT_BYTES = {"float16": 2, "bfloat16": 2, "float32": 4}
BLOCK = {"Q8_0": (32, 34), "Q4_K": (256, 144), "Q6_K": (256, 210)}      # values, bytes
VOCABULARY = 128256
MAX_LOGITS = 256 * VOCABULARY
MAX_ROTATED = 8192 * 40 * 128
MAX_EMBEDDED = 8192 * 8192
MAX_POSITION = 131072


def listed():
    return [
        # one user: the logits of one token, filters as a chat program sets them
        {"name": "sample_one", "kind": "sample", "dtype": "bfloat16", "rows": 1, "vocabulary": VOCABULARY, "temperature": 0.8, "top_k": 50, "top_p": 0.95, "min_p": 0.0,
         "mixed": False},
        # a served batch, every request with settings of its own, greedy ones among them
        {"name": "sample_batch_mixed", "kind": "sample", "dtype": "bfloat16", "rows": 64, "vocabulary": VOCABULARY, "temperature": 0.9, "top_k": 40, "top_p": 0.9,
         "min_p": 0.05, "mixed": True},
        # float32 logits, an odd vocabulary, the temperature alone
        {"name": "sample_f32_odd", "kind": "sample", "dtype": "float32", "rows": 7, "vocabulary": 50001, "temperature": 1.0, "top_k": 0, "top_p": 1.0, "min_p": 0.0,
         "mixed": False},
        # the largest batch, a wide nucleus
        {"name": "sample_large", "kind": "sample", "dtype": "float16", "rows": 256, "vocabulary": VOCABULARY, "temperature": 1.2, "top_k": 0, "top_p": 0.98, "min_p": 0.0,
         "mixed": False},
        # one new token of one user: latency
        {"name": "rotary_one", "kind": "rotary", "dtype": "bfloat16", "rows": 1, "heads": 32, "kv_heads": 8, "head_dim": 128, "rotary": 128, "interleaved": False,
         "norm": "float32", "padded": 0},
        # a long prompt, heads with norms
        {"name": "rotary_prefill", "kind": "rotary", "dtype": "bfloat16", "rows": 2048, "heads": 32, "kv_heads": 8, "head_dim": 128, "rotary": 128, "interleaved": False,
         "norm": "float32", "padded": 0},
        # float32, a part of each head turned, neighbours as pairs, a batch padded to its capture's size
        {"name": "rotary_partial_f32", "kind": "rotary", "dtype": "float32", "rows": 333, "heads": 10, "kv_heads": 5, "head_dim": 256, "rotary": 64, "interleaved": True,
         "norm": "", "padded": 20},
        # a decode step: one token more for every request, behind one that was rejected and is taken back
        {"name": "pool_decode", "kind": "pool", "sequences": 64, "context": 4000, "new": 1, "block": 16, "finished": 0.0, "layout": 11},
        # finished requests leave, prompts come in their places beside decoding ones
        {"name": "pool_prompts", "kind": "pool", "sequences": 256, "context": 8192, "new": 2001, "block": 64, "finished": 0.5, "layout": 12},
        # one token of one user
        {"name": "embedding_one", "kind": "embedding", "qtype": "Q6_K", "dtype": "bfloat16", "tokens": 1, "width": 4096, "vocabulary": VOCABULARY, "scale": 1.0},
        # float32 activations, a width of whole blocks only, scaled by its root
        {"name": "embedding_q8_0_f32", "kind": "embedding", "qtype": "Q8_0", "dtype": "float32", "tokens": 301, "width": 2880, "vocabulary": 32000, "scale": 53.665631},
        # a long prompt through the widest table
        {"name": "embedding_prefill", "kind": "embedding", "qtype": "Q4_K", "dtype": "bfloat16", "tokens": 8192, "width": 8192, "vocabulary": VOCABULARY, "scale": 1.0},
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    """One more case of the same ranges: rows, widths and vocabularies over their logarithms, every type and form."""
    kind = rng.choices(["sample", "rotary", "pool", "embedding"], [40, 25, 15, 20])[0]
    dtype = rng.choices(["bfloat16", "float16", "float32"], [5, 3, 2])[0]
    if kind == "sample":
        rows, vocabulary = _log_int(rng, 1, 256), _log_int(rng, 100, 200000)
        while rows * vocabulary * ELEMENT_BYTES[dtype] > MAX_LOGITS * 2:
            rows = (rows + 1) // 2
        return {"kind": kind, "dtype": dtype, "rows": rows, "vocabulary": vocabulary, "temperature": rng.choice([0.0, 0.2, 0.7, 1.0, 1.0, 1.7]),
                "top_k": rng.choice([0, 0, 1, 20, _log_int(rng, 2, 1000)]), "top_p": rng.choice([1.0, 1.0, 0.5, 0.9, 0.99]), "min_p": rng.choice([0.0, 0.0, 0.01, 0.1]),
                "mixed": rng.random() < 0.4}
    if kind == "rotary":
        head_dim = rng.choice([64, 80, 96, 128, 128, 256])
        kv_heads = rng.choice([1, 2, 4, 5, 8, 8, 16])
        case = {"kind": kind, "dtype": dtype, "rows": _log_int(rng, 1, 8192), "heads": kv_heads * rng.choice([1, 2, 3, 4, 7, 8]), "kv_heads": kv_heads, "head_dim": head_dim,
                "rotary": head_dim if rng.random() < 0.7 else rng.choice([16, 32, head_dim // 2]), "interleaved": rng.random() < 0.4,
                "norm": rng.choice(["", "float32", dtype])}
        while case["rows"] * (case["heads"] + kv_heads) * head_dim * ELEMENT_BYTES[dtype] > MAX_ROTATED * 2:
            case["rows"] = (case["rows"] + 1) // 2
        return {**case, "padded": rng.randint(0, case["rows"] // 4) if rng.random() < 0.3 else 0}
    if kind == "pool":
        new = 1 if rng.random() < 0.5 else _log_int(rng, 2, 2048)
        return {"kind": kind, "sequences": _log_int(rng, 1, 256), "context": max(new, _log_int(rng, 1, 32768)), "new": new, "block": rng.choice([16, 32, 64, 128]),
                "finished": rng.choice([0.0, 0.1, 0.5]) if new > 1 else 0.0, "layout": rng.randrange(1 << 30)}
    qtype = rng.choice(sorted(BLOCK))
    width = max(BLOCK[qtype][0], _log_int(rng, 256, 8192) // BLOCK[qtype][0] * BLOCK[qtype][0])
    tokens = _log_int(rng, 1, 8192)
    while tokens * width * ELEMENT_BYTES[dtype] > MAX_EMBEDDED * 2:
        tokens = (tokens + 1) // 2
    return {"kind": kind, "qtype": qtype, "dtype": dtype, "tokens": tokens, "width": width, "vocabulary": _log_int(rng, 1000, VOCABULARY),
            "scale": rng.choice([1.0, 1.0, round(width ** 0.5, 6)])}


# ----------------------------------------------------------------------------------------------- who is in the batch
def _sequences(case):
    """(tokens before, taken away, new) of each sequence.  A finished request loses all and a prompt of the same number of blocks takes its place; the others lose what a
    step before gave them (a slot that serves nobody has nothing), so that a pass can follow itself."""
    rng, out = random.Random(case["layout"]), []
    for b in range(case["sequences"]):
        context = case["context"] if b == 0 else _log_int(rng, max(1, case["context"] // 8), case["context"])
        if case["sequences"] >= 4 and rng.random() < 0.1:
            out.append((0, 0, 0))
        elif rng.random() < case["finished"]:
            prompt = min(context, case["new"] if b == 0 else _log_int(rng, 1, case["new"]))
            out.append((prompt, 1 << 30, prompt))
        else:
            new = min(context, 1 if case["new"] == 1 else _log_int(rng, 1, min(case["new"], 8)))
            out.append((context, new, new))
    return out


def _blocks(n, block):
    return -(-n // block)


def _expected_rows(case):
    """Different tokens among those of a pass, whose logarithms are uniform."""
    rank = torch.arange(1, case["vocabulary"] + 1, dtype=torch.float64)
    p = torch.log1p(1 / rank) / math.log(case["vocabulary"] + 1)
    return float((1 - (1 - p) ** case["tokens"]).sum())


def work(case):
    if case["kind"] == "sample":
        values = case["rows"] * case["vocabulary"]
        return {"bytes": values * ELEMENT_BYTES[case["dtype"]] + case["rows"] * 12, "flops": 4 * values}
    if case["kind"] == "rotary":
        values = case["rows"] * (case["heads"] + case["kv_heads"]) * case["head_dim"]
        return {"bytes": 2 * values * ELEMENT_BYTES[case["dtype"]] + case["rows"] * 4, "flops": 8 * values}
    if case["kind"] == "pool":
        sizes = _sequences(case)
        rows = sum(new for _, _, new in sizes)
        moved = sum(_blocks(n, case["block"]) - _blocks(max(0, n - drop), case["block"]) for n, drop, _ in sizes)
        return {"bytes": len(sizes) * 24 + moved * 16 + rows * 8, "flops": 4 * rows}
    values, (of, size) = case["tokens"] * case["width"], BLOCK[case["qtype"]]
    return {"bytes": int(_expected_rows(case) * case["width"] // of * size) + values * ELEMENT_BYTES[case["dtype"]] + case["tokens"] * 4, "flops": 3 * values}


# ----------------------------------------------------------------------------------------------- inputs
class _Maker:
    def __init__(self, case, seed):
        self.case, self.dev = case, torch.device("cuda")
        self.generator = torch.Generator(device=self.dev)
        self.generator.manual_seed(int(seed) * 1000 + 29)

    def normal(self, *shape):
        return torch.randn(*shape, device=self.dev, generator=self.generator)

    def uniform(self, *shape):
        return torch.rand(*shape, device=self.dev, generator=self.generator)

    def below(self, high, *shape):
        return torch.randint(0, high, shape, device=self.dev, generator=self.generator)

    def bytes(self, *shape):
        return torch.randint(0, 256, shape, device=self.dev, generator=self.generator, dtype=torch.uint8)

    def ints(self, values):
        return torch.tensor(values, dtype=torch.int32, device=self.dev)

    def halves(self, spread, *shape):
        """Two bytes each of |normal| * spread."""
        return (self.normal(*shape).abs() * spread).to(torch.float16).view(torch.uint8)

    def logits(self):
        """A wide hill of unlikely tokens and some that stand out."""
        c = self.case
        x = 2.0 * self.normal(c["rows"], c["vocabulary"])
        at = self.below(c["vocabulary"], c["rows"], min(30, c["vocabulary"]))
        return x.scatter_add_(1, at, 6 + 8 * self.uniform(*at.shape)).to(getattr(torch, c["dtype"]))

    def table(self):
        c = self.case
        of, size = BLOCK[c["qtype"]]
        x = self.bytes(c["vocabulary"], c["width"] // of, size)
        flat = x.shape[:2]
        if c["qtype"] == "Q8_0":
            x[..., :2] = self.halves(0.01, *flat, 1)
            x[..., 2:][x[..., 2:] == 128] = 129                                           # quants are -127 .. 127
        elif c["qtype"] == "Q4_K":
            x[..., :4] = self.halves(0.005, *flat, 2)
        else:
            x[..., 192:208] = (self.below(128, *flat, 16) - 64).to(torch.int8).view(torch.uint8)
            x[..., 208:] = self.halves(0.002, *flat, 1)
        return x.view(c["vocabulary"], -1)


def _settings(case, make):
    """The four settings, numbers for a whole batch or a tensor with one for each row."""
    names = ("temperature", "top_k", "top_p", "min_p")
    if not case["mixed"]:
        return {n: case[n] for n in names}
    rows = case["rows"]
    pick = make.below(4, 4, rows)
    temperature = case["temperature"] * (0.25 + make.uniform(rows))
    top_p = 1 - (1 - case["top_p"]) * (0.2 + 1.5 * make.uniform(rows))
    return {"temperature": torch.where(pick[0] == 0, torch.zeros_like(temperature), temperature),                    # zero: the largest
            "top_k": torch.where(pick[1] == 0, torch.zeros_like(pick[1]), 1 + make.below(2 * max(1, case["top_k"]), rows)).to(torch.int32),      # zero: all
            "top_p": torch.where(pick[2] == 0, torch.ones_like(top_p), top_p), "min_p": torch.where(pick[3] == 0, case["min_p"], 0.0).to(torch.float32)}


def _positions(case, make):
    """Positions of packed prompts and single tokens, and -1 for the rows that fill the batch up."""
    rows, out = case["rows"] - case["padded"], []
    rng = random.Random(case["rows"] * 7 + case["padded"])
    while len(out) < rows:
        count = rng.choice([1, 1, _log_int(rng, 1, 4096)])
        first = rng.randrange(MAX_POSITION - count)
        out += range(first, first + min(count, rows - len(out)))
    return make.ints(out + [-1] * case["padded"])


def _pool(case, make):
    """Tables with every sequence's blocks in any order and -1 behind, the free ones as a stack, some of them left over."""
    sizes = _sequences(case)
    held = [_blocks(n, case["block"]) for n, _, _ in sizes]
    need = [max(h, _blocks(max(0, n - drop) + new, case["block"])) for h, (n, drop, new) in zip(held, sizes)]
    blocks, widest = sum(need) + 7, max(1, max(need))
    order = torch.randperm(blocks, device=make.dev, generator=make.generator).to(torch.int32)
    table = torch.full((len(sizes), widest), -1, dtype=torch.int32, device=make.dev)
    table[torch.arange(widest, device=make.dev)[None] < make.ints(held)[:, None]] = order[:sum(held)]
    free = torch.full((blocks,), -1, dtype=torch.int32, device=make.dev)
    free[:blocks - sum(held)] = order[sum(held):]
    return table, make.ints([n for n, _, _ in sizes]), free, make.ints([blocks - sum(held)]), case["block"]


def prepare(case, seed):
    make, state = _Maker(case, seed), {"case": case}
    if case["kind"] == "sample":
        state["logits"], state["uniforms"], state["settings"] = make.logits(), make.uniform(case["rows"]), _settings(case, make)
    elif case["kind"] == "rotary":
        d, heads, kv = case["head_dim"], case["heads"], case["kv_heads"]
        fused = make.normal(case["rows"], (heads + 2 * kv) * d).to(getattr(torch, case["dtype"]))
        state["q"], state["k"] = fused[:, :heads * d].view(-1, heads, d), fused[:, heads * d:(heads + kv) * d].view(-1, kv, d)
        state["positions"] = _positions(case, make)
        pair = torch.arange(case["rotary"] // 2, dtype=torch.float64, device=make.dev)
        state["frequencies"] = 500000.0 ** (-2 * pair / case["rotary"])
        state["weights"] = (None, None)
        if case["norm"]:
            state["weights"] = tuple((1 + 0.2 * make.normal(d)).to(getattr(torch, case["norm"])) for _ in range(2))
    elif case["kind"] == "pool":
        sizes = _sequences(case)
        state["pool"] = _pool(case, make)
        state["new"], state["drop"] = make.ints([new for _, _, new in sizes]), make.ints([drop for _, drop, _ in sizes])
        state["rows"] = None if case["new"] == 1 else sum(new for _, _, new in sizes) + 5      # None: one row per sequence; else some to spare
    else:
        state["table"] = make.table()
        rank = torch.exp(make.uniform(case["tokens"]).double() * math.log(case["vocabulary"] + 1)).long() - 1
        state["tokens"] = rank.clamp(0, case["vocabulary"] - 1).to(torch.int32)
    return state


# ----------------------------------------------------------------------------------------------- the calls of a user's program
def _run_own(state):
    from dinoml_v2_b200 import kernels
    case = state["case"]
    if case["kind"] == "sample":
        tokens, probabilities = kernels.sample(state["logits"], state["uniforms"], **state["settings"])
        return {"tokens": tokens, "probabilities": probabilities}
    if case["kind"] == "rotary":
        return kernels.rotary(state["q"], state["k"], state["positions"], state["frequencies"], q_weight=state["weights"][0], k_weight=state["weights"][1],
                              interleaved=case["interleaved"])
    if case["kind"] == "embedding":
        return kernels.embedding(state["tokens"], state["table"], case["qtype"], case["dtype"], scale=case["scale"])
    pool = kernels.KVPool(*state["pool"])
    step = kernels.kv_pool_step(pool, state["new"], state["rows"], drop=state["drop"])
    return {"table": pool.block_table, "held": pool.lengths, "free": pool.free, "free_count": pool.free_count, "lengths": step.lengths, "positions": step.positions,
            "slots": step.slots, **({} if step.starts is None else {"starts": step.starts})}


# ----------------------------------------------------------------------------------------------- the same in elementary operations
def _column(value, rows, dev):
    return value.double()[:, None] if isinstance(value, torch.Tensor) else torch.full((rows, 1), float(value), dtype=torch.float64, device=dev)


def _plain_sample(state):
    case, s = state["case"], state["settings"]
    x, index = torch.sort(state["logits"].double() + 0.0, dim=-1, descending=True, stable=True)      # (+ 0: -0 and 0 are equal)
    rows, dev = len(x), x.device
    temperature, k, p, min_p = (_column(s[n], rows, dev) for n in ("temperature", "top_k", "top_p", "min_p"))
    p, min_p = p.float().double(), min_p.float().double()
    weight = torch.exp((x - x[:, :1]) / torch.where(temperature > 0, temperature.float().double(), torch.ones_like(temperature)))
    rank = torch.arange(x.shape[1], device=dev)[None]
    weight = weight * ((k <= 0) | (rank < k))
    run = weight.cumsum(-1)
    before = torch.cat([torch.zeros_like(run[:, :1]), run[:, :-1]], -1)
    kept = (p >= 1) | (before < p * run[:, -1:])
    kept &= weight >= min_p
    kept |= rank == 0
    weight = weight * kept
    run = weight.cumsum(-1)
    target = state["uniforms"].double()[:, None] * run[:, -1:]
    pick = torch.minimum((run <= target).sum(-1), kept.sum(-1) - 1)
    pick = torch.where(temperature[:, 0] > 0, pick, torch.zeros_like(pick))[:, None]
    share = torch.where(temperature > 0, weight.gather(1, pick) / run[:, -1:], torch.ones_like(temperature))
    return {"tokens": index.gather(1, pick)[:, 0].to(torch.int32), "probabilities": share[:, 0].float()}


def _plain_rotary(state):
    case = state["case"]
    half = case["rotary"] // 2
    angle = state["positions"].double()[:, None] * state["frequencies"]
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    out = []
    for x, w in zip((state["q"], state["k"]), state["weights"]):
        y = x.float()
        if w is not None:
            y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + 1e-5) * w.float()
        if case["interleaved"]:
            a, b = y[..., 0:2 * half:2], y[..., 1:2 * half:2]
            turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
        else:
            a, b = y[..., :half], y[..., half:2 * half]
            turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
        y = torch.cat([turned, y[..., 2 * half:]], -1)
        out.append(torch.where((state["positions"] >= 0)[:, None, None], y, torch.zeros_like(y)).to(x.dtype))
    return tuple(out)


def _plain_pool(state):
    table, lengths, free, free_count, block = state["pool"]
    new, dev = state["new"].long(), table.device
    each = state["rows"] is None
    rows = len(new) if each else state["rows"]
    old = lengths.long()
    kept = (old - state["drop"]).clamp(min=0)
    held, left = (old + block - 1) // block, (kept + block - 1) // block
    column = torch.arange(table.shape[1], device=dev)[None]
    # give back: the last sequence's last block first
    back = held - left
    count = free_count.long()
    available = count + back.sum()
    gone = (column >= left[:, None]) & (column < held[:, None])
    at = count + (back.sum() - back.cumsum(0))[:, None] + held[:, None] - 1 - column
    free[at[gone]] = table[gone]
    table[gone] = -1
    # hand out
    after = kept + new
    wants = (new > 0) & (after <= table.shape[1] * block)
    need = torch.where(wants, (after + block - 1) // block - left, 0)
    granted = wants & ((need == 0) | (need.cumsum(0) <= available)) & (torch.where(wants, new, 0).cumsum(0) <= rows)
    need, new = torch.where(granted, need, 0), torch.where(granted, new, 0)
    taken = (column >= left[:, None]) & (column < (left + need)[:, None])
    at = available - 1 - ((need.cumsum(0) - need)[:, None] + column - left[:, None])
    table[taken] = free[at[taken]]
    lengths.copy_(kept + new)
    free_count.copy_(available - need.sum())
    out = {"table": table, "held": lengths, "free": free, "free_count": free_count, "lengths": torch.where(new > 0, kept + new, 0).to(torch.int32)}
    row = torch.arange(rows, device=dev)
    if each:
        position, b = torch.where(new > 0, kept, -1), row
    else:
        ends = new.cumsum(0)
        out["starts"] = torch.cat([torch.zeros_like(ends[:1]), ends]).to(torch.int32)
        b = (row[:, None] >= ends[None]).sum(1).clamp(max=len(new) - 1)
        position = torch.where(row < ends[-1], kept[b] + row - (ends - new)[b], -1)
    slot = table[b, position.clamp(min=0) // block].long() * block + position % block
    out["positions"], out["slots"] = position.to(torch.int32), torch.where(position >= 0, slot, -1).to(torch.int32)
    return out


def _half(x):
    return x.contiguous().view(torch.float16).float()


def _plain_embedding(state):
    case = state["case"]
    of, size = BLOCK[case["qtype"]]
    x = state["table"][state["tokens"].long()].view(case["tokens"], -1, size)
    if case["qtype"] == "Q8_0":
        y = _half(x[..., :2]) * x[..., 2:].view(torch.int8).float()
    elif case["qtype"] == "Q4_K":
        s, q = x[..., 4:16].int(), x[..., 16:].int().unflatten(-1, (4, 32))
        low, mid, high = s[..., :4], s[..., 4:8], s[..., 8:]
        scale = torch.cat([low & 63, (high & 15) | (low >> 6 << 4)], -1).float()
        least = torch.cat([mid & 63, (high >> 4) | (mid >> 6 << 4)], -1).float()
        q = torch.stack([q & 15, q >> 4], -2).flatten(-3, -2).float()                     # [.., 8, 32]
        y = (_half(x[..., :2]) * scale)[..., None] * q - (_half(x[..., 2:4]) * least)[..., None]
    else:
        low, high = x[..., :128].int().unflatten(-1, (2, 2, 32)), x[..., 128:192].int().unflatten(-1, (2, 1, 32))
        low = torch.stack([low & 15, low >> 4], -3).flatten(-3, -2)                       # [.., 2, 4, 32]
        shift = torch.arange(0, 8, 2, device=x.device)[:, None]
        q = (low | ((high >> shift) & 3) << 4).float() - 32
        scale = _half(x[..., 208:]) * x[..., 192:208].contiguous().view(torch.int8).float()
        y = scale[..., None] * q.reshape(*x.shape[:2], 16, 16)
    return (y.reshape(case["tokens"], -1) * torch.tensor(case["scale"], dtype=torch.float32, device=y.device)).to(getattr(torch, case["dtype"]))


def run(state):
    if own:
        return _run_own(state)
    return {"sample": _plain_sample, "rotary": _plain_rotary, "pool": _plain_pool, "embedding": _plain_embedding}[state["case"]["kind"]](state)


# ----------------------------------------------------------------------------------------------- the definitions in 64 bits
def _setting(value, row, kind):
    value = value[row] if isinstance(value, torch.Tensor) else torch.tensor(value)
    return value.to(kind).item()


def _exact_sample(case, state):
    """Row by row over the different values of the logits, with how often each is there."""
    tokens, shares = [], []
    for row in range(case["rows"]):
        x = state["logits"][row].double() + 0.0
        s = {n: _setting(v, row, torch.int64 if n == "top_k" else torch.float32) for n, v in state["settings"].items()}
        values, counts = torch.unique(x, return_counts=True)
        values, counts = values.flip(0), counts.flip(0).double()
        if s["temperature"] == 0:
            value, place, share = values[0], 0, torch.ones_like(values[0])
        else:
            w = torch.exp((values - values[0]) / s["temperature"])
            ends = counts.cumsum(0)
            if s["top_k"] > 0:
                counts = torch.minimum(counts, (s["top_k"] - (ends - counts)).clamp(min=0))
            mass = (w * counts).cumsum(0)
            if s["top_p"] < 1:                                                            # of every value as many as it takes
                wanted = s["top_p"] * mass[-1] - (mass - w * counts)
                counts = torch.minimum(counts, torch.ceil(torch.where(w > 0, wanted / w.clamp(min=5e-324), 0.0)).clamp(min=0))
            counts = torch.where(w >= s["min_p"], counts, torch.zeros_like(counts))
            counts[0] = counts[0].clamp(min=1)
            mass = (w * counts).cumsum(0)
            target = state["uniforms"][row].double() * mass[-1]
            i = int((mass <= target).sum())
            value, share = values[i], w[i] / mass[-1]
            place = int(min(torch.floor((target - (mass[i] - w[i] * counts[i])) / w[i]).clamp(min=0), counts[i] - 1))
        tokens.append(torch.nonzero(x == value)[place, 0])
        shares.append(share)
    return {"tokens": torch.stack(tokens).to(torch.int32), "probabilities": torch.stack(shares)}


def _exact_rotary(case, state):
    half, out = case["rotary"] // 2, []
    turn = torch.polar(torch.ones((), dtype=torch.float64, device=state["q"].device), torch.outer(state["positions"].double(), state["frequencies"]))
    for x, w in zip((state["q"], state["k"]), state["weights"]):
        y = x.double()
        if w is not None:
            y = w.double() * y / torch.sqrt(y.pow(2).sum(-1, keepdim=True) / case["head_dim"] + 1e-5)
        first, second = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if case["interleaved"] else (slice(0, half), slice(half, 2 * half))
        z = torch.complex(y[..., first], y[..., second]) * turn[:, None]
        y = y.clone()
        y[..., first], y[..., second] = z.real, z.imag
        y[state["positions"] < 0] = 0
        out.append(y)
    return tuple(out)


def _exact_pool(case, state):
    """A stack and lists."""
    table, lengths, free, free_count, block = (x.tolist() if isinstance(x, torch.Tensor) else x for x in state["pool"])
    sizes, rows = _sequences(case), state["rows"]
    count = free_count[0]
    lists = [[i for i in row if i >= 0] for row in table]
    kept = [max(0, n - drop) for n, drop, _ in sizes]
    for b in reversed(range(len(sizes))):
        while len(lists[b]) > _blocks(kept[b], block):
            free[count] = lists[b].pop()
            count += 1
    starts, positions, slots, step = [0], [], [], []
    for b, (_, _, new) in enumerate(sizes):
        while len(lists[b]) < _blocks(kept[b] + new, block):
            count -= 1
            lists[b].append(free[count])
        at = list(range(kept[b], kept[b] + new))
        if rows is None and not at:
            positions.append(-1)
            slots.append(-1)
        positions += at
        slots += [lists[b][p // block] * block + p % block for p in at]
        starts.append(starts[-1] + new)
        step.append(kept[b] + new if new else 0)
    pad = [-1] * ((rows or len(sizes)) - len(positions))
    out = {"table": [row + [-1] * (len(table[0]) - len(row)) for row in lists], "held": [n + new for n, (_, _, new) in zip(kept, sizes)], "free": free, "free_count": [count],
           "lengths": step, "positions": positions + pad, "slots": slots + pad, **({} if rows is None else {"starts": starts})}
    return {name: torch.tensor(x, dtype=torch.int32, device=state["new"].device) for name, x in out.items()}


def _exact_embedding(case, state):
    """Block by block of 32 or 16 values."""
    (of, size), tokens = BLOCK[case["qtype"]], state["tokens"].long()
    x = state["table"][tokens].reshape(-1, size).long()
    half = lambda i: (x[:, i] | x[:, i + 1] << 8).to(torch.int16).view(torch.float16).double()[:, None]      # noqa: E731
    signed = lambda v: torch.where(v > 127, v - 256, v).double()                          # noqa: E731
    parts = []
    if case["qtype"] == "Q8_0":
        parts.append(half(0) * signed(x[:, 2:]))
    elif case["qtype"] == "Q4_K":
        for j in range(8):
            a, c = x[:, 4 + j], x[:, 8 + j]
            scale, least = (a & 63, c & 63) if j < 4 else ((c & 15) | (x[:, j] >> 6) << 4, (c >> 4) | (a >> 6) << 4)
            q = x[:, 16 + j // 2 * 32:48 + j // 2 * 32] >> 4 * (j % 2) & 15
            parts.append(half(0) * scale[:, None] * q - half(2) * least[:, None])
    else:
        for j in range(16):
            h, quarter, place = j // 8, j % 8 // 2, j % 2 * 16
            low = x[:, 64 * h + 32 * (quarter % 2) + place:][:, :16] >> 4 * (quarter // 2) & 15
            high = x[:, 128 + 32 * h + place:][:, :16] >> 2 * quarter & 3
            parts.append(half(208) * signed(x[:, 192 + j])[:, None] * ((low | high << 4) - 32))
    return torch.cat(parts, 1).reshape(len(tokens), -1) * torch.tensor(case["scale"], dtype=torch.float32).double().item()


def exact(case, seed):
    return {"sample": _exact_sample, "rotary": _exact_rotary, "pool": _exact_pool, "embedding": _exact_embedding}[case["kind"]](case, prepare(case, seed))
