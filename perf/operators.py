"""What a decode loop runs between its quantized linears, as cases that can be timed and compared.

A program that serves a decoder from GGUF weights keeps the keys and values of every sequence in 8 bits and calls, in each layer,
four operators next to `kernels.gemm_rcr`:

* ``attention``: `kernels.kv_cache_attention`, causal attention of the new tokens over a paged cache of 8-bit blocks with one scale per
  block of tokens and head: out = softmax(scale * q K^T) V over positions max(0, p - window + 1) .. p of the token's own sequence;
* ``write``: `kernels.kv_cache_write`, the new tokens quantized into the cache.  A block's scale only grows: s = max(s, largest * (1 / 127))
  (int8) or the power of two that brings the largest value below 448 (float8_e4m3fn); tokens that are already in the block are
  brought to the new scale, and the first token of a block starts it anew.  The pass reads the blocks that it touched back, so
  that what the 8 bits stand for can be compared;
* ``read``: `kernels.kv_cache_read`, a range of every sequence as dense keys and values;
* ``norm``: `kernels.rms_norm`, x + residual and its root-mean-square norm, in the activation type or as Q8_0 blocks.

New tokens are rows of one packed tensor, sequence after sequence, cut out of the result of a fused q / k / v projection (so rows are
further apart than they are long).  `lengths` counts the tokens of a sequence with the new ones among them; a slot of the batch that
serves nobody has length zero.  Cache blocks are handed out in any order, table entries that no token uses are -1, and bytes
behind a sequence's last token are whatever was there."""
from __future__ import annotations

import math
import random

import torch

own = False

ELEMENT_BYTES = {"float16": 2, "bfloat16": 2, "float32": 4}
MAX_CONTEXT, MAX_NEW, MAX_SEQUENCES = 131072, 2048, 256
MAX_SCORES = 2048 * 32 * 8192               # new tokens x heads x positions of one pass, as the plain form lays them out
MAX_CACHED = 4 * 131072 * 8 * 128           # values of K of one pass, likewise


def listed():
    return [
        # one user, one new token after a long prompt: nothing but latency and one SM's share of the cache
        {"name": "decode_one", "kind": "attention", "cache": "int8", "dtype": "bfloat16", "sequences": 1, "new": 1, "context": 4001, "heads": 32,
         "kv_heads": 8, "head_dim": 128, "block": 64, "window": 0, "layout": 1},
        # a served batch of ragged lengths, some slots idle, small blocks
        {"name": "decode_batch_ragged", "kind": "attention", "cache": "int8", "dtype": "bfloat16", "sequences": 64, "new": 1, "context": 8192, "heads": 32,
         "kv_heads": 8, "head_dim": 128, "block": 16, "window": 0, "layout": 2},
        # four users with book-long contexts, e4m3, eight query heads per cached head
        {"name": "decode_long_e4m3", "kind": "attention", "cache": "float8_e4m3fn", "dtype": "float16", "sequences": 4, "new": 1, "context": 131072, "heads": 64,
         "kv_heads": 8, "head_dim": 128, "block": 128, "window": 0, "layout": 3},
        # float32 activations, a cached head per query head, a sliding window
        {"name": "decode_f32_window", "kind": "attention", "cache": "int8", "dtype": "float32", "sequences": 5, "new": 1, "context": 6000, "heads": 32,
         "kv_heads": 32, "head_dim": 64, "block": 32, "window": 2500, "layout": 4},
        # prompts that arrive in pieces beside decoding sequences
        {"name": "mixed_chunks", "kind": "attention", "cache": "float8_e4m3fn", "dtype": "bfloat16", "sequences": 8, "new": 300, "context": 3000, "heads": 32,
         "kv_heads": 8, "head_dim": 128, "block": 32, "window": 0, "layout": 5},
        # the last 2048 tokens of a long prompt
        {"name": "prefill_2048", "kind": "attention", "cache": "int8", "dtype": "bfloat16", "sequences": 1, "new": 2048, "context": 8192, "heads": 32,
         "kv_heads": 8, "head_dim": 128, "block": 64, "window": 0, "layout": 6},
        # a decode step's new tokens, and the blocks that they came into
        {"name": "write_decode", "kind": "write", "cache": "int8", "dtype": "bfloat16", "sequences": 64, "new": 1, "context": 4000, "kv_heads": 8,
         "head_dim": 128, "block": 16, "layout": 7, "out": "bfloat16"},
        # a prompt of odd length and shorter ones beside it, read back in full precision
        {"name": "write_prefill_e4m3", "kind": "write", "cache": "float8_e4m3fn", "dtype": "float16", "sequences": 6, "new": 2001, "context": 4096, "kv_heads": 8,
         "head_dim": 128, "block": 64, "layout": 8, "out": "float32"},
        # a shared prefix handed to a program of its own, short and odd
        {"name": "read_short_f32", "kind": "read", "cache": "float8_e4m3fn", "dtype": "float32", "sequences": 3, "context": 333, "kv_heads": 8, "head_dim": 128,
         "block": 16, "layout": 9},
        # long contexts read back as dense keys and values
        {"name": "read_long", "kind": "read", "cache": "int8", "dtype": "bfloat16", "sequences": 4, "context": 32768, "kv_heads": 8, "head_dim": 128, "block": 64,
         "layout": 10},
        # the norm of a decode step, weights in float32 as GGUF files hold them
        {"name": "norm_one", "kind": "norm", "dtype": "bfloat16", "rows": 1, "width": 4096, "residual": True, "weight": "float32", "q8_0": False},
        # the norm of a long prefill, handed on in 8 bits
        {"name": "norm_prefill_q8_0", "kind": "norm", "dtype": "float16", "rows": 2048, "width": 8192, "residual": True, "weight": "float32", "q8_0": True},
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    """One more case of the same ranges: lengths, batches and widths over their logarithms, every type, block and head size."""
    kind = rng.choices(["attention", "write", "read", "norm"], [50, 20, 15, 15])[0]
    dtype = rng.choices(["bfloat16", "float16", "float32"], [5, 3, 2])[0]
    if kind == "norm":
        q8_0 = rng.random() < 0.4
        rows, width = _log_int(rng, 1, 2048), _log_int(rng, 256, 8192)
        if q8_0 or rng.random() < 0.8:
            width = max(32, width // 32 * 32)
        width += 32 * (width == 3072)
        return {"kind": kind, "dtype": dtype, "rows": rows, "width": width, "residual": rng.random() < 0.7,
                "weight": "float32" if rng.random() < 0.6 else dtype, "q8_0": q8_0}
    case = {"kind": kind, "cache": rng.choice(["int8", "float8_e4m3fn"]), "dtype": dtype, "sequences": _log_int(rng, 1, MAX_SEQUENCES),
            "kv_heads": rng.choice([1, 2, 4, 5, 8, 8, 16, 32]), "head_dim": rng.choice([64, 128, 128, 256]), "block": rng.choice([16, 32, 64, 128]),
            "layout": rng.randrange(1 << 30)}
    group = rng.choice([1, 1, 2, 3, 4, 4, 7, 8])
    group += group * case["kv_heads"] * case["head_dim"] == 3072
    context = _log_int(rng, 1, MAX_CONTEXT if kind == "attention" else 32768)
    new = 1 if kind == "read" or rng.random() < 0.5 else _log_int(rng, 2, MAX_NEW)
    context = max(context, new)
    row = case["kv_heads"] * case["head_dim"]
    cap = MAX_CACHED if kind == "attention" else MAX_CACHED // 4
    while case["sequences"] * context * row > cap or (kind == "attention" and case["sequences"] * new * group * case["kv_heads"] * context > MAX_SCORES):
        if case["sequences"] > 1 and rng.random() < 0.6:
            case["sequences"] = (case["sequences"] + 1) // 2
        else:
            context = (context + 1) // 2
            new = min(new, context)
    context, new = context - (context == 3072), new - (new == 3072)
    if kind == "write":
        case["out"] = rng.choice(["bfloat16", "float16", "float32"])
    if kind == "attention":
        case.update(heads=group * case["kv_heads"], window=0 if rng.random() < 0.75 else _log_int(rng, 1, context))
    return {**case, "context": context, **({} if kind == "read" else {"new": new})}


# ----------------------------------------------------------------------------------------------- who is in the batch
def _batch(case):
    """(tokens of each sequence, new ones among them).  The first sequence has the case's own sizes; the others have less, and with four
    or more about one in ten is an idle slot."""
    rng, sizes = random.Random(case["layout"]), []
    for b in range(case["sequences"]):
        context, new = case["context"], case.get("new", 1)
        if b > 0:
            context = _log_int(rng, max(1, context // 8), context)
            new = 1 if new == 1 else _log_int(rng, 1, min(new, context))
            if case["sequences"] >= 4 and rng.random() < 0.1:
                context, new = 0, 1 if case.get("new", 1) == 1 else 0
        sizes.append((context, new))
    return sizes


def _touched(case):
    """First position that is read back, per sequence: the start of the block that holds the first new token."""
    return [max(0, n - new) // case["block"] * case["block"] for n, new in _batch(case)]


def work(case):
    e = ELEMENT_BYTES[case["dtype"]]
    if case["kind"] == "norm":
        values = case["rows"] * case["width"]
        out = values // 32 * 34 + 2 * values if case["q8_0"] else values * e              # Q8_0: the blocks, and what they stand for
        read = values // 32 * 34 if case["q8_0"] else 0
        return {"bytes": values * e * (3 if case["residual"] else 1) + out + read + case["width"] * ELEMENT_BYTES[case["weight"]], "flops": 5 * values}
    sizes, row = _batch(case), case["kv_heads"] * case["head_dim"]
    scale_bytes = 8 * case["kv_heads"]                                                    # of a block's keys and values
    blocks = lambda n: -(-n // case["block"])                                             # noqa: E731
    if case["kind"] == "read":
        tokens = sum(n for n, _ in sizes)
        return {"bytes": tokens * 2 * row * (1 + e) + sum(blocks(n) for n, _ in sizes) * (scale_bytes + 4), "flops": tokens * 2 * row}
    if case["kind"] == "write":
        new = sum(min(n, m) for n, m in sizes)
        back = sum(n - first for (n, _), first in zip(sizes, _touched(case)))
        o = ELEMENT_BYTES[case["out"]]
        return {"bytes": new * 2 * row * (e + 1) + back * 2 * row * (1 + o), "flops": (3 * new + back) * 2 * row}
    flops = cached = tables = 0
    for n, m in sizes:
        window = case["window"] or n
        first = max(0, n - m)                                                             # position of the first new token
        seen = max(0, first - window + 1)
        cached += n - seen
        tables += blocks(n) - seen // case["block"]
        p = range(first, n)
        flops += 4 * case["heads"] * case["head_dim"] * sum(min(x + 1, window) for x in p)
    rows = sum(m for _, m in sizes) * case["heads"] * case["head_dim"]
    return {"bytes": cached * 2 * row + tables * (scale_bytes + 4) + 2 * rows * e, "flops": flops}


# ----------------------------------------------------------------------------------------------- inputs
class _Maker:
    def __init__(self, case, seed):
        self.case, self.dev = case, torch.device("cuda")
        self.generator = torch.Generator(device=self.dev)
        self.generator.manual_seed(int(seed) * 1000 + 17)

    def normal(self, *shape):
        return torch.randn(*shape, device=self.dev, generator=self.generator)

    def ints(self, values):
        return torch.tensor(values, dtype=torch.int32, device=self.dev)

    def cache(self, blocks):
        """Keys and values of order one, with channels of different size, in blocks of different scale."""
        c = self.case
        out = []
        for spread in (0.6, 0.2):
            scale = torch.exp(0.3 * self.normal(blocks, c["kv_heads"])) * (3.0 / (127 if c["cache"] == "int8" else 448))
            x = self.normal(blocks, c["kv_heads"], c["block"], c["head_dim"])
            x *= torch.exp(spread * self.normal(c["kv_heads"], 1, c["head_dim"]))
            if c["cache"] == "int8":
                q = (x * 40).round_().clamp_(-127, 127).to(torch.int8)
            else:
                scale = torch.exp2(torch.round(torch.log2(scale)))
                q = (x * 140).clamp_(-448, 448).to(torch.float8_e4m3fn)
            out.append((q, scale.contiguous()))
        return out[0][0], out[1][0], out[0][1], out[1][1]

    def batch(self):
        c = self.case
        sizes = _batch(c)
        need = [-(-n // c["block"]) for n, _ in sizes]
        used, widest = sum(need), max(1, max(need))
        table = torch.full((len(sizes), widest), -1, dtype=torch.int32, device=self.dev)
        at = torch.arange(widest, device=self.dev)[None] < self.ints(need)[:, None]
        blocks = used + max(2, used // 16)                                                # some are free; the last one always is
        order = torch.randperm(blocks - 1, device=self.dev, generator=self.generator).to(torch.int32)
        table[at] = order[:used]
        return {"sizes": sizes, "table": table, "blocks": blocks, "lengths": self.ints([n for n, _ in sizes])}

    def starts(self, counts):
        total, out = 0, [0]
        for n in counts:
            total += n
            out.append(total)
        return self.ints(out), total


def prepare(case, seed):
    make, dtype = _Maker(case, seed), getattr(torch, case["dtype"])
    state = {"case": case}
    if case["kind"] == "norm":
        shape = (case["rows"], case["width"])
        state["x"] = make.normal(*shape).to(dtype)
        state["residual"] = (3 * make.normal(*shape)).to(dtype) if case["residual"] else None
        state["weight"] = (1 + 0.2 * make.normal(case["width"])).to(getattr(torch, case["weight"]))
        return state
    batch = make.batch()
    state.update(cache=make.cache(batch["blocks"]), table=batch["table"], lengths=batch["lengths"])
    if case["kind"] == "read":
        state["begins"] = None
        state["starts"], state["rows"] = make.starts([n for n, _ in batch["sizes"]])
        return state
    one_each = case["new"] == 1
    starts, tokens = make.starts([m for _, m in batch["sizes"]])
    state["starts"] = None if one_each else starts                                        # None: one row per sequence
    state["most_new"] = max(m for _, m in batch["sizes"])
    d, kv = case["head_dim"], case["kv_heads"]
    heads = case.get("heads", kv)
    fused = make.normal(tokens, (heads + 2 * kv) * d)
    fused[:, heads * d:] *= 1 + 2 * torch.rand(tokens, 1, device=make.dev, generator=make.generator)    # tokens of different size: scales grow
    fused = fused.to(dtype)
    state["q"] = fused[:, :heads * d].view(tokens, heads, d)
    state["k"] = fused[:, heads * d:(heads + kv) * d].view(tokens, kv, d)
    state["v"] = fused[:, (heads + kv) * d:].view(tokens, kv, d)
    if case["kind"] == "write":
        first = _touched(case)
        state["begins"] = make.ints(first)
        state["back"], state["rows"] = make.starts([n - f for (n, _), f in zip(batch["sizes"], first)])
    return state


# ----------------------------------------------------------------------------------------------- the calls of a user's program
def _run_own(state):
    from dinoml_v2_b200 import kernels
    case = state["case"]
    if case["kind"] == "norm":
        y, total = kernels.rms_norm(state["x"], state["weight"], residual=state["residual"], q8_0=case["q8_0"])
        if case["q8_0"]:
            y = kernels.dequantize_rows(y, "Q8_0", case["width"], "float16")
        return {"y": y} if total is None else {"y": y, "total": total}
    if case["kind"] == "attention":
        return kernels.kv_cache_attention(state["q"], state["cache"], state["table"], state["lengths"], state["starts"], window=case["window"])
    if case["kind"] == "read":
        return kernels.kv_cache_read(state["cache"], state["table"], state["starts"], state["rows"], case["dtype"])
    kernels.kv_cache_write(state["cache"], state["k"], state["v"], state["table"], state["lengths"], state["starts"])
    k, v = kernels.kv_cache_read(state["cache"], state["table"], state["back"], state["rows"], case["out"], begins=state["begins"])
    return {"k": k, "v": v, "k_scale": state["cache"][2], "v_scale": state["cache"][3]}


# ----------------------------------------------------------------------------------------------- the same in elementary operations
def _row_of(starts, rows):
    """(sequence, place in it) of every packed row."""
    at = torch.arange(rows, device=starts.device)
    b = (at[:, None] >= starts[None, 1:]).sum(1)
    return b, at - starts[b]


def _plain_norm(state):
    case, x = state["case"], state["x"].float()
    total = x + state["residual"].float() if case["residual"] else x
    y = total * torch.rsqrt((total * total).mean(-1, keepdim=True) + 1e-5) * state["weight"].float()
    out = {}
    if case["q8_0"]:
        blocks = y.view(case["rows"], -1, 32)
        d = (blocks.abs().amax(-1, keepdim=True) * (1 / 127)).to(torch.float16).float()
        q = torch.where(d > 0, (blocks / d).round().clamp(-127, 127), torch.zeros_like(blocks))
        out["y"] = (q * d).view_as(y).to(torch.float16)
    else:
        out["y"] = y.to(state["x"].dtype)
    if case["residual"]:
        out["total"] = total.to(state["x"].dtype)
    return out


def _picked(q, *index):
    """q[index], by bytes."""
    return q.view(torch.uint8)[index].view(q.dtype).float()


def _plain_rows(state, which, starts, rows, begins):
    """Dense float32 [rows, kv_heads, head_dim] of the keys (0) or values (1)."""
    block = state["case"]["block"]
    b, at = _row_of(starts, rows)
    p = at if begins is None else at + begins[b]
    ids = state["table"][b, p // block].long()
    return _picked(state["cache"][which], ids, slice(None), p % block) * state["cache"][2 + which][ids][..., None]


def _plain_read(state, starts, rows, begins, dtype):
    dtype = getattr(torch, dtype)
    return _plain_rows(state, 0, starts, rows, begins).to(dtype), _plain_rows(state, 1, starts, rows, begins).to(dtype)


def _new_range(state):
    """(first packed row, first position) of the new tokens of every sequence."""
    lengths = state["lengths"].long()
    starts = state["starts"]
    if starts is None:
        return torch.arange(len(lengths), device=lengths.device), lengths - 1
    starts = starts.long()
    return starts[:-1], lengths - (starts[1:] - starts[:-1])


def _plain_write_one(state, x, which):
    case, q, scale = state["case"], state["cache"][which], state["cache"][2 + which]
    block, lengths = case["block"], state["lengths"].long()
    row, first = _new_range(state)
    last = (lengths - 1).clamp(min=0) // block                                            # the block of the last token
    piece = (state["most_new"] + block - 2) // block + 1                                  # blocks that a sequence's new tokens can reach
    j = torch.minimum(first.clamp(min=0)[:, None] // block + torch.arange(piece, device=q.device), last[:, None])
    ids = torch.where(lengths[:, None] > 0, torch.gather(state["table"].long(), 1, j), torch.full_like(j, len(q) - 1))
    p = j[..., None] * block + torch.arange(block, device=q.device)                       # [sequence, piece, slot]
    fresh = (p >= first[:, None, None]) & (p < lengths[:, None, None]) & (first >= 0)[:, None, None]
    source = (row[:, None, None] + p - first[:, None, None]).clamp(0, len(x) - 1)
    new = x[source].float().transpose(2, 3) * fresh[:, :, None, :, None]                  # [sequence, piece, head, slot, channel]
    largest = new.abs().amax((-1, -2))
    if case["cache"] == "int8":
        wanted = largest * (1 / 127)
    else:                                                                                 # 448 = 0.875 * 2^9
        m, e = torch.frexp(largest)
        e = (e - torch.where(m <= 0.875, 9, 8)).clamp(min=-126)
        wanted = torch.where(largest > 0, ((e + 127) << 23).to(torch.int32).view(torch.float32), torch.zeros_like(largest))
    before = torch.where((fresh & (p % block == 0)).any(-1)[..., None], torch.zeros_like(wanted), scale[ids])
    after = torch.maximum(before, wanted)
    ratio = torch.where(after > 0, before / after, torch.zeros_like(after))[..., None, None]
    inside = torch.where(after > 0, after, torch.ones_like(after))[..., None, None]
    value = torch.where(fresh[:, :, None, :, None], new / inside, _picked(q, ids) * ratio)
    if case["cache"] == "int8":
        value = value.round().clamp(-127, 127)
    q.view(torch.uint8)[ids] = value.clamp(-448, 448).to(q.dtype).view(torch.uint8)
    scale[ids] = after


def _plain_attention(state):
    case, q = state["case"], state["q"]
    kv, d, block = case["kv_heads"], case["head_dim"], case["block"]
    row, first = _new_range(state)
    reach = torch.arange(state["table"].shape[1] * block, device=q.device)
    ids = state["table"].long().clamp(min=0)                                              # [sequence, blocks]
    there = (reach[None] < state["lengths"][:, None])[:, :, None, None]

    def dense(which):                                                                     # [sequence, position, head, channel]
        x = _picked(state["cache"][which], ids) * state["cache"][2 + which][ids][..., None, None]
        return torch.where(there, x.transpose(2, 3).reshape(len(ids), -1, kv, d), torch.zeros((), device=q.device))

    step = torch.arange(state["most_new"], device=q.device)
    p = first[:, None] + step                                                             # [sequence, new token]
    valid = (p < state["lengths"][:, None]) & (p >= 0)
    rows = (row[:, None] + step).clamp(max=len(q) - 1)
    x = q[rows].float().view(len(ids), len(step), kv, -1, d)
    s = torch.einsum("bnhgd,blhd->bhgnl", x, dense(0)) * d ** -0.5
    seen = (reach <= p[..., None]) & (reach > p[..., None] - (case["window"] or len(reach) + 1)) & valid[..., None]
    s = s.masked_fill_(~seen[:, None, None], -math.inf)
    s = torch.exp(s - s.amax(-1, keepdim=True).clamp(min=-1e30))
    total = s.sum(-1, keepdim=True)
    o = torch.einsum("bhgnl,blhd->bnhgd", s / torch.where(total > 0, total, torch.ones_like(total)), dense(1))
    # back to packed rows
    b, at = (torch.arange(len(q), device=q.device), 0) if state["starts"] is None else _row_of(state["starts"], len(q))
    return o[b, at].reshape(len(q), -1, d).to(q.dtype)


def _run_plain(state):
    case = state["case"]
    if case["kind"] == "norm":
        return _plain_norm(state)
    if case["kind"] == "attention":
        return _plain_attention(state)
    if case["kind"] == "read":
        return _plain_read(state, state["starts"], state["rows"], None, case["dtype"])
    _plain_write_one(state, state["k"], 0)
    _plain_write_one(state, state["v"], 1)
    k, v = _plain_read(state, state["back"], state["rows"], state["begins"], case["out"])
    return {"k": k, "v": v, "k_scale": state["cache"][2], "v_scale": state["cache"][3]}


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ----------------------------------------------------------------------------------------------- the definitions in 64 bits
def _exact_norm(case, state):
    total = state["x"].double()
    if case["residual"]:
        total = total + state["residual"].double()
    y = total / torch.sqrt(total.pow(2).sum(-1, keepdim=True) / case["width"] + 1e-5) * state["weight"].double()
    if case["q8_0"]:
        groups = y.reshape(-1, 32)
        d = (groups.abs().max(-1, keepdim=True).values / 127).to(torch.float16).double()      # a block's scale is a float16 by definition
        y = (torch.round(groups / d.clamp(min=2.0 ** -24)) * d).reshape(y.shape)
    return {"y": y, "total": total} if case["residual"] else {"y": y}


def _exact_sequence(state, b, which, count):
    """The first `count` cached keys (0) or values (1) of sequence b: float64 [count, kv_heads, head_dim]."""
    block = state["case"]["block"]
    ids = state["table"][b, :-(-count // block)].long()
    x = state["cache"][which][ids].double() * state["cache"][2 + which][ids].double()[..., None, None]
    return x.permute(0, 2, 1, 3).flatten(0, 1)[:count]


def _exact_attention(case, state):
    group, d = case["heads"] // case["kv_heads"], case["head_dim"]
    out = torch.zeros(state["q"].shape, dtype=torch.float64, device=state["q"].device)
    row = 0
    for b, (n, m) in enumerate(_batch(case)):
        if n > 0 and m > 0:
            k, v = _exact_sequence(state, b, 0, n), _exact_sequence(state, b, 1, n)
            at = torch.arange(n, device=k.device)[None]
            p = torch.arange(n - m, n, device=k.device)[:, None]
            hidden = at > p
            if case["window"]:
                hidden |= at <= p - case["window"]
            for h in range(case["heads"]):
                s = state["q"][row:row + m, h].double() @ k[:, h // group].T / math.sqrt(d)
                out[row:row + m, h] = torch.softmax(s.masked_fill(hidden, -math.inf), -1) @ v[:, h // group]
        row += m
    return out


def _exact_quantized(case, new, old, scale):
    """One block: `new` [tokens, kv_heads, head_dim] behind the `old` quantized ones, scale [kv_heads]: the values that it then stands for, its scales."""
    largest = new.abs().amax((0, 2))
    if case["cache"] == "int8":
        wanted = (largest / 127).float().double()                                             # a scale is a float32 by definition
    else:
        wanted = torch.exp2(torch.ceil(torch.log2(largest / 448)))
    after = torch.maximum(scale, wanted) if len(old) else wanted
    inside = torch.where(after > 0, after, torch.ones_like(after))[:, None]
    q = torch.cat([old * (scale[:, None] / inside), new / inside])
    q = torch.round(q) if case["cache"] == "int8" else q.float().to(torch.float8_e4m3fn).double()
    return q * after[:, None], after


def _exact_write(case, state):
    block, row = case["block"], 0
    outs, scales = ([], []), [state["cache"][2].double(), state["cache"][3].double()]
    for b, (n, m) in enumerate(_batch(case)):
        first = n - m
        for j in range(max(0, first) // block, -(-n // block)):
            low, high = max(first, j * block), min(n, (j + 1) * block)
            i = int(state["table"][b, j])
            for which, x in enumerate((state["k"], state["v"])):
                new = x[row + low - first:row + high - first].double()
                old = state["cache"][which][i, :, :low - j * block].transpose(0, 1).double()
                value, scales[which][i] = _exact_quantized(case, new, old, scales[which][i].clone())
                outs[which].append(value)
        row += m
    return {"k": torch.cat(outs[0]), "v": torch.cat(outs[1]), "k_scale": scales[0], "v_scale": scales[1]}


def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] == "norm":
        return _exact_norm(case, state)
    if case["kind"] == "attention":
        return _exact_attention(case, state)
    if case["kind"] == "write":
        return _exact_write(case, state)
    sizes = _batch(case)
    return tuple(torch.cat([_exact_sequence(state, b, which, n) for b, (n, _) in enumerate(sizes)]) for which in (0, 1))
