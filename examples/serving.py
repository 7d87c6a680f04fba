"""Requests served by the decoder of decoder.py, from tokens to tokens on the device: rows of a GGUF table, queries and keys normed and turned by position, a pool that hands the cache's blocks
out and takes them back, and tokens chosen with settings of each request.

    python examples/serving.py [--slots 8] [--requests 24] [--cache float8_e4m3fn]

A step for prompts takes requests that are done out of the pool and new ones into their slots; between such steps every request gets a token a step, captured once as a CUDA graph.  The pool
is on the device: a replay begins blocks where it has to, and a request that finds none waits a step.  Weights are random: this shows how the calls fit together, not a trained model."""
from __future__ import annotations

import argparse
import sys
from pathlib import Path
from typing import NamedTuple

import torch

if __package__ in (None, ""):
    sys.path.insert(0, str(Path(__file__).resolve().parents[1]))
from dinoml_v2_b200 import kernels, synthetic  # noqa: E402
from examples.decoder import Config, Layer  # noqa: E402


class Request(NamedTuple):
    prompt: list[int]
    most: int                      # tokens to generate
    temperature: float = 0.8
    top_k: int = 0
    top_p: float = 1.0
    min_p: float = 0.0


def tokens_of_rows(step: kernels.KVStep, new: torch.Tensor, packed: torch.Tensor) -> torch.Tensor:
    """The token of each row of a step, -1 of nobody's: `packed` has new[b] tokens of every sequence one after the other, the step only the rows of sequences that got theirs, so that a
    sequence behind one that went without begins earlier there."""
    if not len(packed):
        return torch.full_like(step.positions, -1)
    row = torch.arange(len(step.positions), dtype=torch.int32, device=packed.device)
    b = torch.searchsorted(step.starts[1:].contiguous(), row, right=True).clamp(max=len(new) - 1)
    source = (new.cumsum(0) - new)[b] + row - step.starts[b]
    return torch.where(step.positions >= 0, packed[source.clamp(max=len(packed) - 1)], -1).to(packed.dtype)


class Server:
    """`slots` requests at a time, of at most `most` tokens each, that share `blocks` blocks of cache."""

    def __init__(self, c: Config, slots: int, blocks: int, most: int, device="cuda", seed: int = 1):
        self.c, self.slots, self.device = c, slots, device
        self.layers = [Layer(c, seed + i, device) for i in range(c.layers)]
        g = torch.Generator()
        g.manual_seed(seed)
        self.head_norms = [tuple((1 + 0.1 * torch.randn(c.head_dim, generator=g)).to(device) for _ in range(2)) for _ in self.layers]
        self.embedding, self.head = (torch.from_numpy(synthetic.random_blocks(c.qtype, c.vocabulary, c.width, seed=98 + i)).to(device) for i in range(2))
        self.norm = torch.ones(c.width, device=device)
        self.frequencies = kernels.rotary_frequencies(c.head_dim, 500000.0, device=device)
        self.caches = [kernels.kv_cache(blocks, c.kv_heads, c.block, c.head_dim, c.cache, device) for _ in self.layers]
        self.pool = kernels.kv_pool(blocks, slots, -(-most // c.block), c.block, device)
        self.tokens = torch.full((slots,), -1, dtype=torch.int32, device=device)          # of each slot, the last one chosen
        self.active = torch.zeros(slots, dtype=torch.int32, device=device)                # slots that want a token more
        self.uniforms = torch.zeros(slots, device=device)
        self.settings = {name: torch.full((slots,), value, dtype=dtype, device=device)
                         for name, value, dtype in (("temperature", 0.0, torch.float32), ("top_k", 0, torch.int32), ("top_p", 1.0, torch.float32), ("min_p", 0.0, torch.float32))}
        self.generator = torch.Generator(device=device)
        self.generator.manual_seed(seed)
        self.done = torch.zeros(slots, dtype=torch.bool, device=device)
        self.graph, self.stream = None, torch.cuda.Stream()

    def forward(self, tokens: torch.Tensor, step: kernels.KVStep) -> torch.Tensor:
        c = self.c
        residual = kernels.embedding(tokens, self.embedding, c.qtype, str(c.dtype)[6:])
        x, _ = kernels.rms_norm(residual, self.layers[0].attention_norm, c.eps)
        for i, (layer, cache, (q_norm, k_norm)) in enumerate(zip(self.layers, self.caches, self.head_norms)):
            qkv = kernels.gemm_rcr(x, layer.qkv, c.qtype).view(len(tokens), -1, c.head_dim)
            q, k, v = qkv.split((c.heads, c.kv_heads, c.kv_heads), dim=1)
            kernels.rotary(q, k, step.positions, self.frequencies, q_weight=q_norm, k_weight=k_norm, eps=c.eps, out=(q, k))
            kernels.kv_cache_write(cache, k, v, self.pool.block_table, step.lengths, step.starts)
            y = kernels.kv_cache_attention(q, cache, self.pool.block_table, step.lengths, step.starts)
            y = kernels.gemm_rcr(y.view(len(tokens), -1), layer.o, c.qtype)
            x, residual = kernels.rms_norm(y, layer.ffn_norm, c.eps, residual=residual)
            y = kernels.gemm_rcr(kernels.dual_gemm_rcr(x, layer.gate_up, c.qtype), layer.down, c.qtype)
            after = self.layers[i + 1].attention_norm if i + 1 < c.layers else self.norm
            x, residual = kernels.rms_norm(y, after, c.eps, residual=residual)
        return x

    def choose(self, x: torch.Tensor, step: kernels.KVStep) -> None:
        """The next tokens of the slots that took part in the step."""
        logits = kernels.gemm_rcr(x, self.head, self.c.qtype)
        chosen, _ = kernels.sample(logits, self.uniforms, **self.settings)
        self.tokens.copy_(torch.where(step.lengths > 0, chosen, self.tokens))

    def check(self, r: Request) -> None:
        """A prompt and what is generated after it, but for the last token, have to fit a slot's blocks: the pool would leave such a request out of every step."""
        room = self.pool.block_table.shape[1] * self.c.block
        if not r.prompt or r.most < 1 or len(r.prompt) + r.most - 1 > room:
            raise ValueError(f"a request has a prompt and generates a token at least, of {room} tokens at most in all: got {len(r.prompt)} and {r.most}")

    def admit(self, requests: dict[int, Request]) -> None:
        """Takes requests into their slots, in the place of whoever had them, and chooses their first tokens.  One that finds no blocks has no tokens in the pool after that."""
        for r in requests.values():
            self.check(r)
        new, drop, packed = [0] * self.slots, [0] * self.slots, []
        for slot in sorted(requests):
            r = requests[slot]
            new[slot], drop[slot] = len(r.prompt), 0x7fffffff
            packed += r.prompt
            for name, t in self.settings.items():
                t[slot] = getattr(r, name)
            self.active[slot] = 1
        new, drop, packed = (torch.tensor(v, dtype=torch.int32, device=self.device) for v in (new, drop, packed))
        step = kernels.kv_pool_step(self.pool, new, len(packed), drop=drop)
        x = self.forward(tokens_of_rows(step, new, packed), step)
        last = (step.starts[1:] - 1).clamp(min=0).long()                                  # (a slot that took no part has no row; its choice is not used)
        self.uniforms.uniform_(generator=self.generator)
        self.choose(x[last], step)

    def release(self, slots: list[int]) -> None:
        """Their blocks go back, and they take no part until they are admitted again."""
        drop = torch.zeros(self.slots, dtype=torch.int32, device=self.device)
        drop[slots] = 0x7fffffff
        self.active[slots] = 0
        self.tokens[slots] = -1
        kernels.kv_pool_step(self.pool, torch.zeros_like(drop), 0, drop=drop)

    def _decode(self) -> None:
        step = kernels.kv_pool_step(self.pool, self.active)
        self.choose(self.forward(self.tokens, step), step)
        self.done.copy_(step.lengths > 0)

    def decode(self, captured: bool = True) -> torch.Tensor:
        """One token more for every active slot; which slots got theirs (the others found no block)."""
        self.uniforms.uniform_(generator=self.generator)
        if not captured:
            self._decode()
            return self.done
        self.stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(self.stream):
            if self.graph is None:                                                        # the first one loads the kernels and makes the stream's workspaces
                self._decode()
                self.graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(self.graph, stream=self.stream):
                    self._decode()
            else:
                self.graph.replay()
        torch.cuda.current_stream().wait_stream(self.stream)
        return self.done


def serve(server: Server, requests: list[Request], captured: bool = True) -> list[list[int]]:
    """Generated tokens of each request: as many at a time as there are slots and blocks, the next one whenever one is done.  Where no request finds a block any more the one that came
    last gives its blocks up and begins again later."""
    for r in requests:
        server.check(r)
    out, waiting, running, full = [[] for _ in requests], list(range(len(requests))), {}, False
    while waiting or running:
        free = [s for s in range(server.slots) if s not in running]
        admitted = {} if full and running else dict(zip(free, waiting))
        if admitted:
            waiting = waiting[len(admitted):]
            server.admit({slot: requests[r] for slot, r in admitted.items()})
            held, tokens = server.pool.lengths.tolist(), server.tokens.tolist()
            for slot, r in admitted.items():
                if held[slot] == 0:                                                       # no blocks for the prompt: later
                    server.active[slot] = 0
                    waiting.append(r)
                else:
                    running[slot] = r
                    out[r] = [tokens[slot]]
            waiting.sort()
            full = bool(waiting)
            if not running:
                raise RuntimeError("the pool has not enough blocks for a prompt")
        got, tokens = server.decode(captured).tolist(), server.tokens.tolist()
        for slot, r in running.items():
            if got[slot] and len(out[r]) < requests[r].most:
                out[r].append(tokens[slot])
        leaving = [slot for slot, r in running.items() if len(out[r]) >= requests[r].most]
        full = full and not leaving
        if not leaving and not any(got[slot] for slot in running):
            if len(running) == 1:
                raise RuntimeError("the pool has not enough blocks for a request")
            leaving, full = [list(running)[-1]], True
            waiting = sorted(waiting + [running[leaving[0]]])
        if leaving:
            server.release(leaving)
            for slot in leaving:
                del running[slot]
    return out


def main() -> None:
    parser = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    parser.add_argument("--cache", default="int8", choices=("int8", "float8_e4m3fn"))
    parser.add_argument("--slots", type=int, default=8)
    parser.add_argument("--requests", type=int, default=24)
    args = parser.parse_args()
    c = Config(layers=4, cache=args.cache)
    g = torch.Generator()
    g.manual_seed(5)
    length = lambda low, high: int(torch.randint(low, high, (1,), generator=g))           # noqa: E731
    requests = [Request(torch.randint(0, c.vocabulary, (length(1, 700),), generator=g).tolist(), length(5, 100), 0.0 if i % 4 == 0 else 0.9, top_k=40 * (i % 3), top_p=0.9 + 0.1 * (i % 2))
                for i in range(args.requests)]
    server = Server(c, args.slots, 12 * args.slots, 1024)
    begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    begin.record()
    out = serve(server, requests)
    end.record()
    torch.cuda.synchronize()
    for r, tokens in list(zip(requests, out))[:8]:
        print(f"prompt of {len(r.prompt)}, temperature {r.temperature}: {tokens[:8]} ({len(tokens)} tokens)")
    print(f"{sum(map(len, out))} tokens in {begin.elapsed_time(end):.0f} ms, device status {kernels.device_status()}")


if __name__ == "__main__":
    main()
