"""A small decoder served from GGUF weights with a paged cache in 8 bits: every operator between the quantized linears is one of `kernels`.

    python examples/decoder.py [--cache float8_e4m3fn] [--layers 4] [--steps 64]

Prompts of different lengths go through the layers packed in one call; after that one step appends a token to every sequence.  The step is captured
once as a CUDA graph: lengths live on the device, so that a replay is the next token.  Weights are random and there is no rotary embedding:
this shows how the calls fit together, not a trained model."""
from __future__ import annotations

import argparse
import sys
from pathlib import Path
from typing import NamedTuple

import torch

if __package__ in (None, ""):
    sys.path.insert(0, str(Path(__file__).resolve().parents[1]))
from dinoml_v2_b200 import kernels, synthetic  # noqa: E402


class Config(NamedTuple):
    layers: int = 2
    width: int = 2048
    heads: int = 16
    kv_heads: int = 8
    head_dim: int = 128
    hidden: int = 4096
    vocabulary: int = 8192
    qtype: str = "Q6_K"
    cache: str = "int8"
    block: int = 64
    dtype: torch.dtype = torch.bfloat16
    eps: float = 1e-5


class Layer:
    def __init__(self, c: Config, seed: int, device):
        def weight(rows: int, columns: int, at: int):
            return torch.from_numpy(synthetic.random_blocks(c.qtype, rows, columns, seed=100 * seed + at)).to(device)

        g = torch.Generator()
        g.manual_seed(seed)
        self.attention_norm, self.ffn_norm = (1 + 0.1 * torch.randn(c.width, generator=g).to(device) for _ in range(2))
        self.qkv = weight((c.heads + 2 * c.kv_heads) * c.head_dim, c.width, 1)
        self.o = weight(c.width, c.heads * c.head_dim, 2)
        self.gate, self.up = weight(c.hidden, c.width, 3), weight(c.hidden, c.width, 4)
        self.gate_up = kernels.interleave_rows8(self.gate, self.up)
        self.down = weight(c.width, c.hidden, 5)


class Decoder:
    """Layers, one cache each, and who has which blocks of them: `sequences` of at most `most` tokens."""

    def __init__(self, c: Config, sequences: int, most: int, device="cuda", seed: int = 1):
        self.c = c
        self.layers = [Layer(c, seed + i, device) for i in range(c.layers)]
        g = torch.Generator()
        g.manual_seed(seed)
        self.embedding = torch.randn(c.vocabulary, c.width, generator=g).to(device, c.dtype)
        self.norm = torch.ones(c.width, device=device)
        self.head = torch.from_numpy(synthetic.random_blocks(c.qtype, c.vocabulary, c.width, seed=99)).to(device)
        each = -(-most // c.block)
        self.caches = [kernels.kv_cache(sequences * each, c.kv_heads, c.block, c.head_dim, c.cache, device) for _ in self.layers]
        # Any order does: here the blocks of all sequences lie interleaved.
        self.table = torch.arange(sequences * each, dtype=torch.int32, device=device).reshape(each, sequences).t().contiguous()
        self.lengths = torch.zeros(sequences, dtype=torch.int32, device=device)

    def forward(self, tokens: torch.Tensor, starts: torch.Tensor | None) -> torch.Tensor:
        """Last hidden states of packed new tokens, whose number is in `lengths` already."""
        c = self.c
        residual = self.embedding[tokens]
        x, total = kernels.rms_norm(residual, self.layers[0].attention_norm, c.eps)
        for i, (layer, cache) in enumerate(zip(self.layers, self.caches)):
            qkv = kernels.gemm_rcr(x, layer.qkv, c.qtype).view(len(tokens), -1, c.head_dim)
            q, k, v = qkv.split((c.heads, c.kv_heads, c.kv_heads), dim=1)      # views: rows are as far apart as those of qkv
            kernels.kv_cache_write(cache, k, v, self.table, self.lengths, starts)
            y = kernels.kv_cache_attention(q, cache, self.table, self.lengths, starts)
            y = kernels.gemm_rcr(y.view(len(tokens), -1), layer.o, c.qtype)
            x, residual = kernels.rms_norm(y, layer.ffn_norm, c.eps, residual=residual)
            y = kernels.gemm_rcr(kernels.dual_gemm_rcr(x, layer.gate_up, c.qtype), layer.down, c.qtype)
            after = self.layers[i + 1].attention_norm if i + 1 < c.layers else self.norm
            x, residual = kernels.rms_norm(y, after, c.eps, residual=residual)
        return x

    def prefill(self, prompts: list[list[int]]) -> torch.Tensor:
        """Takes the prompts in; the next token of each."""
        device = self.lengths.device
        counts = torch.tensor([len(p) for p in prompts], dtype=torch.int32)
        starts = torch.zeros(len(prompts) + 1, dtype=torch.int32)
        starts[1:] = counts.cumsum(0)
        self.lengths += counts.to(device)
        x = self.forward(torch.tensor([t for p in prompts for t in p], device=device), starts.to(device))
        return self.choose(x[(starts[1:] - 1).long().to(device)])

    def choose(self, x: torch.Tensor) -> torch.Tensor:
        return kernels.gemm_rcr(x, self.head, self.c.qtype).argmax(dim=-1)

    def step(self, tokens: torch.Tensor) -> torch.Tensor:
        """One token more for every sequence; the next ones."""
        self.lengths += 1
        return self.choose(self.forward(tokens, None))


def generate(decoder: Decoder, prompts: list[list[int]], steps: int) -> torch.Tensor:
    """[sequences, steps + 1] tokens: the prompts' next ones, and those of `steps` replays of one captured step."""
    tokens = decoder.prefill(prompts)
    out = [tokens.clone()]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        lengths = decoder.lengths.clone()
        decoder.step(tokens)                       # workspaces are made outside of a capture; the token that it writes is written again
        decoder.lengths.copy_(lengths)
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        tokens.copy_(decoder.step(tokens))
    with torch.cuda.stream(stream):
        for _ in range(steps):
            graph.replay()
            out.append(tokens.clone())
    torch.cuda.current_stream().wait_stream(stream)
    return torch.stack(out, dim=1)


def main() -> None:
    parser = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    parser.add_argument("--cache", default="int8", choices=("int8", "float8_e4m3fn"))
    parser.add_argument("--layers", type=int, default=4)
    parser.add_argument("--steps", type=int, default=64)
    parser.add_argument("--prompts", type=int, nargs="+", default=[700, 33, 1, 256], help="lengths of the prompts")
    args = parser.parse_args()
    c = Config(layers=args.layers, cache=args.cache)
    g = torch.Generator()
    g.manual_seed(5)
    prompts = [torch.randint(0, c.vocabulary, (n,), generator=g).tolist() for n in args.prompts]
    decoder = Decoder(c, len(prompts), max(args.prompts) + args.steps + 1)
    begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    tokens = generate(decoder, prompts, args.steps)
    begin.record()
    decoder.lengths -= args.steps
    for _ in range(args.steps):
        decoder.step(tokens[:, 0].contiguous())
    end.record()
    torch.cuda.synchronize()
    for n, row in zip(args.prompts, tokens.tolist()):
        print(f"prompt of {n}: {row[:8]}")
    print(f"{begin.elapsed_time(end) / args.steps * 1e3:.0f} us a step outside of the graph, device status {kernels.device_status()}")


if __name__ == "__main__":
    main()
