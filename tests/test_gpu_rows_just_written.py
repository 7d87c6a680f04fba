"""Packed rows that the launch before has only just written, at an address whose earlier bytes were read a moment ago: what the norm writes as Q8_0 goes straight to the embedding and the dequantizer,
launch beside launch, and as a replayed graph.  Everything is equal to what they read after a synchronization."""
import pytest
import torch

from dinoml_v2_b200 import kernels

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


@pytest.mark.parametrize("rows,width", [(1, 256), (4, 256), (40, 1024), (300, 4096), (1000, 2048)])
def test_norm_to_embedding(rows, width):
    g = torch.Generator(device=DEV)
    g.manual_seed(rows)
    weight = torch.ones(width, device=DEV)
    tokens = torch.randint(0, rows, (rows,), device=DEV, generator=g, dtype=torch.int32)
    xs = [torch.randn(rows, width, device=DEV, generator=g).bfloat16() for _ in range(6)]
    packed = torch.empty(rows, width // 32 * 34, dtype=torch.uint8, device=DEV)

    def chain(x):
        kernels.rms_norm(x, weight, q8_0=True, out=packed)
        return kernels.embedding(tokens, packed, "Q8_0", "float32"), kernels.dequantize_rows(packed, "Q8_0", width)

    want = []
    for x in xs:
        blocks, _ = kernels.rms_norm(x, weight, q8_0=True)
        torch.cuda.synchronize()
        dense = kernels.dequantize_rows(blocks, "Q8_0", width)
        want.append((dense[tokens.long()], dense))
    for _ in range(20):
        got = [chain(x) for x in xs]
        assert all(torch.equal(a, b) for pair, both in zip(got, want) for a, b in zip(pair, both))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = [chain(x) for x in xs]
    for _ in range(20):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for pair, both in zip(got, want) for a, b in zip(pair, both))
