"""Rows of GGUF tables for tokens: with scale 1 the bits of `dequantize_rows`, with another one the float32 product rounded once - both exact, so everything is equal.  Every type, tokens of both
widths and any shape, repeated ones, those that are nobody's, tables past 2^31 bytes, addresses that only the type's own alignment has."""
import pytest
import torch

import oracle
from dinoml_v2_b200 import kernels, synthetic
from dinoml_v2_b200.gguf_blocks import QTYPES

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
DTYPES = ("bfloat16", "float16", "float32")


def _table(qtype, rows, width, seed=3):
    return torch.from_numpy(synthetic.random_blocks(qtype, rows, width, seed=seed)).to(DEV)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("qtype", sorted(QTYPES))
def test_rows(qtype, dtype):
    g = torch.Generator(device=DEV)
    g.manual_seed(1)
    for blocks, count in ((1, 1), (3, 5), (9, 300), (40, 1200)):
        width = blocks * QTYPES[qtype].block_size
        table = _table(qtype, 77, width)
        dense = torch.from_numpy(oracle.dequantize(table.cpu().numpy(), qtype, width)).to(DEV)
        for t in (torch.int32, torch.int64):
            tokens = torch.randint(0, 77, (count,), device=DEV, generator=g).to(t)
            got = kernels.embedding(tokens, table, qtype, dtype)
            assert torch.equal(got, dense[tokens.long()].to(got.dtype)) and torch.equal(got, kernels.dequantize_rows(table, qtype, width, dtype)[tokens.long()])
            got = kernels.embedding(tokens, table, qtype, dtype, scale=53.7)
            assert torch.equal(got, (dense[tokens.long()] * torch.tensor(53.7, device=DEV)).to(got.dtype))


def test_shapes_and_given():
    table = _table("Q8_0", 50, 96)
    tokens = torch.arange(24, device=DEV).view(2, 3, 4) % 50
    want = kernels.dequantize_rows(table, "Q8_0", 96, "bfloat16")
    got = kernels.embedding(tokens, table, "q8_0")
    assert got.shape == (2, 3, 4, 96) and torch.equal(got.view(24, 96), want[:24])
    out = torch.empty_like(got)
    assert kernels.embedding(tokens, table, 8, out=out) is out and torch.equal(out, got)
    assert torch.equal(kernels.embedding(tokens[0, 0, 1], table, "Q8_0"), want[1])
    assert torch.equal(kernels.embedding(tokens, table, "Q8_0", scale=2), got * 2)
    assert kernels.embedding(tokens[:0], table, "Q8_0").shape == (0, 3, 4, 96)


@pytest.mark.parametrize("dtype", DTYPES)
def test_tokens_that_are_in_no_table(dtype):
    table = _table("Q4_K", 10, 512)
    want = kernels.dequantize_rows(table, "Q4_K", 512, dtype)
    for t in (torch.int32, torch.int64):
        tokens = torch.tensor([3, -1, 9, -1], device=DEV).to(t)
        got = kernels.embedding(tokens, table, "Q4_K", dtype)
        assert torch.equal(got[[0, 2]], want[[3, 9]]) and not got[[1, 3]].any() and kernels.device_status() == 0      # nobody's
        for bad in (10, -2, torch.iinfo(t).max, torch.iinfo(t).min):
            tokens = torch.tensor([bad, 4], device=DEV, dtype=t)
            got = kernels.embedding(tokens, table, "Q4_K", dtype)
            assert not got[0].any() and torch.equal(got[1], want[4]) and kernels.device_status() == 10


def test_large_tables():
    """Offsets past 32 bits, of the table and of the result."""
    table = torch.zeros(700000, 4608, dtype=torch.uint8, device=DEV)                      # 3.2 GB of Q4_K, rows of 8192
    part = _table("Q4_K", 3, 8192)
    table[[0, 500000, 699999]] = part
    tokens = torch.tensor([699999, 0, 500000], device=DEV)
    want = kernels.dequantize_rows(part, "Q4_K", 8192, "float32")
    assert torch.equal(kernels.embedding(tokens, table, "Q4_K", "float32"), want[[2, 0, 1]])
    many = torch.full((140000,), 5, device=DEV, dtype=torch.int32)                        # 4.6 GB out
    many[-1] = 699999
    got = kernels.embedding(many, table, "Q4_K", "float32")
    assert torch.equal(got[-1], want[2]) and not got[:-1].any()


@pytest.mark.parametrize("qtype", sorted(QTYPES))
def test_tables_at_any_address(qtype):
    at = {"Q4_K": 4, "Q8_0": 2, "Q6_K": 2}.get(qtype, 1)
    table = _table(qtype, 20, 768)
    room = torch.empty(table.numel() + 32, dtype=torch.uint8, device=DEV)
    odd = room[at:at + table.numel()].view(table.shape)
    odd.copy_(table)
    tokens = torch.arange(20, device=DEV)
    assert torch.equal(kernels.embedding(tokens, odd, qtype), kernels.embedding(tokens, table, qtype))
    if at > 1:
        odd = room[1:1 + table.numel()].view(table.shape)
        with pytest.raises(RuntimeError):
            kernels.embedding(tokens, odd, qtype)


def test_refusals():
    table = _table("Q6_K", 10, 512)
    tokens = torch.zeros(4, dtype=torch.int32, device=DEV)
    for args, kwargs in (((tokens.cpu(), table, "Q6_K"), {}), ((tokens, table.cpu(), "Q6_K"), {}), ((tokens.float(), table, "Q6_K"), {}), ((tokens, table[:, :100], "Q6_K"), {}),
                         ((tokens, table[:, :300].contiguous(), "Q6_K"), {}), ((tokens, table, "Q9"), {}), ((tokens, table, "Q6_K", "int8"), {}), ((tokens, table.int(), "Q6_K"), {}),
                         ((tokens[::2], table, "Q6_K"), {}), ((tokens, table, "Q6_K"), {"out": torch.empty(4, 512, device=DEV)}),
                         ((tokens, table, "Q6_K"), {"out": torch.empty(3, 512, dtype=torch.bfloat16, device=DEV)}), ((tokens, table[:0], "Q6_K"), {})):
        with pytest.raises(ValueError):
            kernels.embedding(*args, **kwargs)


def test_other_streams_and_graphs():
    table = _table("Q5_K", 60, 2048)
    tokens = torch.arange(40, device=DEV, dtype=torch.int32)
    want = kernels.dequantize_rows(table, "Q5_K", 2048, "bfloat16")
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    got = kernels.embedding(tokens, table, "Q5_K", stream=stream)
    stream.synchronize()
    assert torch.equal(got, want[:40])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = kernels.embedding(tokens, table, "Q5_K")
    tokens += 20
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want[20:])
