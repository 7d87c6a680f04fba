"""The server of examples/ - embedding, rotation with norms of heads, pool, cache and attention, choice of tokens together, step after step: replayed steps are the steps, the pool ends as it began,
requests that wait for blocks get their tokens all the same, what a prompt left in the cache is what its linear gave, normed and turned, and tokens are chosen from the logits that the last
hidden states give."""
import importlib
import sys
from pathlib import Path

import pytest
import torch

from dinoml_v2_b200 import kernels
from oracle import decode_ends as E

pytestmark = pytest.mark.gpu
ROOT = Path(__file__).resolve().parents[1]


def _example():
    if str(ROOT) not in sys.path:
        sys.path.insert(0, str(ROOT))
    return importlib.import_module("examples.serving")


def _config(cache, **other):
    from examples.decoder import Config
    return Config(**dict(width=512, heads=8, kv_heads=2, head_dim=64, hidden=1024, vocabulary=1024, qtype="Q8_0", cache=cache, block=16) | other)


def _requests(example, count, longest=70):
    g = torch.Generator()
    g.manual_seed(3)
    out = []
    for i in range(count):
        n, most = (int(torch.randint(1, high, (1,), generator=g)) for high in (longest, 40))
        out.append(example.Request(torch.randint(0, 1024, (n,), generator=g).tolist(), most, (0.0, 0.7, 1.3)[i % 3], (0, 30)[i % 2], (1.0, 0.9)[i % 2], (0.0, 0.05)[i % 5 == 4]))
    return out


@pytest.mark.parametrize("cache", ["int8", "float8_e4m3fn"])
def test_replayed_steps_are_the_steps(cache):
    example = _example()
    requests, sides = _requests(example, 11), []
    for captured in (True, False):
        server = example.Server(_config(cache), 4, 40, 128)
        sides.append(example.serve(server, requests, captured))
        torch.cuda.synchronize()
        assert kernels.device_status() == 0
        assert server.pool.lengths.tolist() == [0] * 4 and sorted(server.pool.free.tolist()) == list(range(40)) and server.pool.free_count.tolist() == [40]
        assert (server.pool.block_table == -1).all()
    assert [len(t) for t in sides[0]] == [r.most for r in requests] and all(0 <= t < 1024 for row in sides[0] for t in row)
    assert sides[0] == sides[1]


def test_requests_wait_for_blocks():
    example = _example()
    requests = _requests(example, 9)
    server = example.Server(_config("int8"), 6, 12, 128)                                  # six requests of up to seven blocks: they do not all fit
    out = example.serve(server, requests)
    assert [len(t) for t in out] == [r.most for r in requests] and kernels.device_status() == 0
    assert server.pool.free_count.tolist() == [12]


@pytest.mark.parametrize("cache", ["int8", "float8_e4m3fn"])
def test_prompts_are_in_the_cache(cache):
    """Bound: half a step of int8 or 2^-4 of an e4m3 value (2^-10 of its scale at least); bfloat16's rounding of the linear's result, of what is turned and of what is read, 2^-8
    of a pair's length or the value each, and the rotation's own 2^-18."""
    example = _example()
    c = _config(cache, layers=1)
    server = example.Server(c, 3, 30, 160)
    prompts = {0: list(range(1, 131)), 2: list(range(50, 83))}
    server.admit({slot: example.Request(p, 1) for slot, p in prompts.items()})
    starts = torch.tensor([0, 130, 130, 163], dtype=torch.int32, device="cuda")
    k, v = kernels.kv_cache_read(server.caches[0], server.pool.block_table, starts, 163, "float32")
    tokens = torch.tensor(prompts[0] + prompts[2], device="cuda", dtype=torch.int32)
    x, _ = kernels.rms_norm(kernels.embedding(tokens, server.embedding, c.qtype), server.layers[0].attention_norm, c.eps)
    qkv = kernels.gemm_rcr(x, server.layers[0].qkv, c.qtype).view(163, -1, c.head_dim)
    position = torch.cat([torch.arange(130), torch.arange(33)])
    sequence = torch.repeat_interleave(torch.tensor([0, 2]), torch.tensor([130, 33]))
    block = server.pool.block_table.cpu()[sequence, position // c.block].long().cuda()
    wanted, size = E.rotate(qkv[:, c.heads:c.heads + c.kv_heads], server.head_norms[0][1], position, server.frequencies, c.eps, False, 1.0)
    for got, want, size, scale in ((k, wanted, size, server.caches[0].k_scale), (v, qkv[:, c.heads + c.kv_heads:].cpu().double(), torch.zeros(()), server.caches[0].v_scale)):
        step = scale[block].cpu().double()[:, :, None]
        turned = want.abs() * 2.0 ** -8 + size * 2.0 ** -17
        bound = step * (0.5 + 2.0 ** -14) if cache == "int8" else torch.maximum((want.abs() + turned) * 2.0 ** -4, step * 2.0 ** -10)
        assert bool(((got.cpu().double() - want).abs() <= bound + turned).all())
    assert kernels.device_status() == 0


def test_tokens_come_from_the_logits():
    example = _example()
    server = example.Server(_config("int8"), 4, 60, 128)
    requests = _requests(example, 4)
    seen = {}
    choose = server.choose

    def keep(x, step):
        seen["logits"], seen["step"] = kernels.gemm_rcr(x, server.head, server.c.qtype).cpu(), step
        choose(x, step)

    server.choose = keep
    for i in range(12):
        if i == 0:
            server.admit(dict(enumerate(requests)))
        else:
            server.decode(captured=False)
        u = server.uniforms.tolist()
        assert seen["step"].lengths.tolist() == [len(r.prompt) + i for r in requests]
        for slot, r in enumerate(requests):
            setting = [torch.tensor(v).float().item() for v in (r.temperature, r.top_p, r.min_p)]
            want, _, margin = E.choose(seen["logits"][slot], u[slot], setting[0], r.top_k, *setting[1:])
            assert margin < 2.0 ** -33 or int(server.tokens[slot]) == want
