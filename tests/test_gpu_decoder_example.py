"""The decoder of examples/ - norms, quantized linears, cache and attention together: a captured step replayed is the step, token by token and byte by
byte, and a prompt that came in one call fills the cache with what its layer's linear gave.

Bound of the values read back, from the arithmetic: int8 half a step of the block's scale, e4m3 2^-4 of the value or half of the smallest step, 2^-10 of the
scale; one rounding to bfloat16 on top, 2^-8 of the value."""
import importlib.util
from pathlib import Path

import pytest
import torch

from dinoml_v2_b200 import kernels

pytestmark = pytest.mark.gpu


def _example():
    spec = importlib.util.spec_from_file_location("decoder_example", Path(__file__).resolve().parents[1] / "examples" / "decoder.py")
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


PROMPTS = [list(range(1, 131)), [7], list(range(50, 83))]


@pytest.mark.parametrize("cache", ["int8", "float8_e4m3fn"])
def test_replayed_steps_are_the_steps(cache):
    example = _example()
    c = example.Config(width=512, heads=8, kv_heads=2, head_dim=64, hidden=1024, vocabulary=1024, qtype="Q8_0", cache=cache, block=16)
    steps, sides = 20, []
    for captured in (True, False):
        decoder = example.Decoder(c, len(PROMPTS), 200)
        if captured:
            tokens = example.generate(decoder, PROMPTS, steps)
        else:
            out = [decoder.prefill(PROMPTS)]
            for _ in range(steps):
                out.append(decoder.step(out[-1]))
            tokens = torch.stack(out, dim=1)
        torch.cuda.synchronize()
        sides.append((tokens, decoder))
    assert kernels.device_status() == 0
    (a, x), (b, y) = sides
    assert a.shape == (len(PROMPTS), steps + 1) and int(a.min()) >= 0 and int(a.max()) < c.vocabulary
    assert torch.equal(a, b) and len(set(a.flatten().tolist())) > steps          # (not one token over and over)
    assert x.lengths.tolist() == y.lengths.tolist() == [len(p) + steps for p in PROMPTS]
    for left, right in zip(x.caches, y.caches):
        for s, t in zip(left, right):
            assert torch.equal(s.view(torch.uint8), t.view(torch.uint8))


@pytest.mark.parametrize("cache", ["int8", "float8_e4m3fn"])
def test_prompts_are_in_the_cache(cache):
    example = _example()
    c = example.Config(layers=1, width=512, heads=8, kv_heads=2, head_dim=64, hidden=1024, vocabulary=1024, qtype="Q8_0", cache=cache, block=16)
    decoder = example.Decoder(c, len(PROMPTS), 200)
    decoder.prefill(PROMPTS)
    starts = torch.tensor([0, 130, 131, 164], dtype=torch.int32, device="cuda")
    k, v = kernels.kv_cache_read(decoder.caches[0], decoder.table, starts, 164)
    layer = decoder.layers[0]
    x, _ = kernels.rms_norm(decoder.embedding[torch.tensor(sum(PROMPTS, []), device="cuda")], layer.attention_norm, c.eps)
    wanted = kernels.gemm_rcr(x, layer.qkv, c.qtype).view(164, -1, c.head_dim)[:, c.heads:].double()
    position = torch.cat([torch.arange(len(p)) for p in PROMPTS]).cuda()
    sequence = torch.repeat_interleave(torch.arange(3), torch.tensor([len(p) for p in PROMPTS])).cuda()
    block = decoder.table[sequence, position // c.block].long()
    for got, want, scale in ((k, wanted[:, :c.kv_heads], decoder.caches[0].k_scale), (v, wanted[:, c.kv_heads:], decoder.caches[0].v_scale)):
        step = scale[block].double()[:, :, None]
        bound = step * (0.5 + 2.0 ** -14) if cache == "int8" else torch.maximum(want.abs() * 2.0 ** -4, step * 2.0 ** -10)
        bound = bound + (want.abs() + bound) * 2.0 ** -8
        assert bool(((got.double() - want).abs() <= bound).all())
    assert kernels.device_status() == 0
