"""What reaches each request when a step leaves another one out: the rows of a sequence that got nothing are not there, so that those of the sequences behind it come earlier than their tokens
do in what the host packed.  And requests that no slot could ever take are refused before anything of them is packed."""
import importlib
import sys
from pathlib import Path

import pytest
import torch

from dinoml_v2_b200 import kernels
from oracle import decode_ends as E

ROOT = Path(__file__).resolve().parents[1]


def _example():
    if str(ROOT) not in sys.path:
        sys.path.insert(0, str(ROOT))
    return importlib.import_module("examples.serving")


# blocks, sequences, columns of 16; tokens that are there; tokens that are new, whether they fit (drop: all of the others' tokens)
CASES = [(40, 3, 8, [0, 0, 0], [200, 17, 5], [False, True, True]),                         # a prompt longer than a row of the table, first
         (40, 3, 8, [0, 0, 0], [17, 200, 5], [True, False, True]),
         (3, 3, 8, [0, 20, 0], [40, 1, 16], [False, True, False]),                         # one block left: a prompt goes without, a decode has room in its block
         (3, 4, 8, [0, 20, 0, 0], [40, 1, 0, 9], [False, True, False, False]),
         (40, 4, 8, [0, 0, 0, 0], [200, 0, 129, 3], [False, False, False, True]),
         (40, 2, 8, [0, 0], [500, 129], [False, False]),                                   # nobody
         (40, 1, 8, [0], [128], [True])]


def _packed(new):
    return [1000 * b + i for b, n in enumerate(new) for i in range(n)]


def _reached(rows, starts, positions):
    assert all((t >= 0) == (p >= 0) for t, p in zip(rows, positions))
    return [rows[starts[b]:starts[b + 1]] for b in range(len(starts) - 1)]


@pytest.mark.parametrize("blocks,sequences,columns,held,new,fits", CASES)
def test_tokens_reach_their_sequences(blocks, sequences, columns, held, new, fits):
    model = E.Pool(blocks, sequences, columns, 16)
    model.step(held, sum(held))
    lengths, starts, positions, slots = (torch.tensor(t, dtype=torch.int32) for t in model.step(new, sum(new)))
    step = kernels.KVStep(lengths, starts, positions, slots)
    rows = _example().tokens_of_rows(step, torch.tensor(new, dtype=torch.int32), torch.tensor(_packed(new), dtype=torch.int32)).tolist()
    assert _reached(rows, starts.tolist(), positions.tolist()) == [[1000 * b + i for i in range(n)] if ok else [] for b, (n, ok) in enumerate(zip(new, fits))]


def test_rows_to_spare():
    model = E.Pool(20, 2, 8, 16)
    step = kernels.KVStep(*(torch.tensor(t, dtype=torch.int32) for t in model.step([200, 3], 210)))
    rows = _example().tokens_of_rows(step, torch.tensor([200, 3], dtype=torch.int32), torch.tensor(_packed([200, 3]), dtype=torch.int32))
    assert rows.tolist() == [1000, 1001, 1002] + [-1] * 207
    step = kernels.KVStep(*(torch.tensor(t, dtype=torch.int32) for t in model.step([0, 0], 4)))
    assert _example().tokens_of_rows(step, torch.zeros(2, dtype=torch.int32), torch.zeros(0, dtype=torch.int32)).tolist() == [-1] * 4


@pytest.mark.gpu
@pytest.mark.parametrize("blocks,sequences,columns,held,new,fits", CASES)
def test_tokens_reach_their_sequences_on_the_device(blocks, sequences, columns, held, new, fits):
    ints = lambda t: torch.tensor(t, dtype=torch.int32, device="cuda")                    # noqa: E731
    pool = kernels.kv_pool(blocks, sequences, columns, 16)
    kernels.kv_pool_step(pool, ints(held), sum(held))
    step = kernels.kv_pool_step(pool, ints(new), sum(new))
    rows = _example().tokens_of_rows(step, ints(new), ints(_packed(new)))
    assert rows.dtype == torch.int32
    assert _reached(rows.tolist(), step.starts.tolist(), step.positions.tolist()) == [[1000 * b + i for i in range(n)] if ok else [] for b, (n, ok) in enumerate(zip(new, fits))]
    assert kernels.device_status() == 0


def _server(example, slots, blocks):
    from examples.decoder import Config
    return example.Server(Config(width=512, heads=8, kv_heads=2, head_dim=64, hidden=1024, vocabulary=1024, qtype="Q8_0", cache="int8", block=16, layers=1), slots, blocks, 128)


@pytest.mark.gpu
def test_requests_that_no_slot_takes():
    example = _example()
    server = _server(example, 3, 24)
    short = example.Request(list(range(17)), 3)
    for r in (example.Request([1] * 200, 3), example.Request([1] * 120, 10), example.Request([], 3), example.Request([1], 0)):
        with pytest.raises(ValueError):
            server.admit({0: r, 1: short})
        with pytest.raises(ValueError):
            example.serve(server, [short, r])
    assert not server.active.any() and server.pool.free_count.tolist() == [24]            # nothing was begun
    out = example.serve(server, [short, example.Request([1] * 119, 10)])
    assert [len(t) for t in out] == [3, 10] and kernels.device_status() == 0


@pytest.mark.gpu
def test_admitted_prompts_are_their_own():
    """What `admit` feeds its layers, with a prompt that finds no blocks ahead of an empty slot and behind one that does."""
    example = _example()
    server = _server(example, 4, 5)
    fed = {}
    forward = server.forward

    def keep(tokens, step):
        fed["tokens"], fed["step"] = tokens.tolist(), step
        return forward(tokens, step)

    server.forward = keep
    prompts = {0: list(range(40)), 1: list(range(100, 150)), 3: list(range(200, 203))}    # 3 and 4 blocks of 5, and who comes later does not overtake
    server.admit({slot: example.Request(p, 2) for slot, p in prompts.items()})
    starts, positions = fed["step"].starts.tolist(), fed["step"].positions.tolist()
    assert _reached(fed["tokens"], starts, positions) == [prompts[0], [], [], []]
    assert server.pool.lengths.tolist() == [40, 0, 0, 0] and kernels.device_status() == 0
