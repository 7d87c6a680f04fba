"""Steps of a pool of cache blocks against one of lists: everything is a whole number and equal.  Prompts and single tokens, tokens taken back across blocks, requests that end and others that
come in the same step, a pool that runs out, tables that are full, batches with rows to spare, up to 8192 sequences, numbers that cannot be."""
import random

import pytest
import torch

from dinoml_v2_b200 import kernels
from oracle import decode_ends as E

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _same(pool, step, model, want):
    lengths, starts, positions, slots = want
    width = pool.block_table.shape[1]
    assert pool.block_table.tolist() == [t + [-1] * (width - len(t)) for t in model.tables]
    assert pool.lengths.tolist() == model.lengths and pool.free_count.tolist() == [len(model.free)] and pool.free[:len(model.free)].tolist() == model.free
    assert step.lengths.tolist() == lengths and (step.starts is None) == (starts is None) and (starts is None or step.starts.tolist() == starts)
    assert step.positions.tolist() == positions and step.slots.tolist() == slots


class Both:
    def __init__(self, *shape):
        self.pool, self.model = kernels.kv_pool(*shape), E.Pool(*shape)

    def step(self, new, rows=None, drop=None):
        step = kernels.kv_pool_step(self.pool, _ints(new), rows, drop=None if drop is None else _ints(drop))
        _same(self.pool, step, self.model, self.model.step(new, rows, drop))
        assert kernels.device_status() == 0
        return step


@pytest.mark.parametrize("block", [16, 32, 64, 128])
@pytest.mark.parametrize("sequences", [1, 3, 40, 257, 1500])
def test_random_steps(sequences, block):
    rng = random.Random(sequences + block)
    both = Both(sequences * 4 + 3, sequences, 9, block)
    for i in range(12):
        new, drop = [], []
        for b in range(sequences):
            n = both.model.lengths[b]
            drop.append(rng.choice([0, 0, rng.randint(0, 3), n, rng.randint(0, n), 1 << 30]))
            new.append(rng.choice([0, 1, 1, rng.randint(0, 5 * block)]) if i % 3 else rng.randint(0, 1))
        each = i % 3 == 0
        both.step(new, None if each else sum(new) + rng.randint(0, 40), drop if i % 4 else None)


def test_decode_across_blocks():
    both = Both(12, 3, 4, 16)
    both.step([15, 0, 33], 48)
    for _ in range(20):
        both.step([1, 0, 1])
    both.step([0, 5, 0], 5, [1 << 30, 0, 7])


def test_what_goes_comes_back_to_the_same_places():
    both = Both(64, 5, 8, 16)
    both.step([100, 17, 0, 64, 128], 309)
    table = both.pool.block_table.clone()
    both.step([9, 17, 0, 40, 128], 194, [9, 1000, 5, 40, 128])
    assert torch.equal(both.pool.block_table, table)


def test_pool_runs_out():
    both = Both(6, 5, 8, 16)
    both.step([40, 16, 20, 1, 0], 77)                                                     # 3 + 1 + 2 blocks: the fourth goes without
    assert both.pool.lengths.tolist() == [40, 16, 20, 0, 0]
    step = both.step([1, 1, 1, 1, 1])                                                     # the first and third have room in their blocks, the second wants one
    assert step.lengths.tolist() == [41, 0, 21, 0, 0] and step.positions.tolist() == [40, -1, 20, -1, -1]
    both.step([0, 16, 0, 0, 0], 16, [41, 0, 0, 0, 0])                                     # given back and handed out in one step
    both.step([200, 1, 0, 0, 0], 300)                                                     # more than a table's row has
    both.step([5, 3, 1, 0, 0], 7)                                                         # more than the batch's rows: the third's would be the ninth
    both.step([0, 0, 0, 0, 0], 0, [9, 99, 999, 0, 0])                                     # no rows at all


def test_later_ones_do_not_overtake():
    both = Both(3, 4, 8, 16)
    step = both.step([16, 48, 16, 0], 80)
    assert step.starts.tolist() == [0, 16, 16, 16, 16]


@pytest.mark.parametrize("sequences,block", [(8192, 16), (4097, 128), (1024, 64)])
def test_many_sequences(sequences, block):
    rng = random.Random(5)
    both = Both(3 * sequences, sequences, 5, block)
    new = [rng.randint(0, 2 * block) for _ in range(sequences)]
    both.step(new, sum(new))
    both.step([rng.randint(0, 1) for _ in range(sequences)], None, [rng.choice([0, 1, 1 << 30]) for _ in range(sequences)])


def test_long_prompts():
    both = Both(5000, 3, 4096, 16)
    both.step([65536, 0, 12345], 78000)
    both.step([1, 1, 1], None, [65000, 0, 12000])


def test_table_that_is_a_view():
    wide = torch.full((4, 20), 7, dtype=torch.int32, device=DEV)
    pool = kernels.kv_pool(10, 4, 6, 32)
    pool = pool._replace(block_table=wide[:, 3:9])
    pool.block_table.fill_(-1)
    model = E.Pool(10, 4, 6, 32)
    step = kernels.kv_pool_step(pool, _ints([50, 1, 0, 70]), 130)
    _same(pool, step, model, model.step([50, 1, 0, 70], 130))
    assert (wide[:, :3] == 7).all() and (wide[:, 9:] == 7).all()


def test_numbers_that_cannot_be():
    """They are told by the status, change nothing outside of the pool, and read nothing outside of it."""
    def fresh():
        pool = kernels.kv_pool(8, 3, 4, 16)
        kernels.kv_pool_step(pool, _ints([20, 16, 5]), 41)
        return pool

    pool = fresh()
    step = kernels.kv_pool_step(pool, _ints([1, -5, 2]))                                  # a negative number, and two where one is the most
    assert kernels.device_status() == 10 and pool.lengths.tolist() == [21, 16, 5] and step.lengths.tolist() == [21, 0, 0]
    step = kernels.kv_pool_step(pool, _ints([1, 1, 1]), drop=_ints([0, -3, 0]))           # the second wants a block, there are four
    assert kernels.device_status() == 10 and pool.lengths.tolist() == [22, 17, 6]
    for name, value in (("lengths", [-4, 16, 5]), ("lengths", [20, 1000, 5]), ("free_count", [-2]), ("free_count", [99]), ("lengths", [(1 << 31) - 1] * 3), ("lengths", [-(1 << 31)] * 3)):
        pool = fresh()
        getattr(pool, name).copy_(_ints(value))
        kernels.kv_pool_step(pool, _ints([1, 1, 1]), drop=_ints([100, 0, 3]))
        assert kernels.device_status() == 10
        assert 0 <= int(pool.free_count) <= 8 and int(pool.lengths.min()) >= 0 and int(pool.lengths.max()) <= 64
    pool = fresh()
    pool.block_table[1, 0] = 12345                                                        # a block that is none comes back
    kernels.kv_pool_step(pool, _ints([0, 0, 0]), 4, drop=_ints([0, 16, 0]))
    assert kernels.device_status() == 10
    pool = fresh()
    pool.free.fill_(1 << 30)                                                              # a stack of nothing: no slot
    step = kernels.kv_pool_step(pool, _ints([0, 1, 0]))
    assert step.positions.tolist() == [-1, 16, -1] and step.slots.tolist() == [-1, -1, -1] and kernels.device_status() == 10


def test_refusals():
    pool = kernels.kv_pool(8, 3, 4, 16)
    new = _ints([1, 0, 1])
    for p, args, kwargs in ((pool, (new.long(),), {}), (pool, (new[:2],), {}), (pool, (new.cpu(),), {}), (pool, (new, -1), {}), (pool, (new, 1 << 31), {}), (pool, (new,), {"drop": new[:1]}),
                            (pool._replace(lengths=pool.lengths[:2]), (new,), {}), (pool._replace(free=pool.free.long()), (new,), {}), (pool._replace(free_count=new), (new,), {}),
                            (pool._replace(block_table=pool.block_table.t()), (_ints([1] * 4),), {}), (pool._replace(block_size=24), (new,), {}),
                            (pool._replace(block_table=pool.block_table[:1].expand(3, 4)), (new,), {}), (pool._replace(free=pool.free[:0]), (new,), {})):
        with pytest.raises(ValueError):
            kernels.kv_pool_step(p, *args, **kwargs)
    for args in ((0, 1, 1, 16), (1, 0, 1, 16), (1, 1, 0, 16), (1, 1, 1, 17), (1, 8193, 1, 16), (1 << 28, 1, 1, 16), (1, 1, 1 << 28, 16)):
        with pytest.raises(ValueError):
            kernels.kv_pool(*args)
    assert pool.lengths.tolist() == [0, 0, 0] and pool.free_count.tolist() == [8]


def test_replayed_steps():
    both = Both(40, 4, 8, 16)
    both.step([10, 30, 0, 16], 56)
    new = _ints([1, 1, 0, 1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step = kernels.kv_pool_step(both.pool, new)
    for _ in range(40):                                                                   # over several blocks
        graph.replay()
        want = both.model.step([1, 1, 0, 1])
        torch.cuda.synchronize()
        _same(both.pool, step, both.model, want)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    step = kernels.kv_pool_step(both.pool, new, stream=stream)
    stream.synchronize()
    _same(both.pool, step, both.model, both.model.step([1, 1, 0, 1]))
