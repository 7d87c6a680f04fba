"""CPU tests of what the rotation takes for results that share no memory with what is still read: by addresses, whoever holds the memory."""
import numpy as np
import torch

from dinoml_v2_b200 import kernels


def _views(memory, begin, rows, pitch, heads, dim):
    """[rows, heads, dim] at element `begin` of a row of `pitch`, of a storage that begins there."""
    return torch.from_numpy(memory[begin:]).as_strided((rows, heads, dim), (pitch, dim, 1))


def test_one_memory_in_several_storages():
    memory = np.zeros(10 * 64, dtype=np.float32)
    at = lambda begin, heads=2, rows=5: _views(memory, begin, rows, 128, heads, 16)       # noqa: E731
    q, k = at(0), at(32)
    assert q.untyped_storage().data_ptr() != k.untyped_storage().data_ptr()
    assert kernels._apart(q, k) and kernels._apart(k, q)
    assert not kernels._apart(q, at(0)) and not kernels._apart(q, at(16)) and not kernels._apart(at(16), q)
    assert not kernels._apart(at(0, 4), k) and kernels._apart(at(0, 4), at(64)) and not kernels._apart(at(96, 4, 4), at(0, 2))
    assert kernels._apart(at(0, rows=2), at(256, rows=2)) and not kernels._apart(at(0, rows=3), at(256, rows=2))
    other = np.zeros(10 * 64, dtype=np.float32)
    assert kernels._apart(q, _views(other, 0, 5, 128, 2, 16))


def test_one_storage():
    x = torch.zeros(5, 12, 16, dtype=torch.bfloat16)
    assert kernels._apart(x[:, :4], x[:, 4:6]) and kernels._apart(x[:, 8:], x[:, :8]) and not kernels._apart(x[:, :4], x[:, 3:6])
    assert kernels._apart(x[:2], x[2:]) and not kernels._apart(x[:3], x[2:]) and kernels._apart(x[:0], x)
    assert not kernels._apart(x[:, :4].transpose(0, 1), x[:, :4])
