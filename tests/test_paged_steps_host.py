"""Steps of a paged cache as the Python classes check them, without a GPU: device tensors are stand-ins."""
import numpy as np
import pytest
import torch

import skainet_b200 as skn
from skainet_b200.paged import _host_batch


class OnDevice:
    """what PagedBatch asks of a device tensor"""

    def __init__(self, shape, device, dtype=torch.int32):
        self.shape, self.dtype, self.is_cuda, self.device = torch.Size(shape), dtype, device is not None, torch.device("cuda", device) if device is not None else torch.device("cpu")

    def is_contiguous(self):
        return True

    def get_device(self):
        return self.device.index

    def data_ptr(self):
        return 4096


def test_a_step_lies_on_one_device():
    arrays = [(3, 5), (4,), (3,)]
    b = skn.PagedBatch(*(OnDevice(s, 1) for s in arrays), 7, 7)
    assert (b.device, b.n_seqs, b.max_pages) == (1, 3, 5)
    for other in range(3):
        with pytest.raises(ValueError, match="one device"):
            skn.PagedBatch(*(OnDevice(s, int(i == other)) for i, s in enumerate(arrays)), 7, 7)
        with pytest.raises(ValueError):
            skn.PagedBatch(*(OnDevice(s, None if i == other else 0) for i, s in enumerate(arrays)), 7, 7)


@pytest.mark.parametrize("table,starts,lens", [
    ([[0, 2 ** 32]], [0, 2], [20]), ([[0, 1]], [0, 2 ** 32 + 2], [20]), ([[0, 1]], [0, 2], [2 ** 32 + 20]), ([[0, 1]], [0, 2], [-2 ** 31 - 1]),
    ([[0, 1.5]], [0, 2], [20]), ([[0, 1]], [0, 2], [float("nan")]), ([[0, 1]], [0, float("inf")], [20]), ([[0, 1]], np.array([0, 2 ** 63 + 2], dtype=np.uint64), [20]), ([[0, 1]], [0, 2], [None])])
def test_numbers_that_are_no_int32_are_refused(table, starts, lens):
    """a host step's numbers are taken as they are or not at all: 2^32 + 20 is not 20"""
    with pytest.raises(ValueError, match="int32"):
        _host_batch(table, starts, lens, 2)


def test_steps_of_whole_numbers_are_taken():
    for kind in (list, np.int16, np.int64, np.uint64, np.int32, np.float32):
        make = (lambda a: a) if kind is list else (lambda a: np.array(a, dtype=kind))
        b, (table, starts, lens) = _host_batch(make([[0, 1], [3, 2]]), make([0, 2, 5]), make([20, 3]), 5)
        assert (b.n_seqs, b.n_tokens, b.max_new, b.max_pages) == (2, 5, 3, 2)
        assert table.tolist() == [[0, 1], [3, 2]] and starts.tolist() == [0, 2, 5] and lens.tolist() == [20, 3]
        assert table.dtype == starts.dtype == lens.dtype == np.int32
    b, _ = _host_batch(np.zeros((0, 0)), [0], [], 4)          # nothing is of no type
    assert (b.n_seqs, b.max_new) == (0, 0)
