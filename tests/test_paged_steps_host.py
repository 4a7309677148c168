"""Steps of a paged cache as the Python classes check them, without a GPU: device tensors are stand-ins."""
import numpy as np
import pytest
import torch

import skainet_b200 as skn


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
