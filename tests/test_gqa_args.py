"""CPU tests of the grouped-head entry points' host index arrays: taken as the
integers they are, or refused."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from wave_engine_b200 import gqa


@pytest.mark.parametrize("a", [[0, 3, 2 ** 31 - 1], (0, 3, 2 ** 31 - 1), np.array([0, 3, 2 ** 31 - 1]),
                               np.array([0, 9, 3, 9, 2 ** 31 - 1, 9], dtype=np.int32)[::2],
                               np.array([0, 3, 2 ** 31 - 1], dtype=np.uint64), torch.tensor([0, 3, 2 ** 31 - 1])])
def test_integers_of_any_width(a):
    ptr, keep = gqa._index(a, 3, "cu", 0)
    assert keep.dtype == np.int32 and keep.tolist() == [0, 3, 2 ** 31 - 1] and keep.flags.c_contiguous
    assert ptr == keep.ctypes.data


def test_nothing_and_an_empty_array():
    assert gqa._index(None, 3, "cu", 0) == (0, None)
    assert gqa._index([], 0, "slots", 0)[1].size == 0


@pytest.mark.parametrize("a", [[0, 2 ** 31, 5], np.array([0, 2 ** 32, 5]), np.array([0, -2 ** 31 - 1, 5]), torch.tensor([0, 2 ** 32, 5]),
                               np.array([0, 2 ** 63, 5], dtype=np.uint64), [0.0, 1.5, 2.0], np.array([0, 1, 2.0]),
                               [False, True, True], [[0], [1], [2]], torch.tensor([[0, 1, 2]]), [0, 1], [0, 1, 2, 3]])
def test_refused(a):
    with pytest.raises(ValueError):
        gqa._index(a, 3, "cu", 0)
