"""Numbers that an adapter plan's lists cannot hold are refused, not cut to 32 bits or to whole numbers."""
import numpy as np
import pytest

from roost_b200.kernels import library


@pytest.mark.parametrize("counts,slots", [([1], [2 ** 32]), ([1], [2 ** 31]), ([1, 1], [0, 2 ** 63]), ([1], [0.5]), ([1.5], [0]), ([1], ["0"]), ([2 ** 31], [0]),
                                          ([2 ** 30, 2 ** 30], [0, -1]), ([2 ** 62, 2 ** 62, 2 ** 62], [0, 0, 0]), ([2 ** 64], [0]), (np.ones(1, np.uint64), np.full(1, 2 ** 63, np.uint64))])
def test_refused(counts, slots):
    with pytest.raises(library.KernelError):
        library.adapter_lists(counts, slots)


def test_taken():
    for counts, slots in (([2, 1], [2 ** 31 - 1, -1]), (np.array([2, 1], np.int32), np.array([2 ** 31 - 1, -5], np.int64)), ((2, 1), (2 ** 31 - 1, -2 ** 40))):
        rows, tiles, _ = library.adapter_lists(counts, slots)
        assert rows.tolist() == [0, 1] and tiles.tolist() == [[2 ** 31 - 1, 0, 2]]
