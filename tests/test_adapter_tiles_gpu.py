"""Tiles of an adapter plan whose numbers are wrong reach nothing that is not the list's."""
import itertools

import pytest
import torch

from roost_b200.kernels.library import AdapterPlan
from tests.test_adapters_gpu import rand, want_and_bound

pytestmark = pytest.mark.gpu
LEAST, MOST = -2 ** 31, 2 ** 31 - 1
TYPES = [(torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32), (torch.float32, torch.float32)]


def ints(v):
    return torch.tensor(v, dtype=torch.int32).cuda()


@pytest.mark.parametrize("dtype,out", TYPES)
@pytest.mark.parametrize("tile_rows", [16, 64])
def test_ranges_of_any_numbers(kernels, dtype, out, tile_rows):
    """Every range that has none of the list's three entries, and ranges that hold them all and more."""
    x, y = rand((40, 64), dtype, 1), rand((40, 64), out, 2)
    y[5, 3] = -0.0
    a, b, scale = rand((2, 1, 8, 64), dtype, 3), rand((2, 64, 8), dtype, 4), torch.ones(2, device="cuda")
    rows = ints([7, 2, 30])
    ends = [LEAST, LEAST + 1, LEAST + 60, -70, -1, 0, 1, 2, 3, 4, MOST - 60, MOST - 1, MOST]
    empty = [[1, f, e] for f, e in itertools.product(ends, ends) if max(f, 0) >= min(max(e, 0), 3)]
    assert len(empty) > 100
    before = y.clone()
    kernels.adapters_add_(y, x, a, b, scale, AdapterPlan(rows, ints(empty), 40, tile_rows))
    assert torch.equal(y, before)
    for f, e in ((LEAST, MOST), (-1, 3), (0, MOST - 1)):
        y.copy_(before)
        kernels.adapters_add_(y, x, a, b, scale, AdapterPlan(rows, ints([[1, f, e]]), 40, tile_rows))
        for r in (7, 2, 30):
            want, bound = want_and_bound(before[r:r + 1], x[r:r + 1], a, b, scale, [1], [1], (64,), None, 2.0 ** -17)
            assert bool(((y[r:r + 1].double() - want).abs() <= bound).all())
        others = [r for r in range(40) if r not in (7, 2, 30)]
        assert torch.equal(y[others], before[others])


@pytest.mark.parametrize("dtype,out", TYPES)
def test_an_adapter_of_rank_zero_leaves_its_rows_as_they_are(kernels, dtype, out):
    """To the bit: a zero below zero too."""
    x, y = rand((20, 64), dtype, 1), torch.full((20, 64), -0.0, dtype=out, device="cuda")
    a, b, scale = rand((2, 1, 8, 64), dtype, 3), rand((2, 64, 8), dtype, 4), torch.ones(2, device="cuda")
    kernels.adapters_add_(y, x, a, b, scale, kernels.adapter_plan([20], [1]), ranks=ints([8, 0]))
    assert bool(torch.signbit(y).all()) and not bool(y.any())


@pytest.mark.parametrize("dtype,out", TYPES)
def test_tiles_longer_than_the_plan_says(kernels, dtype, out):
    """What lies beyond ``tile_rows`` is passed over, and the next tile's tokens have their own adapter's h."""
    x, y = rand((40, 264), dtype, 1), rand((40, 64), out, 2)
    a, b, scale = rand((2, 1, 8, 264), dtype, 3, 0.06), rand((2, 64, 8), dtype, 4), torch.ones(2, device="cuda")
    for tile_rows, lists in ((10, [[0, 0, 16], [1, 10, 20]]), (20, [[0, 0, 40], [1, 20, 40]])):
        got = kernels.adapters_add_(y.clone(), x, a, b, scale, AdapterPlan(ints(list(range(40))), ints(lists), 40, tile_rows))
        want, bound = want_and_bound(y, x, a, b, scale, [tile_rows, tile_rows], [0, 1], (64,), None, 2.0 ** -17)
        assert bool(((got.double() - want).abs() <= bound).all())
