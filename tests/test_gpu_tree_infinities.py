"""GPU: infinities and NaN in the V of a 16-bit cache that holds its values as they are. A key that a row sees has a probability above
zero, so that an infinity stands in its column of O with its sign, in every unit of rows, however the tensor cores hold the probability;
both signs, or a NaN, make NaN."""
import numpy as np
import pytest
import torch

from cache_ref import check_tree, tree_reference
from test_gpu_tree import both_paths, problem

pytestmark = pytest.mark.gpu
BAD = (float("inf"), float("-inf"), float("nan"))


def plant(c, b, places, head):
    """Column 1 + k of a head's V gets one value of BAD, column 5 both infinities."""
    for k, x in enumerate(BAD):
        c.V[c.place(b, places[k])][head, 1 + k] = x
    for k in range(2):
        c.V[c.place(b, places[k])][head, 5] = BAD[k]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("rows", [
    [40, 2, 2],    # units of 128 and 32 rows (the second one copied four times), 8 and 8
    [48, 1, 3],    # 128 and 64 (copied twice)
    [55, 9, 0],    # 128 and 92
    [8, 30, 20],   # whole sequences in a unit: two terms of the probabilities
    [80, 100, 5],  # units of 256 rows
])
def test_every_unit_of_rows(pkg, rows, d, dtype):
    c, Q, cu, mask = problem(dtype, "native", [300, 130, 64], rows, 8, 2, d, 16, "hnd", seed=rows[0])
    for b, n in enumerate((300, 130, 64)):
        plant(c, b, (n - 1, 3, n // 2), b % 2)
    want, bound, written = tree_reference(c, Q, cu, mask)
    assert np.isinf(want[2][0, 0, 1]) and np.isnan(want[2][0, 0, 5]) and np.isfinite(want[2][0, 0, 0])
    tags = []
    for tag, got in both_paths(pkg, c, Q, cu, mask):
        tags.append(tag)
        check_tree(got, want, bound, written, tag)
    assert "tiled" in tags


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("rows", [[3], [20], [70]])
def test_small_probabilities_of_infinite_values(pkg, rows, dtype):
    """Scores of about -40 beside 0 and a probability of 2^-58: not zero, though 16 bits beside the others' would say so."""
    c, _, cu, mask = problem(dtype, "native", [200], rows, 8, 2, 64, 16, seed=1)
    g = torch.Generator().manual_seed(2)
    Q = (1 + 0.1 * torch.randn(rows[0], 8, 64, generator=g)).to(c.dtype)
    c.K.mul_(0.1)
    for p in (150, 20, 77):
        c.K[c.place(0, p)] = -5
    plant(c, 0, (150, 20, 77), 1)
    want, bound, written = tree_reference(c, Q, cu, mask)
    assert np.isinf(want[2][:, 4:, 1]).all() and np.isnan(want[2][:, 4:, 5]).all()
    for tag, got in both_paths(pkg, c, Q, cu, mask):
        check_tree(got, want, bound, written, tag)
