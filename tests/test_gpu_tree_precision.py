"""GPU: the attention of drafted trees within bounds that know which kernel ran (tree_tight): probabilities in two terms where they are
promised, one where not, none rounded in the kernels without tensor cores. Pieces of several tiles, and more sequences than threads."""
import numpy as np
import pytest
import torch

from test_gpu_tree import DT, SHAPES, TYPES, both_paths, problem, run
from tree_tight import check_path, few_keys

pytestmark = pytest.mark.gpu


def check_all(pkg, c, Q, cu, mask):
    known, tags = {}, []
    for tag, got in both_paths(pkg, c, Q, cu, mask):
        check_path(pkg, c, Q, cu, mask, tag, got, known)
        tags.append(tag)
    return tags


@pytest.mark.parametrize("dtype,cache", TYPES)
@pytest.mark.parametrize("rows", [[5, 3], [40, 20]])
def test_probabilities_in_the_promised_bits(pkg, rows, dtype, cache):
    c, Q, cu, mask = few_keys(DT[dtype], cache, rows)
    assert ("tiled" in check_all(pkg, c, Q, cu, mask)) == (dtype != "f32")


@pytest.mark.parametrize("dtype,cache", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_shapes(pkg, shape, dtype, cache):
    lens, rows, Hq, Hkv, d, page, layout = shape
    check_all(pkg, *problem(dtype, cache, lens, rows, Hq, Hkv, d, page, layout, seed=d + page))


@pytest.mark.parametrize("dtype,cache", TYPES)
@pytest.mark.parametrize("rows,d,page,q_scale", [(3, 128, 16, 1.0), (20, 64, 24, 6.0), (40, 80, 64, 2.0), (70, 64, 100, 4.0)])
def test_pieces_of_several_tiles(pkg, rows, d, page, q_scale, dtype, cache):
    """Units of 6, 40, 80 and 140 rows, whose running maximum moves from tile to tile."""
    c, Q, cu, mask = problem(dtype, cache, [900, 800, 700], [rows] * 3, 32, 16, d, page, "hnd", seed=rows, q_scale=q_scale)
    check_all(pkg, c, Q, cu, mask)


@pytest.mark.parametrize("dtype,cache", [("f32", "native"), ("bf16", "native"), ("f16", "int8"), ("bf16", "e4m3")])
def test_more_sequences_than_threads(pkg, dtype, cache):
    """The list of key tiles is cut by a scan over the sequences, a CTA's threads at a time: 700 of them, some without rows or keys."""
    rng = np.random.default_rng(3)
    lens, rows = rng.integers(0, 40, 700), rng.integers(0, 4, 700)
    lens[rng.integers(0, 700, 60)] = 0
    lens[[255, 256, 257, 383, 384, 385, 639, 640, 641, 699]] = 39
    rows[[255, 256, 257, 383, 384, 385, 639, 640, 641, 699]] = 2
    c, Q, cu, mask = problem(dtype, cache, lens.tolist(), rows.tolist(), 2, 1, 16, 8, seed=1)
    assert ("tiled" in check_all(pkg, c, Q, cu, mask)) == (dtype != "f32")


@pytest.mark.parametrize("dtype,cache", TYPES)
def test_a_call_repeats_itself_bit_for_bit(pkg, dtype, cache):
    for rows, heads in (([3, 9, 1], 8), ([80, 40, 20], 16), ([1, 0, 2], 2)):
        c, Q, cu, mask = problem(dtype, cache, [1900, 300, 700], rows, heads, 2, 64, 16, seed=rows[0])
        first = run(pkg, c, Q, cu, mask)
        for _ in range(5):
            assert all(torch.equal(x, y) for x, y in zip(run(pkg, c, Q, cu, mask), first))


@pytest.mark.parametrize("dtype,cache", TYPES)
def test_a_chunk_of_a_prompt(pkg, dtype, cache):
    """Hundreds of rows that see the committed positions and one another causally, ragged, beside a single token."""
    rows = [300, 1, 65]
    c, Q, cu, _ = problem(dtype, cache, [200, 90, 0], rows, 4, 2, 64, 16, seed=2)
    mask = torch.zeros(sum(rows), max(rows), dtype=torch.bool)
    for b, T in enumerate(rows):
        mask[cu[b]:cu[b + 1], :T] = torch.ones(T, T, dtype=torch.bool).tril()
    check_all(pkg, c, Q, cu, mask)


@pytest.mark.parametrize("rows", [3, 20, 70])
def test_bfloat16_values_near_the_largest(pkg, rows):
    """V of 2^121 under probabilities that add up to little more than 1: finite in every kernel, whatever reference it holds them to."""
    c, _, cu, mask = problem("bf16", "native", [900, 800, 700], [rows] * 3, 32, 16, 64, 16, "hnd", seed=rows)
    g = torch.Generator().manual_seed(1)
    Q = (1 + 0.1 * torch.randn(3 * rows, 32, 64, generator=g)).to(c.dtype)
    c.K.mul_(0.02)
    c.V.copy_(torch.where(c.V < 0, -1.0, 1.0) * (1 + c.V.abs() / 8) * 2.0 ** 121)
    for b, n in enumerate((900, 800, 700)):  # in a later tile, scores of about 5.2: e^5.2 = 2^7.5 times the others, which are then taken away
        for p in range(n):
            c.K[c.place(b, p)] -= 3.0 if p % 64 else 0.0
        c.K[c.place(b, 300)] = 0.65
    check_all(pkg, c, Q, cu, mask)
