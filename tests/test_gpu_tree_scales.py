"""GPU: V of an 8-bit cache whose rows' scales differ widely. What counts is a row's own largest product of probability and scale: not
the largest scale around, whose key it may not attend to."""
import numpy as np
import pytest
import torch

import cache_ref
from test_gpu_tree import both_paths, problem
from tree_tight import check_path

pytestmark = pytest.mark.gpu
EIGHT = [(t, x) for t in ("f32", "f16", "bf16") for x in ("e4m3", "int8")]
LENS = [900, 800, 700]  # times 16 key heads: a CTA of the tensor cores takes three or five tiles one after the other


def places(c, b, positions):
    at = [c.place(b, p) for p in positions]
    return torch.tensor([x[0] for x in at], device="cuda"), torch.tensor([x[1] for x in at], device="cuda")


def set_rows(c, which, b, positions, factor):
    """K or V of some positions times a power of two (a number, or one for each), in every head."""
    s = getattr(c, which + "_scale")
    s[places(c, b, positions)] *= torch.as_tensor(factor, dtype=torch.float32).expand(len(positions)).cuda()[:, None]


def long_problem(dtype, cache, rows, d=64, seed=0):
    """Three sequences of `rows` drafted tokens each, 32 query heads on 16; all queries near (1, 1, ...)."""
    c, _, cu, mask = problem(dtype, cache, LENS, [rows] * 3, 32, 16, d, 16, "hnd", seed=seed)
    g = torch.Generator().manual_seed(seed + 2)
    return c, (1 + 0.2 * torch.randn(3 * rows, 32, d, generator=g)).to(c.dtype), cu, mask


def set_keys(c, b, positions, score):
    """K of some positions becomes one number throughout: a score of about `score` for queries near (1, 1, ...)."""
    at, x = places(c, b, positions), score / c.d ** 0.5
    c.K.view(torch.uint8 if c.cache == "e4m3" else torch.int8)[at] = (0x68 if x > 0 else 0xe8) if c.cache == "e4m3" else (64 if x > 0 else -64)
    c.K_scale[at] = abs(x) / 64  # the code of +-64


def check_paths(pkg, c, Q, cu, mask):
    known = {}
    for tag, got in both_paths(pkg, c, Q, cu, mask):
        check_path(pkg, c, Q, cu, mask, tag, got, known)
        yield got


@pytest.mark.parametrize("dtype,cache", EIGHT)
@pytest.mark.parametrize("rows", [3, 20, 70])
def test_a_large_row_that_nobody_attends_to(pkg, rows, dtype, cache):
    """V of about 6 x 10^4 beside 10^-3, at a score of -60: it adds nothing, and the others keep their bits. First, in the middle, at the
    end, and two in a tile."""
    c, Q, cu, mask = long_problem(dtype, cache, rows)
    for b, n in enumerate(LENS):
        set_rows(c, "V", b, range(n + rows), 2.0 ** -11)
        large = ((0, 170, n - 1), (300, 301, 600))[b % 2]
        set_rows(c, "V", b, large, 2.0 ** 26)
        set_keys(c, b, large, -60.0)
    for got in check_paths(pkg, c, Q, cu, mask):
        assert got[2].abs().max() < 0.05


@pytest.mark.parametrize("dtype,cache", EIGHT)
@pytest.mark.parametrize("rows", [3, 20, 70])
@pytest.mark.parametrize("spread", [2, 8])
def test_scales_of_a_wide_range(pkg, spread, rows, dtype, cache):
    """Every V row times a power of two between 2^-spread and 2^spread."""
    c, _, cu, mask = long_problem(dtype, cache, rows, seed=spread)
    Q = (torch.randn(3 * rows, 32, 64, generator=torch.Generator().manual_seed(1)) * 4).to(c.dtype)
    rng = np.random.default_rng(spread)
    for b, n in enumerate(LENS):
        set_rows(c, "V", b, range(n + rows), 2.0 ** rng.integers(-spread, spread + 1, n + rows))
    assert len(list(check_paths(pkg, c, Q, cu, mask))) >= 2


@pytest.mark.parametrize("dtype,cache", EIGHT)
@pytest.mark.parametrize("rows", [3, 20, 70])
def test_key_scales_of_a_wide_range(pkg, rows, dtype, cache):
    """Every K row times a power of two between 2^-10 and 2^2: scores from almost nothing to some twenty."""
    c, _, cu, mask = long_problem(dtype, cache, rows, seed=7)
    Q = (torch.randn(3 * rows, 32, 64, generator=torch.Generator().manual_seed(1)) * 2).to(c.dtype)
    rng = np.random.default_rng(rows)
    for b, n in enumerate(LENS):
        set_rows(c, "K", b, range(n + rows), 2.0 ** rng.integers(-10, 3, n + rows))
    assert len(list(check_paths(pkg, c, Q, cu, mask))) >= 2


@pytest.mark.parametrize("dtype,cache", [("f32", "int8"), ("bf16", "e4m3"), ("bf16", "int8")])
@pytest.mark.parametrize("rows", [3, 20, 70])
@pytest.mark.parametrize("low,high", [(-64, 0), (-64, 90), (0, -64), (90, -64), (90, 90)])
def test_scales_from_end_to_end_of_what_is_held(pkg, low, high, rows, dtype, cache):
    """Every other 128 keys lie far from the rest, and attention is on both, or twelve apart: l counts every key, whatever its V."""
    for lift in (0.0, 12.0, -12.0) if low * high < 0 else (0.0,):
        c, Q, cu, mask = long_problem(dtype, cache, rows, seed=5)
        for b, n in enumerate(LENS):
            far = [p for p in range(n + rows) if p // 128 % 2 == 0]
            set_rows(c, "V", b, far, 2.0 ** low)
            set_rows(c, "V", b, [p for p in range(n + rows) if p // 128 % 2], 2.0 ** high)
            if lift:
                set_keys(c, b, far, lift)
        assert len(list(check_paths(pkg, c, Q, cu, mask))) >= 2


@pytest.mark.parametrize("dtype,cache", EIGHT)
@pytest.mark.parametrize("rows", [3, 70])
def test_rows_of_zeros_beside_large_ones(pkg, rows, dtype, cache):
    """A V row of zeros has the smallest scale there is (int8: zero), and its key counts in l all the same."""
    c, Q, cu, mask = long_problem(dtype, cache, rows, seed=4)
    _, scale = cache_ref.quantise(np.zeros((16, 64)), cache)
    for b, n in enumerate(LENS):
        at = places(c, b, list(range(70)) + [n // 2, n - 1] + list(range(320, 320 + 64 * (b % 3))))
        c.V.view(torch.uint8)[at] = 0
        c.V_scale[at] = torch.from_numpy(scale).to(c.V_scale)
    assert len(list(check_paths(pkg, c, Q, cu, mask))) >= 2
    if dtype != "f16":
        for b, n in enumerate(LENS):
            set_rows(c, "V", b, range(100, n + rows), 2.0 ** 50)
        assert len(list(check_paths(pkg, c, Q, cu, mask))) >= 2
