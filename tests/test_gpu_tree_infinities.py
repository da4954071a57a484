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


def test_pieces_of_a_hundred_thousand_keys(pkg):
    """48 sequences of 131072 positions on shared pages, whose pieces are 170000 keys long: looking for the infinities of one must not
    hold its CTA up beyond the limit of the waits. Everything that sees no such value is, bit for bit, what it is without any."""
    B, n, H, d, ps, pool = 48, 131072, 8, 64, 64, 64
    g = torch.Generator().manual_seed(1)
    K, V = (torch.randn(pool, ps, H, d, generator=g).to("cuda", torch.bfloat16) for _ in range(2))
    Q = torch.randn(B, H, d, generator=g).to("cuda", torch.bfloat16)
    table = torch.randint(0, pool - 2, (B, n // ps + 1), generator=g, dtype=torch.int32)
    table[7, 500], table[20, 1500], table[33, 2047] = pool - 1, pool - 2, pool - 1
    lens, cu = torch.full((B,), n, dtype=torch.int32, device="cuda"), torch.arange(B + 1, dtype=torch.int32, device="cuda")
    mask = torch.ones(B, 1, dtype=torch.bool, device="cuda")

    def forward(k, v):
        m, l = (torch.empty(B, H, device="cuda") for _ in range(2))
        O = torch.empty_like(Q)
        pkg.binding("spfa_tree").forward(Q, k, v, table.cuda(), lens, cu, mask, m, l, O, first=True)
        torch.cuda.synchronize()
        assert pkg.capi.last_path() == pkg.capi.PATH_TILED and pkg.capi.last_device_error() == 0
        return m.cpu(), l.cpu(), O.cpu()

    m, l, O = forward(K, V)
    # 64 bits, a page as often as it is there. u = 2^-24: sums of n terms, 2^-8 of a probability's and the result's rounding
    times = torch.stack([torch.bincount(t, minlength=pool) for t in table[:, :-1].long()]).double()
    for b in range(0, B, 9):
        k, v = K.double().cpu(), V.double().cpu()
        last = table[b, -1].long()
        k, v = torch.cat([k.flatten(0, 1), k[last, :1]]), torch.cat([v.flatten(0, 1), v[last, :1]])  # the drafted token itself
        w = torch.cat([times[b].repeat_interleave(ps), torch.ones(1)]).double()
        s = torch.einsum("nhd,hd->hn", k, Q[b].double().cpu()) / d ** 0.5
        p = torch.exp(s - s.masked_fill(w == 0, -np.inf).amax(-1, keepdim=True)) * w
        size = torch.einsum("hn,nhd->hd", p, v.abs()) / p.sum(-1)[:, None]
        want = torch.einsum("hn,nhd->hd", p, v) / p.sum(-1)[:, None]
        rel = n * 2.0 ** -24 + 2.0 ** -18
        assert ((l[b].double() - p.sum(-1)).abs() <= rel * p.sum(-1)).all()
        assert ((O[b].double() - want).abs() <= (2 * rel + 2.0 ** -8) * size + 2.0 ** -8 * (want.abs() + (2 * rel + 2.0 ** -8) * size)).all()

    Vi = V.clone()
    Vi[pool - 1, 3, 2, 1], Vi[pool - 1, 60, 5, 63], Vi[pool - 1, 0, 2, 40] = BAD
    Kn = K.clone()
    Kn[pool - 2, 9, 4, 0] = float("nan")
    mi, li, Oi = forward(Kn, Vi)
    same = torch.ones(B, H, d, dtype=torch.bool)
    for b in (7, 33):
        assert (Oi[b, 2, 1] == np.inf) and (Oi[b, 5, 63] == -np.inf) and torch.isnan(Oi[b, 2, 40])
        same[b, 2, 1] = same[b, 5, 63] = same[b, 2, 40] = False
    assert torch.isnan(Oi[20, 4]).all() and torch.isnan(mi[20, 4]) and torch.isnan(li[20, 4])
    same[20, 4] = False
    assert torch.equal(Oi[same], O[same]) and torch.equal(mi[same[..., 0]], m[same[..., 0]]) and torch.equal(li[same[..., 0]], l[same[..., 0]])

    Vi = V.clone()
    Vi[3, 5, :, 17] = float("inf")  # in every piece
    mi, li, Oi = forward(K, Vi)
    assert (Oi[..., 17] == np.inf).all() and torch.equal(mi, m) and torch.equal(li, l)
    same = torch.arange(d) != 17
    assert torch.equal(Oi[..., same], O[..., same])
