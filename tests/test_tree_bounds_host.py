"""CPU: the bounds that results of the tree attention are held to by the kernel that ran notice a probability in fewer bits than that
kernel promises. The loss is planted in a restatement on the CPU."""
import numpy as np
import pytest
import torch

from cache_ref import check_tree
from tree_tight import few_keys, tree_tight

DT = {"f16": torch.float16, "bf16": torch.bfloat16}


def restate(c, Q, cu, mask, kind, terms):
    """The rows with the committed probabilities (times V's scale) in `terms` numbers of type `kind`, all else in 64 bits."""
    (m, l, O), _, _ = tree_tight(c, Q, cu, mask, "32 bits")
    O = O.copy()
    g = Q.shape[1] // c.heads
    for b in range(len(cu) - 1):
        rows, n = slice(cu[b], cu[b + 1]), int(c.lens[b])
        k, _ = c.dense("K", b, range(n))
        v, _ = c.dense("V", b, range(n))
        scale = np.ones((n, c.heads)) if c.cache == "native" else np.array([c.raw("V")[1].double().numpy()[c.place(b, i)] for i in range(n)])
        for h in range(Q.shape[1]):
            p = np.exp(Q[rows, h].double().numpy() @ k[:, h // g].T / np.sqrt(c.d) - m[rows, h, None])
            P = p * scale[:, h // g]
            unit = 2.0 ** (np.floor(np.log2(P.max(-1, keepdims=True))) - 8)
            left, held = torch.from_numpy(P / unit), 0.0
            for _ in range(terms):
                t = left.to(kind).double()
                held, left = held + t, left - t
            codes = np.divide(v[:, h // g], scale[:, h // g, None], out=np.zeros_like(v[:, h // g]), where=scale[:, h // g, None] != 0)
            O[rows, h] += ((held.numpy() * unit - P) @ codes) / l[rows, h, None]
    return torch.from_numpy(m).float(), torch.from_numpy(l).float(), torch.from_numpy(O).to(Q.dtype)


def within(got, want, bound, written):
    try:
        check_tree(got, want, bound, written)
    except AssertionError:
        return False
    return True


@pytest.mark.parametrize("cache", ["native", "e4m3", "int8"])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("rows", [[5, 3], [40, 20]])
def test_a_lost_term_is_noticed(rows, dtype, cache):
    c, Q, cu, mask = few_keys(DT[dtype], cache, rows, device="cpu")
    tiled, plain = tree_tight(c, Q, cu, mask, "tiled"), tree_tight(c, Q, cu, mask, "32 bits")
    kind = torch.float16 if cache != "native" else DT[dtype]
    two = not (cache != "native" and dtype == "bf16")  # of sequences with at most 128 rows for a key head: all but the first of [40, 20]
    assert within(restate(c, Q, cu, mask, kind, 2), *tiled)
    assert within(restate(c, Q, cu, mask, kind, 1), *tiled) == (not two)
    assert not within(restate(c, Q, cu, mask, kind, 1), *plain)
    assert not within(restate(c, Q, cu, mask, torch.bfloat16, 1), *tiled)
