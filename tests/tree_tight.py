"""Bounds on the attention of drafted trees that know which kernel ran: in how many bits a committed key's probability met V. In 64
bits, on the CPU; used by the tests only. cache_ref.tree_reference has one bound for all kernels of a type."""
import numpy as np
import torch

from cache_ref import HALF, Cache, check_tree

U = 2.0 ** -24


def probability_error(dtype, cache, rows, tag):
    """(relative error of the number that stands for a probability, the same for all; half of its smallest step over the row's largest
    product of probability and V's scale) of committed keys. Kernels without tensor cores round none. The tensor cores take float16 over
    8-bit caches, else Q's type: the rounding and what it left, rounded itself, where a sequence has at most 128 rows for a key head
    (not over 8-bit caches under bfloat16 Q), else the rounding alone. float16's smallest step is 2^-24, and the row's largest product is
    held at 2^8 at least; over 8-bit caches at 2^4, as the scales of a tile may differ by 2^4 before they are told apart."""
    if tag != "tiled":
        return 0.0, 0.0
    half = cache != "native" or dtype == torch.float16
    one = 2.0 ** -11 if half else 2.0 ** -8
    two = rows <= 128 and not (cache != "native" and dtype == torch.bfloat16)
    return (one * one if two else one), (2.0 ** -25 / (2.0 ** 8 if cache == "native" else 2.0 ** 4) if half else 0.0)


def tree_tight(c, Q, cu, mask, tag):
    """(m, l, O) in float64, bounds on each, and the rows that are written, for Q [N, Hq, d] (host tensor) over the cache c. `tag`: "tiled"
    where the tensor cores ran, else anything. The parts of a bound that all kernels share are those of cache_ref.tree_reference."""
    N, Hq, d = Q.shape
    g, half = Hq // c.heads, HALF[Q.dtype]
    q = Q.double().numpy()
    m, l, O = np.full((N, Hq), -np.inf), np.zeros((N, Hq)), np.zeros((N, Hq, d))
    em, el, eO = np.zeros((N, Hq)), np.zeros((N, Hq)), np.zeros((N, Hq, d))
    written = np.zeros(N, dtype=bool)
    vs = None if c.cache == "native" else c.raw("V")[1].double().numpy()
    for b in range(len(cu) - 1):
        n0, n1 = cu[b], cu[b + 1]
        T, n = n1 - n0, int(c.lens[b])
        if T == 0:
            continue
        written[n0:n1] = True
        one, step = probability_error(Q.dtype, c.cache, T * g, tag)
        k, ok = c.dense("K", b, range(n + T))
        v, _ = c.dense("V", b, range(n + T))
        seen = np.ones((T, n + T), dtype=bool)
        seen[:, n:] = False
        w = min(T, mask.shape[1])
        seen[:, n:n + w] = mask[n0:n1, :w].numpy()
        seen &= ok[None]
        if vs is not None:
            v_scale = np.array([vs[c.place(b, i)] if ok[i] else np.zeros(c.heads) for i in range(n)]).reshape(n, c.heads)
        for h in range(Hq):
            x, kk, vv = q[n0:n1, h], k[:, h // g], v[:, h // g]
            some = seen.any(-1)
            s = np.where(seen, x @ kk.T / np.sqrt(d), -np.inf)
            top = np.where(some, s.max(-1), 0.0)
            p = np.exp(s - top[:, None])
            ll = np.where(some, p.sum(-1), 1.0)
            absk = np.where(seen, np.abs(x) @ np.abs(kk).T, 0.0) / np.sqrt(d)
            ds = 2 * (d + 6) * U * absk.max(-1)
            if tag == "tiled" and c.cache != "native" and Q.dtype == torch.bfloat16:
                big = np.abs(x).max(-1, keepdims=True)
                if c.cache == "e4m3":  # two 8-bit terms: exact from 2^-13 of the largest element on, smaller ones to 2^-21 of it
                    off = np.where((np.abs(x) < 2.0 ** -13 * big) & (x != 0), 2.0 ** -21 * big, 0.0)
                else:  # float16 with the largest element at 2^14: half of a smallest step of 2^-24
                    off = np.broadcast_to(2.0 ** -39 * big, x.shape)
                ds = ds + np.where(seen, off @ np.abs(kk).T, 0.0).max(-1) / np.sqrt(d)
            rel = 2 * ds + (np.abs(np.where(seen, s, 0.0)).max(-1) + np.abs(top) + 2) * 2 * U + 2.0 ** -21 + (seen.sum(-1) + 64) * U
            size = p @ np.abs(vv) / ll[:, None]
            e = 2 * rel[:, None] * size + one * (p[:, :n] @ np.abs(vv[:n])) / ll[:, None]
            if step and n:
                scale = np.ones(n) if vs is None else v_scale[:, h // g]
                codes = np.abs(np.divide(vv[:n], scale[:, None], out=np.zeros_like(vv[:n]), where=scale[:, None] != 0))
                e = e + step * (p[:, :n] * scale).max(-1, keepdims=True) * codes.sum(0)[None] / ll[:, None]
            o = p @ vv / ll[:, None]
            m[n0:n1, h] = np.where(some, top, -np.inf)
            l[n0:n1, h] = np.where(some, p.sum(-1), 0.0)
            O[n0:n1, h] = o
            em[n0:n1, h], el[n0:n1, h] = ds + 4 * U * np.abs(top), rel * ll
            eO[n0:n1, h] = e + half * (np.abs(o) + e)
    return (m, l, O), (em, el, eO), written


def few_keys(dtype, cache, rows, device="cuda"):
    """(cache, Q, cu_rows, mask) where little but the rounding of probabilities can move a result: nine and five keys of 16 elements, one
    element of a query that is not zero, and columns of O in which V's signs cancel, so that the result's own rounding is small."""
    lens = [9, 5]
    c = Cache(dtype, cache, [n + r for n, r in zip(lens, rows)], 2, 16, 16, "nhd", 3, lens, device=device)
    g = torch.Generator().manual_seed(4)
    Q = torch.zeros(sum(rows), 8, 16)
    Q.scatter_(2, torch.randint(0, 16, (sum(rows), 8, 1), generator=g), torch.randn(sum(rows), 8, 1, generator=g) * 4)
    mask = torch.rand(sum(rows), max(rows), generator=g) < 0.1
    return c, Q.to(dtype), [0, rows[0], sum(rows)], mask


def check_path(pkg, c, Q, cu, mask, tag, got, known):
    """The rows that a path left, within the bounds of the kernel that ran. `known`: a dict that keeps the bounds of this call."""
    ran = "tiled" if tag == "tiled" or (tag == "auto" and pkg.capi.last_path() == pkg.capi.PATH_TILED) else "32 bits"
    if ran not in known:
        known[ran] = tree_tight(c, Q, cu, mask, ran)
    check_tree(got, *known[ran], (tag, ran))
