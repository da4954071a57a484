"""Plain 64-bit restatement of the paged caches and of the attention of drafted trees over them, on the CPU, and the bounds that
results are held to. Used by the tests only."""
import numpy as np
import torch

CACHE_TYPE = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}
# half a step, relative to the value
HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}

E4M3 = np.array([(m / 8 * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7)) for e in range(16) for m in range(8)][:127])


def e4m3_codes(y):
    """Codes of float64 values |y| <= 448, to nearest, ties to the even code."""
    a = np.abs(y)
    hi = np.clip(np.searchsorted(E4M3, a), 1, 126)
    lo = hi - 1
    down, up = a - E4M3[lo], E4M3[hi] - a
    code = np.where((down < up) | ((down == up) & (lo % 2 == 0)), lo, hi)
    return (code + np.where(np.signbit(y), 128, 0)).astype(np.uint8)


def quantise(x, cache):
    """(codes as uint8 / int8, scales float32) of float64 rows [..., d] that are exact float32 values."""
    with np.errstate(invalid="ignore", over="ignore", divide="ignore"):
        top = np.abs(x).max(-1)
        bad = ~np.isfinite(top)
        top = np.where(bad, 1.0, top)
        if cache == "e4m3":
            e = np.full(top.shape, -126.0)
            for k in range(-126, 121):  # the smallest e with top <= 448 2^e
                e = np.where(top > 448 * 2.0 ** k, k + 1.0, e)
            scale = 2.0 ** e
            codes = e4m3_codes(np.where(bad[..., None], 0.0, x / scale[..., None]))
            return codes, np.where(bad, np.nan, scale).astype(np.float32)
        t32 = top.astype(np.float32)
        some = t32 >= np.float32(2.0 ** -100)
        scale = np.where(some, t32 / np.float32(127), np.float32(0))
        inverse = np.where(some, np.float32(127) / np.where(some, t32, np.float32(1)), np.float32(0)).astype(np.float32)
        y = np.rint(np.where(bad[..., None], np.float32(0), x.astype(np.float32)) * inverse[..., None])
        return y.astype(np.int8), np.where(bad, np.float32(np.nan), scale).astype(np.float32)


def values(codes, scale, cache):
    """float64 values of codes, exactly."""
    if cache == "e4m3":
        v = E4M3[codes & 127] * np.where(codes & 128, -1.0, 1.0)
    else:
        v = codes.astype(np.float64)
    return v * scale.astype(np.float64)[..., None]


class Cache:
    """A paged cache on the host (codes or values and scales as float64 / raw arrays) and its tensors on a device.

    `ends`: positions that each sequence's pages hold. Pages are handed out in a random order; page 0 of the pool is never used."""

    def __init__(self, dtype, cache, ends, heads, d, page, layout, seed, lens, device="cuda", shift=0):
        g = torch.Generator().manual_seed(seed)
        self.cache, self.dtype, self.page, self.heads, self.d = cache, dtype, page, heads, d
        B = len(ends)
        width = max([1] + [-(-e // page) for e in ends])
        n_pages = 1 + sum(-(-e // page) for e in ends)
        order = (torch.randperm(n_pages - 1, generator=g) + 1).to(torch.int32)
        self.table = torch.full((B, width), -1, dtype=torch.int32)
        at = 0
        for b, e in enumerate(ends):
            k = -(-e // page)
            self.table[b, :k] = order[at:at + k]
            at += k
        self.lens = torch.tensor(lens, dtype=torch.int32)
        store = CACHE_TYPE.get(cache, dtype)
        shape = (n_pages, heads, page) if layout == "hnd" else (n_pages, page, heads)
        turn = (lambda t: t.transpose(1, 2)) if layout == "hnd" else (lambda t: t)

        def pages():
            flat = torch.empty(int(np.prod(shape)) * d + shift, dtype=store, device=device)
            t = flat[shift:].view(*shape, d)
            x = torch.randn(*shape, d, generator=g)
            if cache == "native":
                t.copy_(x.to(dtype))
                return turn(t), None
            codes, scale = quantise(x.double().numpy(), cache)
            raw = torch.from_numpy(codes)
            t.view(torch.uint8 if cache == "e4m3" else torch.int8).copy_(raw)
            return turn(t), turn(torch.from_numpy(scale).to(device))

        self.K, self.K_scale = pages()
        self.V, self.V_scale = pages()

    def args(self):
        return self.K, self.V, self.table.to(self.K.device), self.lens.to(self.K.device)

    def scales(self):
        return (self.K_scale, self.V_scale)

    def raw(self, which):
        """Host copies: pages as raw bytes or values [n_pages, page, heads, d], scales."""
        t, s = (self.K, self.K_scale) if which == "K" else (self.V, self.V_scale)
        t = t.view(torch.uint8) if self.cache == "e4m3" else t
        return t.cpu().contiguous(), None if s is None else s.cpu().contiguous()

    def place(self, b, p):
        """(page, slot) of position p of sequence b, or None."""
        if p < 0 or p >= self.table.shape[1] * self.page:
            return None
        page = int(self.table[b, p // self.page])
        return (page, p % self.page) if 0 <= page < self.K.shape[0] else None

    def dense(self, which, b, positions):
        """float64 [n, heads, d] of existing positions of a sequence, and which of them exist."""
        raw, scale = self.raw(which)
        raw = raw.double().numpy() if self.cache == "native" else raw.numpy()
        at = [self.place(b, p) for p in positions]
        ok = np.array([x is not None for x in at], dtype=bool)
        pg = np.array([x[0] if x else 0 for x in at], dtype=np.int64)
        sl = np.array([x[1] if x else 0 for x in at], dtype=np.int64)
        v = raw[pg, sl]
        if self.cache != "native":
            v = values(v, scale.numpy()[pg, sl], self.cache)
        return v, ok


def tree_reference(cache, Q, cu, mask, state=None):
    """(m, l, O) in float64 and bounds on each, for Q [N, Hq, d] (host tensor) over `cache`.

    Bounds (u = 2^-24, products of the operands exact, sums and softmax in 32 bits):
      a score's dot product of d terms, in any order, with one more rounding for each scale:  ds <= (d + 6) u sum|q_e k_e| / sqrt(d)
      (matrix instructions may cut instead of round: twice that); a probability relative to its row's reference: 2 ds + |s| u + 2^-21
      (the exponential, the subtraction of the maximum); sums of n terms: n u; then the number that a 16-bit call rounds each
      probability to (bfloat16 2^-8, float16 2^-11) and the result's own rounding. All of them weigh on sum p |v| / l."""
    N, Hq, d = Q.shape
    g = Hq // cache.heads
    q = Q.double().numpy()
    u = 2.0 ** -24
    m = np.full((N, Hq), -np.inf)
    l = np.zeros((N, Hq))
    O = np.zeros((N, Hq, d))
    em, el, eO = np.zeros((N, Hq)), np.zeros((N, Hq)), np.zeros((N, Hq, d))
    written = np.zeros(N, dtype=bool)
    p_half = 0.0 if Q.dtype == torch.float32 else (2.0 ** -11 if (Q.dtype == torch.float16 and cache.cache == "native") else 2.0 ** -8)
    for b in range(len(cu) - 1):
        n0, n1 = max(0, min(N, cu[b])), max(0, min(N, cu[b + 1]))
        T = n1 - n0
        if T <= 0:
            continue
        cap = cache.table.shape[1] * cache.page
        n = min(max(int(cache.lens[b]), 0), cap)
        k, ok = cache.dense("K", b, range(n + T))
        v, _ = cache.dense("V", b, range(n + T))
        seen = np.zeros((T, n + T), dtype=bool)
        seen[:, :n] = True
        w = min(T, mask.shape[1])
        seen[:, n:n + w] = mask[n0:n1, :w].numpy()
        seen &= ok[None]
        written[n0:n1] = True
        for h in range(Hq):
            for t in range(T):
                j = np.nonzero(seen[t])[0]
                x = q[n0 + t, h]
                with np.errstate(invalid="ignore", over="ignore"):
                    m_in, l_in, O_in = (-np.inf, 0.0, 0.0) if state is None else (state[0][n0 + t, h], state[1][n0 + t, h], state[2][n0 + t, h])
                    if len(j) == 0:
                        if state is not None:
                            m[n0 + t, h], l[n0 + t, h], O[n0 + t, h] = m_in, l_in, O_in
                        continue
                    kk, vv = k[j, h // g], v[j, h // g]
                    s = kk @ x / np.sqrt(d)
                    ds = 2 * (d + 6) * u * (np.abs(kk) @ np.abs(x)).max() / np.sqrt(d)
                    top = s.max()
                    if l_in != 0 and not m_in <= top:
                        top = m_in
                    p = np.exp(s - top)
                    keep = l_in * np.exp(m_in - top) if l_in != 0 else 0.0
                    ll = p.sum() + keep
                    o = (p @ vv + (keep * O_in if keep != 0 else 0.0)) / ll
                    size = (p @ np.abs(vv) + (keep * np.abs(O_in) if keep != 0 else 0.0)) / ll
                    rel = 2 * ds + (np.abs(s).max() + abs(top) + 2) * 2 * u + 2.0 ** -21 + (len(j) + 64) * u
                    m[n0 + t, h], l[n0 + t, h], O[n0 + t, h] = top, ll, o
                    em[n0 + t, h] = ds + 4 * u * abs(top)
                    el[n0 + t, h] = rel * ll
                    eO[n0 + t, h] = (2 * rel + p_half) * size + HALF[Q.dtype] * (np.abs(o) + (2 * rel + p_half) * size)
    return (m, l, O), (em, el, eO), written


def check_tree(got, want, bound, written, tag=""):
    for name, x, y, e in zip(("m", "l", "O"), got, want, bound):
        x = x.double().cpu().numpy()[written]
        y, e = y[written], e[written]
        assert np.array_equal(np.isnan(x), np.isnan(y)), (tag, name, "NaN pattern")
        f = np.isfinite(y)
        assert np.array_equal(x[~f & ~np.isnan(y)], y[~f & ~np.isnan(y)]), (tag, name, "infinities")
        tiny = 2.0 ** -24 if got[2].dtype == torch.float16 and name == "O" else 1e-37  # the smallest steps of the type
        off = np.abs(x[f] - y[f]) - e[f] - tiny
        assert off.size == 0 or off.max() <= 0, (tag, name, float(off.max()), int((off > 0).sum()), off.size)
