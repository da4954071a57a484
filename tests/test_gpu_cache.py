"""GPU: paged caches. Codes, scales and values against the 64-bit restatement, bit for bit (every step is either exact or one
defined float32 operation); what a call does not own stays as it was."""
import numpy as np
import pytest
import torch

import cache_ref
from cache_ref import Cache

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _rows(n, heads, d, dtype, seed, strides="packed"):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(n, 3 * heads, d, generator=g) * torch.exp2(torch.randint(-4, 5, (n, 3 * heads, 1), generator=g).float())).to(dtype)
    if n > 2:
        x[1] = 0
    x = x.cuda()
    if strides == "packed":  # slices of one projection's output
        return x[:, heads:2 * heads], x[:, 2 * heads:]
    if strides == "heads_first":
        return tuple(x[:, a:a + heads].transpose(0, 1).contiguous().transpose(0, 1) for a in (0, heads))
    flat = torch.empty(x[:, :heads].numel() + 1, dtype=dtype, device="cuda")  # no alignment beyond an element's
    flat[1:] = x[:, :heads].reshape(-1)
    return flat[1:].view(n, heads, d), x[:, heads:2 * heads].contiguous()


def _want(cache, x):
    """What the cache holds of rows x: (raw, scale)."""
    if cache.cache == "native":
        return x.cpu(), None
    codes, scale = cache_ref.quantise(x.double().cpu().numpy(), cache.cache)
    return torch.from_numpy(codes), torch.from_numpy(scale)


def _same(a, b):
    return torch.equal(a.view(torch.uint8) if a.dtype != torch.uint8 else a, b.view(torch.uint8) if b.dtype != torch.uint8 else b)


def _check_append(pkg, c, lens, cu, dtype, seed, strides, mod=None):
    N = max(cu[-1], 0) + 2  # two rows behind the last sequence
    K, V = _rows(N, c.heads, c.d, dtype, seed, strides)
    before = {w: c.raw(w) for w in "KV"}
    cu_t = torch.tensor(cu, dtype=torch.int32, device="cuda")
    if mod is None:
        held = c.args()  # the description holds addresses
        pkg.capi.cache_append(pkg.capi.kv_cache(*held, *c.scales()), K, V, cu_t)
    else:
        mod.append(K, V, *c.args(), cu_t, *c.scales())
    torch.cuda.synchronize()
    for w, x in (("K", K), ("V", V)):
        raw, scale = before[w]
        new, s = _want(c, x)
        for b in range(len(lens)):
            for i in range(max(cu[b], 0), min(cu[b + 1], N)):
                at = c.place(b, lens[b] + i - cu[b])
                if at:
                    raw[at] = new[i]
                    if s is not None:
                        scale[at] = s[i]
        got_raw, got_scale = c.raw(w)
        assert _same(got_raw, raw), w
        if s is not None:
            assert torch.equal(got_scale.view(torch.int32), scale.view(torch.int32)) or torch.equal(
                got_scale.nan_to_num(-1), scale.nan_to_num(-1)), w
    return K, V


SHAPES = [  # heads, d, page, layout
    (2, 64, 16, "nhd"), (3, 128, 24, "hnd"), (1, 40, 8, "nhd"), (8, 128, 64, "hnd"), (2, 80, 7, "nhd"), (1, 1, 3, "nhd"), (2, 3, 16, "hnd"),
    (1, 256, 16, "nhd"), (2, 200, 10, "hnd"), (1, 1024, 4, "nhd"), (5, 96, 100, "nhd"), (2, 36, 16, "nhd"),
]


@pytest.mark.parametrize("cache", ["native", "e4m3", "int8"])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("shape", SHAPES)
def test_append_writes_codes_scales_and_nothing_else(pkg, shape, dtype, cache):
    heads, d, page, layout = shape
    lens, rows = [0, 5, 33, 7, 1], [9, 0, 20, 1, 31]
    c = Cache(DT[dtype], cache, [n + r for n, r in zip(lens, rows)], heads, d, page, layout, seed=d + heads, lens=lens)
    cu = np.concatenate([[0], np.cumsum(rows)]).tolist()
    for k, strides in enumerate(("packed", "heads_first", "odd")):
        _check_append(pkg, c, lens, cu, DT[dtype], 7 * d + k, strides, mod=pkg.binding("spfa_cache") if k == 0 else None)


@pytest.mark.parametrize("cache", ["native", "e4m3", "int8"])
def test_positions_that_do_not_exist_are_skipped(pkg, cache):
    lens, rows = [30, -4, 10, 2 ** 31 - 3], [12, 9, 4, 6]  # beyond the page list, below 0, in bad pages, beyond 32 bits
    c = Cache(torch.float16, cache, [32, 16, 16, 16], 2, 64, 16, "nhd", 3, lens)
    c.table[2, 0] = 10 ** 6
    c.table[1, 1] = -2 ** 31
    _check_append(pkg, c, lens, [0, 12, 21, 25, 31], torch.float16, 5, "packed")
    # rows before the first sequence, sequences that do not follow each other, and rows behind the last
    _check_append(pkg, c, lens, [3, 12, 12, 12, 14], torch.float16, 6, "packed")
    K, V = (torch.full((40, 2, 64), 7.0, device="cuda", dtype=torch.float16) for _ in range(2))
    pkg.binding("spfa_cache").read(*c.args(), torch.tensor([3, 15, 24, 28, 34], dtype=torch.int32, device="cuda"), K, V, *c.scales())
    for w, x in (("K", K), ("V", V)):
        x = x.cpu()
        for i in range(40):
            b = next((b for b, (lo, hi) in enumerate(((3, 15), (15, 24), (24, 28), (28, 34))) if lo <= i < hi), None)
            at = None if b is None else c.place(b, lens[b] + i - (3, 15, 24, 28)[b])
            if at is None:
                assert (x[i] == 7).all(), i
            else:
                v, _ = c.dense(w, b, [lens[b] + i - (3, 15, 24, 28)[b]])
                assert torch.equal(x[i], torch.from_numpy(v[0]).to(torch.float32).half()), i


@pytest.mark.parametrize("cache", ["e4m3", "int8"])
@pytest.mark.parametrize("d", [64, 20])
def test_extreme_rows(pkg, cache, d):
    """Rows of one value, the largest and smallest of float32, ties, and values that are not finite."""
    c = Cache(torch.float32, cache, [64], 1, d, 16, "nhd", 1, [0])
    K = torch.zeros(40, 1, d, device="cuda")
    g = torch.Generator().manual_seed(d)
    K[1, 0, 0], K[2, 0, 3], K[3, 0, d - 1], K[4, 0, 2] = 3.4028234663852886e38, -2.0 ** -149, 2.0 ** -126, 448.0
    K[5] = 2.0 ** -100
    K[6] = 2.0 ** -101
    K[7] = torch.tensor([448.0, 449.0] * (d // 2), device="cuda").view(1, d)
    K[8] = torch.tensor([1.0, 17 / 16] * (d // 2), device="cuda").view(1, d)  # a tie of e4m3
    K[9] = torch.tensor([127.0, 0.5, 1.5, -2.5] * (d // 4), device="cuda").view(1, d)  # ties of int8
    K[10, 0, 5], K[11, 0, 6], K[12, 0, 7] = float("nan"), float("inf"), float("-inf")
    for r in range(13, 40):
        K[r] = (torch.randn(1, d, generator=g) * 2.0 ** (9 * (r - 26))).cuda()
    V = K.flip(0).contiguous()
    cu = torch.tensor([0, 40], dtype=torch.int32, device="cuda")
    mod = pkg.binding("spfa_cache")
    mod.append(K, V, *c.args(), cu, *c.scales())
    for dtype in (torch.float32, torch.bfloat16):
        k, v = (torch.empty(40, 1, d, device="cuda", dtype=dtype) for _ in range(2))
        mod.read(*c.args(), cu, k, v, *c.scales())
        for got, x in ((k, K), (v, V)):
            codes, scale = cache_ref.quantise(x.double().cpu().numpy(), cache)
            want = torch.from_numpy(cache_ref.values(codes, scale, cache).astype(np.float32)).to(dtype)
            assert torch.equal(got.cpu().nan_to_num(-7, 8, 9), want.nan_to_num(-7, 8, 9))
            bad = ~np.isfinite(x.cpu().numpy()).all(-1)[:, 0]
            assert torch.isnan(got.cpu()[bad]).all() and not torch.isnan(got.cpu()[~bad]).any()


@pytest.mark.parametrize("cache", ["native", "e4m3", "int8"])
@pytest.mark.parametrize("out", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("shape", SHAPES)
def test_read_returns_the_rounded_values(pkg, shape, out, cache):
    heads, d, page, layout = shape
    ends = [37, 0, 1, 64]
    c = Cache(DT[out], cache, ends, heads, d, page, layout, seed=d, lens=[0, 0, 0, 20])
    rows = [37, 0, 1, 44]
    cu = torch.tensor(np.concatenate([[0], np.cumsum(rows)]).tolist(), dtype=torch.int32, device="cuda")
    N = int(cu[-1])
    big = torch.full((2, heads, N + 1, d), 3.0, dtype=DT[out], device="cuda")  # heads first: what an operator on dense K and V takes
    K, V = big[0].transpose(0, 1), big[1].transpose(0, 1)
    got = pkg.binding("spfa_cache").read(*c.args(), cu, K, V, *c.scales())
    assert got[0].data_ptr() == K.data_ptr()
    for w, x in (("K", K), ("V", V)):
        want = np.concatenate([c.dense(w, b, range(int(c.lens[b]), int(c.lens[b]) + r))[0] for b, r in enumerate(rows)])
        assert torch.equal(x[:N].cpu(), torch.from_numpy(want).to(torch.float32).to(DT[out]))
        assert (x[N] == 3).all()


@pytest.mark.parametrize("cache,dtype", [("native", "f32"), ("native", "bf16"), ("e4m3", "f16"), ("int8", "bf16")])
@pytest.mark.parametrize("shape", [(2, 64, 16, "nhd"), (3, 128, 24, "hnd"), (1, 3, 5, "nhd"), (2, 37, 16, "hnd"), (1, 1024, 8, "nhd")])
def test_keep_moves_rows_in_order(pkg, shape, cache, dtype):
    heads, d, page, layout = shape
    T, lens = 70, [11, 0, 40, 3]
    c = Cache(DT[dtype], cache, [n + T for n in lens], heads, d, page, layout, seed=9, lens=lens)
    g = torch.Generator().manual_seed(4)
    kept = torch.full((4, 66), 10 ** 9, dtype=torch.int32)
    n_kept = [66, 0, 7, 99]  # the last: more than the width
    kept[0] = torch.randperm(T, generator=g)[:66].sort().values
    kept[2, :7] = torch.tensor([0, 1, 5, 6, 30, 31, 69])
    kept[3] = torch.arange(66) + 4
    before = {w: c.raw(w) for w in "KV"}
    pkg.binding("spfa_cache").keep(*c.args(), kept.cuda(), torch.tensor(n_kept, dtype=torch.int32, device="cuda"), *c.scales())
    for w in "KV":
        raw, scale = before[w]
        old, old_scale = raw.clone(), None if scale is None else scale.clone()
        for b in range(4):
            for i in range(min(n_kept[b], 66)):
                src, dst = c.place(b, lens[b] + int(kept[b, i])), c.place(b, lens[b] + i)
                raw[dst] = old[src]
                if scale is not None:
                    scale[dst] = old_scale[src]
        got, got_scale = c.raw(w)
        assert _same(got, raw) and (scale is None or torch.equal(got_scale, scale)), w


def test_keep_skips_what_does_not_exist(pkg):
    c = Cache(torch.float32, "native", [32, 32], 1, 8, 16, "nhd", 1, lens=[4, 20])
    c.table[0, 1] = 99
    before = {w: c.raw(w)[0] for w in "KV"}
    kept = torch.tensor([[-5, 2, 14], [1, 3, 12]], dtype=torch.int32, device="cuda")  # negative, good, in a bad page; good, good, beyond
    pkg.binding("spfa_cache").keep(*c.args(), kept, torch.tensor([3, 3], dtype=torch.int32, device="cuda"))
    for w in "KV":
        raw, old = before[w].clone(), before[w]
        raw[c.place(0, 5)] = old[c.place(0, 6)]
        raw[c.place(1, 20)] = old[c.place(1, 21)]
        raw[c.place(1, 21)] = old[c.place(1, 23)]
        assert torch.equal(c.raw(w)[0], raw)
    for n in (-3, 0):
        pkg.binding("spfa_cache").keep(*c.args(), kept, torch.tensor([n, n], dtype=torch.int32, device="cuda"))
    assert torch.equal(c.raw("K")[0][c.place(1, 21)], before["K"][c.place(1, 23)])


def test_pages_beyond_32_bit_offsets(pkg):
    """2.2e9 elements of K lie before the pages that the sequence uses."""
    n_pages, page, d = 17200, 1024, 128
    K = torch.zeros(n_pages, page, 1, d, dtype=torch.int8, device="cuda")
    V = torch.zeros_like(K)
    ks, vs = (torch.zeros(n_pages, page, 1, device="cuda") for _ in range(2))
    table = torch.tensor([[n_pages - 1, 3, n_pages - 2]], dtype=torch.int32, device="cuda")
    lens, cu = torch.tensor([1000], dtype=torch.int32, device="cuda"), torch.tensor([0, 2000], dtype=torch.int32, device="cuda")
    x, y = (torch.randn(2000, 1, d, device="cuda") for _ in range(2))
    mod = pkg.binding("spfa_cache")
    mod.append(x, y, K, V, table, lens, cu, ks, vs)
    a, b = torch.empty_like(x), torch.empty_like(x)
    mod.read(K, V, table, lens, cu, a, b, ks, vs)
    for got, z in ((a, x), (b, y)):
        codes, scale = cache_ref.quantise(z.double().cpu().numpy(), "int8")
        assert torch.equal(got.cpu(), torch.from_numpy(cache_ref.values(codes, scale, "int8").astype(np.float32)))
    kept = torch.tensor([[1500, 1999]], dtype=torch.int32, device="cuda")
    mod.keep(K, V, table, lens, kept, torch.tensor([2], dtype=torch.int32, device="cuda"), ks, vs)
    c, e = torch.empty(2, 1, d, device="cuda"), torch.empty(2, 1, d, device="cuda")
    mod.read(K, V, table, lens, torch.tensor([0, 2], dtype=torch.int32, device="cuda"), c, e, ks, vs)
    assert torch.equal(c, a[[1500, 1999]]) and torch.equal(e, b[[1500, 1999]])
    assert not K[5:n_pages - 2].any()


def test_streams_and_replayed_graphs(pkg):
    """Calls go to the current stream, can be captured, and read lens and the page table when they run."""
    mod = pkg.binding("spfa_cache")
    c = Cache(torch.bfloat16, "e4m3", [64, 64], 2, 64, 16, "nhd", 1, lens=[0, 0])
    pages, scales = c.args(), c.scales()
    K, V = _rows(6, 2, 64, torch.bfloat16, 3)
    K, V = K.clone(), V.clone()
    cu = torch.tensor([0, 4, 6], dtype=torch.int32, device="cuda")
    k, v = torch.empty_like(K), torch.empty_like(V)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        mod.append(K, V, *pages, cu, *scales)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            mod.append(K, V, *pages, cu, *scales)
            mod.read(*pages, cu, k, v, *scales)
    s.synchronize()
    for step in range(3):
        pages[3].copy_(torch.tensor([step * 4, step * 2 + 1], dtype=torch.int32))
        K.copy_(torch.randn(K.shape))
        graph.replay()
        torch.cuda.synchronize()
        codes, scale = cache_ref.quantise(K.double().cpu().numpy(), "e4m3")
        assert torch.equal(k.double().cpu(), torch.from_numpy(cache_ref.values(codes, scale, "e4m3")))
        c.lens = pages[3].cpu()
        got, _ = c.dense("K", 1, [int(c.lens[1]) + 1])
        assert np.array_equal(got[0], cache_ref.values(codes, scale, "e4m3")[5])


def test_refusals(pkg):
    mod = pkg.binding("spfa_cache")
    c = Cache(torch.bfloat16, "int8", [32, 32], 2, 64, 16, "nhd", 1, lens=[0, 0])
    n = Cache(torch.bfloat16, "native", [32, 32], 2, 64, 16, "nhd", 1, lens=[0, 0])
    K, V = (torch.zeros(4, 2, 64, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    cu = torch.tensor([0, 2, 4], dtype=torch.int32, device="cuda")
    P, T, L = c.args()[:2], c.args()[2], c.args()[3]
    for bad in (lambda: mod.append(K, V, *P, T, L, cu),                                   # no scales
                lambda: mod.append(K, V, *n.args(), cu, *c.scales()),                     # scales of a cache that has none
                lambda: mod.append(K, V.float(), *P, T, L, cu, *c.scales()),
                lambda: mod.append(K.float(), V.float(), *n.args(), cu),                  # float32 rows, bfloat16 cache
                lambda: mod.append(K.to(torch.float64), V.to(torch.float64), *P, T, L, cu, *c.scales()),
                lambda: mod.append(K[:, :1], V[:, :1], *P, T, L, cu, *c.scales()),
                lambda: mod.append(K[..., ::2], V[..., ::2], *P, T, L, cu, *c.scales()),
                lambda: mod.append(K, V[:3], *P, T, L, cu, *c.scales()),
                lambda: mod.append(K, V, *P, T.long(), L, cu, *c.scales()),
                lambda: mod.append(K, V, *P, T, L, cu[:2], *c.scales()),
                lambda: mod.append(K, V, *P, T[:1], L, cu, *c.scales()),
                lambda: mod.append(K, V, P[0], P[1][:1], T, L, cu, *c.scales()),
                lambda: mod.append(K.cpu(), V.cpu(), *P, T, L, cu, *c.scales()),
                lambda: mod.append(K, V, *P, T, L, cu.cpu(), *c.scales()),
                lambda: mod.append(K, V, *P, T, L, cu, c.K_scale.half(), c.V_scale),
                lambda: mod.append(K, V, *P, T, L, cu, c.K_scale[:, :1], c.V_scale),
                lambda: mod.read(*P, T, L, cu, K.char(), V.char(), *c.scales()),
                lambda: mod.keep(*P, T, L, T[:1], L, *c.scales()),
                lambda: mod.keep(*P, T, L, T, L[:1], *c.scales()),
                lambda: mod.keep(*P, T, L, T.long(), L, *c.scales())):
        with pytest.raises(RuntimeError):
            bad()
    empty = torch.zeros(0, 2, 64, dtype=torch.bfloat16, device="cuda")
    mod.append(empty, empty, *c.args(), torch.zeros(3, dtype=torch.int32, device="cuda"), *c.scales())  # nothing to do
    mod.keep(*c.args(), torch.zeros(2, 0, dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda"), *c.scales())
    assert pkg.capi.last_device_error() == 0
