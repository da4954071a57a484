"""CPU: what the cache and tree entry points refuse (no kernel is launched by any call here), the descriptions of a cache, and the
reference of their GPU tests against independent forms."""
import ctypes

import numpy as np
import pytest
import torch

import cache_ref

P = 4096  # an aligned address that is never dereferenced: every call below fails its checks first


def _cache(pkg, **over):
    c = pkg.capi.KvCache()
    c.K = c.V = c.K_scale = c.V_scale = c.page_table = c.lens = P
    c.K_stride[:] = c.V_stride[:] = (16 * 4 * 64, 4 * 64, 64)
    c.K_scale_stride[:] = c.V_scale_stride[:] = (64, 4, 1)
    c.n_pages, c.page_size, c.n_heads, c.n_seq, c.table_width, c.d, c.dtype = 8, 16, 4, 3, 2, 64, 2
    for k, v in over.items():
        if isinstance(v, tuple):
            getattr(c, k)[:] = v
        else:
            setattr(c, k, v)
    return c


BAD_CACHE = [
    (dict(K=None), -1), (dict(V=None), -1), (dict(page_table=None), -1), (dict(lens=None), -1), (dict(dtype=9), -1), (dict(dtype=-1), -1),
    (dict(K=P + 1), -1), (dict(lens=P + 2), -1), (dict(d=0), -2), (dict(d=1025), -2), (dict(n_pages=-1), -1), (dict(page_size=0), -1),
    (dict(n_heads=0), -1), (dict(n_seq=-1), -1), (dict(table_width=-1), -1), (dict(K_stride=(-1, 0, 0)), -1), (dict(n_pages=1 << 31), -11),
    (dict(page_size=1 << 31), -11), (dict(n_heads=70000), -11), (dict(dtype=3, K_scale=None), -1), (dict(dtype=4, V_scale=P + 2), -1),
    (dict(dtype=4, V_scale_stride=(0, -1, 0)), -1),
]


@pytest.mark.parametrize("over,status", BAD_CACHE)
def test_bad_caches_are_refused(pkg, over, status):
    lib, c = pkg.capi.lib(), _cache(pkg, **over)
    s, p = (ctypes.c_int64 * 2)(256, 64), ctypes.c_void_p(P)
    assert lib.spfa_cache_append(ctypes.byref(c), 2, p, s, p, s, p, 5, None) == status
    assert lib.spfa_cache_read(ctypes.byref(c), 2, p, s, p, s, p, 5, None) == status
    assert lib.spfa_cache_keep(ctypes.byref(c), p, 3, p, None) == status
    assert lib.spfa_tree_workspace_bytes(ctypes.byref(c), 2, 5, 8) == 0
    assert lib.spfa_tree_forward(ctypes.byref(c), 2, p, s, p, 5, 8, p, 4, p, p, p, s, 1, p, 1 << 40, None) == status


def test_bad_rows_are_refused(pkg):
    lib, c = pkg.capi.lib(), _cache(pkg)
    s, p, r = (ctypes.c_int64 * 2)(256, 64), ctypes.c_void_p(P), ctypes.byref
    for f in (lib.spfa_cache_append, lib.spfa_cache_read):
        assert f(None, 2, p, s, p, s, p, 5, None) == -1
        assert f(r(c), 0, p, s, p, s, p, 5, None) == -1      # float32 rows, bfloat16 cache
        assert f(r(c), 3, p, s, p, s, p, 5, None) == -1      # rows are never 8-bit
        assert f(r(c), 2, None, s, p, s, p, 5, None) == -1
        assert f(r(c), 2, p, None, p, s, p, 5, None) == -1
        assert f(r(c), 2, p, s, ctypes.c_void_p(P + 1), s, p, 5, None) == -1
        assert f(r(c), 2, p, s, p, (ctypes.c_int64 * 2)(-8, 64), p, 5, None) == -1
        assert f(r(c), 2, p, s, p, s, None, 5, None) == -1
        assert f(r(c), 2, p, s, p, s, p, -1, None) == -1
        assert f(r(c), 2, p, s, p, s, p, 1 << 31, None) == -11
        assert f(r(c), 2, p, s, p, s, p, 0, None) == 0       # nothing to do: nothing is launched
    assert lib.spfa_cache_keep(r(c), None, 3, p, None) == -1
    assert lib.spfa_cache_keep(r(c), p, -1, p, None) == -1
    assert lib.spfa_cache_keep(r(c), p, 3, None, None) == -1
    assert lib.spfa_cache_keep(r(c), p, 0, p, None) == 0
    need = lib.spfa_tree_workspace_bytes(r(c), 2, 5, 8)
    assert need >= 5 * 8 * 66 * 4
    f = lambda **o: lib.spfa_tree_forward(*[{**dict(c=r(c), dtype=2, Q=p, qs=s, cu=p, n=5, hq=8, mask=p, w=4, m=p, l=p, O=p, os=s, first=1,
                                                    ws=p, wb=need, st=None), **o}[k] for k in
                                            ("c", "dtype", "Q", "qs", "cu", "n", "hq", "mask", "w", "m", "l", "O", "os", "first", "ws", "wb", "st")])
    assert f(hq=6) == -1 and f(hq=0) == -1        # not a multiple of the cache's heads
    assert f(n=1 << 31) == -11 and f(n=1 << 28, hq=16) == -11
    assert f(Q=None) == -1 and f(cu=None) == -1 and f(m=None) == -1 and f(O=None) == -1 and f(mask=None) == -1
    assert f(w=-1) == -1 and f(O=ctypes.c_void_p(P + 1)) == -1 and f(l=ctypes.c_void_p(P + 2)) == -1
    assert f(dtype=1) == -1                        # float16 rows, bfloat16 cache
    assert f(wb=need - 1) == -3 and f(ws=None) == -3 and f(ws=ctypes.c_void_p(P + 128)) == -3
    assert f(n=0) == 0


def test_descriptions_refuse_what_does_not_fit(pkg):
    c = pkg.capi
    K = torch.zeros(4, 16, 2, 8)
    table, lens = torch.zeros(3, 2, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    with pytest.raises(c.SpfaError):  # no CPU path
        c.kv_cache(K, K, table, lens)
    for name in ("spfa_cache", "spfa_tree"):
        assert name in pkg.MODULES
    mod = pkg.binding("spfa_cache")
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        mod.append(K, K, K, K, table, lens, torch.zeros(4, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        mod.read(K, K, table, lens, torch.zeros(4, dtype=torch.int32), K, K)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        mod.keep(K, K, table, lens, table, lens)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        pkg.binding("spfa_tree").forward(K, K, K, table, lens, lens, K, K, K, K)


def test_reference_quantisation():
    """The reference's 8-bit types against torch's conversion, and its scales against their definition."""
    g = torch.Generator().manual_seed(1)
    x = torch.randn(500, 64, generator=g) * torch.exp2(torch.randint(-30, 30, (500, 1), generator=g).float())
    x[3], x[4] = 0, 2.0 ** -140
    codes, scale = cache_ref.quantise(x.double().numpy(), "e4m3")
    want = (x / torch.from_numpy(scale)[:, None]).to(torch.float8_e4m3fn)
    assert torch.equal(torch.from_numpy(codes), want.view(torch.uint8))
    top = x.abs().amax(-1).double().numpy()
    assert (top <= 448.0 * scale).all() and ((top > 224.0 * scale) | (scale == 2.0 ** -126)).all()
    codes, scale = cache_ref.quantise(x.double().numpy(), "int8")
    assert codes[3].any() == 0 and scale[4] == 0
    back = cache_ref.values(codes, scale, "int8")
    assert (np.abs(back - x.double().numpy()) <= np.where(scale > 0, 0.5 * scale * (1 + 2.0 ** -15), 2.0 ** -100)[:, None]).all()
    x[5, 7], x[6, 8] = float("nan"), float("-inf")
    for cache in ("e4m3", "int8"):
        codes, scale = cache_ref.quantise(x.double().numpy(), cache)
        assert np.isnan(scale[5]) and np.isnan(scale[6]) and np.isfinite(scale[7])


def test_reference_tree_is_masked_softmax():
    """The reference against torch's attention in float64 on a mask written out, and its chaining against the union."""
    c = cache_ref.Cache(torch.float32, "native", [30, 9], 2, 16, 8, "nhd", 3, [25, 4], device="cpu")
    cu, N = [0, 5, 10], 10
    g = torch.Generator().manual_seed(2)
    Q = torch.randn(N, 4, 16, generator=g)
    mask = torch.rand(N, 5, generator=g) < 0.5
    (m, l, O), bound, written = cache_ref.tree_reference(c, Q, cu, mask)
    for b in range(2):
        n = int(c.lens[b])
        k, ok = c.dense("K", b, range(n + 5))
        v, _ = c.dense("V", b, range(n + 5))
        seen = torch.cat([torch.ones(5, n, dtype=torch.bool), mask[cu[b]:cu[b + 1]]], 1) & torch.from_numpy(ok)
        for h in range(4):
            want = torch.nn.functional.scaled_dot_product_attention(
                Q[cu[b]:cu[b + 1], h].double()[None], torch.from_numpy(k[:, h // 2])[None], torch.from_numpy(v[:, h // 2])[None], seen[None])[0]
            assert np.allclose(O[cu[b]:cu[b + 1], h], want.numpy(), atol=1e-12)
    assert written.all() and all((x >= 0).all() for x in bound)
    none = torch.zeros(N, 0, dtype=torch.bool)
    first, _, _ = cache_ref.tree_reference(c, Q, cu, none)
    c.lens[:] = 0
    cu2 = [0, 5, 10]
    again, _, _ = cache_ref.tree_reference(c, Q, cu2, torch.zeros(N, 5, dtype=torch.bool), state=first)
    assert all(np.array_equal(x, y) for x, y in zip(first, again))  # nothing visible: the state stays
