"""CPU: calls that would write several elements to one place are refused before anything is launched; what is only read may share it."""
import ctypes

import pytest

from test_cache_tree_host import P, _cache


def calls(pkg, c, rows=(256, 64)):
    lib, r, p = pkg.capi.lib(), ctypes.byref(c), ctypes.c_void_p(P)
    s, ok = (ctypes.c_int64 * 2)(*rows), (ctypes.c_int64 * 2)(256, 64)
    need = 1 << 40
    return {"append": lambda n=5: lib.spfa_cache_append(r, 2, p, s, p, ok, p, n, None), "read": lambda n=5: lib.spfa_cache_read(r, 2, p, ok, p, s, p, n, None),
            "keep": lambda: lib.spfa_cache_keep(r, p, 0, p, None),
            "tree": lambda n=5: lib.spfa_tree_forward(r, 2, p, ok, p, n, 8, p, 4, p, p, p, s, 1, p, need, None)}


@pytest.mark.parametrize("which", ["K_stride", "V_stride", "K_scale_stride", "V_scale_stride"])
@pytest.mark.parametrize("dim", [0, 1, 2])
def test_an_expanded_cache_is_not_written(pkg, which, dim):
    strides = list((16 * 4 * 64, 4 * 64, 64) if "scale" not in which else (64, 4, 1))
    strides[dim] = 0
    f = calls(pkg, _cache(pkg, dtype=3, **{which: tuple(strides)}))
    assert f["append"]() == -1 and f["keep"]() == -1
    assert f["read"](0) == 0 and f["tree"](0) == 0  # fine to read from
    one = {0: "n_pages", 1: "page_size", 2: "n_heads"}[dim]
    f = calls(pkg, _cache(pkg, dtype=3, **{which: tuple(strides), one: 1}))
    assert f["append"](0) == 0 and f["keep"]() == 0  # a dimension of one element
    if "scale" in which:  # of no account where the cache holds its values as they are
        f = calls(pkg, _cache(pkg, **{which: tuple(strides)}))
        assert f["append"](0) == 0 and f["keep"]() == 0


@pytest.mark.parametrize("rows", [(0, 64), (256, 0)])
def test_expanded_rows_are_not_written(pkg, rows):
    f = calls(pkg, _cache(pkg), rows)
    assert f["read"]() == -1 and f["tree"]() == -1
    assert f["append"](0) == 0
    if rows[0] == 0:  # one row
        f = calls(pkg, _cache(pkg, n_seq=0), rows)
        assert f["read"](1) == 0 and f["tree"](1) == 0
