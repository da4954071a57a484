"""GPU: descriptions of paged caches made by capi.kv_cache."""
import weakref

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_a_description_keeps_its_tensors(pkg):
    """Described from temporaries, the cache is still there when the calls come."""
    pages = [torch.randn(4, 16, 2, 64, device="cuda") for _ in range(2)]
    want = pages[0][2, :5].clone(), pages[1][2, :5].clone()
    table, lens = torch.tensor([[2, 0]], dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    gone = weakref.ref(pages[0])
    c = pkg.capi.kv_cache(*pages, table.cuda(), lens.cuda())
    del pages
    junk = [torch.full((4, 16, 2, 64), 7.0, device="cuda") for _ in range(4)] + [torch.full((1, 2), 9, dtype=torch.int32, device="cuda") for _ in range(4)]
    assert gone() is not None
    K, V = (torch.zeros(5, 2, 64, device="cuda") for _ in range(2))
    pkg.capi.cache_read(c, K, V, torch.tensor([0, 5], dtype=torch.int32, device="cuda"))
    assert torch.equal(K, want[0]) and torch.equal(V, want[1])
    del c, junk
    assert gone() is None


@pytest.mark.parametrize("dtype,cache", [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.float16, torch.int8),
                                         (torch.bfloat16, torch.float8_e4m3fn)])
@pytest.mark.parametrize("n_pages,width,rows", [(0, 2, 3), (0, 0, 3), (3, 0, 3), (0, 2, 90)])
def test_caches_without_pages_and_empty_page_lists(pkg, n_pages, width, rows, dtype, cache):
    """No position exists: nothing is written, read or attended to, through the modules and capi alike."""
    pages = [torch.zeros(n_pages, 16, 2, 64, device="cuda").to(cache) for _ in range(2)]
    scales = [torch.ones(n_pages, 16, 2, device="cuda") for _ in range(2)] if cache.itemsize == 1 else [None, None]
    table, lens = torch.zeros(1, width, dtype=torch.int32, device="cuda"), torch.full((1,), 20, dtype=torch.int32, device="cuda")
    cu = torch.tensor([0, rows], dtype=torch.int32, device="cuda")
    K, V = (torch.full((rows, 2, 64), 3.0, device="cuda", dtype=dtype) for _ in range(2))
    Q, mask = torch.ones(rows, 8, 64, device="cuda", dtype=dtype), torch.ones(rows, rows, device="cuda", dtype=torch.bool)
    kept = torch.arange(2, dtype=torch.int32, device="cuda")[None]
    described = pkg.capi.kv_cache(*pages, table, lens, *scales)
    mod, args = pkg.binding("spfa_cache"), (*pages, table, lens)
    pkg.capi.cache_append(described, K, V, cu)
    pkg.capi.cache_keep(described, kept, kept[0, :1] + 2)
    pkg.capi.cache_read(described, K, V, cu)
    mod.append(K, V, *args, cu, *scales)
    mod.keep(*args, kept, kept[0, :1] + 2, *scales)
    mod.read(*args, cu, K, V, *scales)
    assert (K == 3).all() and (V == 3).all() and not any(t.float().any() for t in pages)
    for through in ("capi", "module"):
        m, l, O = (torch.full(s, float("nan"), device="cuda", dtype=t) for s, t in (((rows, 8), torch.float32),) * 2 + (((rows, 8, 64), dtype),))
        if through == "capi":
            pkg.capi.tree_forward(described, Q, cu, mask, m, l, O, first=True)
        else:
            pkg.binding("spfa_tree").forward(Q, *args, cu, mask, m, l, O, *scales, first=True)
        assert (m == float("-inf")).all() and not l.any() and not O.any()
    assert pkg.capi.last_device_error() == 0
