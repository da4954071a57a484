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
