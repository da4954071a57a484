"""CPU: a cache described on one device is not given to a call whose tensors are on another."""
import pytest
import torch

from test_cache_tree_host import _cache


def test_rows_of_another_device_are_refused(pkg):
    capi, c = pkg.capi, _cache(pkg)
    c.device = torch.device("cuda", 1)  # as kv_cache notes it
    K, Q = torch.zeros(5, 4, 64, dtype=torch.bfloat16), torch.zeros(5, 8, 64, dtype=torch.bfloat16)
    cu, m = torch.zeros(4, dtype=torch.int32), torch.zeros(5, 8)
    for call in (lambda: capi.cache_append(c, K, K, cu), lambda: capi.cache_read(c, K, K, cu),
                 lambda: capi.cache_keep(c, torch.zeros(3, 2, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)),
                 lambda: capi.tree_forward(c, Q, cu, torch.zeros(5, 2, dtype=torch.bool), m, m.clone(), Q.clone(), first=True)):
        with pytest.raises(capi.SpfaError, match="cache is on cuda:1"):
            call()
