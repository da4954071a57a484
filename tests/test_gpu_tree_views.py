"""GPU: caches and rows that are views of other tensors -- expanded dimensions, whose stride is 0 -- on every path."""
import pytest
import torch

from cache_ref import check_tree, tree_reference
from test_gpu_tree import TYPES, both_paths, problem

pytestmark = pytest.mark.gpu


def expand(c, dim, size):
    """The cache with one dimension of its pages and scales (of one element so far) expanded."""
    shape = [-1, -1, -1, -1]
    shape[dim] = size
    for w in "KV":
        t, s = getattr(c, w), getattr(c, w + "_scale")
        setattr(c, w, t.expand(shape))
        assert getattr(c, w).stride(dim) == 0
        if s is not None:
            setattr(c, w + "_scale", s.expand(shape[:3]))
    return c


@pytest.mark.parametrize("dtype,cache", TYPES)
@pytest.mark.parametrize("layout", ["nhd", "hnd"])
def test_one_key_head_expanded_over_many(pkg, layout, dtype, cache):
    """Every key head is the same memory: small calls, and large ones of 16-bit types that would run on the tensor cores."""
    for lens, rows in (([40], [1]), ([300, 64, 9], [30, 40, 2])):
        c, Q, cu, mask = problem(dtype, cache, lens, rows, 8, 1, 64, 16, layout, seed=len(lens))
        c = expand(c, 2, 4)
        c.heads = 4
        want, bound, written = tree_reference(c, Q, cu, mask)
        tags = []
        for tag, got in both_paths(pkg, c, Q, cu, mask):
            tags.append(tag)
            check_tree(got, want, bound, written, (tag, lens))
        assert tags == ["auto", "gather"]  # the tensor cores are refused, not given other addresses


@pytest.mark.parametrize("dtype,cache", [("bf16", "native"), ("f16", "int8"), ("bf16", "e4m3")])
@pytest.mark.parametrize("dim,page", [(0, 64), (1, 1)])
def test_pages_or_slots_that_share_their_memory(pkg, dim, page, dtype, cache):
    """All pages are one, or all slots of a page: rows of a constant prefix."""
    c, Q, cu, mask = problem(dtype, cache, [30, 25], [40, 9], 8, 2, 64, page, seed=dim)
    if dim == 0:  # the pool's second page, as often as there were pages
        n = c.K.shape[0]
        for w in ("K", "V", "K_scale", "V_scale"):
            t = getattr(c, w)
            setattr(c, w, t if t is None else t[1:2])
        c = expand(c, 0, n)
    else:
        c.table = c.table[:, :9].contiguous()
        c = expand(c, 1, 8)
        c.page = 8
    want, bound, written = tree_reference(c, Q, cu, mask)
    tags = []
    for tag, got in both_paths(pkg, c, Q, cu, mask):
        tags.append(tag)
        check_tree(got, want, bound, written, tag)
    assert "tiled" not in tags


@pytest.mark.parametrize("dtype,cache", [("bf16", "native"), ("f16", "int8"), ("bf16", "e4m3")])
def test_dimensions_of_one_element_keep_the_tensor_cores(pkg, dtype, cache):
    """A stride of 0 says nothing where the dimension has one element."""
    c, Q, cu, mask = problem(dtype, cache, [300, 64], [30, 40], 4, 1, 64, 16, seed=3)
    c.K, c.V = (torch.as_strided(t, t.shape, (*t.stride()[:2], 0, 1), t.storage_offset()) for t in (c.K, c.V))
    want, bound, written = tree_reference(c, Q, cu, mask)
    tags = []
    for tag, got in both_paths(pkg, c, Q, cu, mask):
        tags.append(tag)
        check_tree(got, want, bound, written, tag)
    assert tags == ["auto", "tiled", "gather"]


@pytest.mark.parametrize("dtype,cache", [("f32", "native"), ("bf16", "int8"), ("f16", "e4m3")])
def test_query_rows_that_share_their_memory(pkg, dtype, cache):
    """One query head expanded over a group, one token over all: reads of Q go by its strides."""
    for dim in (0, 1):
        c, Q, cu, mask = problem(dtype, cache, [300, 64], [30, 40], 4, 2, 64, 16, seed=3)
        view = Q.cuda()[:1].expand(70, 4, 64) if dim == 0 else Q.cuda()[:, :1].expand(70, 4, 64)
        want, bound, written = tree_reference(c, view.cpu(), cu, mask)
        m, l = (torch.full((70, 4), float("nan"), device="cuda") for _ in range(2))
        O = torch.empty(70, 4, 64, device="cuda", dtype=view.dtype)
        pkg.binding("spfa_tree").forward(view, *c.args(), torch.tensor(cu, dtype=torch.int32, device="cuda"), mask.cuda(), m, l, O,
                                         *c.scales(), first=True)
        check_tree((m, l, O), want, bound, written, dim)


@pytest.mark.parametrize("dtype,cache", [("bf16", "native"), ("f16", "int8")])
def test_modules_refuse_to_write_expanded_tensors(pkg, dtype, cache):
    c, Q, cu, mask = problem(dtype, cache, [20, 9], [3, 2], 4, 1, 64, 16)
    c = expand(c, 2, 2)
    mod, cu_t = pkg.binding("spfa_cache"), torch.tensor(cu, dtype=torch.int32, device="cuda")
    rows = torch.ones(5, 2, 64, dtype=Q.dtype, device="cuda")
    kept, before = torch.ones(2, 1, dtype=torch.int32, device="cuda"), c.K.clone()
    m, l = (torch.zeros(5, 4, device="cuda") for _ in range(2))
    O = torch.zeros(5, 1, 64, dtype=Q.dtype, device="cuda")
    for bad in (lambda: mod.append(rows, rows, *c.args(), cu_t, *c.scales()), lambda: mod.keep(*c.args(), kept, kept[:, 0], *c.scales()),
                lambda: mod.read(*c.args(), cu_t, rows[:, :1].expand(5, 2, 64), rows, *c.scales()),
                lambda: pkg.binding("spfa_tree").forward(Q.cuda(), *c.args(), cu_t, mask.cuda(), m, l, O.expand(5, 4, 64), *c.scales())):
        with pytest.raises(RuntimeError, match="bad argument"):
            bad()
    assert torch.equal(c.K.view(torch.int8 if cache == "int8" else torch.int16), before.view(torch.int8 if cache == "int8" else torch.int16))
    assert (rows == 1).all() and not O.any()
    mod.read(*c.args(), cu_t, rows, rows.clone(), *c.scales())  # reading from them is fine
    assert torch.equal(rows[:, 0], rows[:, 1]) and not (rows == 1).all()
