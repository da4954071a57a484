"""GPU: attention of drafted token trees over a paged cache, against the 64-bit restatement within the bounds derived there."""
import numpy as np
import pytest
import torch

import cache_ref
from cache_ref import Cache, check_tree, tree_reference

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
TYPES = [(t, c) for t in ("f32", "f16", "bf16") for c in ("native", "e4m3", "int8")]


def tree_mask(rows, width, g, dense=0.0):
    """Ancestors and self, in random trees; with `dense` any entries besides."""
    mask, at = torch.zeros(sum(rows), width, dtype=torch.bool), 0
    for T in rows:
        seen = torch.eye(T, dtype=torch.bool)
        for i in range(1, T):
            p = int(torch.randint(-1, i, (1,), generator=g))
            if p >= 0:
                seen[i] |= seen[p]
        if dense:
            seen |= torch.rand(T, T, generator=g) < dense
        w = min(T, width)
        mask[at:at + T, :w] = seen[:, :w]
        at += T
    return mask


def problem(dtype, cache, lens, rows, Hq, Hkv, d, page, layout="nhd", seed=0, q_scale=2.0, dense=0.0, width=None, shift=0):
    g = torch.Generator().manual_seed(seed)
    c = Cache(DT[dtype], cache, [max(0, n) + r for n, r in zip(lens, rows)], Hkv, d, page, layout, seed + 1, lens, shift=shift)
    Q = (torch.randn(sum(rows), Hq, d, generator=g) * q_scale).to(DT[dtype])
    cu = np.concatenate([[0], np.cumsum(rows)]).tolist()
    return c, Q, cu, tree_mask(rows, max(rows + [1]) if width is None else width, g, dense)


def new_state(N, Hq, d, dtype, junk=False):
    m, l = torch.full((N, Hq), -np.inf, device="cuda"), torch.zeros(N, Hq, device="cuda")
    O = torch.zeros(N, Hq, d, device="cuda", dtype=dtype)
    if junk:
        for t in (m, l, O):
            t.fill_(float("nan"))
    return m, l, O


def run(pkg, c, Q, cu, mask, state=None):
    N, Hq, d = Q.shape
    first = state is None
    m, l, O = new_state(N, Hq, d, Q.dtype, junk=True) if first else state
    out = pkg.binding("spfa_tree").forward(Q.cuda(), *c.args(), torch.tensor(cu, dtype=torch.int32, device="cuda"), mask.cuda(), m, l, O,
                                           *c.scales(), first=first)
    assert out.data_ptr() == O.data_ptr()
    torch.cuda.synchronize()
    assert pkg.capi.last_device_error() == 0
    return m, l, O


def both_paths(pkg, *args, **kw):
    """The automatic choice (small calls: one launch), the tensor cores where they can take the call, and the kernels without."""
    yield "auto", run(pkg, *args, **kw)
    for tag, path in (("tiled", pkg.capi.PATH_TILED), ("gather", pkg.capi.PATH_GATHER)):
        pkg.capi.set_path(path)
        try:
            try:
                got = run(pkg, *args, **kw)
            except RuntimeError as e:
                assert path == pkg.capi.PATH_TILED and "bad argument" in str(e)
                continue
            assert pkg.capi.last_path() == path
        finally:
            pkg.capi.set_path(pkg.capi.PATH_AUTO)
        yield tag, got


SHAPES = [  # lens, rows, Hq, Hkv, d, page, layout
    ([0], [1], 1, 1, 64, 16, "nhd"), ([1], [1], 2, 1, 128, 16, "nhd"), ([500], [1], 8, 8, 64, 16, "nhd"),
    ([63, 64, 65, 0, 1], [3, 1, 7, 5, 2], 8, 2, 128, 16, "hnd"), ([200, 3], [16, 0], 4, 4, 64, 24, "nhd"),
    ([1000, 17, 333], [5, 30, 12], 12, 4, 64, 64, "hnd"), ([130, 700], [33, 9], 8, 1, 128, 100, "nhd"),
    ([257], [64], 6, 2, 80, 32, "nhd"), ([100, 40], [4, 20], 7, 1, 40, 48, "hnd"), ([90], [3], 5, 5, 96, 256, "nhd"),
    ([300, 20], [2, 6], 4, 2, 256, 16, "nhd"), ([33, 80], [3, 2], 3, 1, 3, 5, "nhd"), ([50], [4], 2, 2, 200, 10, "hnd"),
    ([40], [2], 2, 1, 1024, 4, "nhd"), ([70, 10], [2, 5], 2, 1, 37, 7, "nhd"), ([64], [2], 1, 1, 512, 16, "nhd"),
    ([45], [3], 2, 2, 32, 20, "nhd"), ([600], [40], 16, 2, 16, 8, "nhd"),
    # more rows than a row tile holds on average, sequences with fewer among them
    ([600, 100, 0, 300, 70], [40, 70, 33, 5, 33], 16, 2, 128, 16, "hnd"), ([1500, 64], [30, 9], 16, 1, 64, 64, "nhd"),
]


@pytest.mark.parametrize("dtype,cache", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_rows_against_64_bits(pkg, shape, dtype, cache):
    lens, rows, Hq, Hkv, d, page, layout = shape
    c, Q, cu, mask = problem(dtype, cache, lens, rows, Hq, Hkv, d, page, layout, seed=d + page)
    want, bound, written = tree_reference(c, Q, cu, mask)
    for tag, got in both_paths(pkg, c, Q, cu, mask):
        check_tree(got, want, bound, written, tag)


@pytest.mark.parametrize("dtype,cache", TYPES)
def test_many_pieces_are_merged(pkg, dtype, cache):
    """One sequence over every CTA (a row has a piece in each), then ragged ones whose units end inside a CTA's share."""
    for lens, rows in (([9000], [2]), ([1500, 7, 0, 650, 2222, 64], [3, 1, 2, 40, 1, 9])):
        c, Q, cu, mask = problem(dtype, cache, lens, rows, 4, 2, 64, 16, seed=len(lens), q_scale=6.0)
        want, bound, written = tree_reference(c, Q, cu, mask)
        for tag, got in both_paths(pkg, c, Q, cu, mask):
            check_tree(got, want, bound, written, (tag, lens))


@pytest.mark.parametrize("dtype,cache", TYPES)
def test_state_chains(pkg, dtype, cache):
    """Two caches on one state are the attention over both; rows without keys keep their state, and without `first` rows
    behind the last sequence do too."""
    c1, Q, cu, mask = problem(dtype, cache, [100, 31, 64], [4, 6, 2], 4, 2, 64, 16, seed=5)
    c2, _, _, mask2 = problem(dtype, cache, [77, 0, 130], [4, 6, 2], 4, 2, 64, 32, seed=6)
    mask2[5] = False
    one, b1, written = tree_reference(c1, Q, cu, mask)
    for path in (pkg.capi.PATH_AUTO, pkg.capi.PATH_GATHER) + ((pkg.capi.PATH_TILED,) if dtype != "f32" else ()):
        pkg.capi.set_path(path)
        try:
            state = run(pkg, c1, Q, cu, mask)
            check_tree(state, one, b1, written)
            given = tuple(x.double().cpu().numpy() for x in state)
            want, bound, _ = tree_reference(c2, Q, cu, mask2, state=given)  # from what the first call really left
            got = run(pkg, c2, Q, cu, mask2, state=state)
            check_tree(got, want, bound, written)
            # nothing visible: bit for bit what it was, in rows of sequences and in others
            c1.lens[:] = 0
            before = tuple(x.clone() for x in got)
            again = run(pkg, c1, Q, [0, 4, 10, 10], torch.zeros(12, 6, dtype=torch.bool), state=got)
            assert all(torch.equal(x, y) for x, y in zip(before, again))
            c1.lens[:] = torch.tensor([100, 31, 64])
        finally:
            pkg.capi.set_path(pkg.capi.PATH_AUTO)


def test_incoming_rows_of_weight_zero_do_not_count(pkg):
    c, Q, cu, mask = problem("bf16", "native", [100, 31], [4, 6], 4, 2, 64, 16, seed=5)
    want, bound, written = tree_reference(c, Q, cu, mask)
    m, l, O = new_state(10, 4, 64, torch.bfloat16)
    O.fill_(float("nan"))
    check_tree(run(pkg, c, Q, cu, mask, state=(m, l, O)), want, bound, written)


@pytest.mark.parametrize("dtype,cache", TYPES)
def test_rows_without_keys(pkg, dtype, cache):
    """Masks that leave a row nothing, in sequences without a committed key; pages that do not exist; masks narrower and wider than
    the tree; dense masks."""
    c, Q, cu, mask = problem(dtype, cache, [0, 40, 0, 33], [5, 4, 0, 40], 4, 2, 64, 16, seed=9, dense=0.3, width=37)
    mask[2], mask[7] = False, False
    c.table[3, 1], c.table[1, 0], c.table[3, 4] = -1, 10 ** 7, c.K.shape[0]
    want, bound, written = tree_reference(c, Q, cu, mask)
    assert want[1][2].max() == 0
    for tag, got in both_paths(pkg, c, Q, cu, mask):
        check_tree(got, want, bound, written, tag)
        assert torch.isinf(got[0][2]).all() and not got[1][2].any() and not got[2][2].any()
    wide = torch.cat([mask, torch.ones(len(mask), 100, dtype=torch.bool)], 1)  # columns beyond a tree's rows name nothing
    wide[:, 37:40] = False
    for tag, got in both_paths(pkg, c, Q, cu, wide):
        check_tree(got, want, bound, written, tag)
    none = torch.zeros(len(mask), 0, dtype=torch.bool)
    want, bound, _ = tree_reference(c, Q, cu, none)
    for tag, got in both_paths(pkg, c, Q, cu, none):
        check_tree(got, want, bound, written, tag)


@pytest.mark.parametrize("dtype,cache", TYPES)
def test_values_behind_the_end_and_in_masked_places_do_not_count(pkg, dtype, cache):
    """NaN and infinities in every position that nobody sees: behind the sequences, in pages of nobody, in drafted rows that a
    row's mask leaves out."""
    lens, rows = [100, 64, 3], [9, 4, 6]
    c, Q, cu, mask = problem(dtype, cache, lens, rows, 8, 2, 64, 16, seed=3)
    for b, T in enumerate(rows):  # the last drafted row of each is seen by nobody but itself
        mask[cu[b]:cu[b + 1] - 1, T - 1] = False
        mask[cu[b + 1] - 1] = False
        mask[cu[b + 1] - 1, 0] = True
    want, bound, written = tree_reference(c, Q, cu, mask)
    used = torch.zeros(c.K.shape[:2], dtype=torch.bool)
    for b in range(3):
        for p in range(lens[b] + rows[b] - 1):
            used[c.place(b, p)] = True
    for fill in (float("nan"), float("inf"), float("-inf")):
        for t, s in ((c.K, c.K_scale), (c.V, c.V_scale)):
            if s is None:
                t[~used.cuda()] = fill
            else:
                s[~used.cuda()] = fill
                t.view(torch.uint8)[~used.cuda()] = 0x7f
        for tag, got in both_paths(pkg, c, Q, cu, mask):
            check_tree(got, want, bound, written, (tag, fill))


@pytest.mark.parametrize("dtype,cache", TYPES)
def test_values_that_are_not_finite_reach_the_rows_that_see_them(pkg, dtype, cache):
    lens, rows = [100, 64, 70], [3, 4, 2]
    c, Q, cu, mask = problem(dtype, cache, lens, rows, 4, 2, 64, 16, seed=3)
    at, at2 = c.place(0, 50), c.place(1, 64)  # a committed key of the first sequence, the first drafted one of the second
    mask[cu[1]:cu[2], 0] = torch.tensor([True, False, True, False])
    if cache == "native":
        c.V[at][0, 5], c.K[at2][1, 0] = float("inf"), float("nan")
    else:
        c.V_scale[at[0], at[1], 0], c.K_scale[at2[0], at2[1], 1] = float("nan"), float("nan")
    want, bound, written = tree_reference(c, Q, cu, mask)
    assert not np.isfinite(want[2][0, 0, 5]) and np.isnan(want[2][3, 2]).all() and np.isfinite(want[2][4]).all()
    for tag, got in both_paths(pkg, c, Q, cu, mask):
        check_tree(got, want, bound, written, tag)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_strides_and_alignment(pkg, dtype):
    """Q and O as slices of larger tensors, O in the place of Q, K and V interleaved, pages off a 16-byte boundary."""
    lens, rows = [150, 70], [5, 9]
    c, Q, cu, mask = problem(dtype, "native", lens, rows, 4, 2, 64, 16, seed=8)
    want, bound, written = tree_reference(c, Q, cu, mask)
    N = len(Q)
    both = torch.empty(*c.K.shape[:2], 2, 2, 64, dtype=DT[dtype], device="cuda")  # [page, slot, K or V, head, d]
    both[:, :, 0], both[:, :, 1] = c.K, c.V
    packed = torch.zeros(N, 8, 64, dtype=DT[dtype], device="cuda")
    packed[:, 4:] = Q.cuda()
    m, l, _ = new_state(N, 4, 64, DT[dtype], junk=True)
    fwd = pkg.binding("spfa_tree").forward
    rest = (*c.args()[2:], torch.tensor(cu, dtype=torch.int32, device="cuda"), mask.cuda())
    fwd(packed[:, 4:], both[:, :, 0], both[:, :, 1], *rest, m, l, packed[:, :4], first=True)
    check_tree((m, l, packed[:, :4]), want, bound, written)
    fwd(packed[:, 4:], c.K, c.V, *rest, m, l, packed[:, 4:], first=True)  # in place
    check_tree((m, l, packed[:, 4:]), want, bound, written)
    assert pkg.capi.last_device_error() == 0
    c, Q, cu, mask = problem(dtype, "native", lens, rows, 4, 2, 64, 16, seed=8, shift=1)  # rows start one element off
    want, bound, written = tree_reference(c, Q, cu, mask)
    check_tree(run(pkg, c, Q, cu, mask), want, bound, written)
    odd = torch.empty(N * 4 * 64 + 1, dtype=DT[dtype], device="cuda")
    odd[1:] = Q.cuda().reshape(-1)
    O = torch.empty(N * 4 * 64 + 3, dtype=DT[dtype], device="cuda")[3:].view(N, 4, 64)
    c.lens = torch.tensor(lens, dtype=torch.int32)
    fwd(odd[1:].view(N, 4, 64), *c.args(), *rest[2:], m, l, O, first=True)
    check_tree((m, l, O), want, bound, written)


@pytest.mark.parametrize("dtype,cache", [("f32", "native"), ("bf16", "native"), ("f16", "int8"), ("bf16", "e4m3")])
def test_ranges(pkg, dtype, cache):
    """Scores from all alike to one that takes everything, lengths that a device-side value cuts, and sequences the call does not hold."""
    for q_scale in (0.0, 0.01, 40.0):
        c, Q, cu, mask = problem(dtype, cache, [260, 33], [6, 3], 4, 2, 64, 32, seed=2, q_scale=q_scale)
        want, bound, written = tree_reference(c, Q, cu, mask)
        for tag, got in both_paths(pkg, c, Q, cu, mask):
            check_tree(got, want, bound, written, (tag, q_scale))
    c.lens[:] = torch.tensor([10 ** 9, -7])  # more than the pages hold: all of them; below zero: none
    want, bound, written = tree_reference(c, Q, cu, mask)
    for tag, got in both_paths(pkg, c, Q, cu, mask):
        check_tree(got, want, bound, written, tag)
    c.lens[:] = torch.tensor([100, 20])
    for cu2 in ([2, 5, 7], [0, 0, 9], [4, 4, 4], [0, 9, 9]):
        want, bound, written = tree_reference(c, Q, cu2, mask)
        for tag, got in both_paths(pkg, c, Q, cu2, mask):
            check_tree(got, want, bound, written, (tag, cu2))
            assert torch.isnan(got[2][torch.from_numpy(~written).cuda()]).all()  # rows of no sequence are left as they were


def test_streams_and_replayed_graphs(pkg):
    """Two captured calls of different sizes, replayed with other lengths in turn and at once on two streams: no shared scratch."""
    graphs = []
    for seed, (lens, rows) in enumerate((([300, 100], [5, 7]), ([700], [40]))):
        c, Q, cu, mask = problem("bf16", "native", lens, rows, 8, 2, 128, 16, seed=seed)
        args = c.args()
        st = new_state(len(Q), 8, 128, torch.bfloat16)
        q, cu_t, mk = Q.cuda(), torch.tensor(cu, dtype=torch.int32, device="cuda"), mask.cuda()
        fwd = pkg.binding("spfa_tree").forward
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            fwd(q, *args, cu_t, mk, *st, first=True)
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):
                fwd(q, *args, cu_t, mk, *st, first=True)
        s.synchronize()
        graphs.append((c, Q, cu, mask, args, st, g, s, q, cu_t, mk))
    for step in range(3):
        for c, Q, cu, mask, args, st, g, s, *_ in graphs:
            c.lens = torch.clamp(c.lens - 50 * step, min=0)
            args[3].copy_(c.lens)
            for t in st:
                t.fill_(float("nan"))
        torch.cuda.synchronize()
        for _ in range(4):
            for *_, g, s, _, _, _ in graphs:
                with torch.cuda.stream(s):
                    g.replay()
        torch.cuda.synchronize()
        for c, Q, cu, mask, args, st, *_ in graphs:
            want, bound, written = tree_reference(c, Q, cu, mask)
            check_tree(st, want, bound, written, step)
    assert pkg.capi.last_device_error() == 0


def test_a_step_of_drafted_decoding(pkg):
    """Write drafted rows, attend, keep the accepted path, go on: against the same step on dense float64 K and V, in a cache of each
    type. The rows of the next step see the kept ones where they were moved to."""
    cache_mod, fwd = pkg.binding("spfa_cache"), pkg.binding("spfa_tree").forward
    for dtype, cache in TYPES:
        lens = [40, 17, 0]
        c = Cache(DT[dtype], cache, [n + 60 for n in lens], 2, 64, 16, "hnd", 11, lens)
        pages = c.args()
        g = torch.Generator().manual_seed(1)
        for step in range(3):
            rows = [7, 1 + step, 12]
            N, cu = sum(rows), np.concatenate([[0], np.cumsum(rows)]).tolist()
            K, V = (torch.randn(N, 2, 64, generator=g).to(DT[dtype]) for _ in range(2))
            Q = (torch.randn(N, 4, 64, generator=g) * 2).to(DT[dtype])
            mask, cu_t = tree_mask(rows, 12, g), torch.tensor(cu, dtype=torch.int32, device="cuda")
            st = new_state(N, 4, 64, DT[dtype], junk=True)
            cache_mod.append(K.cuda(), V.cuda(), *pages, cu_t, *c.scales())
            fwd(Q.cuda(), *pages, cu_t, mask.cuda(), *st, *c.scales(), first=True)
            c.lens = pages[3].cpu()
            held = {"K": K.double().numpy(), "V": V.double().numpy()}
            if cache != "native":
                held = {w: cache_ref.values(*cache_ref.quantise(x, cache), cache) for w, x in held.items()}
            for w, x in held.items():
                for b in range(3):
                    assert np.array_equal(c.dense(w, b, range(int(c.lens[b]), int(c.lens[b]) + rows[b]))[0], x[cu[b]:cu[b + 1]])
            want, bound, written = tree_reference(c, Q, cu, mask)
            check_tree(st, want, bound, written, (dtype, cache, step))
            kept, n_kept = torch.zeros(3, 4, dtype=torch.int32), torch.tensor([min(4, r) for r in rows], dtype=torch.int32)
            for b in range(3):
                kept[b, :n_kept[b]] = torch.randperm(rows[b], generator=g)[:int(n_kept[b])].sort().values
            cache_mod.keep(*pages, kept.cuda(), n_kept.cuda(), *c.scales())
            for w, x in held.items():
                for b in range(3):
                    k = int(n_kept[b])
                    assert np.array_equal(c.dense(w, b, range(int(c.lens[b]), int(c.lens[b]) + k))[0], x[cu[b]:cu[b + 1]][kept[b, :k].numpy()])
            pages[3].add_(n_kept.cuda())
    assert pkg.capi.last_device_error() == 0


def test_read_rows_feed_the_dense_operators(pkg):
    """A cache read back head by head is K and V of the windowed operator: the last 2 w + 1 positions of a chain of drafted tokens."""
    L, d, w = 300, 64, 20
    c, Q, cu, _ = problem("f32", "int8", [0], [L], 2, 1, d, 16, seed=4)
    i = torch.arange(L)
    mask = (i[:, None] - i[None]).abs() <= w
    want, bound, written = tree_reference(c, Q, cu, mask)
    K, V = (torch.empty(1, L, d, device="cuda") for _ in range(2))
    pkg.binding("spfa_cache").read(*c.args(), torch.tensor(cu, dtype=torch.int32, device="cuda"), K.transpose(0, 1), V.transpose(0, 1),
                                   *c.scales())
    m, l, O = run(pkg, c, Q, cu, mask)
    check_tree((m, l, O), want, bound, written)
    pkg.capi.set_path(pkg.capi.PATH_GATHER)
    try:
        for h in range(2):
            st = pkg.capi.new_state(L, d)
            pkg.binding("spfa_local").forward(Q[:, h].contiguous().cuda(), K[0], V[0], *st, w)
            check_tree(tuple(t[:, None] for t in st), tuple(x[:, h:h + 1] for x in want),
                       tuple(x[:, h:h + 1] * 4 for x in bound), written)  # another order of operations: four times the bound
    finally:
        pkg.capi.set_path(pkg.capi.PATH_AUTO)


def test_refusals(pkg):
    fwd = pkg.binding("spfa_tree").forward
    c, Q, cu, mask = problem("bf16", "native", [20, 5], [3, 2], 4, 2, 64, 16)
    q, cu_t, mk = Q.cuda(), torch.tensor(cu, dtype=torch.int32, device="cuda"), mask.cuda()
    m, l, O = new_state(5, 4, 64, torch.bfloat16)
    a = c.args()
    for bad in (lambda: fwd(q.cpu(), *a, cu_t, mk, m, l, O), lambda: fwd(q.half(), *a, cu_t, mk, m, l, O.half()),
                lambda: fwd(q, *a, cu_t, mk, m, l, O.float()), lambda: fwd(q[:, :3], *a, cu_t, mk, m[:, :3], l[:, :3], O[:, :3]),
                lambda: fwd(q[..., :32], *a, cu_t, mk, m, l, O[..., :32]), lambda: fwd(q[:4], *a, cu_t, mk, m, l, O),
                lambda: fwd(q, *a, cu_t[:2], mk, m, l, O), lambda: fwd(q, *a, cu_t.long(), mk, m, l, O),
                lambda: fwd(q, *a, cu_t, mk.float(), m, l, O), lambda: fwd(q, *a, cu_t, mk[:4], m, l, O),
                lambda: fwd(q, *a, cu_t, mk.cpu(), m, l, O), lambda: fwd(q, *a, cu_t, mk, m.half(), l, O),
                lambda: fwd(q, *a, cu_t, mk, m[:, :2], l, O), lambda: fwd(q, *a, cu_t, mk, m, l.t().contiguous().t(), O),
                lambda: fwd(q, *a, cu_t, mk, m, l, O, m, l), lambda: fwd(q[0], *a, cu_t, mk, m, l, O)):
        with pytest.raises(RuntimeError):
            bad()
    none = torch.zeros(0, 4, 64, dtype=torch.bfloat16, device="cuda")
    fwd(none, *a, torch.zeros(3, dtype=torch.int32, device="cuda"), mk[:0], m[:0], l[:0], none)
    assert pkg.capi.last_device_error() == 0


def test_which_kernel_takes_a_call(pkg):
    """The tensor-core path takes 16-bit calls on rows and pages that the copy engine can address; the others go without."""
    tiled = pkg.capi.PATH_TILED
    for dtype, cache, d, page, shift, want in (("bf16", "native", 128, 16, 0, True), ("f16", "native", 40, 8, 0, True),
                                               ("f16", "int8", 80, 24, 0, True), ("bf16", "e4m3", 64, 100, 0, True),
                                               ("bf16", "e4m3", 64, 20, 0, False), ("bf16", "e4m3", 40, 16, 0, False),
                                               ("bf16", "native", 64, 65, 0, True), ("bf16", "native", 136, 16, 0, False),
                                               ("bf16", "native", 64, 16, 1, False), ("f32", "int8", 64, 16, 0, False)):
        c, Q, cu, mask = problem(dtype, cache, [70], [2], 2, 1, d, page, shift=shift)
        run(pkg, c, Q, cu, mask)
        assert pkg.capi.last_path() == pkg.capi.PATH_GATHER  # small: one launch, or the kernels without tensor cores
        pkg.capi.set_path(tiled)
        try:
            if want:
                run(pkg, c, Q, cu, mask)
            else:
                with pytest.raises(RuntimeError):
                    run(pkg, c, Q, cu, mask)
        finally:
            pkg.capi.set_path(pkg.capi.PATH_AUTO)
        c, Q, cu, mask = problem(dtype, cache, [2048], [150], 2, 1, d, page, shift=shift)
        run(pkg, c, Q, cu, mask)
        assert (pkg.capi.last_path() == tiled) == want, (dtype, cache, d, page, shift)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("cache", ["e4m3", "int8"])
def test_every_code_is_taken_as_its_value(pkg, cache, dtype):
    """One committed key: O is its V row, whatever the score, and the score is q . k. All 256 codes, on both paths; NaN codes make
    NaN of their column of O, and as K of the whole row."""
    codes = torch.arange(256, dtype=torch.uint8).view(4, 64)
    c, Q, cu, mask = problem(dtype, cache, [1], [1], 4, 4, 64, 16)
    at = c.place(0, 0)
    none = torch.zeros(1, 0, dtype=torch.bool)
    value = torch.from_numpy(np.concatenate([cache_ref.E4M3, [np.nan], -cache_ref.E4M3, [np.nan]])) if cache == "e4m3" else \
        codes.view(torch.int8).double().flatten()
    raw = lambda t: t.view(torch.uint8)  # noqa: E731
    raw(c.V)[at] = codes.cuda()
    raw(c.K)[at] = 0x18
    c.V_scale[at], c.K_scale[at] = 2.0 ** -9, 0.25
    for tag, (m, l, O) in both_paths(pkg, c, Q, cu, none):
        # the reference of the row is its score rounded to float32, the exponent its unrounded product less that: |x| <= |m log2 e| 2^-24,
        # and l = 2^x, from an instruction good to 2^-22
        assert ((l.cpu() - 1).abs() <= m.cpu().abs() * 2.0 ** -24 + 2.0 ** -22).all()
        assert torch.equal(O.cpu()[0].nan_to_num(7), (value.view(4, 64) * 2.0 ** -9).to(DT[dtype]).nan_to_num(7)), tag
    raw(c.V)[at] = 1
    Q = torch.zeros(1, 4, 64, dtype=DT[dtype])
    for e in range(64):  # m is one code of each head at a time
        Q.zero_()
        Q[0, :, e] = 8
        raw(c.K)[at] = codes.cuda()
        if cache == "e4m3":
            raw(c.K)[at][codes.cuda() % 128 == 127] = 0
        for tag, (m, l, O) in both_paths(pkg, c, Q, cu, none):
            want = value.view(4, 64)[:, e].nan_to_num(0) * 0.25  # 8 / sqrt(64) = 1
            assert np.allclose(m.cpu()[0].double(), want, rtol=2.0 ** -22, atol=0), (tag, e)
    if cache == "e4m3":
        raw(c.K)[at][2, 5] = 0xff
        for tag, (m, l, O) in both_paths(pkg, c, Q, cu, none):
            bad = torch.tensor([[False, False, True, False]])
            assert torch.equal(torch.isnan(m.cpu()), bad) and torch.equal(torch.isnan(O.cpu()).all(-1), bad), tag


@pytest.mark.parametrize("dtype,cache", [("f32", "native"), ("bf16", "native"), ("f16", "int8"), ("bf16", "e4m3")])
@pytest.mark.parametrize("Hq,Hkv", [(4, 2), (6, 2), (12, 3), (5, 1), (12, 2), (14, 2), (18, 2), (20, 1), (67, 1), (130, 1)])
def test_many_rows_are_merged_together(pkg, Hq, Hkv, dtype, cache):
    """Calls of many rows merge several query heads at a time: groups that four divides and others, groups that no row tile divides,
    units that end inside a token; twice, on the state that the first call left."""
    tokens = 2400 // Hq + 1  # more rows than the machine holds warps
    rows = [tokens // 2, 0, 1, tokens - tokens // 2]
    c, Q, cu, mask = problem(dtype, cache, [70, 9, 0, 33], rows, Hq, Hkv, 64, 16, "hnd", seed=Hq, width=40)
    want, bound, written = tree_reference(c, Q, cu, mask)
    got = run(pkg, c, Q, cu, mask)
    check_tree(got, want, bound, written, "first")
    given = tuple(x.double().cpu().numpy() for x in got)
    want, bound, _ = tree_reference(c, Q, cu, mask, state=given)
    check_tree(run(pkg, c, Q, cu, mask, state=got), want, bound, written, "again")


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("rows", [3, 40])
def test_query_rows_of_a_wide_range_over_e4m3(pkg, dtype, rows):
    """bfloat16 Q meets an e4m3 cache as an e4m3 and an e5m2 number an element, the row's largest between 2^7 and 2^8 (float16 Q meets
    it as it is, well within these bounds). Elements from 2^-6 on are held exactly; of smaller ones e4m3 leaves at most 2^-10, and e5m2 (a half step of 2^-3
    below the power of two) 2^-14 of that: 2^-21 of the row's largest. A score is off by dq = 2^-21 max|q| sum|k| / sqrt(d) then, a
    probability by 2 dq, O by 4 dq max|v|. Rows that are not finite are NaN."""
    c, Q, cu, mask = problem(dtype, "e4m3", [700], [rows], 8, 2, 128, 16, seed=rows)
    g = torch.Generator().manual_seed(1)
    low = -12 if dtype == "f16" else -24
    Q = Q * torch.exp2(torch.randint(low, 1, Q.shape, generator=g).float()).to(Q.dtype)
    want, bound, written = tree_reference(c, Q, cu, mask)
    k = np.abs(c.dense("K", 0, range(700 + rows))[0]).sum(-1).max()
    v = np.abs(c.dense("V", 0, range(700 + rows))[0]).max()
    dq = 2.0 ** -21 * np.abs(Q.double().numpy()).max(-1) * k / np.sqrt(128)
    bound = (bound[0] + dq, bound[1] + 2 * dq * want[1], bound[2] + 4 * (dq * v)[..., None])
    pkg.capi.set_path(pkg.capi.PATH_TILED)
    try:
        check_tree(run(pkg, c, Q, cu, mask), want, bound, written)
        Q[1, 2, 5], Q[2, 1, 0] = float("inf"), float("nan")
        m, l, O = run(pkg, c, Q, cu, mask)
        assert torch.isnan(O[1, 2]).all() and torch.isnan(O[2, 1]).all()
        others = torch.ones(rows, 8, dtype=torch.bool)
        others[1, 2] = others[2, 1] = False
        assert torch.isfinite(O[others.cuda()]).all() and torch.isfinite(m[others.cuda()]).all()
    finally:
        pkg.capi.set_path(pkg.capi.PATH_AUTO)
