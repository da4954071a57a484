"""What is measured of the cached-decoding operators: a paged key / value cache and the attention of drafted token trees over it.

Position p of sequence b lies in page `table[b, p // page]`, slot `p % page`, of `K_pages` / `V_pages`
[n_pages, page, kv heads, d]. Row i of a call belongs to the sequence b with `cu[b] <= i < cu[b + 1]` and stands for the
position `lens[b] + i - cu[b]`. Kinds of cases:

  append  the rows of new tokens are written into the cache, in the cache's type, and read back: what a step that goes on
          with the stored values does
  read    whole sequences are read back from their pages
  commit  drafted rows are written, the accepted ones are moved to the front, and these are read back
  tree    attention of drafted tokens: each row sees the whole of its sequence and, of the drafted rows, those its mask names

Caches hold the input's type ("native"), 8-bit floating point (e4m3, a power of two as the scale of each row and head) or
8-bit integers (scale max / 127, multiplied by 127 / max and rounded).
"""
import importlib
import math

import torch

own = False

PACKAGE = "graph-processing-attention-ipdps-2025_b200"
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2, "e4m3": 1, "int8": 1}
_modules = {}


def module(name):
    if name not in _modules:
        _modules[name] = importlib.import_module(PACKAGE).binding(name)
    return _modules[name]


# ---- cases -------------------------------------------------------------------------------------------------------------

def listed():
    return [
        # one new token for each of a full batch: the write of every plain decoding step, latency only
        {"name": "append_step", "kind": "append", "dtype": "bf16", "cache": "e4m3", "B": 64, "rows": 1, "len": 4096, "Hkv": 8, "d": 128, "page": 16, "layout": "nhd"},
        # a few ragged prompts that arrive together, small heads, values kept as they are
        {"name": "append_prompts_f32", "kind": "append", "dtype": "f32", "cache": "native", "B": 5, "rows": 777, "len": 0, "Hkv": 4, "d": 64, "page": 32, "layout": "hnd"},
        # a long prompt, quantised as it is written
        {"name": "append_long_int8", "kind": "append", "dtype": "f16", "cache": "int8", "B": 1, "rows": 131072, "len": 0, "Hkv": 8, "d": 128, "page": 64, "layout": "hnd"},
        # a short prefix read back for a full-precision step, odd length
        {"name": "read_prefix_int8", "kind": "read", "dtype": "f32", "cache": "int8", "B": 1, "len": 257, "Hkv": 4, "d": 64, "page": 16, "layout": "nhd"},
        # ragged sequences read back whole, as an operator on dense K and V takes them
        {"name": "read_batch_e4m3", "kind": "read", "dtype": "bf16", "cache": "e4m3", "B": 8, "len": 32768, "Hkv": 8, "d": 128, "page": 64, "layout": "hnd"},
        # one verified draft of one sequence
        {"name": "commit_one", "kind": "commit", "dtype": "f16", "cache": "int8", "B": 1, "rows": 16, "kept": 5, "len": 1000, "Hkv": 8, "d": 64, "page": 16, "layout": "hnd"},
        # the verified drafts of a large batch
        {"name": "commit_batch", "kind": "commit", "dtype": "bf16", "cache": "native", "B": 128, "rows": 64, "kept": 12, "len": 2048, "Hkv": 8, "d": 128, "page": 32, "layout": "nhd"},
        # one token, one short sequence: latency only
        {"name": "tree_one_token", "kind": "tree", "dtype": "bf16", "cache": "native", "B": 1, "rows": 1, "len": 500, "Hq": 8, "Hkv": 8, "d": 64, "page": 16, "layout": "nhd"},
        # full precision, a few small trees
        {"name": "tree_f32", "kind": "tree", "dtype": "f32", "cache": "native", "B": 4, "rows": 16, "len": 4096, "Hq": 8, "Hkv": 4, "d": 64, "page": 32, "layout": "nhd"},
        # an ordinary ragged batch in half precision, small pages
        {"name": "tree_bf16_ragged", "kind": "tree", "dtype": "bf16", "cache": "native", "B": 16, "rows": 32, "len": 32768, "Hq": 32, "Hkv": 8, "d": 128, "page": 16, "layout": "nhd"},
        # wide trees on many heads that share keys: arithmetic counts
        {"name": "tree_f16_int8_wide", "kind": "tree", "dtype": "f16", "cache": "int8", "B": 8, "rows": 64, "len": 16384, "Hq": 32, "Hkv": 4, "d": 128, "page": 64, "layout": "hnd"},
        # long sequences with short drafts in 8 bits: reading the cache counts
        {"name": "tree_bf16_e4m3_long", "kind": "tree", "dtype": "bf16", "cache": "e4m3", "B": 32, "rows": 8, "len": 65536, "Hq": 32, "Hkv": 8, "d": 128, "page": 64, "layout": "hnd"},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "read", "commit", "tree", "tree", "tree"])
    c = {"kind": kind, "dtype": rng.choice(["f32", "f16", "bf16", "bf16"]), "cache": rng.choice(["native", "e4m3", "int8"]),
         "Hkv": rng.choice([1, 2, 4, 5, 8]), "d": rng.choice([64, 64, 128, 128, 96, 80, 40]),
         "page": rng.choice([16, 24, 32, 48, 64, 100, 128, 256]), "layout": rng.choice(["nhd", "hnd"])}
    if kind in ("append", "read"):
        c["B"] = _log_int(rng, 1, 64)
        most = 131072 * 8 // (c["Hkv"] * c["B"])
        if kind == "append":
            c["rows"], c["len"] = _log_int(rng, 1, most), rng.choice([0, rng.randint(1, 3000)])
        else:
            c["len"] = _log_int(rng, 17, most)
    elif kind == "commit":
        c["B"], c["rows"], c["len"] = _log_int(rng, 1, 128), _log_int(rng, 1, 64), _log_int(rng, 1, 4096)
        c["kept"] = rng.randint(1, max(1, c["rows"] // 2))
    else:
        g = rng.choice([1, 2, 3, 4, 7, 8])
        c["Hq"], c["B"], c["rows"] = g * c["Hkv"], _log_int(rng, 1, 48), _log_int(rng, 1, 64)
        slow = 8 if c["dtype"] == "f32" else 1
        most = min(32 * 65536 * 8 * 128 // (c["B"] * c["Hkv"] * c["d"]),
                   8 * 64 * 32 * 16384 * 128 // (slow * c["B"] * c["rows"] * c["Hq"] * c["d"]), 131072)
        c["len"] = _log_int(rng, 1, max(2, most))
    return c


def spread(case):
    """Lengths and rows of the sequences: the first has the case's, the others fall evenly to a quarter (half) of it."""
    B, n, r = case["B"], case["len"], case.get("rows", 0)
    return [n - (n * 3 // 4) * b // B for b in range(B)], [r - (r // 2) * b // B for b in range(B)]


def _lists(case):
    """(committed lengths, rows that the call handles, positions that the pages must hold) of every sequence."""
    lens, rows = spread(case)
    if case["kind"] == "read":
        return [0] * case["B"], lens, lens
    return lens, rows, [n + r for n, r in zip(lens, rows)]


def work(case):
    lens, rows, _ = _lists(case)
    Hkv, d, kind = case["Hkv"], case["d"], case["kind"]
    wide = BYTES[case["dtype"]]
    held = wide if case["cache"] == "native" else BYTES[case["cache"]]
    one_in, one_held = 2 * Hkv * d * wide, 2 * Hkv * (d * held + (0 if case["cache"] == "native" else 4))
    N = sum(rows)
    if kind == "append":
        return {"bytes": N * (2 * one_in + one_held), "flops": 4.0 * N * Hkv * d}
    if kind == "read":
        return {"bytes": N * (one_in + one_held), "flops": 2.0 * N * Hkv * d}
    if kind == "commit":
        kept = sum(min(case["kept"], r) for r in rows)
        return {"bytes": N * (one_in + one_held) + kept * (one_in + one_held), "flops": 4.0 * N * Hkv * d}
    Hq = case["Hq"]
    keys = sum(n + r for n, r in zip(lens, rows))
    pairs = sum(r * (n + 1) for n, r in zip(lens, rows))
    return {"bytes": keys * one_held + N * Hq * (2 * d * wide + 8), "flops": 4.0 * d * Hq * pairs}


# ---- inputs ------------------------------------------------------------------------------------------------------------

def _tree(T, gen):
    """Ancestors (and self) of T drafted tokens: the parent of token i is one of the tokens before it, or the last
    committed token."""
    par = (torch.rand(T, generator=gen) * (torch.arange(T) + 1)).long() - 1
    par = torch.maximum(par, torch.arange(T) // 3 - 1).tolist()
    seen = torch.eye(T, dtype=torch.bool)
    for i in range(T):
        if par[i] >= 0:
            seen[i] |= seen[par[i]]
    return seen


def _pages(shape, case, cache_type, gen):
    """Pages [n_pages, page, heads, d] that hold N(0, 1) values, and the scales of their rows, in the case's memory order."""
    n, page, H, d = shape
    lead = (n, H, page) if case["layout"] == "hnd" else (n, page, H)
    turn = (lambda t: t.transpose(1, 2)) if case["layout"] == "hnd" else (lambda t: t)
    out = torch.empty(*lead, d, dtype=cache_type, device="cuda")
    scale = None if case["cache"] == "native" else torch.empty(*lead, device="cuda")
    for a in range(0, n, 4096):  # pieces: the float32 values are larger than the pages
        x = torch.randn(out[a:a + 4096].shape, generator=gen, device="cuda")
        if scale is None:
            out[a:a + 4096] = x
        elif case["cache"] == "e4m3":  # rows as a cache holds them: near the top of the type's range, powers of two as scales
            out[a:a + 4096] = (x * 96).clamp(-448, 448).to(cache_type)
            scale[a:a + 4096] = 1.0 / 128
        else:
            out[a:a + 4096] = (x * 32).round().clamp(-127, 127).to(cache_type)
            scale[a:a + 4096] = torch.rand(scale[a:a + 4096].shape, generator=gen, device="cuda") * 0.02 + 0.02
    return turn(out), None if scale is None else turn(scale)


def prepare(case, seed):
    host = torch.Generator().manual_seed(int(seed))
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    lens, rows, ends = _lists(case)
    B, Hkv, d, page = case["B"], case["Hkv"], case["d"], case["page"]
    dtype = DTYPES[case["dtype"]]
    cache_type = {"native": dtype, "e4m3": torch.float8_e4m3fn, "int8": torch.int8}[case["cache"]]
    width = max(1, max(-(-e // page) for e in ends))
    n_pages = sum(-(-e // page) for e in ends) + 1
    table = torch.zeros(B, width, dtype=torch.int32)
    order, at = torch.randperm(n_pages, generator=host).to(torch.int32), 0
    for b, e in enumerate(ends):
        k = -(-e // page)
        table[b, :k] = order[at:at + k]
        at += k
    K_pages, K_scale = _pages((n_pages, page, Hkv, d), case, cache_type, gen)
    V_pages, V_scale = _pages((n_pages, page, Hkv, d), case, cache_type, gen)
    N = sum(rows)
    s = {"case": case, "K_pages": K_pages, "V_pages": V_pages, "K_scale": K_scale, "V_scale": V_scale,
         "table": table.cuda(), "lens": torch.tensor(lens, dtype=torch.int32).cuda(),
         "cu": torch.tensor([sum(rows[:b]) for b in range(B + 1)], dtype=torch.int32).cuda()}
    if case["kind"] in ("append", "commit"):
        s["K"] = torch.randn(N, Hkv, d, generator=gen, device="cuda").to(dtype)
        s["V"] = torch.randn(N, Hkv, d, generator=gen, device="cuda").to(dtype)
    if case["kind"] == "commit":
        most = case["kept"]
        kept, n_kept, begin = torch.zeros(B, most, dtype=torch.int32), [], [0]
        for b in range(B):
            k = min(most, rows[b])
            kept[b, :k] = torch.randperm(rows[b], generator=host)[:k].sort().values.to(torch.int32)
            n_kept.append(k)
            begin.append(begin[-1] + k)
        s["kept"], s["n_kept"] = kept.cuda(), torch.tensor(n_kept, dtype=torch.int32).cuda()
        s["cu_kept"], N = torch.tensor(begin, dtype=torch.int32).cuda(), begin[-1]
    if case["kind"] == "tree":
        Hq, T = case["Hq"], max(rows)
        s["Q"] = (torch.randn(N, Hq, d, generator=gen, device="cuda") * 2).to(dtype)
        mask, at = torch.zeros(N, T, dtype=torch.bool), 0
        for r in rows:
            mask[at:at + r, :r] = _tree(r, host)
            at += r
        s["mask"] = mask.cuda()
        s["m"], s["l"] = torch.empty(N, Hq, device="cuda"), torch.empty(N, Hq, device="cuda")
        s["O"] = torch.empty(N, Hq, d, dtype=dtype, device="cuda")
    else:
        s["K_out"] = torch.empty(N, Hkv, d, dtype=dtype, device="cuda")
        s["V_out"] = torch.empty(N, Hkv, d, dtype=dtype, device="cuda")
    return s


# ---- plain forms -------------------------------------------------------------------------------------------------------

def _bytes(t):
    return t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t


def _places(s, cu, n):
    """Sequence of each of n rows, and the page and slot of its position."""
    i = torch.arange(n, device="cuda", dtype=torch.int32)
    seq = torch.bucketize(i, cu[1:], right=True)
    pos = s["lens"][seq] + i - cu[seq]
    return s["table"][seq, pos // s["K_pages"].shape[1]].long(), pos % s["K_pages"].shape[1]


def _quantise(x, cache):
    top = x.abs().amax(-1)
    if cache == "e4m3":
        f, e = torch.frexp(top)
        e = torch.where(f <= 0.875, e - 9, e - 8)
        e = torch.where(top == 0, -126, e).clamp(min=-126)
        scale = ((e + 127) << 23).view(torch.float32)
        return (x / scale[..., None]).to(torch.float8_e4m3fn), scale
    seven_bits = torch.full_like(top, 127)  # as a tensor: a division by a number multiplies by its rounded reciprocal
    some = top >= 2.0 ** -100  # smaller rows count as zeros
    scale, inverse = torch.where(some, top / seven_bits, 0), torch.where(some, seven_bits / top, 0)
    return (x * inverse[..., None]).round().clamp(-127, 127).to(torch.int8), scale


def _plain_append(s):
    page, slot = _places(s, s["cu"], s["K"].shape[0])
    for x, pages, scales in ((s["K"], s["K_pages"], s["K_scale"]), (s["V"], s["V_pages"], s["V_scale"])):
        if scales is None:
            pages[page, slot] = x
        else:
            q, scale = _quantise(x.float(), s["case"]["cache"])
            _bytes(pages)[page, slot] = _bytes(q)
            scales[page, slot] = scale


def _values(pages, scales, page, slot):
    x = _bytes(pages)[page, slot]
    x = (x.view(pages.dtype) if x.dtype != pages.dtype else x).float()
    return x if scales is None else x * scales[page, slot][..., None]


def _plain_read(s, cu):
    page, slot = _places(s, cu, s["K_out"].shape[0])
    return (_values(s["K_pages"], s["K_scale"], page, slot).to(s["K_out"].dtype),
            _values(s["V_pages"], s["V_scale"], page, slot).to(s["V_out"].dtype))


def _plain_keep(s):
    page_size = s["K_pages"].shape[1]
    i = torch.arange(s["K_out"].shape[0], device="cuda", dtype=torch.int32)
    seq = torch.bucketize(i, s["cu_kept"][1:], right=True)
    i = i - s["cu_kept"][seq]
    src, dst = s["lens"][seq] + s["kept"][seq, i], s["lens"][seq] + i
    from_page, to_page = s["table"][seq, src // page_size].long(), s["table"][seq, dst // page_size].long()
    for t in (s["K_pages"], s["V_pages"], s["K_scale"], s["V_scale"]):
        if t is not None:
            t = _bytes(t)
            t[to_page, dst % page_size] = t[from_page, src % page_size]


def _plain_tree(s):
    Q, mask, lens, cu, table = s["Q"], s["mask"], s["lens"], s["cu"], s["table"]
    page_size, Hkv = s["K_pages"].shape[1:3]
    N, Hq, d = Q.shape
    B, T, S = lens.shape[0], mask.shape[1], table.shape[1] * page_size
    row = cu[:-1, None] + torch.arange(T, device="cuda", dtype=torch.int32)
    row = torch.minimum(row, cu[1:, None] - 1).long()  # short trees repeat their last row
    pos = torch.arange(S, device="cuda", dtype=torch.int32)
    page, slot = table[:, pos // page_size].long(), (pos % page_size).expand(B, S)
    j = pos[None] - lens[:, None]
    drafted = (j >= 0) & (j < (cu[1:] - cu[:-1])[:, None])
    at = j.clamp(0, T - 1).long()[:, None, :].expand(B, T, S)
    seen = (j < 0)[:, None] | (drafted[:, None] & mask[row].gather(2, at))
    g = Hq // Hkv
    q = Q.float()[row].view(B, T, Hkv, g, d).permute(0, 2, 3, 1, 4).reshape(B, Hkv, g * T, d)
    k = _values(s["K_pages"], s["K_scale"], page, slot).permute(0, 2, 3, 1)
    score = (q @ k).view(B, Hkv, g, T, S) / math.sqrt(d)
    del k
    score = score.masked_fill_(~seen[:, None, None], float("-inf"))
    m = score.amax(-1)
    p = score.sub_(m[..., None]).exp_()
    l = p.sum(-1)
    v = _values(s["V_pages"], s["V_scale"], page, slot).permute(0, 2, 1, 3)
    O = (p.view(B, Hkv, g * T, S) @ v).view(B, Hkv, g, T, d) / l[..., None]
    i = torch.arange(N, device="cuda", dtype=torch.int32)
    seq = torch.bucketize(i, cu[1:], right=True)
    t = (i - cu[seq]).long()
    take = lambda x: x.permute(0, 3, 1, 2, *range(4, x.dim()))[seq, t]  # noqa: E731
    return take(O).reshape(N, Hq, d).to(Q.dtype), take(m).reshape(N, Hq), take(l).reshape(N, Hq)


def run(s):
    kind = s["case"]["kind"]
    if own:
        scales = (s["K_scale"], s["V_scale"])
        if kind == "tree":
            module("spfa_tree").forward(s["Q"], s["K_pages"], s["V_pages"], s["table"], s["lens"], s["cu"], s["mask"],
                                        s["m"], s["l"], s["O"], *scales, first=True)
            return {"O": s["O"], "m": s["m"], "l": s["l"]}
        cache = module("spfa_cache")
        if kind != "read":
            cache.append(s["K"], s["V"], s["K_pages"], s["V_pages"], s["table"], s["lens"], s["cu"], *scales)
        if kind == "commit":
            cache.keep(s["K_pages"], s["V_pages"], s["table"], s["lens"], s["kept"], s["n_kept"], *scales)
        cache.read(s["K_pages"], s["V_pages"], s["table"], s["lens"], s["cu_kept"] if kind == "commit" else s["cu"],
                   s["K_out"], s["V_out"], *scales)
        return {"K": s["K_out"], "V": s["V_out"]}
    if kind == "tree":
        O, m, l = _plain_tree(s)
        return {"O": O, "m": m, "l": l}
    if kind != "read":
        _plain_append(s)
    if kind == "commit":
        _plain_keep(s)
    K, V = _plain_read(s, s["cu_kept"] if kind == "commit" else s["cu"])
    return {"K": K, "V": V}


# ---- 64 bits -----------------------------------------------------------------------------------------------------------

def _power(e):
    """2^e as float64, built from its bits: the library's power is not exact everywhere."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _stored(x, cache):
    """What the cache holds of rows x (float64), from the definition of its type."""
    if cache == "native":
        return x
    top = x.abs().amax(-1, keepdim=True)
    if cache == "int8":
        return torch.round(x * (127 / torch.where(top > 0, top, 1))) * (top / 127).float().double()
    e = torch.floor(torch.log2(torch.where(top > 0, top, 1) / 448)) - 1
    e = (e + (top > 448 * _power(e)) + (top > 448 * _power(e + 1)) + (top > 448 * _power(e + 2))).clamp(min=-126)
    y = x / _power(e)
    step = _power(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)  # 3 bits behind the leading one, 2^-9 at the least
    return torch.round(y / step) * step * _power(e)


def exact(case, seed):
    s = prepare(case, seed)
    lens, rows, _ = _lists(case)
    page, kind, cache = case["page"], case["kind"], case["cache"]

    def sequence(pages, scales, b, lo, hi):
        """Positions [lo, hi) of sequence b as float64."""
        p = torch.arange(lo, hi, device="cuda")
        where = (s["table"][b].long()[p // page], p % page)
        raw = pages.view(torch.uint8)[where].view(pages.dtype) if pages.dtype == torch.float8_e4m3fn else pages[where]
        return raw.double() if scales is None else raw.double() * scales[where].double()[..., None]

    if kind in ("append", "commit"):
        out = {}
        for name in ("K", "V"):
            x = _stored(s[name].double(), cache)
            if kind == "commit":
                at, parts = 0, []
                for b, r in enumerate(rows):
                    parts.append(x[at:at + r][s["kept"][b, :min(case["kept"], r)].long()])
                    at += r
                x = torch.cat(parts)
            out[name] = x
        return out
    if kind == "read":
        return {name: torch.cat([sequence(s[name + "_pages"], s[name + "_scale"], b, 0, n) for b, n in enumerate(rows)])
                for name in ("K", "V")}
    Hq, Hkv, d = case["Hq"], case["Hkv"], case["d"]
    g, at, O, m, l = Hq // Hkv, 0, [], [], []
    for b, (n, r) in enumerate(zip(lens, rows)):
        k, v = (sequence(s[x + "_pages"], s[x + "_scale"], b, 0, n + r).transpose(0, 1) for x in ("K", "V"))
        q = s["Q"][at:at + r].double().transpose(0, 1)  # [Hq, r, d]
        hidden = torch.zeros(r, n + r, dtype=torch.bool, device="cuda")
        hidden[:, n:] = ~s["mask"][at:at + r, :r]
        for h in range(Hq):
            a = (q[h] @ k[h // g].T / math.sqrt(d)).masked_fill(hidden, -math.inf)
            top = a.amax(-1, keepdim=True)
            a = torch.exp(a - top)
            m.append(top[:, 0])
            l.append(a.sum(-1))
            O.append(a @ v[h // g] / l[-1][:, None])
        for x in (O, m, l):  # the heads of this sequence as [r, Hq, ...]
            x[-Hq:] = [torch.stack(x[-Hq:], 1)]
        at += r
    return {"O": torch.cat(O), "m": torch.cat(m), "l": torch.cat(l)}
