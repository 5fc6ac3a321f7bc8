"""Measured cases of the 8-bit K/V cache operators: one call a pass, in the plain form (elementary torch operations in
32 bits) or through the package's own entry points.

The cache of one layer is a pool of pages.  A page holds page_size consecutive tokens of one request for every KV
head, K and V in 8 bits (int8 or float8 e4m3) with one float32 scale per page, KV head and tensor.  A request is a row
of the page table and a length.  Four operators work on it:

  append   quantise new rows (a prompt, or the accepted path of a verified tree) into each request's pages
  attend   attention of n query nodes over the cached tokens and the n nodes' own bf16 keys under an ancestor mask
           (n = 1: an ordinary decode step), with the log-sum-exp of every row
  weigh    the attention weight each page received from the accepted nodes, added to the running mass of the pages
  evict    drop the pages of least mass from every request that is over its budget of pages
"""

import math
import random

import torch

own = False

DEV = "cuda"
QMAX = {"int8": 127.0, "e4m3": 448.0}
FLOOR = 2.0 ** -100  # the least scale of a page, so that an all-zero page divides by something


# ------------------------------------------------------------------------------------------------------- the cases

def listed():
    return [
        # a chat's decode step at batch 1: nothing but latency
        {"name": "attend 1x1 ctx 1000", "op": "attend", "bs": 1, "n": 1, "heads": 32, "kv_heads": 8, "page": 64,
         "dtype": "int8", "lo": 1000, "hi": 1000},
        # decode of a full serving batch, lengths as they come
        {"name": "attend 64x1 ctx 1K-8K", "op": "attend", "bs": 64, "n": 1, "heads": 32, "kv_heads": 8, "page": 64,
         "dtype": "e4m3", "lo": 1024, "hi": 8192},
        # one long document
        {"name": "attend 1x1 ctx 128K", "op": "attend", "bs": 1, "n": 1, "heads": 32, "kv_heads": 8, "page": 128,
         "dtype": "int8", "lo": 131072, "hi": 131072},
        # the verify step of one 64-node tree and its root behind a 4096-token prefix
        {"name": "attend 1x65 ctx 4096", "op": "attend", "bs": 1, "n": 65, "heads": 32, "kv_heads": 8, "page": 64,
         "dtype": "int8", "lo": 4096, "hi": 4096},
        # the verify step of a serving batch
        {"name": "attend 32x65 ctx 1K-8K", "op": "attend", "bs": 32, "n": 65, "heads": 32, "kv_heads": 8, "page": 32,
         "dtype": "e4m3", "lo": 1024, "hi": 8192},
        # short drafts over short ragged contexts, seven query heads to a KV head, the smallest page
        {"name": "attend 9x5 ctx 1-2001", "op": "attend", "bs": 9, "n": 5, "heads": 28, "kv_heads": 4, "page": 16,
         "dtype": "int8", "lo": 1, "hi": 2001},
        # the commit of a serving batch's accepted paths
        {"name": "append 32 paths", "op": "append", "bs": 32, "n": 65, "rows": 17, "path": True, "kv_heads": 8,
         "page": 64, "dtype": "int8", "lo": 1024, "hi": 8192},
        # two prompts
        {"name": "append 2 prompts", "op": "append", "bs": 2, "n": 8192, "rows": 8192, "path": False, "kv_heads": 8,
         "page": 128, "dtype": "e4m3", "lo": 0, "hi": 100},
        # page weights of one request's accepted path
        {"name": "weigh 1 ctx 4096", "op": "weigh", "bs": 1, "n": 65, "rows": 17, "heads": 32, "kv_heads": 8,
         "page": 64, "dtype": "int8", "lo": 4096, "hi": 4096},
        # and of a serving batch
        {"name": "weigh 32 ctx 1K-8K", "op": "weigh", "bs": 32, "n": 65, "rows": 17, "heads": 32, "kv_heads": 8,
         "page": 32, "dtype": "e4m3", "lo": 1024, "hi": 8192},
        # one long document over its budget
        {"name": "evict 1x1024", "op": "evict", "bs": 1, "pages": 1024, "keep": 768, "sink": 4, "recent": 16,
         "page": 64},
        # a large batch of long requests, most over their budget
        {"name": "evict 128x4095", "op": "evict", "bs": 128, "pages": 4095, "keep": 2048, "sink": 4, "recent": 32,
         "page": 16},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))


def draw(rng):
    most = {k: max(work(c)[k] for c in listed()) for k in ("bytes", "flops")}
    while True:
        op = rng.choice(["attend", "attend", "attend", "append", "weigh", "evict"])
        page = rng.choice([16, 32, 64, 128])
        if op == "evict":
            pages = _log(rng, 8, 4095)
            sink, recent = rng.randint(0, 4), rng.randint(1, 32)
            case = {"op": op, "bs": _log(rng, 1, 128), "pages": pages, "sink": sink, "recent": recent,
                    "keep": max(sink + recent, int(pages * rng.uniform(0.3, 1.1))), "page": page}
        else:
            heads, kv = rng.choice([(32, 8), (32, 8), (16, 16), (28, 4), (40, 8), (16, 2), (64, 4), (12, 4)])
            hi = _log(rng, 16, 131072)
            case = {"op": op, "bs": _log(rng, 1, 64), "kv_heads": kv, "page": page,
                    "dtype": rng.choice(["int8", "e4m3"]), "lo": max(0, int(hi * rng.choice([0.0, 0.125, 0.5, 1.0]))),
                    "hi": hi}
            if op == "attend":
                case.update(n=rng.choice([1, 1, _log(rng, 2, 129)]), heads=heads)
            elif op == "weigh":
                rows = _log(rng, 1, 17)
                case.update(n=rng.randint(rows, 129), rows=rows, heads=heads)
            else:
                path = rng.random() < 0.5
                rows = _log(rng, 1, 17) if path else _log(rng, 1, 8192)
                case.update(n=rng.randint(rows, 129) if path else rows, rows=rows, path=path)
        w = work(case)
        if w["bytes"] <= most["bytes"] and w["flops"] <= most["flops"]:
            return case


def _spread(case, lo, hi, what):
    """One length per request, spread over [lo, hi]; the same for every seed, so that a case's work is its own."""
    rng = random.Random("%s %d %d %d" % (what, case["bs"], lo, hi))
    return [hi if b == 0 else rng.randint(lo, hi) for b in range(case["bs"])]


def _lens(case):
    if case["op"] == "evict":
        return [max(0, case["page"] * p - b % case["page"])
                for b, p in enumerate(_spread(case, case["pages"] // 2, case["pages"], "pages"))]
    return _spread(case, case["lo"], case["hi"], "lens")


def _counts(case):
    return _spread(case, 1 if case.get("path", True) else case["rows"] // 2, case["rows"], "rows")


def work(case):
    bs, lens = case["bs"], _lens(case)
    if case["op"] == "evict":  # table and mass in and out, the freed pages and the lengths out
        n = sum((t + case["page"] - 1) // case["page"] for t in lens)
        return {"bytes": 16 * n + 12 * bs, "flops": n}
    kv, page, d = case["kv_heads"], case["page"], 128
    pages = sum((t + page - 1) // page for t in lens)
    if case["op"] == "append":  # new rows in (bf16) and out (8 bits), the open page's rows in and out, scales
        rows = _counts(case)
        old = sum(t % page for t in lens)
        touched = sum((t % page + r + page - 1) // page for t, r in zip(lens, rows))
        return {"bytes": 2 * kv * d * (3 * sum(rows) + 2 * old) + 8 * kv * touched, "flops": 4 * kv * d * sum(rows)}
    table = 4 * pages
    if case["op"] == "weigh":  # K once, the accepted nodes' queries and log-sum-exps, the masses in and out
        rows = _counts(case)
        return {"bytes": kv * (d * sum(lens) + 4 * pages) + table + case["heads"] * (2 * d + 4) * sum(rows) + 8 * pages,
                "flops": 2 * d * case["heads"] * sum(r * t for r, t in zip(rows, lens))}
    n, heads = case["n"], case["heads"]
    words = (n + 63) // 64
    io = bs * n * (heads * (4 * d + 4) + kv * 4 * d + 8 * words)
    return {"bytes": 2 * kv * (d * sum(lens) + 4 * pages) + table + io,
            "flops": 4 * d * heads * (n * sum(lens) + bs * n * (n + 1) // 2)}


# ------------------------------------------------------------------------------------------------------ the inputs

def _codes(gen, shape, dtype):
    x = torch.empty(shape, dtype=torch.float16, device=DEV)
    q = QMAX[dtype]
    for part in x.view(-1).split(1 << 27):  # a page's values: bell-shaped, its largest near the type's largest code
        part.normal_(0, q / 3.5, generator=gen).clamp_(-q, q)
    return x.round_().to(torch.int8) if dtype == "int8" else x.to(torch.float8_e4m3fn)


def _scales(gen, shape, dtype):
    return torch.exp(0.25 * torch.randn(shape, generator=gen, device=DEV)) * (3.5 / QMAX[dtype])


def _randn(gen, *shape, std=1.0):
    return (torch.randn(shape, generator=gen, device=DEV) * std).to(torch.bfloat16)


def _table(rng, lens, page, spare):
    """A page table with room for `spare` more tokens a request, its pages scattered over the pool; unused entries -1.
    The pool's last page belongs to nobody."""
    need = [(t + s + page - 1) // page for t, s in zip(lens, spare)]
    ids = list(range(sum(need)))
    rng.shuffle(ids)
    width = max(1, max(need))
    rows, at = [], 0
    for n in need:
        rows.append(ids[at:at + n] + [-1] * (width - n))
        at += n
    return torch.tensor(rows, dtype=torch.int32, device=DEV), len(ids) + 1


def _trees(rng, bs, n):
    """Ancestor-or-self bitsets of random trees (int64 words), as the tree builder gives them."""
    words = (n + 63) // 64
    out = []
    for _ in range(bs):
        sets = [1]
        for i in range(1, n):
            sets.append(sets[rng.randint(max(0, i - 9), i - 1)] | (1 << i))
        out.append([[((s >> (64 * w)) & (2 ** 64 - 1)) - ((s >> (64 * w + 63)) & 1) * 2 ** 64 for w in range(words)]
                    for s in sets])
    return torch.tensor(out, dtype=torch.int64, device=DEV)


def _paths(rng, bs, n, rows, counts):
    """Accepted node ids in order, node 0 first, then -1."""
    return torch.tensor([[0] + sorted(rng.sample(range(1, n), c - 1)) + [-1] * (rows - c) for c in counts],
                        dtype=torch.int64, device=DEV)


def prepare(case, seed):
    rng = random.Random(seed)
    gen = torch.Generator(device=DEV).manual_seed(seed)
    lens = _lens(case)
    s = dict(case)
    s["seq_lens"] = torch.tensor(lens, dtype=torch.int32, device=DEV)
    if case["op"] == "evict":
        s["table"], _ = _table(rng, lens, case["page"], [0] * case["bs"])
        # attention mass: few pages carry most of it, and many have never been looked at
        mass = torch.empty(s["table"].shape, device=DEV).exponential_(generator=gen).pow_(3)
        s["mass"] = torch.where(mass < 0.01, torch.zeros_like(mass), mass) * (s["table"] >= 0)
        return s
    bs, n, kv, page = case["bs"], case["n"], case["kv_heads"], case["page"]
    counts = _counts(case) if case["op"] != "attend" else [0] * bs
    s["table"], pool = _table(rng, lens, page, counts if case["op"] == "append" else [0] * bs)
    s["k"] = _codes(gen, (pool, kv, page, 128), case["dtype"])
    s["k_scale"] = _scales(gen, (pool, kv), case["dtype"])
    s["v"] = _codes(gen, (pool, kv, page, 128), case["dtype"])
    s["v_scale"] = _scales(gen, (pool, kv), case["dtype"])
    s["scale"] = 128 ** -0.5
    if case["op"] == "append":
        s["k_new"], s["v_new"] = _randn(gen, bs, n, kv, 128), _randn(gen, bs, n, kv, 128)
        s["counts"] = torch.tensor(counts, dtype=torch.int32, device=DEV)
        s["path"] = _paths(rng, bs, n, case["rows"], counts) if case["path"] else None
        return s
    s["q"] = _randn(gen, bs, n, case["heads"], 128, std=2.0)
    if case["op"] == "attend":
        s["k_new"], s["v_new"] = _randn(gen, bs, n, kv, 128), _randn(gen, bs, n, kv, 128)
        s["anc"] = _trees(rng, bs, n)
        return s
    s["counts"] = torch.tensor(counts, dtype=torch.int32, device=DEV)
    s["path"] = _paths(rng, bs, n, case["rows"], counts)
    s["mass"] = torch.empty(s["table"].shape, device=DEV).exponential_(generator=gen)
    s["decay"] = 0.99
    # the attention's log-sum-exps: those of the cached tokens, and a share that the nodes' own keys took
    lse = torch.rand((bs, n, case["heads"]), generator=gen, device=DEV) * 0.5 + 8
    for b in range(bs):
        if lens[b]:
            at = s["path"][b, :counts[b]]
            one = {**s, "q": s["q"][b:b + 1, at], "table": s["table"][b:b + 1], "seq_lens": s["seq_lens"][b:b + 1]}
            top = torch.logsumexp(_scores(one), -1)
            lse[b, at] = top.view(kv, counts[b], -1).transpose(0, 1).reshape(counts[b], -1) + \
                torch.rand((counts[b], case["heads"]), generator=gen, device=DEV) * 0.5
    s["lse"] = lse
    return s


# --------------------------------------------------------------------------------------------------- the plain form

def _rows(codes, scale, table):
    """Cached rows of every request in order, in 32 bits: [bs, kv, pages * page, 128]."""
    ids = table.long().clamp_min(0)
    x = codes.view(torch.uint8)[ids].view(codes.dtype).float() * scale[ids][..., None, None]
    bs, pages, kv, page, d = x.shape
    return x.transpose(1, 2).reshape(bs, kv, pages * page, d)


def _scores(s):
    """Scores of the queries s["q"] over the cached tokens: [bs, kv, nodes * group, tokens], -inf past the length."""
    q = s["q"].float()
    bs, n, h, d = q.shape
    kv = s["k"].shape[1]
    q = q.view(bs, n, kv, h // kv, d).transpose(1, 2).reshape(bs, kv, n * (h // kv), d)
    sc = (q @ _rows(s["k"], s["k_scale"], s["table"]).transpose(2, 3)) * s["scale"]
    at = torch.arange(sc.shape[-1], device=sc.device)
    return torch.where(at < s["seq_lens"][:, None, None, None], sc, torch.full_like(sc, -math.inf))


def _plain_attend(s):
    q = s["q"].float()
    bs, n, h, d = q.shape
    kv = s["k"].shape[1]
    g = h // kv
    old = _scores(s)
    qn = q.view(bs, n, kv, g, d).permute(0, 2, 1, 3, 4)
    new = torch.einsum("bkigd,bjkd->bkigj", qn, s["k_new"].float()) * s["scale"]
    at = torch.arange(n, device=q.device)
    seen = (s["anc"][:, :, at // 64] >> (at % 64)) & 1
    new = torch.where(seen[:, None, :, None, :] != 0, new, torch.full_like(new, -math.inf)).reshape(bs, kv, n * g, n)
    sc = torch.cat([old, new], -1)
    top = sc.amax(-1, keepdim=True)
    p = torch.exp(sc - top)
    total = p.sum(-1, keepdim=True)
    v = torch.cat([_rows(s["v"], s["v_scale"], s["table"]), s["v_new"].float().transpose(1, 2)], 2)
    out = (p @ v) / total
    lse = (torch.log(total) + top).squeeze(-1)

    def back(x):
        return x.view(bs, kv, n, g, -1).transpose(1, 2).reshape(bs, n, h, -1)

    return {"out": back(out).to(torch.bfloat16), "lse": back(lse).squeeze(-1).contiguous()}


def _plain_quantise(x, fresh, open_scale, keep, qmax, dtype):
    """x: the new rows' values in the touched pages; keep: the rows already there, in their page's old scale."""
    finite = torch.where(torch.isfinite(x), x.abs(), torch.zeros_like(x)) * fresh
    scale = torch.maximum(finite.amax((2, 4)) / qmax, open_scale).clamp_min(FLOOR)
    x = torch.nan_to_num(torch.where(fresh, x, keep) / scale[:, :, None, :, None], nan=0.0, posinf=qmax, neginf=-qmax)
    x = x.clamp(-qmax, qmax)
    return scale, (x.round().to(torch.int8) if dtype == torch.int8 else x.to(dtype))


def _plain_append(s):
    bs, n, kv, d = s["k_new"].shape
    page, pool = s["k"].shape[2], s["k"].shape[0]
    lens, counts = s["seq_lens"].long(), s["counts"].long()
    rows = s["rows"]
    touched = (rows + page - 1) // page + 1
    first = lens // page
    slot = torch.arange(touched, device=DEV)[:, None] * page + torch.arange(page, device=DEV)  # [touched, page]
    row = slot[None] - (lens % page)[:, None, None]  # the new row that goes there, if any
    fresh = (row >= 0) & (row < counts[:, None, None])
    row = row.clamp(0, rows - 1)
    node = row if s["path"] is None else s["path"].gather(1, row.view(bs, -1)).view_as(row).clamp_min(0)
    at = first[:, None] + torch.arange(touched, device=DEV)
    ids = s["table"].long().gather(1, at.clamp_max(s["table"].shape[1] - 1))
    used = fresh.any(2)
    ids = torch.where(used, ids, torch.full_like(ids, pool - 1))  # pages without a new row: the page of nobody
    kept = (at == first[:, None]) & (lens % page > 0)[:, None]  # the open page, with rows already in it
    old = slot[None] < (lens % page)[:, None, None]
    b = torch.arange(bs, device=DEV)[:, None, None]
    out = {}
    for name in ("k", "v"):
        codes, scales = s[name], s[name + "_scale"]
        was = codes.view(torch.uint8)[ids].view(codes.dtype)
        x = s[name + "_new"][b, node].float()  # [bs, touched, page, kv, d]
        keep = was.float().transpose(2, 3) * scales[ids][:, :, None, :, None]
        open_scale = scales[ids] * kept[:, :, None]
        scale, new = _plain_quantise(x, fresh[..., None, None], open_scale, keep, QMAX[s["dtype"]], codes.dtype)
        write = (fresh | (old & kept[:, :, None]))[..., None, None]
        new = torch.where(write, new.view(torch.uint8), was.transpose(2, 3).view(torch.uint8)).transpose(2, 3)
        new = torch.where(used[:, :, None, None, None], new, was.view(torch.uint8))
        codes.view(torch.uint8)[ids] = new
        scales[ids] = torch.where(used[:, :, None], scale, scales[ids])
        out[name], out[name + "_scale"] = codes, scales
    out["seq_lens"] = (lens + counts).to(torch.int32)
    return out


def _plain_weigh(s):
    bs, rows = s["path"].shape
    b = torch.arange(bs, device=DEV)[:, None]
    at = s["path"].clamp_min(0)
    kv, page, pages = s["k"].shape[1], s["k"].shape[2], s["table"].shape[1]
    lse = s["lse"][b, at]
    h = lse.shape[-1]
    lse = lse.view(bs, rows, kv, h // kv).transpose(1, 2).reshape(bs, kv, -1, 1)
    w = torch.exp(_scores({**s, "q": s["q"][b, at]}) - lse)
    live = (torch.arange(rows, device=DEV) < s["counts"][:, None]).repeat_interleave(h // kv, 1)
    w = torch.where(live[:, None, :, None], w, torch.zeros_like(w)).sum((1, 2)).view(bs, pages, page).sum(2)
    inside = torch.arange(pages, device=DEV) * page < s["seq_lens"][:, None]
    return torch.where(inside, s["mass"] * s["decay"] + w, torch.zeros_like(w))


def _plain_evict(s):
    table, mass, page, keep = s["table"], s["mass"], s["page"], s["keep"]
    bs, width = table.shape
    pages = (s["seq_lens"].long() + page - 1) // page
    at = torch.arange(width, device=DEV)[None]
    inside = at < pages[:, None]
    fixed = inside & ((at < s["sink"]) | (at >= pages[:, None] - s["recent"]))
    key = torch.where(inside & ~fixed, mass, torch.full_like(mass, -math.inf))
    order = torch.sort(key, dim=1, descending=True, stable=True).indices
    rank = torch.empty_like(order).scatter_(1, order, at.expand(bs, width).contiguous())
    stay = fixed | (inside & ~fixed & (rank < keep - s["sink"] - s["recent"]))
    stay = torch.where((pages <= keep)[:, None], inside, stay)
    gone = inside & ~stay

    def packed(values, mask, fill):
        to = torch.where(mask, mask.cumsum(1) - 1, torch.full_like(at, width).expand(bs, width))
        out = torch.full((bs, width + 1), fill, dtype=values.dtype, device=DEV).scatter_(1, to, values)
        return out[:, :width].contiguous()

    freed = gone.sum(1)
    return {"table": packed(table, stay, -1), "mass": packed(mass, stay, 0.0),
            "seq_lens": (s["seq_lens"] - freed * page).to(torch.int32), "freed": packed(table, gone, -1),
            "freed_counts": freed.to(torch.int32)}


# ------------------------------------------------------------------------------------------------------- one pass

def run(state):
    s = state
    op = s["op"]
    if not own:
        return {"attend": _plain_attend, "append": _plain_append, "weigh": _plain_weigh, "evict": _plain_evict}[op](s)
    from mfd_b200 import ops
    if op == "attend":
        out, lse = ops.kv8_attention(s["q"], s["k"], s["v"], s["k_scale"], s["v_scale"], s["table"], s["seq_lens"],
                                     s["scale"], k_new=s["k_new"], v_new=s["v_new"], anc=s["anc"], return_lse=True)
        return {"out": out, "lse": lse}
    if op == "append":
        lens = ops.kv8_append(s["k"], s["v"], s["k_scale"], s["v_scale"], s["k_new"], s["v_new"], s["table"],
                              s["seq_lens"], path=s["path"], counts=s["counts"])
        return {"k": s["k"], "k_scale": s["k_scale"], "v": s["v"], "v_scale": s["v_scale"], "seq_lens": lens}
    if op == "weigh":
        return ops.kv8_page_weights(s["q"], s["lse"], s["k"], s["k_scale"], s["table"], s["seq_lens"], s["scale"],
                                    s["mass"], path=s["path"], counts=s["counts"], decay=s["decay"])
    table, mass, lens, freed, counts = ops.kv8_evict(s["table"], s["mass"], s["seq_lens"], s["page"], s["keep"],
                                                     s["sink"], s["recent"])
    return {"table": table, "mass": mass, "seq_lens": lens, "freed": freed, "freed_counts": counts}


# ------------------------------------------------------------------------------------------------ in 64 bits, apart

def _request(s, b, name):
    """Request b's cached rows in 64 bits: [kv, tokens, 128]."""
    t = int(s["seq_lens"][b])
    page = s[name].shape[2]
    ids = s["table"][b, :(t + page - 1) // page].long()
    x = s[name].view(torch.uint8)[ids].view(s[name].dtype).double() * s[name + "_scale"][ids].double()[:, :, None, None]
    return x.permute(1, 0, 2, 3).flatten(1, 2)[:, :t]


def _exact_attend(s):
    bs, n, h, d = s["q"].shape
    kv = s["k"].shape[1]
    g = h // kv
    out = torch.zeros(bs, n, h, d, dtype=torch.float64, device=DEV)
    lse = torch.zeros(bs, n, h, dtype=torch.float64, device=DEV)
    for b in range(bs):
        keys = torch.cat([_request(s, b, "k"), s["k_new"][b].double().transpose(0, 1)], 1)
        values = torch.cat([_request(s, b, "v"), s["v_new"][b].double().transpose(0, 1)], 1)
        t = int(s["seq_lens"][b])
        hide = torch.stack([((s["anc"][b, :, j // 64] >> (j % 64)) & 1) == 0 for j in range(n)], 1)
        for c in range(h):
            sc = s["q"][b, :, c].double() @ keys[c // g].T * s["scale"]
            sc[:, t:][hide] = -math.inf
            lse[b, :, c] = torch.logsumexp(sc, 1)
            out[b, :, c] = torch.exp(sc - lse[b, :, c, None]) @ values[c // g]
    return {"out": out, "lse": lse}


def _e4m3(x):
    """The nearest value with a 3-bit fraction and exponents from 2^-6 (ties to even), at most 448 in size."""
    e = torch.floor(torch.log2(x.abs().clamp_min(2.0 ** -6)))
    step = torch.exp2(e - 3)
    return (torch.round(x / step) * step).clamp(-448, 448)


def _exact_append(s):
    page, dtype = s["page"], s["dtype"]
    out = {}
    for name in ("k", "v"):
        codes, scales = s[name].double(), s[name + "_scale"].double()
        for b in range(s["bs"]):
            t, c = int(s["seq_lens"][b]), int(s["counts"][b])
            at = s["path"][b, :c] if s["path"] is not None else slice(0, c)
            new = s[name + "_new"][b, at].double()  # [c, kv, 128]
            i = 0
            while i < c:
                slot = (t + i) % page
                m = min(page - slot, c - i)
                p = int(s["table"][b, (t + i) // page])
                x = new[i:i + m].transpose(0, 1)  # [kv, m, 128]
                scale = x.abs().amax((1, 2)) / QMAX[dtype]
                rows = x
                if slot:
                    scale = torch.maximum(scale, scales[p])
                    rows = torch.cat([codes[p, :, :slot] * scales[p][:, None, None], x], 1)
                rows = rows / scale[:, None, None]
                codes[p, :, :slot + m] = torch.round(rows) if dtype == "int8" else _e4m3(rows)
                scales[p] = scale
                i += m
        out[name], out[name + "_scale"] = codes, scales
    out["seq_lens"] = None
    return out


def _exact_weigh(s):
    bs, h, page = s["bs"], s["q"].shape[2], s["page"]
    g = h // s["k"].shape[1]
    out = torch.zeros_like(s["mass"], dtype=torch.float64)
    for b in range(bs):
        t = int(s["seq_lens"][b])
        pages = (t + page - 1) // page
        at = s["path"][b, :int(s["counts"][b])]
        keys = _request(s, b, "k")
        w = torch.zeros(pages * page, dtype=torch.float64, device=DEV)
        for c in range(h):
            sc = s["q"][b, at, c].double() @ keys[c // g].T * s["scale"]
            w[:t] += torch.exp(sc - s["lse"][b, at, c, None].double()).sum(0)
        out[b, :pages] = s["mass"][b, :pages].double() * s["decay"] + w.view(pages, page).sum(1)
    return out


def exact(case, seed):
    if case["op"] == "evict":
        return None  # it moves its inputs, and computes no number
    s = prepare(case, seed)
    return {"attend": _exact_attend, "append": _exact_append, "weigh": _exact_weigh}[case["op"]](s)
