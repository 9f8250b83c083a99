"""Timed cases of the operators for prompts that are answered several times.

* ``prompt``: causal attention over whole prompts that lie behind one another, without a cache;
* ``copy``: pages of a K/V cache, or the first tokens of pages, copied in every layer;
* ``fork``: rows of a page table that continue other rows' sequences: whole pages shared, the last part page copied;
* ``count``: how many rows hold each page, and the pages that nobody holds;
* ``compact``: the pages in use moved to the front of the pool, and the page table renamed.

Head layouts and depths are those of the models that this repository's benchmark runs (16 / 8, 32 / 8 and 32 / 4 heads of 128, 28
layers) and generic ones.
"""
from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False   # False: the plain form; True: the framework's operators


def _prompt(name, heads, kv_heads, dim, count, lo, hi):
    """count sequences of lo to hi tokens."""
    return {"name": name, "kind": "prompt", "heads": heads, "kv_heads": kv_heads, "dim": dim, "count": count, "lo": lo, "hi": hi}


def _pages(name, kind, page, layers, kv_heads, dim, pages, **more):
    """A pool of `pages` pages of `page` tokens."""
    return {"name": name, "kind": kind, "page": page, "layers": layers, "kv_heads": kv_heads, "dim": dim, "pages": pages, **more}


LISTED = [
    # one short question: latency is all there is
    _prompt("prompt_short", 16, 8, 128, 1, 41, 41),
    # a scoring batch of texts of very different lengths, single tokens among them
    _prompt("prompt_batch", 32, 8, 128, 64, 1, 700),
    # documents for an embedding model of small heads
    _prompt("prompt_small_heads", 24, 8, 64, 7, 333, 2100),
    # two long documents
    _prompt("prompt_long", 32, 8, 128, 2, 7900, 8192),
    # the part pages of four samples
    _pages("copy_few", "copy", 16, 28, 8, 128, 40, pairs=4, whole=False),
    # many requests' pages moved aside: whole pages, all layers
    _pages("copy_many", "copy", 16, 28, 8, 128, 1500, pairs=700, whole=True),
    # four samples of one prompt
    _pages("fork_samples", "fork", 16, 28, 8, 128, 60, parents=1, children=4, lo=300, hi=310),
    # beams of several long prompts, large pages
    _pages("fork_beams", "fork", 64, 16, 8, 128, 560, parents=6, children=96, lo=3500, hi=4600),
    # the end of some answers of a batch that shares prompts: which pages are free?
    _pages("count_batch", "count", 16, 1, 1, 8, 9000, rows=64, lo=100, hi=2000, shared=0.5),
    # the same for a large pool of pages of one token
    _pages("count_large", "count", 1, 1, 1, 8, 1 << 20, rows=256, lo=200, hi=12000, shared=0.6),
    # a few short requests left in a small pool
    _pages("compact_few", "compact", 16, 28, 8, 128, 64, rows=6, lo=30, hi=150, shared=0.0),
    # half of a pool's requests have ended
    _pages("compact_half", "compact", 16, 28, 8, 128, 1600, rows=40, lo=100, hi=800, shared=0.2),
]


def listed():
    return [dict(case) for case in LISTED]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _cheap(case, like):
    cost, most = work(case), work(like)
    return cost["bytes"] <= most["bytes"] and cost["flops"] <= most["flops"]


def draw(rng):
    kind = rng.choice(["prompt", "prompt", "copy", "fork", "count", "compact"])
    while True:
        if kind == "prompt":
            heads, kv_heads = rng.choice([(16, 8), (32, 8), (32, 4), (16, 2), (8, 1), (24, 8), (12, 12), (14, 2)])
            hi = _log(rng, 1, 8192)
            case = _prompt("", heads, kv_heads, rng.choice([128, 128, 64, 80, 96]), _log(rng, 1, 128), max(1, hi // rng.choice([1, 3, 50])), hi)
            if case["count"] * hi <= 40000 and _cheap(case, LISTED[3]):
                break
            continue
        page, layers = rng.choice([1, 4, 16, 64]), _log(rng, 1, 32)
        kv_heads, dim = rng.choice([(8, 128), (4, 128), (2, 64), (1, 128)])
        token = 4 * layers * kv_heads * dim
        room = int(2.7e9 / (token * page))                # pages of a pool of that many bytes
        if kind == "copy":
            pages = min(room, 200000)
            pairs = _log(rng, 1, max(1, pages // 2 - 1)) if pages > 3 else 0
            case = _pages("", kind, page, layers, kv_heads, dim, pages, pairs=pairs, whole=rng.random() < 0.5)
            if pairs >= 1 and _cheap(case, LISTED[5]):
                break
        elif kind == "fork":
            parents, hi = _log(rng, 1, 12), _log(rng, 2, 8000)
            children = parents + _log(rng, 1, 120)
            need = parents * -(-hi // page) + children + 1
            case = _pages("", kind, page, layers, kv_heads, dim, need, parents=parents, children=children, lo=max(1, hi // 2), hi=hi)
            if need <= room and _cheap(case, LISTED[5]):
                break
        elif kind == "count":
            pages, rows, hi = _log(rng, 200, 1 << 20), _log(rng, 1, 300), _log(rng, 2, 14000)
            case = _pages("", kind, page, 1, 1, 8, pages, rows=rows, lo=max(1, hi // 20), hi=hi, shared=round(rng.uniform(0, 0.8), 2))
            if rows * -(-hi // page) <= pages and pages * page <= 1 << 24 and rows * hi <= 1 << 22:
                break
        else:
            rows, hi = _log(rng, 1, 100), _log(rng, 2, 4000)
            held = rows * -(-hi // page)
            pages = max(2, int(held * rng.uniform(1.05, 2.5)))
            case = _pages("", kind, page, layers, kv_heads, dim, pages, rows=rows, lo=max(1, hi // 8), hi=hi, shared=round(rng.uniform(0, 0.5), 2))
            if pages <= room and held <= pages and _cheap(case, LISTED[11]):
                break
    del case["name"]
    return case


# ---- sizes that belong to a case: the same for every seed ------------------------------------------------------

def _lengths(case, count):
    rng = random.Random(count * 1000003 + case["lo"] * 1009 + case["hi"])
    return [rng.randint(case["lo"], case["hi"]) for _ in range(count)]


def _token_bytes(case):
    """Of one token's keys and values in every layer."""
    return 4 * case["layers"] * case["kv_heads"] * case["dim"]


def _tokens(case):
    """copy: how many tokens of each page."""
    rng = random.Random(case["pairs"] * 17 + case["page"])
    return [case["page"] if case["whole"] else rng.randint(1, case["page"]) for _ in range(case["pairs"])]


def _rows(case, seed):
    """count, compact: per row its length and the pages that it holds.  Rows share the pages of one prompt that half of the shortest
    row has room for, and then follow pages of their own; all lie in the pool in no order."""
    lens, page = _lengths(case, case["rows"]), case["page"]
    free = np.random.default_rng(seed).permutation(case["pages"])
    shared = int(case["lo"] * case["shared"]) // page
    prompt, at, out = free[:shared], shared, []
    for n in lens:
        mine = -(-n // page) - shared
        out.append((n, np.concatenate([prompt, free[at:at + mine]])))
        at += mine
    return out


def _moved(case, rows):
    used = np.zeros(case["pages"], bool)
    for _, held in rows:
        used[held] = True
    return int(used[int(used.sum()):].sum())


def work(case):
    kind = case["kind"]
    if kind == "prompt":
        lens = _lengths(case, case["count"])
        h, k, d = case["heads"], case["kv_heads"], case["dim"]
        return {"bytes": sum(lens) * (4 * d * (h + k) + 4 * h), "flops": 4 * d * h * sum(n * (n + 1) // 2 for n in lens)}
    if kind == "copy":
        return {"bytes": 2 * _token_bytes(case) * sum(_tokens(case)), "flops": 0}
    if kind == "fork":
        lens = _lengths(case, case["parents"])
        of = [i % case["parents"] for i in range(case["children"])]
        page = case["page"]
        part = _token_bytes(case) * (sum(n % page for n in lens) + sum(lens[i] % page for i in of))
        return {"bytes": part + 4 * (sum(lens) + sum(lens[i] for i in of)), "flops": 0}
    rows = _rows(case, 0)
    held = sum(len(pages) for _, pages in rows)
    if kind == "count":
        return {"bytes": 4 * held + 8 * case["pages"], "flops": held + case["pages"]}
    return {"bytes": 2 * _token_bytes(case) * case["page"] * _moved(case, rows) + 4 * held + 4 * held * case["page"] + 4 * case["pages"],
            "flops": held + case["pages"]}


# ---- inputs -----------------------------------------------------------------------------------------------------

def _pkg():
    from __graft_entry__ import load_package
    pkg = load_package()
    pkg.load_library()
    return pkg.layers


def _cuda(values, dtype=torch.int32):
    return torch.as_tensor(np.asarray(values), dtype=dtype).cuda()


def _slots(pages, page):
    return (np.asarray(pages, dtype=np.int64)[:, None] * page + np.arange(page)).reshape(-1)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    if case["kind"] == "prompt":
        lens, h, k, d = _lengths(case, case["count"]), case["heads"], case["kv_heads"], case["dim"]
        # the rows that a joint projection leaves; scores spread over a few units, as a trained model's do
        qkv = torch.randn(sum(lens), (h + 2 * k) * d, device="cuda", generator=gen)
        qkv[:, :h * d] *= 2
        q, key, v = (x.unflatten(1, (-1, d)) for x in qkv.to(torch.bfloat16).split([h * d, k * d, k * d], 1))
        return {"kind": "prompt", "q": q, "k": key, "v": v, "lens": lens, "indptr": _cuda(np.cumsum([0] + lens)), "scale": d ** -0.5}
    page, pages = case["page"], case["pages"]
    s = {"kind": case["kind"], "page": page, "pages": pages}
    if own:
        L = _pkg()
        cache = L.MHAKVCache(case["kv_heads"], case["layers"], case["dim"], pages, page)
        s |= {"cache": L.CachePages(cache), "kv": cache.kv_buffer_}
    else:
        s["kv"] = torch.zeros(2, case["layers"], pages * page, case["kv_heads"], case["dim"], dtype=torch.bfloat16, device="cuda")
    if case["kind"] != "count":
        s["kv"].normal_(generator=gen)
    rng = np.random.default_rng(seed)
    if case["kind"] == "copy":
        order = rng.permutation(pages)
        n = case["pairs"]
        s |= {"src": _cuda(order[:n]), "dst": _cuda(order[n:2 * n]), "tokens": None if case["whole"] else _cuda(_tokens(case))}
    elif case["kind"] == "fork":
        lens, free = _lengths(case, case["parents"]), rng.permutation(pages)
        table = np.zeros((case["parents"] + case["children"], -(-(max(lens) + page) // 32) * 32), np.int32)
        at = 0
        for r, n in enumerate(lens):
            held = free[at:at + -(-n // page)]
            at += len(held)
            table[r, :len(held) * page] = _slots(held, page)[:table.shape[1]]
        of = [i % case["parents"] for i in range(case["children"])]
        s |= {"table": _cuda(table), "parents": _cuda(of), "children": _cuda(np.arange(len(of)) + case["parents"]),
              "lens": _cuda([lens[i] for i in of]), "new": _cuda(free[at:at + len(of)])}
    else:
        rows = _rows(case, seed)
        width = -(-max(len(held) for _, held in rows) * page // 32) * 32
        table = np.zeros((len(rows), width), np.int32)
        for r, (_, held) in enumerate(rows):
            table[r, :len(held) * page] = _slots(held, page)
        s |= {"table": _cuda(table), "rows": _cuda(np.arange(len(rows))), "lens": _cuda([n for n, _ in rows])}
        if case["kind"] == "compact":
            s["out"] = s["table"].clone()   # the renamed table, so that a pass can be made again
    return s


# ---- one pass ---------------------------------------------------------------------------------------------------

def run(s):
    if own:
        if s["kind"] == "prompt":
            return _pkg().prompt_attention(s["q"], s["k"], s["v"], s["indptr"], s["scale"], return_lse=True)
        if s["kind"] == "copy":
            s["cache"].copy(s["src"], s["dst"], s["tokens"])
            return s["kv"]
        if s["kind"] == "fork":
            s["cache"].fork(s["table"], s["parents"], s["children"], s["lens"], s["new"])
            return s["kv"], s["table"]
        if s["kind"] == "count":
            return s["cache"].count(s["table"], s["rows"], s["lens"])
        return (s["kv"], s["out"]) + s["cache"].compact(s["table"], s["rows"], s["lens"], out=s["out"])
    return {"prompt": _plain_prompt, "copy": _plain_copy, "fork": _plain_fork, "count": _plain_count, "compact": _plain_compact}[s["kind"]](s)


def _plain_prompt(s):
    """Every sequence by itself, up to 1024 query rows at a time: scores, masked softmax, sum."""
    q, k, v = s["q"], s["k"], s["v"]
    tokens, heads, dim = q.shape
    kv_heads = k.shape[1]
    out = torch.empty(tokens, heads * dim, dtype=torch.bfloat16, device="cuda")
    lse = torch.empty(tokens, heads, dtype=torch.float32, device="cuda")
    at = 0
    for n in s["lens"]:
        key, val = (x[at:at + n].float().transpose(0, 1) for x in (k, v))                      # [kv_heads, n, dim]
        for lo in range(0, n, 1024):
            hi = min(n, lo + 1024)
            rows = q[at + lo:at + hi].float().reshape(hi - lo, kv_heads, heads // kv_heads, dim).permute(1, 2, 0, 3)
            score = torch.matmul(rows, key[:, None, :hi].transpose(2, 3)) * s["scale"]          # [kv_heads, group, rows, hi]
            late = torch.arange(hi, device="cuda")[None, :] > torch.arange(lo, hi, device="cuda")[:, None]
            score = score.masked_fill(late, -math.inf)
            most = score.amax(-1, keepdim=True)
            weight = torch.exp(score - most)
            total = weight.sum(-1, keepdim=True)
            o = torch.matmul(weight, val[:, None, :hi]) / total
            out[at + lo:at + hi] = o.permute(2, 0, 1, 3).reshape(hi - lo, heads * dim).to(torch.bfloat16)
            lse[at + lo:at + hi] = (most + torch.log(total))[..., 0].permute(2, 0, 1).reshape(hi - lo, heads)
        at += n
    return out, lse


def _plain_copy(s):
    kv = s["kv"].view(2, s["kv"].shape[1], s["pages"], s["page"], -1)
    src, dst = s["src"].long(), s["dst"].long()
    if s["tokens"] is None:
        kv[:, :, dst] = kv[:, :, src]
    else:
        there = torch.arange(s["page"], device="cuda")[None, :] < s["tokens"][:, None]
        kv[:, :, dst] = torch.where(there[None, None, :, :, None], kv[:, :, src], kv[:, :, dst])
    return s["kv"]


def _plain_fork(s):
    page, table = s["page"], s["table"]
    kv = s["kv"].view(2, s["kv"].shape[1], s["pages"], page, -1)
    parents, children, lens, new = (s[k].long() for k in ("parents", "children", "lens", "new"))
    full, part = lens // page * page, lens % page
    where = torch.arange(table.shape[1], device="cuda")[None, :]
    mine = new[:, None] * page + where - full[:, None]
    row = torch.where(where < full[:, None], table[parents].long(), mine)
    written = where < torch.where(part > 0, full + page, full)[:, None]
    table[children] = torch.where(written, row, table[children].long()).to(torch.int32)
    src = table[parents, torch.where(part > 0, full, 0)].long() // page
    there = torch.arange(page, device="cuda")[None, :] < part[:, None]
    kv[:, :, new] = torch.where(there[None, None, :, :, None], kv[:, :, src], kv[:, :, new])
    return s["kv"], table


def _plain_refs(s):
    first = s["table"][s["rows"].long()][:, ::s["page"]].long() // s["page"]                  # a page per column
    there = torch.arange(first.shape[1], device="cuda")[None, :] * s["page"] < s["lens"][:, None]
    refs = torch.zeros(s["pages"], dtype=torch.int32, device="cuda")
    return refs.index_add_(0, first.reshape(-1), there.reshape(-1).to(torch.int32)), first, there


def _plain_count(s):
    refs = _plain_refs(s)[0]
    free = refs == 0
    place = torch.cumsum(free, 0)
    listed = torch.full((s["pages"] + 1,), -1, dtype=torch.int32, device="cuda")
    at = torch.where(free, place - 1, s["pages"])                                               # (the others behind the list)
    listed.scatter_(0, at, torch.arange(s["pages"], dtype=torch.int32, device="cuda"))
    return refs, torch.where(torch.arange(s["pages"], device="cuda") < place[-1], listed[:-1], -1), place[-1:].to(torch.int32)


def _plain_compact(s):
    page = s["page"]
    refs, first, there = _plain_refs(s)
    used, number = refs > 0, torch.arange(s["pages"], device="cuda")
    count = used.sum()
    src, dst = (torch.nonzero(x)[:, 0] for x in (used & (number >= count), ~used & (number < count)))
    kv = s["kv"].view(2, s["kv"].shape[1], s["pages"], page, -1)
    kv[:, :, dst] = kv[:, :, src]
    to = torch.where(used, number, -1)
    to[src] = dst
    slots = (to[first][:, :, None] * page + torch.arange(page, device="cuda")).reshape(first.shape[0], -1)
    held = there[:, :, None].expand(-1, -1, page).reshape(first.shape[0], -1)
    out = s["out"]
    rows, width = s["rows"].long(), min(out.shape[1], slots.shape[1])
    out[rows, :width] = torch.where(held[:, :width], slots[:, :width].to(torch.int32), out[rows, :width])
    return s["kv"], out, to.to(torch.int32), count.reshape(1).to(torch.int32)


# ---- the definitions in 64 bits ---------------------------------------------------------------------------------

def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    return {"prompt": _exact_prompt, "copy": _exact_copy, "fork": _exact_fork, "count": _exact_count, "compact": _exact_compact}[case["kind"]](s)


def _exact_prompt(s):
    """One head at a time; a handful of rows at a time where a sequence is long."""
    tokens, heads, dim = s["q"].shape
    out = torch.zeros(tokens, heads, dim, dtype=torch.float64, device="cuda")
    lse = torch.zeros(tokens, heads, dtype=torch.float64, device="cuda")
    at = 0
    for n in s["lens"]:
        for h in range(heads):
            g = h * s["k"].shape[1] // heads
            q, k, v = s["q"][at:at + n, h].double(), s["k"][at:at + n, g].double(), s["v"][at:at + n, g].double()
            for lo in range(0, n, 2048):
                e = q[lo:lo + 2048] @ k.T * s["scale"]
                e += torch.triu(torch.full_like(e, -math.inf), diagonal=lo + 1)
                out[at + lo:at + lo + e.shape[0], h] = torch.softmax(e, -1) @ v
                lse[at + lo:at + lo + e.shape[0], h] = torch.logsumexp(e, -1)
        at += n
    return out.reshape(tokens, heads * dim), lse


def _exact_copy(s):
    """A page at a time."""
    p = s["page"]
    tokens = [p] * s["src"].numel() if s["tokens"] is None else s["tokens"].tolist()
    for a, b, n in zip(s["src"].tolist(), s["dst"].tolist(), tokens):
        s["kv"][:, :, b * p:b * p + n] = s["kv"][:, :, a * p:a * p + n]
    return s["kv"]


def _exact_fork(s):
    """A child at a time, on the host."""
    p, table = s["page"], s["table"].cpu().numpy()
    for a, b, n, page in zip(*(s[k].tolist() for k in ("parents", "children", "lens", "new"))):
        full = n // p * p
        table[b, :full] = table[a, :full]
        if n > full:
            end = min(full + p, table.shape[1])
            table[b, full:end] = np.arange(page * p, page * p + end - full)
            for i in range(n - full):
                s["kv"][:, :, page * p + i] = s["kv"][:, :, int(table[a, full]) + i]
    return s["kv"], torch.from_numpy(table)


def _held(s):
    """Per row the pages that it holds, on the host."""
    p, table = s["page"], s["table"].cpu().numpy()
    return [[int(table[r, j]) // p for j in range(0, n, p)] for r, n in zip(s["rows"].tolist(), s["lens"].tolist())]


def _exact_count(s):
    refs = np.zeros(s["pages"], np.int32)
    for pages in _held(s):
        for g in pages:
            refs[g] += 1
    free = [g for g in range(s["pages"]) if refs[g] == 0]
    return (torch.from_numpy(refs), torch.tensor(free + [-1] * (s["pages"] - len(free)), dtype=torch.int32),
            torch.tensor([len(free)], dtype=torch.int32))


def _exact_compact(s):
    p, held = s["page"], _held(s)
    used = sorted({g for pages in held for g in pages})
    late, holes = [g for g in used if g >= len(used)], sorted(set(range(len(used))) - set(used))
    to = {g: g for g in used} | dict(zip(late, holes))
    for a, b in zip(late, holes):
        s["kv"][:, :, b * p:(b + 1) * p] = s["kv"][:, :, a * p:(a + 1) * p]
    out = s["out"].cpu().numpy()
    for r, pages in zip(s["rows"].tolist(), held):
        for j, g in enumerate(pages):
            end = min((j + 1) * p, out.shape[1])
            out[r, j * p:end] = np.arange(to[g] * p, to[g] * p + end - j * p)
    new = np.full(s["pages"], -1, np.int32)
    for g in used:
        new[g] = to[g]
    return s["kv"], torch.from_numpy(out), torch.from_numpy(new), torch.tensor([len(used)], dtype=torch.int32)
