"""Timed cases of the operators of a drafted decoding step for requests that share a prompt.

* ``attention``: decode attention of a batch whose requests share a long prefix of their KV slots (parallel samples of a
  prompt, requests behind one system prompt), with one or a few query rows per request;
* ``probs``: the probabilities that a row of logits stands for after temperature, top-k and top-p;
* ``verify``: which drafted tokens the target's probabilities accept, and the token that follows them.

Head layouts and vocabularies are those of the models that this repository's benchmark runs (16 / 8, 32 / 8 and 32 / 4 heads of
128; 151936 and 128256 tokens) and generic ones.
"""
from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False   # False: the plain form; True: the framework's operators

HEAD_DIM = 128
GREEDY = 1e-6      # temperatures up to here mean the largest logit
TOP = 2 ** 30      # a top-k that keeps everything


def _attention(name, heads, kv_heads, page, sizes, prefixes, rows, suffix):
    """sizes, prefixes: requests and shared keys per group, as texts; rows, suffix: the smallest and largest per request."""
    return {"name": name, "kind": "attention", "heads": heads, "kv_heads": kv_heads, "page": page, "sizes": sizes,
            "prefixes": prefixes, "rows_lo": rows[0], "rows_hi": rows[1], "suffix_lo": suffix[0], "suffix_hi": suffix[1]}


LISTED = [
    # four samples of a short prompt a few tokens on: latency is all there is
    _attention("attention_fork4", 16, 8, 16, "4", "300", (1, 1), (1, 40)),
    # a decode batch behind one system prompt that ends inside a page
    _attention("attention_batch64", 16, 8, 16, "64", "2051", (1, 1), (1, 512)),
    # several prompts in a batch, one of them nobody else's; pages of one token, eight query heads per KV head
    _attention("attention_groups", 32, 4, 1, "40 1 23", "4096 700 1505", (1, 1), (10, 1000)),
    # drafted tokens of a batch behind a long document: one to six rows a request
    _attention("attention_drafts", 32, 8, 16, "48", "16001", (1, 6), (8, 400)),
    # a large batch behind a very long prompt, long continuations
    _attention("attention_long", 32, 8, 16, "128", "32768", (1, 1), (64, 2048)),
    # one request's drafts: a handful of rows
    {"name": "probs_few", "kind": "probs", "rows": 6, "vocab": 32000, "filters": "k"},
    # a drafted step of 64 requests, all filters in use, some requests greedy
    {"name": "probs_batch", "kind": "probs", "rows": 320, "vocab": 151936, "filters": "kpg"},
    # a large step at a temperature alone
    {"name": "probs_large", "kind": "probs", "rows": 512, "vocab": 128256, "filters": ""},
    # one request
    {"name": "verify_one", "kind": "verify", "batch": 1, "drafts_lo": 4, "drafts_hi": 4, "vocab": 128256, "lookup": False},
    # a batch whose requests bring up to five drafts each, some none
    {"name": "verify_batch", "kind": "verify", "batch": 64, "drafts_lo": 0, "drafts_hi": 5, "vocab": 151936, "lookup": False},
    # drafts that were looked up in the text (no probabilities of their own), odd vocabulary
    {"name": "verify_lookup", "kind": "verify", "batch": 200, "drafts_lo": 1, "drafts_hi": 8, "vocab": 50001, "lookup": True},
]


def listed():
    return [dict(case) for case in LISTED]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attention", "attention", "probs", "verify"])
    if kind == "attention":
        while True:
            heads, kv_heads = rng.choice([(16, 8), (32, 8), (32, 4), (16, 2), (8, 1), (24, 8)])
            sizes = [_log(rng, 1, 128) for _ in range(_log(rng, 1, 6))]
            prefixes = [_log(rng, 30, 32768) for _ in sizes]
            rows_hi, suffix_hi = rng.choice([1, 1, 2, 5, 8]), _log(rng, 8, 2048)
            case = _attention("", heads, kv_heads, rng.choice([1, 4, 16, 64]), " ".join(map(str, sizes)), " ".join(map(str, prefixes)),
                              (1, rows_hi), (max(rows_hi, suffix_hi // 50), suffix_hi + rows_hi))
            cost, most = work(case), work(LISTED[4])
            if sum(sizes) <= 256 and cost["bytes"] <= most["bytes"] and cost["flops"] <= most["flops"]:
                del case["name"]
                return case
    if kind == "probs":
        vocab = _log(rng, 1000, 152000)
        return {"kind": "probs", "rows": _log(rng, 1, min(1024, max(2, 60_000_000 // vocab))), "vocab": vocab,
                "filters": rng.choice(["", "k", "p", "kp", "kpg"])}
    batch, lo = _log(rng, 1, 200), rng.choice([0, 1, 2, 4])
    return {"kind": "verify", "batch": batch, "drafts_lo": lo, "drafts_hi": lo + rng.choice([0, 1, 3, 4]),
            "vocab": _log(rng, 1000, min(152000, 70_000_000 // (batch * (lo + 5)))), "lookup": rng.random() < 0.3}


# ---- sizes that belong to a case: the same for every seed ------------------------------------------------------

def _lengths(case):
    """Per request: its group, its shared keys, its query rows, all of its keys."""
    rng = random.Random(case["sizes"] + "/" + case["prefixes"])
    sizes, prefixes = ([int(x) for x in case[k].split()] for k in ("sizes", "prefixes"))
    out = []
    for g, (n, prefix) in enumerate(zip(sizes, prefixes)):
        for _ in range(n):
            rows = rng.randint(case["rows_lo"], case["rows_hi"])
            out.append((g, prefix, rows, prefix + max(rows, rng.randint(case["suffix_lo"], case["suffix_hi"]))))
    return out


def _drafts(case):
    rng = random.Random(case["batch"] * 1000 + case["vocab"])
    return [rng.randint(case["drafts_lo"], case["drafts_hi"]) for _ in range(case["batch"])]


def work(case):
    if case["kind"] == "attention":
        lens = _lengths(case)
        keys = sum(int(x) for x in case["prefixes"].split()) + sum(n - p for _, p, _, n in lens)
        tokens = sum(r for _, _, r, _ in lens)
        seen = sum(n - r + 1 + i for _, _, r, n in lens for i in range(r))
        return {"bytes": keys * case["kv_heads"] * HEAD_DIM * 4 + tokens * case["heads"] * HEAD_DIM * 4,
                "flops": seen * case["heads"] * HEAD_DIM * 4}
    if case["kind"] == "probs":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * 6, "flops": n * 4}
    # one row of the target's probabilities per request, and one of the draft's where not every draft is accepted (three in
    # four are)
    refused = 0.0 if case["lookup"] else sum(1 - 0.75 ** n for n in _drafts(case))
    n = (case["batch"] + refused) * case["vocab"]
    return {"bytes": int(n * 4), "flops": int(n * 2)}


# ---- inputs -----------------------------------------------------------------------------------------------------

def _pkg():
    from __graft_entry__ import load_package
    pkg = load_package()
    pkg.load_library()
    return pkg.layers


def _cuda(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device="cuda")


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return {"attention": _prepare_attention, "probs": _prepare_probs, "verify": _prepare_verify}[case["kind"]](case, seed, gen)


def _prepare_attention(case, seed, gen):
    """A KV pool whose pages lie in no order; requests of a group have the pages of the shared keys in common."""
    lens, page = _lengths(case), case["page"]
    prefixes = [int(x) for x in case["prefixes"].split()]
    pages_of = lambda keys: -(-keys // page)
    # a page that the shared keys fill in part is the first request's own page too: the others have copied it
    need = sum(pages_of(p) for p in prefixes) + sum(pages_of(n) - p // page for _, p, _, n in lens)
    free = np.random.default_rng(seed).permutation(need + 1).tolist()
    width = -(-max(n for _, _, _, n in lens) // 32) * 32
    table = np.zeros((len(lens) + 1, width), dtype=np.int32)
    shared, first = {}, set()
    for b, (g, prefix, _, n) in enumerate(lens):
        if g not in shared:
            shared[g] = [free.pop() for _ in range(pages_of(prefix))]
        pages = list(shared[g][:prefix // page])
        if prefix % page:
            pages.append(shared[g][-1] if g not in first else free.pop())
        first.add(g)
        pages += [free.pop() for _ in range(pages_of(n) - len(pages))]
        slots = (np.asarray(pages, dtype=np.int64)[:, None] * page + np.arange(page)).reshape(-1)
        table[b, :n] = slots[:n]
    tokens = sum(r for _, _, r, _ in lens)
    slots = (need + 1) * page
    kv = torch.empty(2, 1, slots, case["kv_heads"], HEAD_DIM, dtype=torch.bfloat16, device="cuda").normal_(generator=gen)
    for b, (g, prefix, _, _) in enumerate(lens):      # the copied part of a page
        if prefix % page and b > 0 and lens[b - 1][0] == g:
            leader = next(i for i, x in enumerate(lens) if x[0] == g)
            part = slice(prefix // page * page, prefix)
            kv[:, 0, table[b, part].tolist()] = kv[:, 0, table[leader, part].tolist()]
    # scores spread over a few units, as a trained model's do
    q = (torch.randn(tokens, case["heads"], HEAD_DIM, device="cuda", generator=gen) * 2).to(torch.bfloat16)
    sizes = [int(x) for x in case["sizes"].split()]
    s = {"kind": "attention", "q": q, "kv": kv, "table": torch.from_numpy(table).cuda(), "lens": lens,
         "table_idx": _cuda(list(range(len(lens)))), "seq_lens": _cuda([n for _, _, _, n in lens]),
         "qo_indptr": _cuda(np.cumsum([0] + [r for _, _, r, _ in lens]).tolist()),
         "group_indptr": _cuda(np.cumsum([0] + sizes).tolist()), "prefix_lens": _cuda(prefixes), "scale": HEAD_DIM ** -0.5}
    if own:
        L = _pkg()
        cache = L.MHAKVCache(case["kv_heads"], 1, HEAD_DIM, need + 1, page)
        cache.kv_buffer_.copy_(kv)
        s["kv"] = None
        s["attention"] = L.SharedPrefixAttention(cache, case["heads"], case["kv_heads"], HEAD_DIM, max_tokens=tokens,
                                                 max_batch=len(lens))
    return s


def _prepare_probs(case, seed, gen):
    rows, vocab, f = case["rows"], case["vocab"], case["filters"]
    rng = random.Random(seed)
    # an output head's logits: a wide bulk, a few tokens well ahead of it
    logits = torch.randn(rows, vocab, device="cuda", generator=gen) * 2
    ahead = torch.randint(vocab, (rows, min(32, vocab)), device="cuda", generator=gen)
    logits.scatter_(1, ahead, 8 + 3 * torch.randn(ahead.shape, device="cuda", generator=gen))
    temperature = [GREEDY if "g" in f and rng.random() < 0.2 else rng.choice([0.6, 0.7, 0.8, 1.0, 1.2]) for _ in range(rows)]
    return {"kind": "probs", "logits": logits.to(torch.bfloat16), "temperatures": _cuda(temperature, torch.float32),
            "top_k": _cuda([rng.choice([20, 40, 50, 200, TOP]) for _ in range(rows)]) if "k" in f else None,
            "top_p": _cuda([rng.choice([0.8, 0.9, 0.95, 1.0]) for _ in range(rows)], torch.float32) if "p" in f else None}


def _prepare_verify(case, seed, gen):
    """Draft rows are softmaxes, drafted tokens are drawn from them, target rows lie about them."""
    drafts, vocab = _drafts(case), case["vocab"]
    total, batch = sum(drafts), case["batch"]
    indptr = np.cumsum([0] + drafts)
    before = torch.randn(total, vocab, device="cuda", generator=gen) * 2.5
    rows = [int(indptr[b]) + b + j for b, n in enumerate(drafts) for j in range(n)]   # the target's row of every draft
    logits = torch.randn(total + batch, vocab, device="cuda", generator=gen) * 2.5
    if total:
        logits[rows] = before + 0.6 * torch.randn(total, vocab, device="cuda", generator=gen)
    target = torch.softmax(logits, -1)
    draft_probs = torch.softmax(before, -1)
    if total == 0:
        tokens = torch.zeros(0, device="cuda")
    else:   # looked up: mostly what the target would have said
        tokens = (target[rows] ** 4 if case["lookup"] else draft_probs).multinomial(1, generator=gen)[:, 0]
    return {"kind": "verify", "target": target, "draft_probs": None if case["lookup"] else draft_probs,
            "tokens": tokens.to(torch.int32), "indptr": _cuda(indptr.tolist()), "drafts": drafts, "most": max(drafts),
            "accept": torch.rand(total, device="cuda", generator=gen), "draw": torch.rand(batch, device="cuda", generator=gen)}


# ---- one pass ---------------------------------------------------------------------------------------------------

def run(s):
    if own:
        L = _pkg()
        if s["kind"] == "attention":
            return s["attention"].forward(s["q"], 0, s["table"], s["table_idx"], s["seq_lens"], s["qo_indptr"], s["group_indptr"],
                                          s["prefix_lens"])
        if s["kind"] == "probs":
            return L.sampling_probs(s["logits"], s["temperatures"], s["top_k"], s["top_p"])
        return L.verify_drafts(s["target"], s["tokens"], s["indptr"], s["accept"], s["draw"], s["most"], draft_probs=s["draft_probs"])
    return {"attention": _plain_attention, "probs": _plain_probs, "verify": _plain_verify}[s["kind"]](s)


def _plain_attention(s):
    """Every request by itself: its keys and values gathered, scores, masked softmax, sum."""
    heads, kv_heads = s["q"].shape[1], s["kv"].shape[3]
    out = torch.empty(s["q"].shape[0], heads * HEAD_DIM, dtype=torch.bfloat16, device="cuda")
    at = 0
    for b, (_, _, rows, n) in enumerate(s["lens"]):
        slots = s["table"][b, :n].long()
        k, v = (s["kv"][i, 0][slots].float().transpose(0, 1) for i in (0, 1))             # [kv_heads, n, 128]
        q = s["q"][at:at + rows].float().reshape(rows, kv_heads, heads // kv_heads, HEAD_DIM).permute(1, 2, 0, 3)
        score = torch.matmul(q, k.transpose(1, 2)[:, None]) * s["scale"]                      # [kv_heads, group, rows, n]
        if rows > 1:
            last = torch.arange(n - rows, n, device="cuda")[:, None]
            score = score.masked_fill(torch.arange(n, device="cuda")[None, :] > last, -math.inf)
        weight = torch.exp(score - score.amax(-1, keepdim=True))
        o = torch.matmul(weight, v[:, None]) / weight.sum(-1, keepdim=True)
        out[at:at + rows] = o.permute(2, 0, 1, 3).reshape(rows, heads * HEAD_DIM).to(torch.bfloat16)
        at += rows
    return out


def _plain_probs(s):
    """Sorted, cut, divided by what is left.  In 64 bits: where a row is cut depends on sums next to a border."""
    x = s["logits"].double()
    t = s["temperatures"].double()[:, None]
    greedy = t <= 1.0000001e-6
    best = s["logits"].float().max(-1, keepdim=True)
    w = torch.exp((x - best.values.double()) / torch.where(greedy, 1.0, t))
    if s["top_k"] is not None or s["top_p"] is not None:
        order = torch.sort(s["logits"].float(), dim=-1, descending=True, stable=True).indices
        ordered = torch.gather(w, 1, order)
        place = torch.arange(x.shape[1], device="cuda")[None, :]
        if s["top_k"] is not None:
            ordered = ordered * (place < s["top_k"].long()[:, None])
        if s["top_p"] is not None:
            p = s["top_p"].double()[:, None]
            total = ordered.sum(-1, keepdim=True)
            ordered = ordered * ((torch.cumsum(ordered, -1) <= p * total) | (place == 0) | (p >= 1))
        w = torch.zeros_like(w).scatter_(1, order, ordered)
    out = (w / w.sum(-1, keepdim=True)).float()
    first = torch.zeros_like(out).scatter_(1, torch.argmax(s["logits"].float(), -1, keepdim=True), 1.0)
    return torch.where(greedy, first, out)


def _plain_verify(s):
    """All drafts are tested at once; the first that is refused decides the row to draw from.  In 64 bits: tests and sums."""
    target, indptr, most = s["target"], s["indptr"].long(), s["most"]
    batch = indptr.numel() - 1
    n = indptr[1:] - indptr[:-1]
    place = torch.arange(most, device="cuda")[None, :].expand(batch, most)
    there = place < n[:, None]
    draft = torch.where(there, indptr[:-1, None] + place, 0)
    row = torch.where(there, indptr[:-1, None] + torch.arange(batch, device="cuda")[:, None] + place, 0)
    if most:
        x = s["tokens"][draft].long()
        p = target[row, x].double()
        q = torch.ones_like(p) if s["draft_probs"] is None else s["draft_probs"][draft, x].double()
        ok = there & (s["accept"][draft].double() * q < p)
        accepted = torch.cumprod(ok.long(), 1).sum(1)
    else:
        x = torch.zeros(batch, 0, dtype=torch.long, device="cuda")
        accepted = torch.zeros(batch, dtype=torch.long, device="cuda")
    refused = accepted < n
    last = target[indptr[:-1] + torch.arange(batch, device="cuda") + accepted].double()
    if most:
        at = torch.where(refused, indptr[:-1] + accepted, 0)
        if s["draft_probs"] is None:
            minus = torch.zeros_like(last).scatter_(1, s["tokens"][at].long()[:, None], 1.0)
        else:
            minus = s["draft_probs"][at].double()
        rest = (last - minus * refused[:, None]).clamp_min(0)
        last = torch.where(rest.sum(-1, keepdim=True) > 0, rest, last)
    c = torch.cumsum(last, -1)
    drawn = (c <= s["draw"].double()[:, None] * c[:, -1:]).sum(-1).clamp_max(target.shape[1] - 1)
    column = torch.arange(most + 1, device="cuda")[None, :]
    tokens = torch.where(column < accepted[:, None], torch.cat([x, torch.zeros_like(drawn)[:, None]], 1), -1)
    tokens = torch.where(column == accepted[:, None], drawn[:, None], tokens)
    return tokens.to(torch.int32), accepted.to(torch.int32)


# ---- the definitions in 64 bits ---------------------------------------------------------------------------------

def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    return {"attention": _exact_attention, "probs": _exact_probs, "verify": _exact_verify}[case["kind"]](s)


def _exact_attention(s):
    """Row by row from the definition, key heads one at a time."""
    tokens, heads, _ = s["q"].shape
    kv_heads = s["kv"].shape[3]
    group = heads // kv_heads
    out = torch.zeros(tokens, heads, HEAD_DIM, dtype=torch.float64, device="cuda")
    at = 0
    for b, (_, _, rows, n) in enumerate(s["lens"]):
        slots = s["table"][b, :n].long()
        for h in range(kv_heads):
            k, v = s["kv"][0, 0][slots, h].double(), s["kv"][1, 0][slots, h].double()
            for i in range(rows):
                see = n - rows + 1 + i
                e = s["q"][at + i, h * group:(h + 1) * group].double() @ k[:see].T * s["scale"]
                out[at + i, h * group:(h + 1) * group] = torch.softmax(e, -1) @ v[:see]
        at += rows
    return out.reshape(tokens, heads * HEAD_DIM)


def _exact_probs(s):
    """A row at a time on the host: the bf16 patterns in order of value are sorted, then cut."""
    logits = s["logits"].cpu()
    bits = logits.view(torch.int16).numpy().astype(np.int32) & 0xffff
    order_key = np.where(bits & 0x8000, ~bits & 0xffff, bits | 0x8000).astype(np.uint16)
    values = logits.double().numpy()
    out = np.zeros(values.shape)
    for r in range(values.shape[0]):
        t = float(s["temperatures"][r])
        if t <= 1.0000001e-6:
            out[r, int(np.argmax(values[r]))] = 1.0
            continue
        keep = np.argsort(np.uint16(0xffff) - order_key[r], kind="stable")   # largest first, equal ones by index
        if s["top_k"] is not None:
            keep = keep[:int(s["top_k"][r])]
        w = np.exp((values[r, keep] - values[r, keep[0]]) / t)
        if s["top_p"] is not None and float(s["top_p"][r]) < 1:
            inside = max(1, int(np.searchsorted(np.cumsum(w), float(s["top_p"][r]) * w.sum(), side="right")))
            keep, w = keep[:inside], w[:inside]
        out[r, keep] = w / w.sum()
    return torch.from_numpy(out)


def _exact_verify(s):
    """A request at a time, a draft at a time, on the host."""
    starts, x, accept, draw_at = (s[k].cpu().numpy() for k in ("indptr", "tokens", "accept", "draw"))
    batch = len(starts) - 1
    tokens = np.full((batch, s["most"] + 1), -1, dtype=np.int32)
    count = np.zeros(batch, dtype=np.int32)
    for b in range(batch):
        left = None
        for j in range(starts[b], starts[b + 1]):
            p = s["target"][j + b].cpu().numpy().astype(np.float64)
            q = np.zeros_like(p)
            if s["draft_probs"] is None:
                q[x[j]] = 1.0
            else:
                q = s["draft_probs"][j].cpu().numpy().astype(np.float64)
            if float(accept[j]) * q[x[j]] < p[x[j]]:
                tokens[b, count[b]] = x[j]
                count[b] += 1
                continue
            left = np.maximum(p - q, 0)
            if not left.any():
                left = p
            break
        if left is None:
            left = s["target"][starts[b + 1] + b].cpu().numpy().astype(np.float64)
        c = np.cumsum(left)
        tokens[b, count[b]] = min(int(np.searchsorted(c, float(draw_at[b]) * c[-1], side="right")), len(c) - 1)
    return torch.from_numpy(tokens), torch.from_numpy(count)
