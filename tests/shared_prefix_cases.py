"""Set-ups and plain 64-bit forms for the tests of attention over a shared prefix, sampling probabilities and draft verification.

Nothing here is collected by pytest.
"""
from __future__ import annotations

import math

import numpy as np
import torch

bf16 = torch.bfloat16
D = 128


class SharedSetup:
    """Requests of `groups` (lists of (own keys, query rows)) behind `prefixes` shared keys each.  Pages lie in no order; a page that a
    prefix fills in part belongs to the group's first request, the others have copies of that part.  Slots that nobody's sequence
    reaches hold NaN."""

    def __init__(self, groups, prefixes, page, heads, kv_heads, seed=0, device="cuda", q_scale=1.0, extra_slots=0):
        rng = np.random.default_rng(seed)
        gen = torch.Generator().manual_seed(seed)
        self.page, self.heads, self.kv_heads = page, heads, kv_heads
        self.reqs = [(g, prefixes[g], own, rows) for g, members in enumerate(groups) for own, rows in members]
        self.lens = [prefix + own for _, prefix, own, _ in self.reqs]
        self.rows = [rows for _, _, _, rows in self.reqs]
        B = len(self.reqs)
        pages_of = lambda n: -(-n // page)
        total = sum(pages_of(n) for n in self.lens) + sum(pages_of(p) for p in prefixes) + 2
        order = (rng.permutation(total) + extra_slots // page).tolist()
        self.num_slots = total * page + extra_slots // page * page
        cols = -(-(max(self.lens + [1]) + 32) // max(page, 32)) * max(page, 32)
        self.table = np.zeros((B + 2, cols), dtype=np.int32)
        self.table_idx = rng.permutation(B + 2)[:B].astype(np.int32)
        k = torch.randn(total * page, kv_heads, D, generator=gen).to(bf16)
        v = torch.randn(total * page, kv_heads, D, generator=gen).to(bf16)
        used = np.zeros(total * page, dtype=bool)
        low = self.num_slots - total * page
        shared = {}
        for b, (g, prefix, own, _) in enumerate(self.reqs):
            n, r = prefix + own, self.table_idx[b]
            leader = g not in shared
            if leader:
                shared[g] = [order.pop() for _ in range(pages_of(prefix))]
            pages = shared[g][:prefix // page] + ([shared[g][-1] if leader else order.pop()] if prefix % page else [])
            pages += [order.pop() for _ in range(pages_of(n) - len(pages))]
            slots = (np.asarray(pages, dtype=np.int64).reshape(-1, 1) * page + np.arange(page)).reshape(-1)
            self.table[r, :len(slots)] = slots
            if leader:
                first = slots
            elif prefix % page:
                part = slice(prefix // page * page, prefix)
                k[slots[part] - low] = k[first[part] - low]
                v[slots[part] - low] = v[first[part] - low]
            used[slots[:n] - low] = True
        unused = torch.from_numpy(~used)
        k[unused] = float("nan")
        v[unused] = float("nan")
        self.k, self.v, self.low = k, v, low
        self.q = (torch.randn(sum(self.rows), heads, D, generator=gen) * q_scale).to(bf16)
        self.qo = np.concatenate([[0], np.cumsum(self.rows)]).astype(np.int32)
        self.group_indptr = np.concatenate([[0], np.cumsum([len(m) for m in groups])]).astype(np.int32)
        self.prefixes = np.asarray(prefixes, dtype=np.int32)
        self.device = device

    def cache(self, L):
        c = L.MHAKVCache(self.kv_heads, 1, D, self.num_slots // self.page, self.page, device=self.device)
        c.kv_buffer_[0, 0, self.low:].copy_(self.k)
        c.kv_buffer_[1, 0, self.low:].copy_(self.v)
        return c

    def index(self, *arrays):
        return [torch.from_numpy(np.asarray(a, dtype=np.int32)).to(self.device) for a in arrays]

    def run(self, L, attn=None, q=None, out=None):
        cache = self.cache(L) if attn is None else None
        attn = attn or L.SharedPrefixAttention(cache, self.heads, self.kv_heads, D, max(self.q.shape[0], 1), max(len(self.reqs), 1))
        q = self.q.to(self.device) if q is None else q
        got = attn.forward(q, 0, *self.index(self.table, self.table_idx, self.lens, self.qo, self.group_indptr, self.prefixes), out=out)
        return got

    def want(self):
        """The formula in 64 bits: (out, sum of the weighted |v|), both [rows, heads * 128]."""
        group = self.heads // self.kv_heads
        out = torch.zeros(self.q.shape[0], self.heads, D, dtype=torch.float64)
        size = torch.zeros_like(out)
        for b, n in enumerate(self.lens):
            slots = torch.from_numpy(self.table[self.table_idx[b], :n].astype(np.int64) - self.low)
            k, v = self.k[slots].double(), self.v[slots].double()
            for i in range(self.rows[b]):
                see = n - self.rows[b] + 1 + i
                if see <= 0:
                    continue
                r = int(self.qo[b]) + i
                q = self.q[r].double().reshape(self.kv_heads, group, D)
                s = torch.einsum("hgd,khd->hgk", q, k[:see]) / math.sqrt(D)
                w = torch.softmax(s, -1)
                out[r] = torch.einsum("hgk,khd->hgd", w, v[:see]).reshape(self.heads, D)
                size[r] = torch.einsum("hgk,khd->hgd", w, v[:see].abs()).reshape(self.heads, D)
        return out.reshape(-1, self.heads * D), size.reshape(-1, self.heads * D)


def assert_attention(got, want, size):
    """Half a step of the output, and of every weight (rounded to bf16 before it meets its value): 2^-8 each; scores, exponentials
    and sums are fp32, together below 2^-12 of the weights for scores of a few units."""
    got = got.double().cpu()
    bad = ~((got - want).abs() <= 2.0 ** -8 * want.abs() + (2.0 ** -8 + 2.0 ** -12) * size)
    assert not bool(bad.any()), f"{int(bad.sum())} of {bad.numel()} off, by up to {float((got - want).abs().max())}"


def probs_oracle(logits, temperatures, top_k=None, top_p=None):
    """[rows, vocab] in 64 bits, a row at a time."""
    x = logits.double().cpu().numpy()
    out = np.zeros(x.shape)
    for r in range(x.shape[0]):
        row = np.where(np.isnan(x[r]), -np.inf, x[r])
        t = float(temperatures[r])
        if not t > 1.0000001e-6:
            out[r, int(np.argmax(row))] = 1.0
            continue
        order = np.argsort(-row, kind="stable")
        k = x.shape[1] if top_k is None else int(top_k[r])
        if 1 <= k < x.shape[1]:
            order = order[:k]
        top = row[order[0]]
        if top == -np.inf:
            continue
        with np.errstate(invalid="ignore"):
            w = np.where(row[order] == top, 1.0, np.exp((row[order] - top) / t))
        w = np.where(row[order] == -np.inf, 0.0, w)
        p = 1.0 if top_p is None else float(top_p[r])
        if p < 1:
            keep = max(1, int(np.searchsorted(np.cumsum(w), max(p, 0.0) * w.sum(), side="right")))
            order, w = order[:keep], w[:keep]
        out[r, order] = w / w.sum()
    return torch.from_numpy(out)


def assert_probs(got, want):
    """Zero where it should be, and elsewhere right to 2^-19 of itself and 2^-23 for every power of two that it lies below the
    row's largest.  The exponent e = (x - max) log2(e) / T is formed in fp32: half a last place of it and of the factor, 2 * 2^-24 |e|, so
    ln 2 of that of the weight; a weight's exponential is right to 2^-22, the sum that it is divided by as its terms (nearly all
    of it within 2^-10 of the largest: 2^-21) and 8 additions (2^-21), products and quotient 3 * 2^-24: below 2^-20 together."""
    got = got.double().cpu()
    assert bool(((got > 0) <= (want > 0)).all()), "probability outside the kept set"
    largest = want.amax(-1, keepdim=True).clamp_min(1e-300)
    below = -torch.log2(want.clamp_min(1e-300) / largest)
    bad = ~((got - want).abs() <= (2.0 ** -19 + 2.0 ** -23 * below) * want + 2.0 ** -126)
    assert not bool(bad.any()), f"{int(bad.sum())} off, relative {float(((got - want).abs() / want.clamp_min(1e-300))[bad].max())}"


def verify_oracle(target, draft, tokens, indptr, accept, draw, most):
    """(tokens, accepted) in 64 bits, a draft at a time."""
    clean = lambda p: np.where(p.astype(np.float64) > 0, p.astype(np.float64), 0.0)
    unit = lambda u: min(max(float(u), 0.0), float(np.float32(0.99999994))) if u == u else 0.0
    target = target.cpu().numpy()
    draft = None if draft is None else draft.cpu().numpy()
    tokens, indptr, accept, draw = (a.cpu().numpy() for a in (tokens, indptr, accept, draw))
    batch, vocab = len(indptr) - 1, target.shape[1]
    out = np.full((batch, most + 1), -1, dtype=np.int32)
    count = np.zeros(batch, dtype=np.int32)
    for b in range(batch):
        n = min(int(indptr[b + 1] - indptr[b]), most)
        rest = None
        for j in range(int(indptr[b]), int(indptr[b]) + n):
            p, x = clean(target[j + b]), int(tokens[j])
            q = np.zeros(vocab) if draft is None else clean(draft[j])
            known = 0 <= x < vocab
            if draft is None and known:
                q[x] = 1.0
            if known and unit(accept[j]) * q[x] < p[x]:
                out[b, count[b]] = x
                count[b] += 1
                continue
            rest = np.maximum(p - q, 0.0)
            if not rest.any():
                rest = p
            break
        if rest is None:
            rest = clean(target[int(indptr[b]) + b + n])
        c = np.cumsum(rest)
        out[b, count[b]] = 0 if c[-1] == 0 else int(np.searchsorted(c, unit(draw[b]) * c[-1], side="right"))
    return torch.from_numpy(out), torch.from_numpy(count)
