"""Set-ups and plain forms for the tests of attention over whole prompts and of the operators on cache pages.

Nothing here is collected by pytest.
"""
from __future__ import annotations

import math

import numpy as np
import torch

bf16 = torch.bfloat16


class PromptSetup:
    """Sequences of `lens` tokens behind one another in rows [q | k | v], `before` and `behind` rows of nobody (NaN) around them."""

    def __init__(self, lens, heads, kv_heads, dim, seed=0, q_scale=1.5, before=0, behind=0, pad=0):
        gen = torch.Generator().manual_seed(seed)
        self.lens, self.heads, self.kv_heads, self.dim, self.before = list(lens), heads, kv_heads, dim, before
        n, self.width = sum(lens), (heads + 2 * kv_heads) * dim + pad
        self.rows = torch.full((before + n + behind, self.width), float("nan"), dtype=bf16)
        x = torch.randn(n, self.width, generator=gen)
        x[:, :heads * dim] *= q_scale
        self.rows[before:before + n] = x.to(bf16)
        self.indptr = (before + np.concatenate([[0], np.cumsum(self.lens)])).astype(np.int32)
        self.scale = 1.0 / math.sqrt(dim)

    def parts(self, rows):
        h, k, d = self.heads, self.kv_heads, self.dim
        return tuple(rows[:, a:b].unflatten(1, (-1, d)) for a, b in ((0, h * d), (h * d, (h + k) * d), ((h + k) * d, (h + 2 * k) * d)))

    def run(self, L, rows=None, indptr=None, **more):
        rows = self.rows.cuda() if rows is None else rows
        indptr = torch.from_numpy(self.indptr).cuda() if indptr is None else indptr
        return L.prompt_attention(*self.parts(rows), indptr, return_lse=True, **more)

    def want(self, device="cpu"):
        """The formula in 64 bits for the rows of all sequences: (out, sum of the weighted |v|, lse, how large the terms of a row's
        scores are at most)."""
        q, k, v = (x.to(device).double() for x in self.parts(self.rows))
        group = self.heads // self.kv_heads
        out, size, lse, terms = [], [], [], []
        for a, b in zip(self.indptr[:-1], self.indptr[1:]):
            n = int(b - a)
            for lo in range(0, n, 512):
                hi = min(n, lo + 512)
                late = torch.arange(hi, device=device)[None, :] > torch.arange(lo, hi, device=device)[:, None]
                x = q[a + lo:a + hi].reshape(hi - lo, self.kv_heads, group, self.dim)
                s = torch.einsum("rhgd,khd->rhgk", x, k[a:a + hi]) * self.scale
                s = s.masked_fill(late[:, None, None, :], -math.inf)
                t = torch.einsum("rhgd,khd->rhgk", x.abs(), k[a:a + hi].abs()).masked_fill(late[:, None, None, :], 0.0) * self.scale
                w = torch.softmax(s, -1)
                out.append(torch.einsum("rhgk,khd->rhgd", w, v[a:a + hi]).reshape(hi - lo, self.heads, self.dim))
                size.append(torch.einsum("rhgk,khd->rhgd", w, v[a:a + hi].abs()).reshape(hi - lo, self.heads, self.dim))
                lse.append(torch.logsumexp(s, -1).reshape(hi - lo, self.heads))
                terms.append(t.amax(-1).reshape(hi - lo, self.heads))
        none = torch.zeros(0, self.heads, self.dim, dtype=torch.float64, device=device)
        return tuple(torch.cat(x + [e]) for x, e in ((out, none), (size, none), (lse, none[..., 0]), (terms, none[..., 0])))


def assert_prompt(got, want):
    """A score is a sum of up to 128 exact products in fp32: off by at most 130 * 2^-24 of the sum of their sizes T, with scaling and
    subtraction of the reference (of a size up to T again) 3 * 2^-24 more: below 2^-16 T, the exponential another 2^-22.  So weights
    are right to e = 2^-15 T + 2^-20 of themselves (theirs and the sum's), and besides each is rounded to bf16 before it meets its value
    (2^-8) and the output once more (2^-8).  lse: the sum's error, an addition and a logarithm of numbers up to T + 20, 4 * 2^-24 each."""
    (out, lse), (want, size, want_lse, terms) = got, want
    n = want.shape[0]
    out, lse = out[:n].double().reshape(want.shape).to(want.device), lse[:n].double().to(want.device)
    e = 2.0 ** -15 * terms + 2.0 ** -20
    bad = ~((out - want).abs() <= 2.0 ** -8 * want.abs() + (2.0 ** -8 + e[..., None]) * (1 + 2.0 ** -7) * size)
    assert not bool(bad.any()), f"{int(bad.sum())} of {bad.numel()} off, by up to {float((out - want).abs().max())}"
    bad = ~((lse - want_lse).abs() <= e + 2.0 ** -22 * (terms + 20))
    assert not bool(bad.any()), f"{int(bad.sum())} of {bad.numel()} logarithms off, by up to {float((lse - want_lse).abs().max())}"


# ---- pages ---------------------------------------------------------------------------------------------------------

class PageSetup:
    """A pool of `pages` pages whose contents tell (plane, slot, place in the slot) apart, and a page table."""

    def __init__(self, page, pages, layers=2, kv_heads=2, dim=64, spare=0, seed=0):
        self.page, self.pages, self.layers, self.kv_heads, self.dim, self.spare = page, pages, layers, kv_heads, dim, spare
        self.rng = np.random.default_rng(seed)
        slots = (pages + spare) * page
        self.kv = torch.from_numpy(self.rng.integers(-2 ** 15, 2 ** 15, size=(2, layers, slots, kv_heads, dim)).astype(np.int16))

    def cache(self, L):
        c = L.MHAKVCache(self.kv_heads, self.layers, self.dim, self.pages + self.spare, self.page)
        c.kv_buffer_.copy_(self.kv.view(bf16))   # (bit patterns of every kind: compared as integers)
        return c

    def contents(self, cache):
        return cache.kv_buffer_.view(torch.int16).cpu()

    def slots_of(self, pages):
        return (np.asarray(pages, dtype=np.int64)[:, None] * self.page + np.arange(self.page)).reshape(-1).astype(np.int32)

    def table(self, held, cols, rows=None, fill=-7):
        """Row r names the slots of held[r]."""
        t = np.full((rows or len(held), cols), fill, np.int32)
        for r, pages in enumerate(held):
            s = self.slots_of(pages) if len(pages) else np.zeros(0, np.int32)
            t[r, :len(s)] = s[:cols]
        return t


def ints(*arrays):
    return [torch.from_numpy(np.ascontiguousarray(np.asarray(a, dtype=np.int32))).cuda() for a in arrays]


def copy_oracle(kv, page, pages, src, dst, tokens=None):
    """(contents afterwards, destinations that are left out)."""
    n = [page] * len(src) if tokens is None else [min(max(int(x), 0), page) for x in tokens]
    real = [i for i in range(len(src)) if src[i] >= 0 and dst[i] >= 0 and src[i] != dst[i] and src[i] < pages and dst[i] < pages and n[i] > 0]
    out, left = kv.clone(), set()
    for i in real:
        if any(j != i and dst[j] == dst[i] for j in real) or any(src[j] == dst[i] for j in real):
            left.add(dst[i])
            continue
        a, b = src[i] * page, dst[i] * page
        out[:, :, b:b + n[i]] = kv[:, :, a:a + n[i]]
    return out, left


def fork_oracle(kv, table, page, pages, parents, children, lens, new):
    """(contents, table, entries that are left out)."""
    rows, cols = table.shape
    kv2, t2, left = kv.clone(), table.copy(), set()

    def source(j):
        n = lens[j]
        if not (0 < n <= cols and 0 <= parents[j] < rows and n % page):
            return None
        slot = int(table[parents[j], n // page * page])
        return slot // page if slot >= 0 and slot % page == 0 and slot // page < pages else None

    count = len(parents)
    for i in range(count):
        a, b, n = parents[i], children[i], lens[i]
        part = n % page if n >= 0 else 0
        bad = not (0 <= a < rows and 0 <= b < rows and 0 <= n <= cols and a != b)
        bad = bad or any(j != i and b in (children[j], parents[j]) for j in range(count))
        if not bad and part:
            bad = source(i) is None or not 0 <= new[i] < pages or any(source(j) == new[i] for j in range(count))
            bad = bad or any(j != i and lens[j] > 0 and lens[j] % page and new[j] == new[i] for j in range(count))
        if bad:
            left.add(i)
            continue
        full = n - part
        t2[b, :full] = table[a, :full]
        if part:
            end = min(full + page, cols)
            t2[b, full:end] = new[i] * page + np.arange(end - full)
            at = source(i) * page
            kv2[:, :, new[i] * page:new[i] * page + part] = kv[:, :, at:at + part]
    return kv2, t2, left


def held_pages(table, rows, lens, page, pages):
    """Per entry the pages that it holds (those that there are), with their places."""
    out = []
    for r, n in zip(rows, lens):
        mine = []
        if 0 <= r < table.shape[0]:
            for at in range(0, min(max(int(n), 0), table.shape[1]), page):
                slot = int(table[r, at])
                if slot >= 0 and slot % page == 0 and slot // page < pages:
                    mine.append((at, slot // page))
        out.append(mine)
    return out


def count_oracle(table, rows, lens, page, pages, held=()):
    refs = np.zeros(pages, np.int32)
    for mine in held_pages(table, rows, lens, page, pages):
        for _, g in mine:
            refs[g] += 1
    for g in held:
        if 0 <= g < pages:
            refs[g] += 1
    free = [g for g in range(pages) if refs[g] == 0]
    return refs, np.asarray(free + [-1] * (pages - len(free)), np.int32), len(free)


def compact_oracle(kv, table, rows, lens, page, pages, held=(), out=None):
    """(contents, table, map, used)."""
    refs = count_oracle(table, rows, lens, page, pages, held)[0]
    used = [g for g in range(pages) if refs[g] > 0]
    late, holes = [g for g in used if g >= len(used)], [g for g in range(len(used)) if refs[g] == 0]
    to = {g: g for g in used} | dict(zip(late, holes))
    kv2, t2 = kv.clone(), (table if out is None else out).copy()
    for a, b in zip(late, holes):
        kv2[:, :, b * page:(b + 1) * page] = kv[:, :, a * page:(a + 1) * page]
    for r, mine in zip(rows, held_pages(table, rows, lens, page, pages)):
        for at, g in mine:
            end = min(at + page, table.shape[1])
            t2[r, at:end] = to[g] * page + np.arange(end - at)
    return kv2, t2, np.asarray([to.get(g, -1) for g in range(pages)], np.int32), len(used)
