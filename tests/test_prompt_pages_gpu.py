"""Attention over whole prompts and the operators on cache pages on the GPU, against plain forms (tests/prompt_pages_cases.py, where
the tolerances are derived)."""
import numpy as np
import pytest
import torch

from tests.prompt_pages_cases import (PageSetup, PromptSetup, assert_prompt, compact_oracle, copy_oracle, count_oracle, fork_oracle, ints)

pytestmark = pytest.mark.gpu
bf16 = torch.bfloat16


# ---- attention over whole prompts ---------------------------------------------------------------------------------

PROMPTS = {   # lengths, heads, KV heads, head dimension
    "one token": ([1], 16, 8, 128),
    "one key fewer than a tile": ([127], 16, 8, 128),
    "a tile": ([128], 16, 8, 128),
    "a tile and a token": ([129], 16, 8, 128),
    "two blocks": ([257], 16, 8, 128),
    "single tokens": ([1] * 9, 32, 8, 128),
    "odd lengths": ([3, 130, 1, 0, 64, 65, 200, 0, 77], 32, 8, 128),
    "nobody's rows between": ([0, 0, 5, 0], 16, 8, 128),
    "one head per KV head": ([300, 1, 129, 255, 256, 257], 12, 12, 128),
    "three heads per KV head": ([300, 43, 42, 85, 500], 24, 8, 128),
    "five heads per KV head": ([260, 26, 51, 7], 10, 2, 128),
    "seven heads per KV head": ([300, 19, 37], 14, 2, 128),
    "sixteen heads per KV head": ([200, 9, 17], 32, 2, 128),
    "heads of 128 on one": ([3, 2, 140], 128, 1, 128),
    "hundred heads on one": ([3, 2, 140], 100, 1, 64),
    "heads of 64": ([300, 64, 1, 128, 129, 511], 16, 4, 64),
    "heads of 96": ([300, 64, 1], 16, 8, 96),
    "heads of 80": ([150, 33], 8, 8, 80),
    "heads of 72": ([150, 33], 8, 2, 72),
    "heads of 8": ([150, 33], 8, 2, 8),
    "heads of 40": ([150, 33], 6, 2, 40),
    "long": ([2500, 700], 16, 2, 128),
    "three heads per KV head, long": ([1700, 800], 6, 2, 64),
    "five heads per KV head, long": ([1500], 10, 2, 128),
    "six heads per KV head, long": ([1300, 900], 12, 2, 96),
    "eleven heads per KV head, long": ([1100], 22, 2, 64),
    "forty heads per KV head, long": ([700], 40, 1, 128),
    "sixty-five heads per KV head": ([400], 65, 1, 64),
    "many of all lengths": ([1 + 37 * i % 211 for i in range(90)], 8, 4, 64),
    "a long one among short ones": ([5] * 20 + [1700] + [9] * 30, 8, 8, 128),
}


@pytest.mark.parametrize("name", PROMPTS)
def test_prompt_attention(L, name):
    s = PromptSetup(*PROMPTS[name], seed=len(name))
    got = s.run(L)
    assert_prompt(got, s.want("cuda"))
    assert L.read_device_status() == (0, 0)


def test_prompt_attention_equals_the_paged_one(L):
    s = PromptSetup([130, 1, 300], 16, 8, 128, seed=2)
    out, _ = s.run(L)
    n = sum(s.lens)
    cache = L.MHAKVCache(8, 1, 128, n, 1)
    q, k, v = s.parts(s.rows.cuda())
    cache.store_kv(k.reshape(n, -1), v.reshape(n, -1), torch.arange(n, dtype=torch.int32, device="cuda"), 0)
    table = np.zeros((3, 320), np.int32)
    for r, (a, b) in enumerate(zip(s.indptr[:-1], s.indptr[1:])):
        table[r, :b - a] = np.arange(a, b)
    table, idx, lens, qo = ints(table, [0, 1, 2], s.lens, s.indptr)
    paged = L.PagedAttention(cache, 16, 8, 128).prefill(q, 0, table, idx, lens, qo, 300)
    want = s.want("cuda")
    assert_prompt((out, want[2].float()), want)
    assert_prompt((paged, want[2].float()), want)


def test_prompt_attention_leaves_other_rows(L):
    """Rows before the first sequence and behind the last one, NaN themselves; q, k and v are columns of wider rows."""
    s = PromptSetup([130, 3, 77], 16, 8, 128, seed=3, before=5, behind=9, pad=24)
    out = torch.full((s.rows.shape[0], 16 * 128), 7.0, dtype=bf16, device="cuda")
    got, lse = s.run(L, out=out)
    assert got is out
    n = sum(s.lens)
    assert_prompt((out[5:5 + n], lse[5:5 + n]), s.want("cuda"))
    assert bool((out[:5] == 7).all()) and bool((out[5 + n:] == 7).all())


@pytest.mark.parametrize("heads,kv_heads", [(16, 8), (8, 8), (6, 2)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_prompt_attention_odd_values_reach_only_what_sees_them(L, bad, heads, kv_heads):
    """An infinity or NaN among keys and values: other sequences and earlier rows do not see it, the rows from its own on do."""
    lens = [200, 131, 60, 300]
    s = PromptSetup(lens, heads, kv_heads, 128, seed=4)
    want = s.want("cuda")
    _, _, v = s.parts(s.rows)
    k = s.parts(s.rows)[1]
    at = [int(s.indptr[0]) + 199, int(s.indptr[1]) + 40, int(s.indptr[3]) + 257]
    v[at[0], :, 5] = bad
    v[at[1], 0, 7] = bad
    k[at[2], 1] = bad
    out, lse = s.run(L)
    row = torch.arange(sum(lens), device="cuda")
    group = heads // kv_heads
    hit = torch.zeros(sum(lens), heads, 128, dtype=torch.bool, device="cuda")
    hit[at[0], :, 5] = True
    hit[(row >= at[1]) & (row < int(s.indptr[2])), :group, 7] = True
    hit[at[2]:, group:2 * group] = True
    got = out.reshape(hit.shape)
    want = list(want)
    clean = torch.where(hit, want[0].to(bf16), got)
    assert_prompt((clean.reshape(out.shape), torch.where(hit.any(-1), want[2].float(), lse)), want)
    assert not bool(torch.isfinite(got[at[0], :, 5]).any())
    assert not bool(torch.isfinite(got[at[1]:int(s.indptr[2]), :group, 7]).any())
    assert not bool(torch.isfinite(got[at[2]:, group:2 * group]).all(-1).any())
    # an infinite value stays one
    if bad != bad:
        assert bool(torch.isnan(got[at[0], :, 5]).all())
    else:
        assert bool((got[at[0], :, 5] == bad).all()) and bool((got[at[1]:int(s.indptr[2]), :group, 7] == bad).all())


def test_prompt_attention_of_large_and_small_scores(L):
    """Scores of hundreds (one key takes all), of one value throughout, and ones that grow along the keys."""
    s = PromptSetup([300, 140], 8, 4, 128, seed=5, q_scale=60.0)
    assert_prompt(s.run(L), s.want("cuda"))
    s = PromptSetup([300, 140], 8, 4, 128, seed=6, q_scale=0.0)
    assert_prompt(s.run(L), s.want("cuda"))
    s = PromptSetup([700], 8, 4, 128, seed=7)
    q, k, _ = s.parts(s.rows)
    q[:, :, :] = 1.0
    k[:] = (torch.arange(700)[:, None, None] / 64.0).to(bf16)
    assert_prompt(s.run(L), s.want("cuda"))
    k[:] = -(torch.arange(700)[:, None, None] / 64.0).to(bf16)
    assert_prompt(s.run(L), s.want("cuda"))


@pytest.mark.parametrize("at,value", [(0, -1), (1, 400), (2, 3), (3, 211)])
def test_prompt_attention_reports_an_odd_indptr(L, at, value):
    s = PromptSetup([100, 50, 60], 16, 8, 128, seed=8)
    s.indptr[at] = value
    out = torch.full((210, 16 * 128), 7.0, dtype=bf16, device="cuda")
    s.run(L, out=out)
    torch.cuda.synchronize()
    assert L.read_device_status() == (0, 211) and bool((out == 7).all())


def test_prompt_attention_of_nobody(L):
    s = PromptSetup([0, 0], 16, 8, 128)
    assert s.run(L)[0].shape == (0, 2048)
    s = PromptSetup([9], 16, 8, 128)
    s.indptr = np.zeros(1, np.int32)
    assert s.run(L)[0].shape == (9, 2048)
    assert L.read_device_status() == (0, 0)


def test_prompt_attention_of_most_sequences(L):
    s = PromptSetup([(5 * i) % 13 for i in range(1023)] + [150], 8, 1, 64, seed=9)
    assert_prompt(s.run(L), s.want("cuda"))


def test_prompt_attention_of_any_strides(L):
    """Heads outside and tokens inside; each tensor by itself; a single token and a single head, whose strides say nothing."""
    s = PromptSetup([150, 33], 8, 4, 96, seed=10)
    q, k, v = (x.contiguous().cuda() for x in s.parts(s.rows))
    turn = lambda x: x.transpose(0, 1).contiguous().transpose(0, 1)
    indptr = torch.from_numpy(s.indptr).cuda()
    assert_prompt(L.prompt_attention(turn(q), k, turn(v), indptr, return_lse=True), s.want("cuda"))
    one = PromptSetup([1], 8, 1, 128, seed=11)
    q, k, v = (x.contiguous().cuda() for x in one.parts(one.rows))
    odd = lambda x: x.as_strided(x.shape, (3, x.stride(1) if x.size(1) > 1 else 5, 1))
    assert_prompt(L.prompt_attention(odd(q), odd(k), odd(v), torch.from_numpy(one.indptr).cuda(), return_lse=True), one.want("cuda"))


def test_prompt_attention_captured(L):
    """A captured call follows the lengths at its replay, whatever they are; on a stream of its own."""
    first = PromptSetup([300, 40, 111], 16, 8, 128, seed=12)
    rows, indptr = first.rows.cuda(), torch.from_numpy(first.indptr).cuda()
    out = torch.zeros(451, 16 * 128, dtype=bf16, device="cuda")
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        first.run(L, rows, indptr, out=out)
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        _, lse = first.run(L, rows, indptr, out=out)
    for lens in ([300, 40, 111], [451, 0, 0], [1, 449, 1], [150, 150, 151]):
        s = PromptSetup(lens, 16, 8, 128, seed=13)
        rows.copy_(s.rows)
        indptr.copy_(torch.from_numpy(s.indptr))
        out.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert_prompt((out, lse), s.want("cuda"))


def test_prompt_attention_on_two_streams_repeats_itself(L):
    setups = [PromptSetup([700, 30, 5], 16, 8, 128, seed=14), PromptSetup([90] * 20, 8, 8, 64, seed=15)]
    streams = [torch.cuda.Stream() for _ in setups]
    data = [(s.rows.cuda(), torch.from_numpy(s.indptr).cuda()) for s in setups]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(setups):
            with torch.cuda.stream(streams[i]):
                got[i].append(s.run(L, *data[i]))
    torch.cuda.synchronize()
    for s, outs in zip(setups, got):
        assert_prompt(outs[0], s.want("cuda"))
        assert all(torch.equal(outs[0][j], o[j]) for o in outs for j in (0, 1))


def test_prompt_attention_beyond_32_bits(L):
    """Rows whose offsets pass 2^31 elements."""
    s = PromptSetup([200, 60], 16, 8, 128, seed=16)
    wide = torch.zeros(260, 9_000_000, dtype=bf16, device="cuda")
    at = 9_000_000 - s.width
    wide[:, at:] = s.rows.cuda()
    assert 259 * wide.stride(0) > 2 ** 31
    assert_prompt(s.run(L, wide[:, at:]), s.want("cuda"))


def test_prompt_attention_checks_its_arguments(L):
    s = PromptSetup([30, 20], 16, 8, 128, seed=17)
    q, k, v = s.parts(s.rows.cuda())
    indptr = torch.from_numpy(s.indptr).cuda()

    def refused(**change):
        with pytest.raises(L.B200Error):
            L.prompt_attention(**{**dict(q=q, k=k, v=v, indptr=indptr), **change})

    refused(q=q.float())
    refused(q=q.cpu())
    refused(q=q[:40])
    refused(q=q[0])
    refused(k=k[:, :4])
    refused(k=k.half())
    refused(v=v[:40])
    refused(v=v[:, :, :64])
    refused(q=q[..., :120:2], k=k[..., :120:2], v=v[..., :120:2])
    refused(q=q[..., :60], k=k[..., :60], v=v[..., :60])
    refused(q=q[..., 4:12], k=k[..., :8], v=v[..., :8])          # not 16-byte aligned
    refused(q=q[:, :12])
    refused(k=k[:, :1].expand(-1, 8, -1))
    refused(indptr=indptr.long())
    refused(indptr=indptr.cpu())
    refused(indptr=indptr[:0])
    refused(indptr=indptr[None])
    refused(indptr=torch.zeros(1026, dtype=torch.int32, device="cuda"))
    refused(out=torch.empty(50, 16, 128, dtype=bf16, device="cuda"))
    refused(out=torch.empty(50, 2048, device="cuda"))
    refused(out=torch.empty(50, 4096, dtype=bf16, device="cuda")[:, ::2])
    refused(sm_scale=0.0)
    assert_prompt(L.prompt_attention(q, k, v, indptr, return_lse=True), s.want("cuda"))


# ---- copy ------------------------------------------------------------------------------------------------------------

COPIES = {   # page, pages, layers, KV heads, dimension, pairs
    "one page": (16, 4, 2, 2, 64, 1),
    "pages of one token": (1, 300, 3, 1, 8, 120),
    "pages of three": (3, 50, 2, 3, 24, 20),
    "pages of 64": (64, 20, 3, 8, 128, 8),
    "one layer": (16, 200, 1, 8, 128, 99),
    "many layers": (4, 30, 40, 1, 16, 14),
    "many pairs": (2, 9000, 1, 1, 8, 4300),
    "a huge page": (3000, 4, 1, 2, 128, 2),
}


def _check_copy(L, s, src, dst, tokens=None):
    cache = s.cache(L)
    L.CachePages(cache, s.pages).copy(*ints(src, dst), None if tokens is None else ints(tokens)[0])
    want, left = copy_oracle(s.kv, s.page, s.pages, list(src), list(dst), None if tokens is None else list(tokens))
    assert torch.equal(s.contents(cache), want)
    return left


@pytest.mark.parametrize("name", COPIES)
@pytest.mark.parametrize("whole", [True, False])
def test_copy_pages(L, name, whole):
    page, pages, layers, kv_heads, dim, pairs = COPIES[name]
    s = PageSetup(page, pages, layers, kv_heads, dim, seed=len(name))
    order = s.rng.permutation(pages)
    src = s.rng.choice(order[pairs:], size=pairs) if name == "many pairs" else order[pairs:2 * pairs]   # (a page may be read twice)
    tokens = None if whole else s.rng.integers(-2, page + 3, size=pairs)
    assert not _check_copy(L, s, src, order[:pairs], tokens)
    assert L.read_device_status() == (0, 0)


@pytest.mark.parametrize("n", [6, 3000])
def test_copy_pages_that_clash(L, n):
    """A page written twice, or written and read: left alone and reported; pairs of nothing: nothing."""
    s = PageSetup(2, 4 * n, 2, 1, 8, seed=3)
    order = s.rng.permutation(4 * n)
    src, dst = order[:n].copy(), order[n:2 * n].copy()
    dst[n // 2] = dst[1]
    assert _check_copy(L, s, src, dst) == {dst[1]}
    assert L.read_device_status() == (0, dst[1] + 1)
    src, dst = order[:n].copy(), order[n:2 * n].copy()
    src[0] = dst[n - 1]
    assert _check_copy(L, s, src, dst) == {dst[n - 1]}
    assert L.read_device_status() == (0, dst[n - 1] + 1)
    src[0], dst[n - 1] = -1, -9
    src[1] = dst[1]                                     # onto itself
    tokens = np.full(n, 2)
    tokens[2] = 0                                       # of nothing: may be named twice
    dst[2] = dst[3]
    assert not _check_copy(L, s, src, dst, tokens)
    assert L.read_device_status() == (0, 0)
    src[4] = 4 * n
    assert not _check_copy(L, s, src, dst, tokens)
    assert L.read_device_status() == (0, 4 * n + 1)


def test_copy_pages_behind_the_last_one(L):
    """Pages of the allocation that do not take part are none."""
    s = PageSetup(4, 10, 2, 2, 16, spare=2, seed=4)
    assert not _check_copy(L, s, [10, 1, 2], [3, 11, 4])
    assert L.read_device_status() in ((0, 11), (0, 12))


# ---- fork --------------------------------------------------------------------------------------------------------------

def _check_fork(L, s, table, parents, children, lens, new, cols=None):
    cache = s.cache(L)
    t = ints(table)[0]
    view = t if cols is None else t[:, :cols]
    L.CachePages(cache, s.pages).fork(view, *ints(parents, children, lens, new))
    want, rows, left = fork_oracle(s.kv, table[:, :cols].copy(), s.page, s.pages, *(list(map(int, x)) for x in (parents, children, lens, new)))
    assert torch.equal(s.contents(cache), want)
    got = t.cpu().numpy()
    assert np.array_equal(got[:, :cols], rows)
    if cols is not None:
        assert np.array_equal(got[:, cols:], table[:, cols:])
    return left


@pytest.mark.parametrize("page", [1, 3, 16, 64])
@pytest.mark.parametrize("children", [1, 5, 70])
def test_fork_rows(L, page, children):
    s = PageSetup(page, 400, 3, 2, 64, seed=page)
    order = s.rng.permutation(400).tolist()
    held = [[order.pop() for _ in range(n)] for n in (20, 7, 1)]
    cols = 20 * page + 2
    table = s.table(held, cols, rows=3 + children)
    rows = s.rng.permutation(children) + 3
    parents = s.rng.integers(0, 3, size=children)
    lens = [int(s.rng.integers(0, len(held[p]) * page + 1)) for p in parents]
    lens[0] = len(held[parents[0]]) * page            # ends with a page
    if children > 4:
        lens[1], lens[2], lens[3] = 0, 1, page
    new = [order.pop() for _ in range(children)]
    assert not _check_fork(L, s, table, parents, rows, lens, new)
    assert L.read_device_status() == (0, 0)


def test_fork_rows_to_the_end_of_the_table(L):
    """A last page that the table's columns cut; columns of a wider table."""
    s = PageSetup(16, 20, 2, 2, 64, seed=5)
    table = s.table([[3, 9, 11]], 48, rows=4)
    assert not _check_fork(L, s, table, [0, 0, 0], [1, 2, 3], [37, 40, 33], [0, 1, 2], cols=40)
    assert L.read_device_status() == (0, 0)


@pytest.mark.parametrize("what", ["child twice", "child is a parent", "own child", "page twice", "page read", "row", "child row", "length",
                                  "negative length", "new page", "slot"])
def test_fork_rows_reports(L, what):
    """An entry that cannot be is left out, the others are not."""
    s = PageSetup(16, 30, 2, 2, 64, seed=6)
    table = s.table([[3, 9, 11], [4, 5, 6]], 64, rows=9)
    parents, children, lens, new = [0, 0, 1, 0], [2, 3, 4, 5], [40, 17, 33, 32], [20, 21, 22, 23]
    left, said = {1}, None
    if what == "child twice":
        children[1], left, said = 2, {0, 1}, 2
    elif what == "child is a parent":
        children[1], left, said = 1, {1}, 1
    elif what == "own child":
        children[1], left, said = 0, {1}, 0
    elif what == "page twice":
        new[1], left, said = 20, {0, 1}, 20
    elif what == "page read":
        new[1], said = 6, 6
    elif what == "row":
        parents[1], said = 9, 9
    elif what == "child row":
        children[1], said = -4, -4
    elif what == "length":
        lens[1], said = 65, 65
    elif what == "negative length":
        lens[1], said = -3, -3
    elif what == "new page":
        new[1], said = 30, 30
    elif what == "slot":
        table[1, 32], left, said = 999, {2}, 999
    assert _check_fork(L, s, table, parents, children, lens, new) == left
    assert L.read_device_status() == (0, said + 1)


# ---- count and compact -----------------------------------------------------------------------------------------------

HOLDERS = {   # page, pages, rows, longest, how many of a row's pages are another's
    "one token": (16, 8, 1, 1, 0.0),
    "pages of one token": (1, 700, 9, 60, 0.3),
    "pages of three": (3, 200, 20, 40, 0.4),
    "pages of sixteen": (16, 300, 30, 300, 0.5),
    "large pages": (64, 70, 12, 300, 0.2),
    "a full pool": (4, 60, 6, 40, 0.0),
    "more pages than a CTA's": (2, 30000, 40, 900, 0.1),
    "a large pool of few": (1, 100000, 3, 50, 0.0),
    "words of bits": (16, 33, 3, 90, 0.0),
}


def _holders(name, kv_heads=1, dim=8, layers=2):
    page, pages, rows, most, shared = HOLDERS[name]
    s = PageSetup(page, pages, layers, kv_heads, dim, seed=len(name))
    order, held, lens = s.rng.permutation(pages).tolist(), [], []
    for r in range(rows):
        n = int(s.rng.integers(0, most + 1)) if r else most
        mine = -(-n // page)
        take = int(mine * shared) if r else 0
        held.append((held[0][:take] if r else []) + [order.pop() for _ in range(mine - take)] if len(order) >= mine else [])
        lens.append(n if held[-1] or n == 0 else 0)
    if name == "a full pool":
        held.append(order)
        lens.append(len(order) * page)
    table = s.table(held, max(len(h) for h in held) * page + 3, rows=len(held) + 2)
    rows = s.rng.permutation(len(held)).astype(np.int32)
    return s, table, rows, np.asarray(lens, np.int32)[rows]


@pytest.mark.parametrize("name", HOLDERS)
def test_count_pages(L, name):
    s, table, rows, lens = _holders(name)
    held = s.rng.integers(0, s.pages, size=5).astype(np.int32)
    pages = L.CachePages(s.cache(L), s.pages)
    for more in (None, held):
        refs, free, number = pages.count(*ints(table, rows, lens), None if more is None else ints(more)[0])
        want = count_oracle(table, rows, lens, s.page, s.pages, () if more is None else more)
        assert np.array_equal(refs.cpu().numpy(), want[0]) and np.array_equal(free.cpu().numpy(), want[1]) and int(number) == want[2]
    assert L.read_device_status() == (0, 0)


@pytest.mark.parametrize("name", HOLDERS)
@pytest.mark.parametrize("in_place", [True, False])
def test_compact_pages(L, name, in_place):
    s, table, rows, lens = _holders(name, *((2, 64, 2) if HOLDERS[name][1] < 1000 else (1, 8, 1)))
    held = np.unique(s.rng.integers(0, s.pages, size=3)).astype(np.int32) if not in_place else np.zeros(0, np.int32)
    cache = s.cache(L)
    t = ints(table)[0]
    out = None if in_place else torch.full_like(t, -3)
    where, used = L.CachePages(cache, s.pages).compact(t, *ints(rows, lens), ints(held)[0], out=out)
    want = compact_oracle(s.kv, table, rows, lens, s.page, s.pages, held, None if in_place else np.full_like(table, -3))
    n = want[3]
    moved = want[2][want[2] >= 0]
    assert sorted(moved.tolist()) == list(range(n))
    assert int(used) == n and np.array_equal(where.cpu().numpy(), want[2])
    assert np.array_equal((t if in_place else out).cpu().numpy(), want[1])
    assert in_place or np.array_equal(t.cpu().numpy(), table)
    assert torch.equal(s.contents(cache), want[0])
    assert L.read_device_status() == (0, 0)


def test_compact_again_moves_nothing(L):
    s, table, rows, lens = _holders("pages of sixteen", 2, 64)
    cache = s.cache(L)
    pages = L.CachePages(cache)
    t, r, n = ints(table, rows, lens)
    pages.compact(t, r, n)
    before, names = s.contents(cache), t.clone()
    where, used = pages.compact(t, torch.cat([r, r]), torch.cat([n, n]))        # (rows named twice)
    assert torch.equal(names, t) and torch.equal(before, s.contents(cache))
    u = int(used)
    assert where.tolist() == list(range(u)) + [-1] * (s.pages - u)


def test_compact_another_pool_by_the_map(L):
    """A pool of another shape behind the same table follows with a copy from page g to map[g]."""
    s, table, rows, lens = _holders("pages of three", 2, 64)
    other = PageSetup(s.page, s.pages, 1, 1, 24, seed=9)
    cache, cache2 = s.cache(L), other.cache(L)
    t, r, n = ints(table, rows, lens)
    where, _ = L.CachePages(cache).compact(t, r, n)
    L.CachePages(cache2).copy(torch.arange(s.pages, dtype=torch.int32, device="cuda"), where)
    assert torch.equal(other.contents(cache2), compact_oracle(other.kv, table, rows, lens, s.page, s.pages)[0])
    assert L.read_device_status() == (0, 0)


def test_pages_of_nobody(L):
    s = PageSetup(4, 40, 1, 1, 8)
    pages = L.CachePages(s.cache(L))
    table = ints(np.zeros((2, 8)))[0]
    none = ints([])[0]
    refs, free, number = pages.count(table, none, none)
    assert not bool(refs.any()) and free.tolist() == list(range(40)) and int(number) == 40
    where, used = pages.compact(table, none, none)
    assert where.tolist() == [-1] * 40 and int(used) == 0
    refs, free, number = pages.count(table, none, none, ints([39, 39, 0])[0])
    assert refs.tolist() == [1] + [0] * 38 + [2] and int(number) == 38 and free.tolist()[:38] == list(range(1, 39))
    pages.copy(none, none)
    pages.fork(table, none, none, none, none)
    refs, free, number = pages.count(table[:, :0], *ints([0], [3]))
    assert int(number) == 40
    assert L.read_device_status() == (0, 0)


@pytest.mark.parametrize("what,said", [("row", 8), ("negative row", -2), ("slot", 641), ("middle of a page", 18), ("held", 41)])
def test_count_and_compact_report(L, what, said):
    """Rows, slots and pages that there are not count for nothing."""
    s = PageSetup(16, 40, 1, 1, 8, seed=7)
    table = s.table([[3, 30, 11], [4, 35]], 64, rows=4)
    rows, lens, held = [0, 1, 1], [40, 17, 99], [7]
    lens[2] = 0
    if what == "row":
        rows[2], lens[2] = 7, 5
    elif what == "negative row":
        rows[2], lens[2] = -3, 5
    elif what == "slot":
        table[1, 16] = 640
    elif what == "middle of a page":
        table[1, 16] = 17
    else:
        held = [7, 40]
    cache = s.cache(L)
    pages = L.CachePages(cache)
    refs, free, number = pages.count(*ints(table, rows, lens), ints(held)[0])
    want = count_oracle(table, rows, lens, 16, 40, held)
    assert np.array_equal(refs.cpu().numpy(), want[0]) and np.array_equal(free.cpu().numpy(), want[1]) and int(number) == want[2]
    assert L.read_device_status() == (0, said)
    t = ints(table)[0]
    where, used = pages.compact(t, *ints(rows, lens), ints(held)[0])
    want = compact_oracle(s.kv, table, rows, lens, 16, 40, held)
    assert torch.equal(s.contents(cache), want[0]) and np.array_equal(t.cpu().numpy(), want[1]) and np.array_equal(where.cpu().numpy(), want[2])
    assert L.read_device_status() == (0, said)


def test_pages_beyond_32_bits(L):
    """Offsets in a plane pass 2^31 bytes and elements; the pool's last pages."""
    s = PageSetup(16, 150_000, 1, 8, 128)
    cache = L.MHAKVCache(8, 1, 128, 150_000, 16)
    assert cache.kv_buffer_.numel() > 2 ** 32
    pages = L.CachePages(cache)
    kv = cache.kv_buffer_.view(2, 150_000, 16, 8, 128)
    a, b = 149_999, 140_000
    kv[:, a] = 3
    kv[0, a, 5] = 4
    pages.copy(*ints([a], [b]))
    assert torch.equal(kv[:, b], kv[:, a]) and not bool(kv[:, b - 1].any()) and not bool(kv[:, b + 1].any())
    table = ints(s.table([[b, a], []], 64))[0]
    pages.fork(table, *ints([0], [1], [16 + 6], [149_998]))
    assert torch.equal(kv[:, 149_998, :6], kv[:, a, :6]) and not bool(kv[:, 149_998, 6:].any())
    where, used = pages.compact(table, *ints([0, 1], [32, 22]))
    assert int(used) == 3 and where[[b, 149_998, a]].tolist() == [0, 1, 2]
    assert table[0, [0, 16, 31]].tolist() == [0, 32, 47] and table[1, [0, 16, 21]].tolist() == [0, 16, 21]
    assert torch.equal(kv[:, 0], kv[:, a]) and torch.equal(kv[:, 2], kv[:, a]) and torch.equal(kv[:, 1, :6], kv[:, a, :6])


def test_pages_captured(L):
    """Captured calls follow what their arrays hold at the replay."""
    s, table, rows, lens = _holders("pages of sixteen", 2, 64)
    cache = s.cache(L)
    pages = L.CachePages(cache)
    t, r, n = ints(table, rows, lens)
    out, src, dst = torch.full_like(t, -3), *ints([1, 2, 3], [4, 5, 6])
    pages.count(t, r, n)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        refs, free, number = pages.count(t, r, n)
        where, used = pages.compact(t, r, n, out=out)
        pages.copy(src, dst)
    for seed in range(3):
        rng = np.random.default_rng(seed)
        lens2 = np.minimum(lens, rng.integers(0, 300, size=len(lens))).astype(np.int32)
        pair = rng.permutation(s.pages)[:6]
        n.copy_(torch.from_numpy(lens2))
        src.copy_(torch.from_numpy(pair[:3].astype(np.int32)))
        dst.copy_(torch.from_numpy(pair[3:].astype(np.int32)))
        out.fill_(-3)
        cache.kv_buffer_.copy_(s.kv.view(bf16))
        graph.replay()
        torch.cuda.synchronize()
        want = count_oracle(table, rows, lens2, s.page, s.pages)
        assert np.array_equal(refs.cpu().numpy(), want[0]) and np.array_equal(free.cpu().numpy(), want[1]) and int(number) == want[2]
        kv, t2, where2, used2 = compact_oracle(s.kv, table, rows, lens2, s.page, s.pages, out=np.full_like(table, -3))
        assert np.array_equal(out.cpu().numpy(), t2) and np.array_equal(where.cpu().numpy(), where2) and int(used) == used2
        assert torch.equal(s.contents(cache), copy_oracle(kv, s.page, s.pages, pair[:3].tolist(), pair[3:].tolist())[0])
    assert L.read_device_status() == (0, 0)


def test_pages_on_two_streams(L):
    """Two objects on one cache's copies and another's compaction at once."""
    s, table, rows, lens = _holders("more pages than a CTA's")
    other = PageSetup(16, 400, 4, 2, 64, seed=8)
    order = other.rng.permutation(400)
    caches, streams = (s.cache(L), other.cache(L)), (torch.cuda.Stream(), torch.cuda.Stream())
    one, two = (L.CachePages(c) for c in caches)
    one.workspace.fill_(255)
    two.workspace.fill_(255)
    t, r, n = ints(table, rows, lens)
    src, dst = ints(order[:200], order[200:])
    out = torch.full_like(t, -3)
    torch.cuda.synchronize()
    for _ in range(5):
        with torch.cuda.stream(streams[0]):
            where, used = one.compact(t, r, n, out=out)
        with torch.cuda.stream(streams[1]):
            two.copy(src, dst)
    torch.cuda.synchronize()
    want = compact_oracle(s.kv, table, rows, lens, s.page, s.pages, out=np.full_like(table, -3))
    assert np.array_equal(out.cpu().numpy(), want[1]) and np.array_equal(where.cpu().numpy(), want[2])
    assert torch.equal(other.contents(caches[1]), copy_oracle(other.kv, 16, 400, order[:200].tolist(), order[200:].tolist())[0])


def test_pages_check_their_arguments(L):
    s = PageSetup(16, 20, 1, 1, 8)
    cache = s.cache(L)
    pages = L.CachePages(cache)
    table, a, b = ints(np.zeros((4, 64)), [1, 2], [3, 4])
    for bad in (a.long(), a.cpu(), a[None], torch.zeros(4, dtype=torch.int32, device="cuda")[::2]):
        for call in (lambda: pages.copy(bad, b), lambda: pages.copy(a, bad), lambda: pages.copy(a, b, bad),
                     lambda: pages.fork(table, bad, b, a, b), lambda: pages.fork(table, a, b, a, bad), lambda: pages.count(table, bad, a),
                     lambda: pages.count(table, a, bad), lambda: pages.count(table, a, b, bad), lambda: pages.compact(table, bad, a)):
            with pytest.raises(L.B200Error):
                call()
    for bad in (table.long(), table.cpu(), table[0], table.t()):
        for call in (lambda: pages.fork(bad, a, b, a, b), lambda: pages.count(bad, a, b), lambda: pages.compact(bad, a, b),
                     lambda: pages.compact(table, a, b, out=bad)):
            with pytest.raises(L.B200Error):
                call()
    for call in (lambda: pages.copy(a, b[:1]), lambda: pages.fork(table, a, b, a, b[:1]), lambda: pages.count(table, a, b[:1]),
                 lambda: pages.compact(table, a, b, out=table[:2]), lambda: L.CachePages(cache, 21), lambda: L.CachePages(cache, 0),
                 lambda: L.CachePages(L.MHAKVCache(1, 1, 4, 8, 16)).copy(a, b)):
        with pytest.raises(L.B200Error):
            call()
    assert torch.equal(s.contents(cache), s.kv)


# ---- all of them, as they are used --------------------------------------------------------------------------------

@pytest.mark.parametrize("page", [1, 16])
def test_a_prompt_answered_several_times(L, page):
    """Two prompts are read, stored, forked for some answers, decoded behind their shared prefixes; some answers end, the pool is
    counted and compacted, and the others go on as before."""
    heads, kv_heads, dim, prompts, answers = 16, 8, 128, [203, 90], [3, 2]
    s = PromptSetup(prompts, heads, kv_heads, dim, seed=20)
    rows = s.rows.cuda()
    q, k, v = s.parts(rows)
    out, _ = s.run(L, rows)
    cache = L.MHAKVCache(kv_heads, 2, dim, 40 * 16 // page, page)
    pages = L.CachePages(cache)
    order = np.random.default_rng(1).permutation(cache.num_pages_).tolist()
    slots_of = lambda held: (np.asarray(held)[:, None] * page + np.arange(page)).reshape(-1)
    table = np.zeros((7, 320), np.int32)
    for r, n in enumerate(prompts):
        at = slots_of([order.pop() for _ in range(-(-n // page))])
        table[r, :len(at)] = at
    where = np.concatenate([table[r, :n] for r, n in enumerate(prompts)])
    t, loc = ints(table, where)
    for layer in (0, 1):
        cache.store_kv(k.reshape(len(where), -1), v.reshape(len(where), -1), loc, layer)
    paged = L.PagedAttention(cache, heads, kv_heads, dim)
    seq, idx, qo = ints(prompts, [0, 1], s.indptr)
    want = s.want("cuda")
    for got in (out, paged.prefill(q, 1, t, idx, seq, qo, max(prompts))):
        assert_prompt((got, want[2].float()), want)

    of = np.repeat([0, 1], answers)
    children, lens = np.arange(5) + 2, np.asarray(prompts)[of]
    new = np.asarray([order.pop() for _ in of])
    pages.fork(t, *ints(of, children, lens, new))
    host = t.cpu().numpy()
    # a token more each: in the copied part page, or a new one
    gen = torch.Generator().manual_seed(2)
    more = torch.randn(5, (heads + 2 * kv_heads) * dim, generator=gen).to(bf16)
    full = lens % page == 0
    for i in np.flatnonzero(full):
        host[children[i], lens[i]:lens[i] + page] = slots_of([order.pop()])
    t.copy_(torch.from_numpy(host))
    nq, nk, nv = s.parts(more.cuda())
    loc = ints(host[children, lens])[0]
    for layer in (0, 1):
        cache.store_kv(nk.reshape(5, -1), nv.reshape(5, -1), loc, layer)
    shared = L.SharedPrefixAttention(cache, heads, kv_heads, dim, 5, 5)
    qo, groups, prefix = ints(np.arange(6), [0, 3, 5], lens[[0, 3]] // page * page)
    idx, seq = ints(children, lens + 1)

    whole = PromptSetup(lens + 1, heads, kv_heads, dim)
    for i, p in enumerate(of):
        a = whole.indptr[i]
        whole.rows[a:a + lens[i]] = s.rows[s.indptr[p]:s.indptr[p + 1]]
        whole.rows[a + lens[i]] = more[i]
    want = [x[whole.indptr[1:] - 1] for x in whole.want("cuda")]
    first = shared.forward(nq, 1, t, idx, seq, qo, groups, prefix)
    assert_prompt((first, want[2].float()), want)

    # answers 0 and 3 end, and the prompts' own rows: what is left?
    stay = np.asarray([1, 2, 4])
    keep = ints(children[stay], lens[stay] + 1)
    refs, free, number = pages.count(t, *keep)
    held = [sorted({int(x) // page for x in host[children[i], :lens[i] + 1]}) for i in stay]
    used = sorted(set().union(*held))
    assert int(number) == cache.num_pages_ - len(used) and free[:int(number)].tolist() == sorted(set(range(cache.num_pages_)) - set(used))
    assert int(refs.sum()) == sum(map(len, held)) and int(refs.max()) == 2
    where, count = pages.compact(t, *keep)
    assert int(count) == len(used) and int(t[children[stay].tolist()][:, :50].max()) < len(used) * page
    got = paged.decode(nq[stay.tolist()], 1, t, *keep)
    assert_prompt((got, want[2][stay].float()), [x[stay] for x in want])
    assert torch.equal(paged.decode(nq[stay.tolist()], 0, t, *keep), got)
    assert L.read_device_status() == (0, 0)


@pytest.mark.parametrize("page,length", [(1, 37), (16, 37), (16, 48)])
def test_an_engine_request_forked(pkg, page, length):
    """Forked requests go on as requests with the same tokens in pages of their own do, whatever the others write."""
    from oracle import token_loop_oracle as O
    from sglang_cpp_b200.engine import Engine, EngineConfig
    from sglang_cpp_b200.host_batch import HostBatcher

    cfg = O.ModelConfig(3, 256, 4, 2, 128, 512, 2048, 1e-6, 1e6, 512, True, True, True)
    weights = O.init_weights(cfg, seed=0, std=0.02)
    ids = np.random.default_rng(5).integers(0, 2048, size=length).astype(np.int32)

    def start(prefix_cache):
        e = Engine(cfg, EngineConfig(page, 512 // page, 8, 512, 1024))
        e.load_weights(weights)
        return e, HostBatcher(e, 512 // page, page, 8, enable_prefix_cache=prefix_cache)

    def decode(hb, reqs, steps):
        out = []
        for _ in range(steps):
            next_token = hb.decode(reqs)
            next_token.synchronize()
            out.append(hb.engine.logits(len(reqs)).float())
            for r, t in zip(reqs, next_token.next_tokens_cpu[:len(reqs)].tolist()):
                r.append_host_token(t)
        return torch.stack(out)

    engine, hb = start(True)
    first = hb.add_request(ids, 30)
    tokens = hb.prefill([first])
    tokens.synchronize()
    answer = int(tokens.next_tokens_cpu[0])
    first.append_host_token(answer)
    kids = hb.fork(first, 3)
    reqs = [first] + kids
    said = [answer, 11, 1500, answer]              # two go on as they would have, two with another token
    for r, t in zip(reqs, said):
        r.input_ids = np.append(r.input_ids[:length], np.int32(t))
    hb.tables.write_tokens([r.table_idx for r in reqs], [length] * 4, said)
    got = decode(hb, reqs, 6)
    assert torch.equal(got[:, 0], got[:, 3])
    table = hb.tables.page_table
    assert np.array_equal(engine.read_table("page_table")[:-1, :length], table[:-1, :length])   # (the last row is the dummy request's)
    # a fork of a fork, in mid-answer
    more = hb.fork(kids[0], 2)
    again = decode(hb, kids[:1] + more, 3)
    assert torch.equal(again[:, 0], again[:, 1]) and torch.equal(again[:, 0], again[:, 2])

    plain, hb2 = start(False)
    alone = [hb2.add_request(np.append(ids, np.int32(t)), 29) for t in said[:3]]
    first_logits = []
    for r in alone:                                # (prompts of one more token: their last row is the forked ones' first step)
        tokens = hb2.prefill([r])
        tokens.synchronize()
        first_logits.append(plain.logits(1).float()[0])
        r.append_host_token(int(tokens.next_tokens_cpu[0]))
    assert float((got[0, :3] - torch.stack(first_logits)).abs().max()) <= 2e-2
    tail = decode(hb2, alone, 5)
    same = [i for i in range(3) if np.array_equal(reqs[i].input_ids[:length + 6], alone[i].input_ids[:length + 6])]
    assert len(same) >= 2                          # (near ties of the logits may part them)
    for i in same:
        assert float((got[1:, i] - tail[:, i]).abs().max()) <= 2e-2
    for r in reqs + more:
        hb.release(r)
    hb.cache_manager.check_integrity()
    engine.synchronize()


def test_an_engine_pool_counted_and_compacted(pkg, L):
    """CachePages over an engine's pool, on its stream: the dummy request's page takes no part."""
    from oracle import token_loop_oracle as O
    from sglang_cpp_b200.engine import Engine, EngineConfig
    from sglang_cpp_b200.host_batch import HostBatcher

    cfg = O.ModelConfig(2, 256, 4, 2, 128, 512, 1024, 1e-6, 1e6, 512, True, True, True)
    engine = Engine(cfg, EngineConfig(16, 32, 4, 512, 1024))
    engine.load_weights(O.init_weights(cfg, seed=1, std=0.02))
    hb = HostBatcher(engine, 32, 16, 4, enable_prefix_cache=False)
    reqs = [hb.add_request(np.arange(n, dtype=np.int32) + 7, 20) for n in (50, 33, 70)]
    hb.prefill(reqs).synchronize()
    for r in reqs:
        r.append_host_token(3)
        hb.tables.write_tokens([r.table_idx], [r.cached_len], [3])
    hb.release(reqs.pop(0))
    hb.decode(reqs).synchronize()
    before = engine.logits(2).clone()
    pages = engine.cache_pages()
    assert pages.pages_ == 32
    stream = engine.cuda_stream()
    rows, lens = [r.table_idx for r in reqs], [r.cached_len for r in reqs]
    with torch.cuda.stream(stream):
        refs, free, number = pages.count(engine.page_table(), *ints(rows, lens))
        where, used = pages.compact(engine.page_table(), *ints(rows, lens))
        stream.synchronize()
    held = sum(-(-n // 16) for n in lens)
    assert int(used) == held and int(number) == 32 - held and int(refs.sum()) == held
    table = engine.read_table("page_table")
    for r, n in zip(rows, lens):
        assert np.array_equal(table[r, :n], where.cpu().numpy()[hb.tables.page_table[r, :n] // 16] * 16 + np.arange(n) % 16)
    # the same step once more, from the moved pages
    for r in reqs:
        r.cached_len -= 1
        r.device_len -= 1
    engine.forward_batch(1, rows, [r.cached_len for r in reqs], [1] * 2, write_pos=[-1] * 2).synchronize()
    assert torch.equal(engine.logits(2), before)
    with pytest.raises(L.B200Error):
        L.MHAKVCache.over(torch.zeros(2, 1, 30, 2, 64, dtype=bf16, device="cuda"), 16)


@pytest.mark.parametrize("name", ["more pages than a CTA's", "a large pool of few"])
@pytest.mark.parametrize("in_place", [True, False])
def test_pages_captured_where_many_ctas_count(L, name, in_place):
    """Pools that more than one CTA looks through, and pairs that are compared ahead of the copies: count, compact and copy behind one another
    on one workspace, in a graph."""
    s, table, rows, lens = _holders(name, 1, 8, 1)
    n_pairs, longest = 300, int(lens.max())
    assert s.pages > 24000 and n_pairs > 32
    cache = s.cache(L)
    pages = L.CachePages(cache)
    pages.workspace.fill_(255)
    t, r, n = ints(table, rows, lens)
    out = t.clone() if in_place else torch.full_like(t, -3)
    target = t if in_place else out
    src, dst, held, tokens = ints(np.zeros(n_pairs), np.zeros(n_pairs), np.zeros(7), np.zeros(n_pairs))
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.stream(stream):
        pages.count(t, r, n)
    stream.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        refs, free, number = pages.count(t, r, n, held)
        where, used = pages.compact(t, r, n, held, out=None if in_place else out)
        pages.copy(src, dst, tokens)
        refs2, free2, number2 = pages.count(target, r, n)
    for seed in range(3):
        rng = np.random.default_rng(seed)
        lens2 = np.minimum(lens, rng.integers(0, longest + 1, size=len(lens))).astype(np.int32)
        pair = rng.permutation(s.pages)[:2 * n_pairs]
        few, more = rng.integers(-1, s.page + 1, size=n_pairs), rng.integers(0, s.pages, size=7)
        t.copy_(torch.from_numpy(table))
        if not in_place:
            out.fill_(-3)
        for a, b in zip((n, src, dst, tokens, held), (lens2, pair[:n_pairs], pair[n_pairs:], few, more)):
            a.copy_(torch.from_numpy(b.astype(np.int32)))
        cache.kv_buffer_.copy_(s.kv.view(bf16))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        want = count_oracle(table, rows, lens2, s.page, s.pages, more)
        assert np.array_equal(refs.cpu().numpy(), want[0]) and np.array_equal(free.cpu().numpy(), want[1]) and int(number) == want[2]
        kv, t2, where2, used2 = compact_oracle(s.kv, table, rows, lens2, s.page, s.pages, more, None if in_place else np.full_like(table, -3))
        assert np.array_equal(target.cpu().numpy(), t2) and np.array_equal(where.cpu().numpy(), where2) and int(used) == used2
        assert torch.equal(s.contents(cache), copy_oracle(kv, s.page, s.pages, pair[:n_pairs].tolist(), pair[n_pairs:].tolist(), few.tolist())[0])
        want = count_oracle(t2, rows, lens2, s.page, s.pages)
        assert np.array_equal(refs2.cpu().numpy(), want[0]) and np.array_equal(free2.cpu().numpy(), want[1]) and int(number2) == want[2]
    assert L.read_device_status() == (0, 0)


@pytest.mark.parametrize("page", [1, 16])
def test_an_engine_compacted_with_the_hosts_books(pkg, L, page):
    """Two engines take the same steps, one of them with its pages compacted in between: the logits are the same, requests that begin
    later among them."""
    from oracle import token_loop_oracle as O
    from sglang_cpp_b200.engine import Engine, EngineConfig
    from sglang_cpp_b200.host_batch import HostBatcher

    cfg = O.ModelConfig(2, 256, 4, 2, 128, 512, 1024, 1e-6, 1e6, 512, True, True, True)
    weights = O.init_weights(cfg, seed=2, std=0.02)

    def steps(compacts):
        engine = Engine(cfg, EngineConfig(page, 640 // page, 6, 512, 1024))
        engine.load_weights(weights)
        hb, logits, rng = HostBatcher(engine, 640 // page, page, 6), [], np.random.default_rng(3)

        def run(call, reqs):
            tokens = call(reqs)
            tokens.synchronize()
            logits.append(engine.logits(len(reqs)).clone())
            for r, t in zip(reqs, tokens.next_tokens_cpu[:len(reqs)].tolist()):
                r.append_host_token(t)

        def begin(n):
            r = hb.add_request(rng.integers(0, 1024, size=n), 30)
            run(hb.prefill, [r])
            hb.cache_prefix(r)
            return r

        reqs = [begin(n) for n in (50, 33, 70)]
        reqs += hb.fork(reqs[1], 2)
        for _ in range(3):
            for _ in range(4):
                run(hb.decode, reqs)
            hb.release(reqs.pop(0))
            tree = hb.cache_manager.prefix_cache
            hb.cache_manager.free_indices(tree.evict(min(page, tree.evictable_size)))    # (holes in the pool)
            if compacts:
                used = hb.compact()
                assert sorted(hb.cache_manager.free_pages) == [g * page for g in range(used, 640 // page)]
                table = engine.read_table("page_table")
                for r in reqs:
                    assert np.array_equal(table[r.table_idx, :r.cached_len], hb.slots_of(r)[:r.cached_len])
            reqs.append(begin(int(rng.integers(20, 60))))
        for r in reqs:
            hb.release(r)
        hb.cache_manager.check_integrity()
        engine.synchronize()
        return logits

    for a, b in zip(steps(False), steps(True)):
        assert torch.equal(a, b)
    assert L.read_device_status() == (0, 0)
