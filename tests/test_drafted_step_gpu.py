"""Attention over a shared prefix, the probabilities to sample from and the verification of drafted tokens on the GPU, against plain
forms in 64 bits (tests/shared_prefix_cases.py, where the tolerances are derived)."""
import numpy as np
import pytest
import torch

from tests.shared_prefix_cases import D, SharedSetup, assert_attention, assert_probs, bf16, probs_oracle, verify_oracle

pytestmark = pytest.mark.gpu


# ---- attention over a shared prefix ------------------------------------------------------------------------------

ONE = [(1, 1)]
ATTENTION = {
    "one key": ([ONE], [0], 16, 16, 8),
    "nothing shared": ([[(40, 1)], [(1, 1)], [(300, 1)]], [0, 0, 0], 16, 16, 8),
    "two samples": ([[(1, 1), (17, 1)]], [33], 16, 16, 8),
    "prefix ends inside a page": ([[(5, 1), (130, 1), (16, 1), (1, 1)]], [203], 16, 16, 8),
    "prefix ends with a page": ([[(5, 1), (130, 1), (16, 1)]], [256], 16, 16, 8),
    "groups": ([[(9, 1)] * 5, [(70, 1)], [(3, 1), (200, 1)]], [700, 90, 1], 16, 32, 8),
    "pages of one token": ([[(9, 1), (40, 2), (1, 1)], [(12, 3), (5, 1)]], [150, 260], 1, 32, 4),
    "pages of four": ([[(9, 2), (40, 1)]], [151], 4, 8, 2),
    "large pages": ([[(9, 2), (400, 1), (30, 1)]], [1000], 256, 16, 8),
    "one KV head": ([[(9, 1), (33, 4), (200, 1)]], [517], 16, 4, 1),
    "sixteen heads per KV head": ([[(20, 3), (33, 1)]], [300], 16, 16, 1),
    "three heads per KV head": ([[(20, 5), (33, 1), (7, 7)]], [300], 16, 24, 8),
    "one head per KV head": ([[(20, 5), (33, 1), (7, 7)]], [130], 16, 8, 8),
    "drafts": ([[(8, 6), (300, 3), (70, 5), (1, 1), (6, 6)] * 3], [900], 16, 32, 8),
    "some bring no rows": ([[(8, 0), (30, 2), (9, 0)], [(5, 0)], [(7, 1), (3, 0)]], [100, 40, 60], 16, 16, 8),
    "more rows than own keys": ([[(3, 5), (30, 2), (1, 9)]], [200], 16, 16, 8),
    "many rows": ([[(70, 64), (100, 90), (50, 1)]], [400], 16, 16, 8),
    "wide group": ([[(3 + i % 50, 1) for i in range(150)]], [2100], 16, 16, 8),
    "wide groups of drafts": ([[(6 + i % 40, 1 + i % 5) for i in range(40)], [(9, 3)] * 30, [(5, 1)] * 3], [1500, 129, 777], 16, 32, 4),
    "pages of one token, every layout": ([[(40, 2), (17, 1), (3, 3)], [(21, 1), (90, 1)]], [75, 310], 1, 32, 8),
    "pages of two, two KV heads": ([[(40, 3), (17, 1), (300, 1)]], [211], 2, 8, 2),
    "pages of four, one KV head, many heads": ([[(40, 2), (17, 1), (300, 5)]], [1021], 4, 14, 1),
    "pages of one token, wide group": ([[(3 + i % 20, 1 + i % 3) for i in range(40)]], [515], 1, 16, 4),
    "pages of eight": ([[(40, 2), (17, 1), (3, 3)], [(21, 1), (90, 1)]], [75, 310], 8, 32, 8),
    "long": ([[(40, 1), (5, 1), (600, 1)] * 8], [9000], 16, 16, 8),
    "some rows behind long prefixes": ([[(5, 1), (20, 1)] * 3, [(7, 2), (9, 3)], [(4, 1)] * 8, [(3, 1)] * 4], [4100, 3000, 4001, 50], 16, 32, 8),
    "some rows behind short prefixes": ([[(5, 1), (20, 1)] * 3, [(7, 2), (9, 3)], [(4, 1)] * 30], [100, 130, 300], 16, 32, 8),
    "few rows, hundreds of parts": ([[(1, 1), (2, 1)], [(12000, 1)]], [30000, 0], 16, 16, 8),
    "a few of many rows with hundreds of parts": ([[(9, 2), (20, 1)], [(5, 1)] * 70, [(11000, 3)]], [20000, 100, 0], 16, 16, 8),
    "many rows of an odd number of heads": ([[(3 + i % 50, 1) for i in range(110)]], [400], 16, 5, 1),
    "many rows, seven heads per KV head": ([[(1 + i % 70, 1 + i % 2) for i in range(50)], [(300, 9)]], [130, 0], 8, 14, 2),
    "hundreds of rows, dozens of parts": ([[(2000 + 100 * i, 1 + i % 2) for i in range(12)]], [1200], 16, 32, 8),
}


@pytest.mark.parametrize("name", ATTENTION)
def test_shared_prefix_attention(L, name):
    groups, prefixes, page, heads, kv_heads = ATTENTION[name]
    s = SharedSetup(groups, prefixes, page, heads, kv_heads, seed=len(name))
    got = s.run(L)
    torch.cuda.synchronize()
    assert_attention(got, *s.want())
    assert L.read_device_status() == (0, 0)


def test_shared_prefix_equals_prefill_and_decode(L):
    """The same batch through the kernels that read the prefix once per request."""
    s = SharedSetup([[(20, 1), (300, 1), (1, 1)], [(40, 1)] * 6], [500, 130], 16, 32, 8, seed=3)
    cache = s.cache(L)
    plain = L.PagedAttention(cache, 32, 8, D, max_batch=16)
    table, idx, lens, qo = s.index(s.table, s.table_idx, s.lens, s.qo)
    want, size = s.want()
    for got in (s.run(L), plain.decode(s.q.cuda(), 0, table, idx, lens)):
        assert_attention(got, want, size)
    cache.kv_buffer_.nan_to_num_()   # (prefill takes numbers for granted in a page behind the last key)
    assert_attention(plain.prefill(s.q.cuda(), 0, table, idx, lens, qo, 1), want, size)


def test_shared_prefix_that_is_longer_than_a_request(L):
    """prefix_lens beyond what lies before some request's rows: as much is shared as lies before all of them."""
    s = SharedSetup([[(0, 1), (300, 2), (0, 4)]], [260], 16, 16, 8, seed=4)
    want = s.want()
    for named in (260, 100000, 257, 256, 1, 0, -5):
        s.prefixes[:] = named
        assert_attention(s.run(L), *want)


def test_shared_prefix_short_sequences(L):
    """A request of no keys, and one of fewer keys than rows: rows that see nothing are zeros."""
    s = SharedSetup([[(0, 0), (2, 4), (0, 2), (9, 1)]], [0], 16, 16, 8, seed=5)
    want, size = s.want()
    got = s.run(L)
    assert_attention(got, want, size)
    assert not bool(got[:2].any()) and not bool(got[4:6].any())


def test_shared_prefix_without_groups(L):
    s = SharedSetup([[(20, 1), (300, 3)], [(40, 2)]], [64, 32], 16, 16, 8, seed=6)
    want = s.want()
    s.group_indptr, s.prefixes = np.zeros(1, np.int32), np.zeros(0, np.int32)
    assert_attention(s.run(L), *want)
    s.group_indptr, s.prefixes = np.asarray([0, 2], np.int32), np.asarray([64], np.int32)   # the last request in no group
    assert_attention(s.run(L), *want)
    s.group_indptr, s.prefixes = np.asarray([0, 0, 2, 3, 3], np.int32), np.asarray([9, 64, 32, 5], np.int32)[:4]   # groups of nobody
    with pytest.raises(Exception):
        s.run(L)   # more groups than requests
    s.group_indptr, s.prefixes = np.asarray([0, 0, 2, 3], np.int32), np.asarray([9, 64, 32], np.int32)
    assert_attention(s.run(L), *want)


def test_shared_prefix_leaves_other_rows(L):
    """Rows before the first request's, behind the last one's and between stay; q lies in wider rows."""
    s = SharedSetup([[(20, 2), (30, 1), (9, 3)]], [100], 16, 16, 8, seed=7)
    want, size = s.want()
    wide = torch.full((s.q.shape[0] + 7, 16 + 2 * 8, D), float("nan"), dtype=bf16, device="cuda")
    wide[3:3 + s.q.shape[0], :16] = s.q.cuda()
    s.qo = s.qo + 3
    out = torch.full((wide.shape[0], 16 * D), 7.0, dtype=bf16, device="cuda")
    attn = L.SharedPrefixAttention(s.cache(L), 16, 8, D, wide.shape[0], 3)
    s.run(L, attn, q=wide[:, :16], out=out)
    n = s.q.shape[0]
    assert_attention(out[3:3 + n], want, size)
    assert bool((out[:3] == 7).all()) and bool((out[3 + n:] == 7).all())


def test_shared_prefix_masked_values_may_be_anything(L):
    """An infinity or NaN among the keys and values of a later draft reaches the rows that see it and no others."""
    for bad, seed in ((float("inf"), 8), (float("nan"), 9)):
        s = SharedSetup([[(40, 4), (21, 6), (3, 3)]], [100], 16, 16, 8, seed=seed)
        want, size = s.want()
        for b, last in enumerate((s.lens[0] - 1, s.lens[1] - 2, s.lens[2] - 1)):
            slot = int(s.table[s.table_idx[b], last])
            s.v[slot, :, 5] = bad
            if b == 1:
                s.k[slot, 0] = bad
        got = s.run(L).double().cpu()
        clean = [0, 1, 2, 4, 5, 6, 7, 10, 11]     # rows before the odd keys
        assert_attention(got[clean], want[clean], size[clean])
        for r in (3, 8, 9, 12):
            assert not bool(torch.isfinite(got[r].reshape(16, D)[:, 5]).any())


def test_shared_prefix_one_object_many_shapes(L):
    """Calls in turn on one workspace, never initialised."""
    big = SharedSetup([[(30, 2)] * 20], [800], 16, 16, 8, seed=10)
    cache = big.cache(L)
    attn = L.SharedPrefixAttention(cache, 16, 8, D, 64, 24)
    attn.workspace.fill_(255)
    first = big.run(L, attn).clone()
    table, idx, lens, qo, gi, pl = big.index(big.table, big.table_idx, big.lens, big.qo, big.group_indptr, big.prefixes)
    one = attn.forward(big.q[:2].cuda(), 0, table, idx[:1], lens[:1], qo[:2], gi[:0].new_tensor([0, 1]), pl)
    again = big.run(L, attn)
    want, size = big.want()
    assert_attention(first, want, size)
    assert torch.equal(first, again)
    assert_attention(one, want[:2], size[:2])
    empty = attn.forward(big.q[:0].cuda(), 0, table, idx[:0], lens[:0], qo[:1], gi[:1], pl[:0])
    assert empty.shape == (0, 16 * D)


def test_shared_prefix_captured(L):
    """A captured call follows lengths, groups and prefixes that change between replays; on a stream of its own."""
    s = SharedSetup([[(60, 2), (90, 1), (33, 1)], [(40, 3), (20, 1)]], [400, 150], 16, 32, 8, seed=11)
    attn = L.SharedPrefixAttention(s.cache(L), 32, 8, D, s.q.shape[0], 5)
    q = s.q.cuda()
    table, idx, lens, qo, gi, pl = s.index(s.table, s.table_idx, s.lens, s.qo, s.group_indptr, s.prefixes)
    out = torch.zeros(s.q.shape[0], 32 * D, dtype=bf16, device="cuda")
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        attn.forward(q, 0, table, idx, lens, qo, gi, pl, out=out)
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        attn.forward(q, 0, table, idx, lens, qo, gi, pl, out=out)
    for change in range(3):
        if change == 1:
            s.lens = [n - 7 for n in s.lens]
            s.prefixes = np.asarray([399, 3], np.int32)
        if change == 2:
            s.prefixes = np.asarray([0, 150], np.int32)
        lens.copy_(s.index(s.lens)[0])
        pl.copy_(s.index(s.prefixes)[0])
        out.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert_attention(out, *s.want())


def test_shared_prefix_reports_slots_outside_the_pool(L):
    s = SharedSetup([[(20, 1), (30, 1)]], [100], 16, 16, 8, seed=12)
    s.table[s.table_idx[0], :16] = 10 ** 6 + np.arange(16)
    s.run(L)
    assert L.read_device_status() == (0, 10 ** 6 + 1)
    s = SharedSetup([[(20, 1), (30, 1)]], [100], 16, 16, 8, seed=12)
    s.table[s.table_idx[1], 112:128] = -3
    s.run(L)
    assert L.read_device_status() == (0, -2)
    for own in (20, 700):   # the prefix by either kernel
        s = SharedSetup([[(own, 1)] * 20], [100], 16, 16, 8, seed=12)
        s.table[s.table_idx[3], 112:128] = -1
        s.run(L)
        assert L.read_device_status() == (0, -2 ** 31)


@pytest.mark.parametrize("name,at,value", [("qo", 1, 64), ("qo", 64, 65), ("qo", 0, -1), ("qo", 30, 28), ("groups", 1, 65),
                                           ("groups", 0, -1), ("groups", 1, 1)])
def test_shared_prefix_reports_odd_index_arrays(L, name, at, value):
    """Requests or groups that overlap, or lie outside the rows there are: reported, nothing written."""
    n = 64
    s = SharedSetup([[(20, 1)] * 40, [(20, 1)] * 24], [100, 100], 16, 16, 8, seed=13)
    (s.qo if name == "qo" else s.group_indptr)[at] = value
    if (name, value) == ("groups", 1):
        s.group_indptr[:] = (2, 1, n)
    out = torch.full((n, 16 * D), 7.0, dtype=bf16, device="cuda")
    s.run(L, out=out)
    torch.cuda.synchronize()
    assert L.read_device_status() == (0, n + 1) and bool((out == 7).all())


def test_shared_prefix_in_a_pool_beyond_32_bits(L):
    """Slots whose offsets pass 2^31 elements."""
    s = SharedSetup([[(20, 2), (30, 1), (9, 1)]], [300], 16, 16, 8, seed=14, extra_slots=2_200_000)
    assert s.low * 8 * D > 2 ** 31
    assert_attention(s.run(L), *s.want())


def test_shared_prefix_most_requests(L):
    """As many requests as there may be: groups of two and of hundreds, some of nobody's rows, in pages of any order."""
    members = [[(1 + (7 * i) % 30, 1), (3, (i % 4) // 2)] for i in range(300)] + [[(2 + i % 9, 1) for i in range(400)]] + [[(5, 1)] for _ in range(24)]
    s = SharedSetup(members, [(13 * i) % 90 for i in range(300)] + [700] + [40] * 24, 16, 16, 8, seed=15)
    assert len(s.reqs) == 1024
    got = s.run(L)
    assert_attention(got, *s.want())
    assert L.read_device_status() == (0, 0)


def test_shared_prefix_on_two_streams(L):
    """Two objects at once: calls of one change nothing for the other's."""
    setups = [SharedSetup([[(60, 2)] * 30, [(9, 1)]], [1700, 20], 16, 16, 8, seed=16), SharedSetup([[(700, 1), (30, 3)]] * 9, [260] * 9, 16, 32, 4, seed=17)]
    streams = [torch.cuda.Stream() for _ in setups]
    work = [(s, L.SharedPrefixAttention(s.cache(L), s.heads, s.kv_heads, D, s.q.shape[0], len(s.reqs)), s.q.cuda(),
             s.index(s.table, s.table_idx, s.lens, s.qo, s.group_indptr, s.prefixes)) for s in setups]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, (s, attn, q, index) in enumerate(work):
            with torch.cuda.stream(streams[i]):
                got[i].append(attn.forward(q, 0, *index))
    torch.cuda.synchronize()
    for s, outs in zip(setups, got):
        assert_attention(outs[0], *s.want())
        assert all(torch.equal(outs[0], o) for o in outs)


def test_shared_prefix_checks_its_arguments(L):
    s = SharedSetup([[(20, 1), (30, 2)]], [100], 16, 16, 8, seed=18)
    attn = L.SharedPrefixAttention(s.cache(L), 16, 8, D, 3, 2)
    q, index = s.q.cuda(), s.index(s.table, s.table_idx, s.lens, s.qo, s.group_indptr, s.prefixes)
    good = attn.forward(q, 0, *index)
    assert_attention(good, *s.want())

    def refused(q=q, layer=0, out=None, **change):
        names = ("page_table", "table_idx", "seq_lens", "qo_indptr", "group_indptr", "prefix_lens")
        with pytest.raises(L.B200Error):
            attn.forward(q, layer, *[change.get(n, t) for n, t in zip(names, index)], out=out)

    refused(q=q.float())
    refused(q=q.cpu())
    refused(q=q[:, :8])
    refused(q=q.transpose(0, 1))
    refused(q=torch.zeros(3, 16, D + 4, dtype=bf16, device="cuda")[:, :, 4:])      # rows that are not 16-byte aligned
    refused(q=torch.zeros(4, 16, D, dtype=bf16, device="cuda"))                     # more rows than the workspace is for
    refused(layer=1)
    refused(layer=-1)
    refused(out=good[:2])
    refused(out=good.float())
    refused(page_table=index[0].long())
    refused(page_table=index[0].t())
    refused(table_idx=index[1][:1])
    refused(seq_lens=index[2].cpu())
    refused(qo_indptr=index[3][:2])
    refused(group_indptr=index[4][:1])
    refused(prefix_lens=index[5].expand(2).contiguous())
    with pytest.raises(L.B200Error):
        L.SharedPrefixAttention(s.cache(L), 16, 4, D, 3, 2)
    with pytest.raises(L.B200Error):
        L.SharedPrefixAttention(s.cache(L), 16, 8, D, 3, 1025)
    assert torch.equal(attn.forward(q, 0, *index), good)


@pytest.mark.parametrize("page", [1, 16])
@pytest.mark.parametrize("rows", [1, 3])
def test_shared_prefix_most_heads(L, page, rows):
    """Sixteen query heads on each of eight KV heads: the rows kernel's largest shared memory."""
    s = SharedSetup([[(9, rows), (130, 1)], [(40, rows)]], [300, 0], page, 128, 8, seed=19)
    assert_attention(s.run(L), *s.want())
    assert L.read_device_status() == (0, 0)


def test_shared_prefix_queries_of_any_strides(L):
    """Heads outside, tokens inside; and rows that are part of wider ones, heads too."""
    s = SharedSetup([[(20, 2), (30, 5), (9, 3)], [(700, 1)]], [140, 0], 16, 16, 8, seed=20)
    want = s.want()
    attn = L.SharedPrefixAttention(s.cache(L), 16, 8, D, s.q.shape[0], 4)
    turned = s.q.transpose(0, 1).contiguous().cuda().transpose(0, 1)
    assert turned.stride(0) < turned.stride(1)
    wide = torch.full((s.q.shape[0] + 1, 18, D + 8), float("nan"), dtype=bf16, device="cuda")
    wide[1:, 1:17, 8:] = s.q.cuda()
    for q in (turned, wide[1:, 1:17, 8:]):
        assert_attention(s.run(L, attn, q=q), *want)


def test_shared_prefix_calls_repeat_themselves(L):
    """Which CTA does which item changes from call to call, the result does not."""
    for groups, prefixes, heads, kv_heads in (([[(1 + 13 * i % 300, 1 + i % 4) for i in range(60)]], [3000], 32, 8),
                                              ([[(1, 1), (900, 2)], [(5000, 1)]], [9000, 0], 8, 1)):
        s = SharedSetup(groups, prefixes, 16, heads, kv_heads, seed=22)
        attn = L.SharedPrefixAttention(s.cache(L), heads, kv_heads, D, s.q.shape[0], len(s.reqs))
        q, index = s.q.cuda(), s.index(s.table, s.table_idx, s.lens, s.qo, s.group_indptr, s.prefixes)
        other, busy = torch.cuda.Stream(), torch.randn(4096, 4096, device="cuda")
        first = attn.forward(q, 0, *index)
        for i in range(20):
            if i % 3 == 1:   # other work holds some of the SMs
                with torch.cuda.stream(other):
                    torch.mm(busy, busy)
            assert torch.equal(attn.forward(q, 0, *index), first)


# ---- probabilities ----------------------------------------------------------------------------------------------

def _logits(rows, vocab, seed, spread=2.0, step=0.0):
    x = torch.randn(rows, vocab, generator=torch.Generator().manual_seed(seed)) * spread
    if step:
        x = (x / step).round() * step
    return x.to(bf16)


def _f32(v):
    return torch.tensor(v, dtype=torch.float32, device="cuda")


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("vocab", [1, 2, 7, 64, 1000, 4099, 32000, 50257, 128256, 151936, 327680])
@pytest.mark.parametrize("filters", ["", "k", "p", "kp"])
def test_sampling_probs(L, vocab, filters):
    rows = 5
    x = _logits(rows, vocab, vocab + len(filters), step=0.5 if vocab % 2 else 0.0)   # (odd ones: many equal logits)
    t = [0.7, 1.0, 0.3, 2.0, 1e-6]
    k = [1, 40, 7, 2 ** 30, 3] if "k" in filters else None
    p = [0.9, 0.5, 1.0, 0.99, 0.1] if "p" in filters else None
    got = L.sampling_probs(x.cuda(), _f32(t), None if k is None else _i32(k), None if p is None else _f32(p))
    want = probs_oracle(x, np.asarray(t, np.float32), k, None if p is None else np.asarray(p, np.float32))
    assert bool(((got.cpu() > 0) == (want > 1e-37)).all()) or filters == ""
    assert_probs(got, want)


@pytest.mark.parametrize("rows", [1, 3, 40, 200])
def test_sampling_probs_rows_and_strides(L, rows):
    vocab = 9001
    wide = _logits(rows, vocab + 13, rows).cuda()
    for x in (wide[:, :vocab], wide[:, 5:5 + vocab], wide[:, :9000], wide[:, 8:9008]):
        t, k, p = [0.8] * rows, [50] * rows, np.asarray([0.95] * rows, np.float32)
        assert_probs(L.sampling_probs(x, _f32(t), _i32(k), _f32(p.tolist())), probs_oracle(x.cpu(), np.asarray(t, np.float32), k, p))
        assert_probs(L.sampling_probs(x, _f32(t)), probs_oracle(x.cpu(), np.asarray(t, np.float32)))


@pytest.mark.parametrize("vocab", [24, 8200, 40000, 100001])
def test_sampling_probs_ties(L, vocab):
    """Equal logits everywhere: what is kept is decided by index alone, across threads and CTAs."""
    k = [1, 5, vocab // 2, vocab - 1, vocab, 17]
    p = np.asarray([1, 1, 1, 0.4999, 0.7501, 0.25], np.float32)
    x = torch.full((6, vocab), 1.5, dtype=bf16)
    x[5, 1::2] = -2.0
    t = np.ones(6, np.float32)
    assert_probs(L.sampling_probs(x.cuda(), _f32(t.tolist()), _i32(k), _f32(p.tolist())), probs_oracle(x, t, k, p))


@pytest.mark.parametrize("filtered", [False, True])
def test_sampling_probs_odd_values(L, filtered):
    """Infinities, NaN, both zeros, the type's ends, rows with nothing to choose from, odd temperatures."""
    inf, nan, big = float("inf"), float("nan"), float(torch.finfo(bf16).max)
    vocab = 70
    rows = [[-inf] * vocab, [nan] * vocab, [-inf] * 69 + [3.0], [inf] * 3 + [1.0] * 67, [nan, 2.0] * 35, [-big] * 70, [big, -big] * 35,
            [0.0, -0.0] * 35, [-inf] * 70, [1.0, nan] * 35]
    x = torch.tensor(rows).to(bf16)
    t = [1.0, 1.0, 0.5, 1.0, 1.0, 2.0, 1.0, 1.0, 1e-6, inf]
    k = [8, 8, 8, 2, 9, 11, 30, 3, 4, 5] if filtered else None
    p = [0.9, 0.5, 0.9, 1.0, 0.55, 1.0, 0.35, 1.0, 1.0, 0.9] if filtered else None
    got = L.sampling_probs(x.cuda(), _f32(t), None if k is None else _i32(k), None if p is None else _f32(p))
    assert_probs(got, probs_oracle(x, np.asarray(t, np.float32), k, None if p is None else np.asarray(p, np.float32)))
    cold = L.sampling_probs(x.cuda(), _f32([nan, -1.0, 0.0] + [1e-6] * 7), None if k is None else _i32(k))
    assert_probs(cold, probs_oracle(x, np.zeros(10, np.float32)))
    extreme = L.sampling_probs(x[:6].cuda(), _f32([1.0] * 6), _i32([0, -3, 71, 2 ** 31 - 1, 70, 1]), _f32([0.0, -1.0, 2.0, nan, 1.0, 0.0]))
    want = probs_oracle(x[:6], np.ones(6, np.float32), [0, -3, 71, 2 ** 31 - 1, 70, 1], np.asarray([0, -1, 2, 2, 1, 0], np.float32))
    assert_probs(extreme, want)


@pytest.mark.parametrize("vocab", [9000, 9001, 70000])
def test_sampling_probs_masked_vocabulary(L, vocab):
    """Most of the vocabulary at the type's lowest number, or at -inf; all of it; and temperatures from nearly 0 to nearly infinite."""
    low = float(torch.finfo(bf16).min)
    for mask in (low, -float("inf"), -1e4):
        x = _logits(7, vocab, vocab)
        keep = torch.zeros(vocab, dtype=torch.bool)
        keep[5::vocab // 40] = True
        x[:, ~keep] = mask
        x[6] = mask
        t = [0.7, 1.0, 2e-6, 1e-5, 1e6, 1e38, 1.0]
        for k, p in ((None, None), ([50] * 7, None), ([3] * 7, [0.9] * 7), (None, [0.6] * 7), ([1000] * 7, [0.95] * 7)):
            got = L.sampling_probs(x.cuda(), _f32(t), None if k is None else _i32(k), None if p is None else _f32(p))
            want = probs_oracle(x, np.asarray(t, np.float32), k, None if p is None else np.asarray(p, np.float32))
            assert_probs(got, want)


@pytest.mark.parametrize("vocab", [70, 430, 9000, 9001, 70000])
@pytest.mark.parametrize("mask", [-3.3895313892515355e38, -3e33, -1e30, -1e12, -1e10, -5e9, -1e8])
def test_sampling_probs_masked_by_low_numbers_at_any_temperature(L, vocab, mask):
    """Stretches of low numbers ahead of the row's largest, whose scaled values are far from any fp32 exponent; some rows all of
    them."""
    t = [1.0, 1.2, 1.45, 1.5, 1.6, 1.7, 1.9, 2.0, 2.5, 3.0, 5.0, 10.0, 33.0, 1e3, 1e4, 3e5, 0.7, 2e-6]
    x = _logits(len(t), vocab, vocab)
    x[:, :-vocab // 40] = mask
    x[::5] = mask
    x[1::5, vocab // 2] = 3.0
    want = probs_oracle(x, np.asarray(t, np.float32))
    assert_probs(L.sampling_probs(x.cuda(), _f32(t)), want)
    assert_probs(L.sampling_probs(x.cuda(), _f32(t), _i32([0] * len(t)), _f32([1.0] * len(t))), want)


def test_sampling_probs_is_what_sample_draws_from(L):
    """The kept set is b200_sample's candidate set (rows whose border is not within its 40-bit sums' reach)."""
    rows, vocab = 32, 32000
    x, t, k, p = _logits(rows, vocab, 77), [0.9] * rows, [300] * rows, [0.9] * rows
    got = L.sampling_probs(x.cuda(), _f32(t), _i32(k), _f32(p))
    _, mask = L.sample(x.cuda(), _f32(t), _i32(k), _f32(p), return_mask=True)
    assert int(((got > 0) != (mask > 0)).sum()) <= 1


# ---- verification -----------------------------------------------------------------------------------------------

def _drafted(counts, vocab, seed, lookup=False, near=0.5):
    gen = torch.Generator().manual_seed(seed)
    total, batch = sum(counts), len(counts)
    indptr = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    before = torch.randn(total, vocab, generator=gen) * 2
    rows = torch.tensor([int(indptr[b]) + b + j for b, n in enumerate(counts) for j in range(n)], dtype=torch.long)
    logits = torch.randn(total + batch, vocab, generator=gen) * 2
    logits[rows] = before + near * torch.randn(total, vocab, generator=gen)
    target, draft = torch.softmax(logits, -1), torch.softmax(before, -1)
    tokens = draft.multinomial(1, generator=gen)[:, 0].to(torch.int32) if total else torch.zeros(0, dtype=torch.int32)
    return {"target": target, "draft": None if lookup else draft, "tokens": tokens, "indptr": torch.from_numpy(indptr),
            "accept": torch.rand(total, generator=gen), "draw": torch.rand(batch, generator=gen), "most": max(counts + [0])}


def _verify(L, s, cuda=None):
    d = {k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in s.items()} if cuda is None else cuda
    return L.verify_drafts(d["target"], d["tokens"], d["indptr"], d["accept"], d["draw"], d["most"], draft_probs=d["draft"])


def _same(got, want):
    assert torch.equal(got[1].cpu(), want[1]), f"accepted {got[1].tolist()} for {want[1].tolist()}"
    assert torch.equal(got[0].cpu(), want[0]), f"{int((got[0].cpu() != want[0]).sum())} tokens differ"


@pytest.mark.parametrize("vocab", [1, 2, 31, 1000, 4099, 32000, 50001, 151936])
@pytest.mark.parametrize("counts,lookup", [([4], False), ([0], False), ([3, 0, 5, 1], False), ([3, 0, 5, 1], True), ([2] * 50, False),
                                           ([40, 0, 33], False)])
def test_verify_drafts(L, vocab, counts, lookup):
    s = _drafted(counts, vocab, vocab + len(counts), lookup, near=0.05 if max(counts) > 9 else 0.5)
    _same(_verify(L, s), verify_oracle(**s))
    assert L.read_device_status() == (0, 0)


def test_verify_drafts_edges(L):
    """Equal distributions are always accepted; a draft the target excludes never; a target that is nowhere above the draft."""
    vocab = 5000
    s = _drafted([3] * 8, vocab, 5, near=0.0)
    s["accept"][:] = 0.99999994
    rows = [3 * b + b + j for b in range(8) for j in range(3)]
    s["draft"] = s["target"][rows].clone()
    got = _verify(L, s)
    _same(got, verify_oracle(**s))
    assert got[1].tolist() == [3] * 8
    s["target"][rows, s["tokens"].long()] = 0.0
    s["accept"][:] = 0.0
    got = _verify(L, s)
    _same(got, verify_oracle(**s))
    assert got[1].tolist() == [0] * 8
    s["target"] *= 0.5      # p < q throughout: the token is drawn from p
    s["accept"][:] = 0.9
    _same(_verify(L, s), verify_oracle(**s))
    s["target"][:] = 0.0    # nothing to draw from
    got = _verify(L, s)
    _same(got, verify_oracle(**s))
    assert got[0][:, 0].tolist() == [0] * 8


def test_verify_drafts_draws_at_the_ends(L):
    vocab = 3000
    s = _drafted([0] * 6, vocab, 6)
    s["target"][:, :7] = 0.0
    s["target"][:, -9:] = 0.0
    s["draw"] = torch.tensor([0.0, 0.99999994, 1.0, -1.0, float("nan"), 2.0])
    got = _verify(L, s)
    _same(got, verify_oracle(**s))
    assert got[0][0, 0] == 7 and got[0][1, 0] == vocab - 10


@pytest.mark.parametrize("vocab", [4096, 131072])
def test_verify_drafts_draws_between_runs_of_the_row(L, vocab):
    """1, 2^-53, 2^-53, 1 at places all over the row and u = 1/2: the goal is 1 + 2^-53, or 1 where the sum of all is rounded to 2.
    However the sums are grouped, one of the four places is drawn."""
    for step in (1, 33, 128, 512, 520, 1024, vocab // 8):
        at = [5, vocab // 8, vocab // 8 + step, vocab // 8 + 2 * step]
        p = torch.zeros(1, vocab)
        p[0, at] = torch.tensor([1.0, 2.0 ** -53, 2.0 ** -53, 1.0])
        tokens, accepted = L.verify_drafts(p.cuda(), _i32([]), _i32([0, 0]), _f32([]), _f32([0.5]), 0)
        assert int(accepted[0]) == 0 and int(tokens[0, 0]) in at, (step, tokens)


def test_verify_drafts_odd_values(L):
    vocab = 600
    s = _drafted([2, 3, 1], vocab, 7)
    for name, at in (("target", 3), ("draft", 5)):
        s[name][:, at::7] = float("nan")
        s[name][:, at + 1::7] = -0.25
    _same(_verify(L, s), verify_oracle(**s))


def test_verify_drafts_tokens_outside_the_vocabulary(L):
    for lookup in (False, True):
        s = _drafted([3, 2], 400, 8, lookup)
        s["tokens"][1], s["tokens"][3] = 400, -7
        s["accept"][:] = 0.0
        _same(_verify(L, s), verify_oracle(**s))
        assert L.read_device_status()[1] in (401, -6)
        s["tokens"][1], s["tokens"][3] = -1, 2
        _same(_verify(L, s), verify_oracle(**s))
        assert L.read_device_status()[1] == -2 ** 31


def test_verify_drafts_strides_and_fewer_than_brought(L):
    s = _drafted([5, 2, 4], 1001, 9)
    want = verify_oracle(**s)
    d = {k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in s.items()}
    for pad in (3, 23):
        wide = torch.full((14, 1001 + pad), float("nan"), device="cuda")
        wide[:, :1001] = d["target"]
        narrow = torch.full((11, 1001 + pad + 5), float("nan"), device="cuda")
        narrow[:, 2:1003] = d["draft"]
        _same(_verify(L, s, {**d, "target": wide[:, :1001], "draft": narrow[:, 2:1003]}), want)
    for most in (0, 1, 3):
        few = {**s, "most": most}
        _same(_verify(L, few), verify_oracle(**few))
    many = {**s, "most": 70}
    _same(_verify(L, many), verify_oracle(**many))


def test_verify_drafts_draws_from_the_target(L):
    """The first token of a step is distributed as the target's first row says, whatever drafted it (five standard deviations)."""
    vocab, batch = 6, 40000
    gen = torch.Generator().manual_seed(10)
    p, q = torch.softmax(torch.randn(vocab, generator=gen), 0), torch.softmax(torch.randn(vocab, generator=gen), 0)
    after = torch.full((vocab,), 1.0 / vocab)
    target = torch.stack([p, after]).repeat(batch, 1).cuda()
    tokens = q.expand(batch, vocab).multinomial(1, generator=gen)[:, 0].to(torch.int32)
    got, accepted = L.verify_drafts(target, tokens.cuda(), torch.arange(batch + 1, dtype=torch.int32).cuda(),
                                    torch.rand(batch, generator=gen).cuda(), torch.rand(batch, generator=gen).cuda(), 1,
                                    draft_probs=q.expand(batch, vocab).contiguous().cuda())
    share = torch.bincount(got[:, 0].cpu().long(), minlength=vocab).double() / batch
    assert bool(((share - p.double()).abs() < 5 * (p.double() * (1 - p.double()) / batch).sqrt()).all())
    assert abs(float(accepted.double().mean()) - float(torch.minimum(p, q).sum())) < 5 * 0.5 / batch ** 0.5


def test_verify_drafts_captured(L):
    s = _drafted([3, 0, 5, 1], 4099, 11)
    d = {k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in s.items()}
    _verify(L, s, d)
    graph = torch.cuda.CUDAGraph()
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        got = _verify(L, s, d)
    for seed in (11, 12, 13):
        s = _drafted([3, 0, 5, 1], 4099, seed)
        for k in ("target", "draft", "tokens", "accept", "draw"):
            d[k].copy_(s[k])
        graph.replay()
        torch.cuda.synchronize()
        _same(got, verify_oracle(**s))


# ---- together ---------------------------------------------------------------------------------------------------

def test_a_drafted_step(L):
    """A step as a server runs it: rows of drafted tokens over a shared prompt, the output head, the probabilities behind
    temperature, top-k and top-p, and what of the drafts stands; captured and replayed as well.  Each operator is checked on what the
    one before it returned."""
    vocab, counts = 4096, [3, 0, 5, 1, 2, 4]
    rows = [n + 1 for n in counts]
    s = SharedSetup([[(10 + 3 * i, rows[i]) for i in range(4)], [(9, rows[4]), (40, rows[5])]], [333, 64], 16, 16, 8, seed=21)
    gen = torch.Generator().manual_seed(22)
    head = (torch.randn(vocab, 16 * D, generator=gen) * 0.3).to(bf16).cuda()
    total, batch = sum(counts), len(counts)
    indptr = _i32(np.concatenate([[0], np.cumsum(counts)]).tolist())
    of_row = [b for b, n in enumerate(rows) for _ in range(n)]
    t, k, p = ([[0.7, 1.0, 0.9, 1e-6, 1.3, 0.8][b] for b in of_row], [[50, 2 ** 30, 20, 5, 200, 100][b] for b in of_row],
               [[0.95, 0.9, 1.0, 1.0, 0.8, 0.99][b] for b in of_row])
    tt, kk, pp = _f32(t), _i32(k), _f32(p)
    accept, draw = torch.rand(total, generator=gen), torch.rand(batch, generator=gen)
    attn = L.SharedPrefixAttention(s.cache(L), 16, 8, D, sum(rows), batch)
    index = s.index(s.table, s.table_idx, s.lens, s.qo, s.group_indptr, s.prefixes)
    q, accept_d, draw_d = s.q.cuda(), accept.cuda(), draw.cuda()
    # drafts that the target half believes in: from its own probabilities, blurred
    out0 = attn.forward(q, 0, *index)
    probs0 = L.sampling_probs(L.linear(out0, head), tt, kk, pp).cpu()
    at = [int(indptr[b]) + b + j for b, n in enumerate(counts) for j in range(n)]
    draft = 0.7 * probs0[at] + 0.3 / vocab
    tokens = draft.multinomial(1, generator=gen)[:, 0].to(torch.int32)
    draft_d, tokens_d = draft.cuda(), tokens.cuda()

    def step():
        out = attn.forward(q, 0, *index)
        logits = L.linear(out, head)
        probs = L.sampling_probs(logits, tt, kk, pp)
        return out, logits, probs, *L.verify_drafts(probs, tokens_d, indptr, accept_d, draw_d, max(counts), draft_probs=draft_d)

    def check(got):
        out, logits, probs, said, stood = (x.cpu() for x in got)
        assert_attention(out, *s.want())
        assert_probs(probs, probs_oracle(logits, np.asarray(t, np.float32), k, np.asarray(p, np.float32)))
        _same((said, stood), verify_oracle(probs, draft, tokens, indptr, accept, draw, max(counts)))

    eager = step()
    check(eager)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        captured = step()
    graph.replay()
    torch.cuda.synchronize()
    check(captured)
    assert all(torch.equal(a, b) for a, b in zip(eager, captured))
