"""Attention over a shared prefix: every key of long rows is weighed once, whatever items, stages, tiles, chunks and parts it falls into
(tests/shared_prefix_counts.py).  Rows of more parts than one round of the joining takes are among them."""
import pytest
import torch

from tests.shared_prefix_cases import D, assert_attention
from tests.shared_prefix_counts import CountedSetup, parts_of_rows

pytestmark = pytest.mark.gpu

# groups, prefixes, page, query heads, KV heads, and the parts that some row has at least (on 148 SMs)
CASES = {
    # a row's parts by sixteen warps, by four and (rows of dozens of parts among many) by eight: 32 for each warp in a round
    "sixteen warps, second round": ([[(1, 1), (2, 1)]], [32768], 16, 8, 1, 32 * 16 + 1),
    "four warps, second round": ([[(3 + i, 1) for i in range(29)], [(20001, 1)]], [130, 0], 16, 8, 1, 32 * 4 + 1),
    "four warps, second round, two KV heads": ([[(3 + i, 1) for i in range(20)], [(16000, 2)]], [130, 0], 16, 16, 2, 32 * 4 + 1),
    "a CTA of eight, second round": ([[(1 + i % 40, 1) for i in range(80)], [(17000, 1)]], [100, 0], 16, 8, 1, 32 * 8 + 1),
    # half a warp: 16 in a round
    "half a warp, second round": ([[(380 + i % 40, 1) for i in range(80)]], [700], 16, 8, 1, 17),
    "few rows, hundreds of parts": ([[(1, 1), (2, 1)], [(12000, 1)]], [30000, 0], 16, 16, 8, 100),
    "a prefix that ends inside a page and a stage": ([[(130, 2), (1, 1), (77, 3)]], [9001], 16, 16, 8, 30),
    "pages of one token": ([[(1, 1), (300, 1)]], [5003], 1, 8, 2, 10),
    "a wide group behind a long prefix": ([[(1 + 7 * i % 90, 1) for i in range(40)]], [20011], 16, 8, 1, 20),
    "a wide group, two chains": ([[(5, 3), (40, 2)] * 16], [6007], 16, 32, 4, 5),
    "a wide group, pages of one token": ([[(5, 3), (40, 2)] * 8], [3001], 1, 32, 8, 5),
    "long continuations": ([[(3000 + 17 * i, 1 + i % 2) for i in range(6)]], [1500], 64, 32, 8, 5),
    "more units than chunks": ([[(3, 1)] * 20, [(9, 2)] * 30, [(2, 1)] * 33, [(4, 3)] * 12, [(1, 1)] * 40], [2500, 129, 4000, 1111, 300], 16, 32, 8, 2),
}


@pytest.mark.parametrize("name", CASES)
def test_every_key_counts_once(L, name):
    groups, prefixes, page, heads, kv_heads, least = CASES[name]
    s = CountedSetup(groups, prefixes, page, heads, kv_heads, seed=len(name))
    cache = s.cache(L)
    attn = L.SharedPrefixAttention(cache, heads, kv_heads, D, s.q.shape[0], len(s.reqs))
    q, index = s.q.cuda(), s.index(s.table, s.table_idx, s.lens, s.qo, s.group_indptr, s.prefixes)
    weights = s.weights()
    for turn in range(s.passes):
        cache.kv_buffer_[1, 0, s.low:].copy_(s.values(turn))
        got = attn.forward(q, 0, *index)
        want = s.shares(weights, turn)
        assert_attention(got, want, want)
    assert L.read_device_status() == (0, 0)
    parts = parts_of_rows(attn, s.q.shape[0], len(s.reqs), len(groups), torch.cuda.get_device_properties(0).multi_processor_count)
    assert max(parts) >= least, (max(parts), least)
