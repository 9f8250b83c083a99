"""What attention over whole prompts and the operators on cache pages refuse (checked before any CUDA call), and their plain forms on cases
worked out by hand."""
import ctypes
import math

import numpy as np
import pytest
import torch

from tests.prompt_pages_cases import PromptSetup, compact_oracle, copy_oracle, count_oracle, fork_oracle

P = ctypes.c_void_p(256)   # never dereferenced: the calls below are refused


def _prompt(pkg, **change):
    from sglang_cpp_b200 import _lib
    a = dict(out=256, lse=None, q=256, k=256, v=256, q_stride_token=4096, q_stride_head=128, k_stride_token=4096, k_stride_head=128,
             v_stride_token=4096, v_stride_head=128, indptr=256, tokens=9, batch=2, q_heads=16, kv_heads=8, head_dim=128, sm_scale=0.1)
    a.update(change)
    lib = pkg.load_library()
    rc = lib.b200_attention_prompt(ctypes.byref(_lib.PromptAttentionArgs(**a)), None)
    return rc, lib.b200_last_error().decode()


@pytest.mark.parametrize("change,text", [
    (dict(head_dim=136), "head_dim"), (dict(head_dim=0), "head_dim"), (dict(head_dim=60), "head_dim"), (dict(batch=1025), "batch"),
    (dict(batch=-1), "batch"), (dict(tokens=-1), "tokens"), (dict(kv_heads=0), "kv_heads"), (dict(kv_heads=3), "q_heads"), (dict(q_heads=0), "q_heads"),
    (dict(q_heads=129, kv_heads=1), "q_heads"), (dict(q_stride_token=4100), "strides"), (dict(q_stride_head=0), "strides"),
    (dict(k_stride_token=-4096), "strides"), (dict(k_stride_head=4), "strides"), (dict(v_stride_token=1 << 40), "strides"), (dict(v_stride_head=129), "strides"),
    (dict(sm_scale=0.0), "sm_scale"), (dict(sm_scale=-1.0), "sm_scale"), (dict(sm_scale=float("nan")), "sm_scale"), (dict(sm_scale=float("inf")), "sm_scale"),
    (dict(tokens=1 << 28), "too many"), (dict(out=None), "NULL"), (dict(q=None), "NULL"), (dict(k=None), "NULL"), (dict(v=None), "NULL"),
    (dict(indptr=None), "NULL"), (dict(out=264), "aligned"), (dict(q=264), "aligned"), (dict(k=258), "aligned"), (dict(v=260), "aligned"),
])
def test_prompt_attention_refusals(pkg, change, text):
    rc, said = _prompt(pkg, **change)
    assert rc == 1 and text in said, (rc, said)


def test_prompt_attention_null_arguments_and_nothing_to_do(pkg):
    assert pkg.load_library().b200_attention_prompt(None, None) == 1
    assert _prompt(pkg, batch=0)[0] == 0
    assert _prompt(pkg, tokens=0)[0] == 0


POOL = dict(planes=256, plane_stride=1 << 20, num_planes=4, slot_bytes=256, page_size=16, num_pages=64)


def _pool(**change):
    from sglang_cpp_b200 import _lib
    return ctypes.byref(_lib.PagePool(**{**POOL, **change}))


def _calls(lib, pool, **change):
    """Each of the calls on a pool, with arguments that it would take."""
    a = dict(src=P, dst=P, tokens=None, copies=4, table=P, rows=8, stride=128, cols=100, parents=P, children=P, lens=P, new=P, count=4, which=P,
             held=None, held_count=0, out=P, out_stride=128, map=P, used=P, refs=P, free=P, free_count=P, page_size=16, num_pages=64, ws=P,
             ws_bytes=1 << 20)
    a.update(change)
    g = lambda names: [a[n] for n in names.split()]
    return {
        "copy": lambda: lib.b200_copy_pages(pool, *g("src dst tokens copies ws ws_bytes"), None),
        "fork": lambda: lib.b200_fork_rows(pool, *g("table rows stride cols parents children lens new count"), None),
        "count": lambda: lib.b200_count_pages(*g("refs free free_count table rows stride cols which lens count held held_count page_size num_pages ws ws_bytes"), None),
        "compact": lambda: lib.b200_compact_pages(pool, *g("out out_stride map used table rows stride cols which lens count held held_count ws ws_bytes"), None),
    }


@pytest.mark.parametrize("call", ["copy", "fork", "compact"])
@pytest.mark.parametrize("change,text", [
    (dict(planes=None), "planes"), (dict(planes=264), "aligned"), (dict(plane_stride=(1 << 20) + 8), "plane_stride"), (dict(plane_stride=16 * 64 * 256 - 16), "plane_stride"),
    (dict(num_planes=0), "num_planes"), (dict(num_planes=1 << 26), "num_planes"), (dict(slot_bytes=0), "slot_bytes"), (dict(slot_bytes=24), "slot_bytes"),
    (dict(page_size=0), "page_size"), (dict(num_pages=0), "num_pages"), (dict(page_size=1 << 26), "2^31"),
])
def test_pool_refusals(pkg, call, change, text):
    lib = pkg.load_library()
    assert _calls(lib, _pool(**change))[call]() == 1 and text in lib.b200_last_error().decode()
    assert _calls(lib, None)[call]() == 1 and "NULL pool" in lib.b200_last_error().decode()


@pytest.mark.parametrize("call,change,text", [
    ("copy", dict(copies=-1), "count"), ("copy", dict(copies=65), "count"), ("copy", dict(src=None), "NULL"), ("copy", dict(dst=None), "NULL"),
    ("copy", dict(ws=None), "workspace"), ("copy", dict(ws_bytes=100), "workspace"),
    ("fork", dict(count=-1), "count"), ("fork", dict(count=1025), "count"), ("fork", dict(table=None), "NULL"), ("fork", dict(parents=None), "NULL"),
    ("fork", dict(children=None), "NULL"), ("fork", dict(lens=None), "NULL"), ("fork", dict(new=None), "NULL"), ("fork", dict(stride=99), "overlap"),
    ("fork", dict(rows=-1), "table"), ("fork", dict(cols=-1), "table"), ("fork", dict(cols=1 << 31, stride=1 << 31), "table"),
    ("count", dict(refs=None), "NULL"), ("count", dict(free=None), "NULL"), ("count", dict(free_count=None), "NULL"), ("count", dict(table=None), "NULL"),
    ("count", dict(which=None), "NULL"), ("count", dict(lens=None), "NULL"), ("count", dict(count=-1), "count"), ("count", dict(held_count=-1), "count"),
    ("count", dict(held_count=3), "NULL"), ("count", dict(page_size=0), "page_size"), ("count", dict(num_pages=0), "num_pages"),
    ("count", dict(num_pages=1 << 28), "2^31"), ("count", dict(ws=None), "workspace"), ("count", dict(ws_bytes=64), "workspace"), ("count", dict(stride=50), "overlap"),
    ("compact", dict(map=None), "NULL"), ("compact", dict(used=None), "NULL"), ("compact", dict(out=None), "NULL"), ("compact", dict(out_stride=99), "overlap"),
    ("compact", dict(table=None), "NULL"), ("compact", dict(which=None), "NULL"), ("compact", dict(lens=None), "NULL"), ("compact", dict(count=-1), "count"),
    ("compact", dict(held_count=2), "NULL"), ("compact", dict(ws=None), "workspace"), ("compact", dict(ws_bytes=512), "workspace"),
])
def test_page_refusals(pkg, call, change, text):
    lib = pkg.load_library()
    assert _calls(lib, _pool(), **change)[call]() == 1 and text in lib.b200_last_error().decode(), lib.b200_last_error()


def test_page_calls_of_nothing(pkg):
    lib = pkg.load_library()
    assert _calls(lib, _pool(), copies=0, src=None, dst=None)["copy"]() == 0
    assert _calls(lib, _pool(), count=0, parents=None, children=None)["fork"]() == 0


def test_pages_workspace_sizes(pkg):
    size = pkg.load_library().b200_pages_workspace_bytes
    assert size(1) > 0 and size(0) == -1 and size(-5) == -1
    sizes = [size(n) for n in (1, 31, 32, 33, 1000, 1 << 20)]
    assert sizes == sorted(sizes) and size(1 << 20) < 32 << 20


def test_oracles_on_known_answers():
    s = PromptSetup([1, 2], 2, 1, 8, seed=1)
    out, size, lse, _ = s.want()
    q, k, v = (x.double() for x in s.parts(s.rows))
    assert torch.allclose(out[0], v[0].expand(2, 8)) and torch.allclose(lse[0], (q[0] * k[0]).sum(-1) / math.sqrt(8))
    assert torch.allclose(out[1], v[1].expand(2, 8))
    a, b = ((q[2] * k[j]).sum(-1) / math.sqrt(8) for j in (1, 2))
    w = torch.sigmoid(a - b)[:, None]
    assert torch.allclose(out[2], w * v[1] + (1 - w) * v[2]) and torch.allclose(lse[2], torch.logaddexp(a, b))

    kv = torch.arange(12).reshape(1, 1, 12, 1, 1).expand(2, 1, 12, 1, 1).clone()
    # page 0 -> 2; 1 -> 3 twice named; 4 -> 5 whose page is read by the last pair, which writes page 1 (read by the second and third)
    got, left = copy_oracle(kv, 2, 6, [0, 1, 1, 4, 5, -1, 7], [2, 3, 3, 5, 1, 0, 0])
    assert got[0, 0, :, 0, 0].tolist() == [0, 1, 2, 3, 0, 1, 6, 7, 8, 9, 10, 11] and left == {3, 5, 1}
    got, left = copy_oracle(kv, 2, 6, [0, 1], [2, 3], [1, 0])
    assert got[0, 0, :, 0, 0].tolist() == [0, 1, 2, 3, 0, 5, 6, 7, 8, 9, 10, 11] and not left

    table = np.full((4, 6), -1, np.int32)
    table[0, :4] = [4, 5, 0, 1]                    # pages 2 and 0
    got, t, left = fork_oracle(kv, table, 2, 6, [0, 0], [1, 3], [3, 2], [4, 9])
    assert t[1].tolist() == [4, 5, 8, 9, -1, -1] and t[3].tolist() == [4, 5, -1, -1, -1, -1] and not left
    assert got[0, 0, 8:10, 0, 0].tolist() == [0, 9]

    refs, free, n = count_oracle(t, [0, 1, 3], [4, 3, 1], 2, 6, held=[5, 0])
    assert refs.tolist() == [2, 0, 3, 0, 1, 1] and free.tolist() == [1, 3, -1, -1, -1, -1] and n == 2
    got, t2, where, used = compact_oracle(got, t, [0, 1, 3], [4, 3, 1], 2, 6, held=[5, 0])
    assert used == 4 and where.tolist() == [0, -1, 2, -1, 1, 3]
    assert t2[1].tolist() == [4, 5, 2, 3, -1, -1] and got[0, 0, 2:4, 0, 0].tolist() == [0, 9] and got[0, 0, 6:8, 0, 0].tolist() == [10, 11]


def _batcher(pkg, page, pages=40, rows=8):
    from sglang_cpp_b200.host_batch import HostBatcher
    return HostBatcher(None, pages, page, rows, max_seq_len=64)


@pytest.mark.parametrize("page", [1, 4, 16])
@pytest.mark.parametrize("length", [21, 32])
def test_forked_requests_share_whole_pages(pkg, page, length):
    hb = _batcher(pkg, page, pages=128 // page)
    r = hb.add_request(np.arange(length), 20)
    hb.allocate([r])
    r.complete_one()
    hb.tables.token_pool[r.table_idx, length] = 77
    free = len(hb.cache_manager.free_pages)
    kids = hb.fork(r, 3)
    full, part = length // page * page, length % page
    assert free - len(hb.cache_manager.free_pages) == (3 if part else 0)
    mine = hb.slots_of(r)
    own = set()
    for k in kids:
        row = hb.slots_of(k)
        assert np.array_equal(row[:full], mine[:full]) and k.cached_len == length and k.device_len == length + 1
        assert np.array_equal(hb.tables.token_pool[k.table_idx, :length + 1], list(range(length)) + [77])
        if part:
            assert row[full] % page == 0 and np.array_equal(row[full:full + page], np.arange(row[full], row[full] + page))
            own.add(int(row[full]))
    assert len(own) == (3 if part else 0) and not own & set(mine[:length].tolist())
    # each goes on with tokens of its own, two of them with the same ones
    reqs = [r] + kids
    for step in range(9):
        hb.allocate(reqs)
        for i, q in enumerate(reqs):
            q.append_host_token(100 * min(i, 2) + step)
            q.complete_one()
    used = [set(hb.slots_of(q)[full:q.cached_len].tolist()) for q in reqs]
    assert all(not a & b for i, a in enumerate(used) for b in used[:i])
    for q in reqs:
        hb.release(q)
    hb.cache_manager.check_integrity()
    assert hb.cache_manager.prefix_cache.protected_size == 0 and len(hb.table_manager.free_rows) == 8


def test_fork_of_a_prompt_that_is_cached_elsewhere(pkg):
    """Two requests with one prompt in pages of their own: the second one, forked behind the first, goes over to the first one's pages."""
    hb = _batcher(pkg, 4)
    a, b = hb.add_request(np.arange(14), 9), hb.add_request(np.arange(14), 9)
    hb.allocate([a, b])
    for r in (a, b):
        r.complete_one()
    assert not set(hb.slots_of(a)[:14].tolist()) & set(hb.slots_of(b)[:14].tolist())
    x = hb.fork(a, 1) + hb.fork(b, 2)
    assert all(np.array_equal(hb.slots_of(k)[:12], hb.slots_of(a)[:12]) for k in x + [b])
    for r in [a, b] + x:
        hb.release(r)
    hb.cache_manager.check_integrity()


def test_fork_refusals(pkg):
    hb = _batcher(pkg, 16, pages=4, rows=4)
    r = hb.add_request(np.arange(20), 9)
    with pytest.raises(ValueError):
        hb.fork(r, 1)                 # nothing read yet
    hb.allocate([r])
    r.complete_one()
    for copies in (-1, 4, 3, 1025):   # (four rows, one of them taken; two free pages)
        with pytest.raises(ValueError):
            hb.fork(r, copies)
    r.complete_one()
    with pytest.raises(ValueError):
        hb.fork(r, 1)                 # a token that the host has not been told
    r.append_host_token(5)
    assert hb.fork(r, 0) == [] and len(hb.fork(r, 2)) == 2
    hb.cache_manager.enabled = False
    with pytest.raises(ValueError):
        hb.fork(r, 1)


@pytest.mark.parametrize("call,pool,change,text", [
    ("count", {}, dict(count=(1 << 20) + 1), "count"), ("count", {}, dict(count=0x7fffffff), "count"),
    ("count", {}, dict(held=P, held_count=(1 << 30) + 1), "count"), ("count", {}, dict(held=P, held_count=0x7fffffff), "count"),
    ("compact", {}, dict(count=0x7fffffff), "count"), ("compact", {}, dict(held=P, held_count=0x7fffffff), "count"),
    ("count", {}, dict(page_size=1, num_pages=(1 << 30) + 1, ws_bytes=1 << 40), "num_pages"),
    ("copy", dict(page_size=1, num_planes=1, num_pages=0x7fffffff), dict(copies=0x7fffffff, ws_bytes=1 << 40), "num_pages"),
    ("compact", dict(page_size=1, num_planes=1, num_pages=0x7fffffff), dict(ws_bytes=1 << 40), "num_pages"),
])
def test_numbers_that_loop_counters_would_pass(pkg, call, pool, change, text):
    """Counters of int go on by up to 2^22 behind the last number: 2^30 leaves room."""
    lib = pkg.load_library()
    assert _calls(lib, _pool(**pool), **change)[call]() == 1 and text in lib.b200_last_error().decode(), lib.b200_last_error()


class _Refuses:
    """An engine whose fork fails; ``stack``: one that has a pool per layer."""

    def __init__(self, cols, stack):
        self.pt_cols, self.stack, self.forks = cols, stack, 0

    def write_page_table(self, *a):
        pass

    write_token_pool = write_page_table

    def fork_rows(self, *a):
        self.forks += 1
        raise RuntimeError("no")


@pytest.mark.parametrize("stack", [False, True])
@pytest.mark.parametrize("length", [21, 32])
def test_a_fork_that_the_engine_refuses_takes_nothing(pkg, stack, length):
    from sglang_cpp_b200.host_batch import HostBatcher
    engine = _Refuses(64, stack)
    hb = HostBatcher(engine, 8, 16, 4)
    cm = hb.cache_manager
    r = hb.add_request(np.arange(length), 9)
    hb.allocate([r])
    r.complete_one()
    hb.cache_prefix(r)
    rows, pages, table, uid = list(hb.table_manager.free_rows), list(cm.free_pages), hb.tables.page_table.copy(), hb._next_uid
    protected = cm.prefix_cache.protected_size
    with pytest.raises(ValueError if stack else RuntimeError):
        hb.fork(r, 3)
    assert engine.forks == (0 if stack else 1)
    assert hb.table_manager.free_rows == rows and cm.free_pages == pages and hb._next_uid == uid
    assert cm.prefix_cache.protected_size == protected and np.array_equal(hb.tables.page_table, table)
    hb.release(r)
    cm.check_integrity()
    assert cm.prefix_cache.protected_size == 0 and len(hb.table_manager.free_rows) == 4 and not hb._held


def test_pages_workspace_of_more_pages_than_there_may_be(pkg):
    size = pkg.load_library().b200_pages_workspace_bytes
    assert size(1 << 30) > size((1 << 30) - 100_000) > 3 * 4 * ((1 << 30) - 100_000)
    assert [size(n) for n in ((1 << 30) + 1, 2 ** 31 - 2048, 2 ** 31 - 1)] == [-1] * 3


@pytest.mark.parametrize("page", [1, 4, 16])
def test_compacted_books(pkg, page):
    """Requests, forks and cached prefixes read the same contents behind a compaction, and nothing that is allocated later is theirs."""
    rng = np.random.default_rng(page)
    hb = _batcher(pkg, page, pages=320 // page, rows=10)
    cm, memory = hb.cache_manager, np.full(320, -1)

    def check(reqs):               # (a position's contents: the tokens up to it)
        for r in reqs:
            for i in range(r.cached_len):
                assert memory[hb.slots_of(r)[i]] == hash(tuple(r.input_ids[:i + 1].tolist()))

    def start(ids):
        r = hb.add_request(ids, 20)
        hb.allocate([r])
        for i in range(r.cached_len, len(ids)):
            memory[hb.slots_of(r)[i]] = hash(tuple(ids[:i + 1].tolist()))
        r.complete_one()
        hb.cache_prefix(r)
        return r

    first = [start(rng.integers(0, 99, size=n)) for n in (21, 32, 7, 18)]
    kids = hb.fork(first[1], 2) + hb.fork(first[0], 2)
    for k, parent in zip(kids, [first[1]] * 2 + [first[0]] * 2):    # the copied part page
        full = k.cached_len // page * page
        memory[hb.slots_of(k)[full:k.cached_len]] = memory[hb.slots_of(parent)[full:k.cached_len]]
    live = first + kids
    for step in range(3):
        for r in live:
            r.append_host_token(int(rng.integers(99)))
        hb.allocate(live)
        for r in live:
            memory[hb.slots_of(r)[r.cached_len]] = hash(tuple(r.input_ids.tolist()))
            r.complete_one()
        check(live)
        for r in (live.pop(0), live.pop()):
            hb.release(r)
        before = {g: memory[g * page:(g + 1) * page].copy() for g in range(cm.num_pages)}
        moved = {}
        real = cm.pages_moved
        cm.pages_moved = lambda where, *a: (moved.update(enumerate(where.tolist())), real(where, *a))
        used = hb.compact()
        del cm.pages_moved
        memory[:] = -1
        for g, to in moved.items():
            if to >= 0:
                memory[to * page:(to + 1) * page] = before[g]
        assert sorted(to for to in moved.values() if to >= 0) == list(range(used))
        assert cm.free_pages == [g * page for g in range(used, cm.num_pages)]
        check(live)
        assert hb.compact() == used                      # (nothing moves again)
        check(live)
    again = start(first[0].input_ids[:21].copy())        # from the prefix cache, in its new place
    assert again.cache_handle.cached_len >= 20 // page * page
    check(live + [again])
    for r in live + [again]:
        hb.release(r)
    cm.check_integrity()
    assert cm.prefix_cache.protected_size == 0 and hb.compact() == len(cm.cached_pages())
    with pytest.raises(ValueError):
        cm.pages_moved(np.full(cm.num_pages, -1), [], [])


def test_compaction_that_the_engine_refuses_changes_no_books(pkg):
    from sglang_cpp_b200.host_batch import HostBatcher
    engine = _Refuses(64, True)
    engine.compact_pages = lambda *a: (_ for _ in ()).throw(RuntimeError("no"))
    hb = HostBatcher(engine, 8, 16, 4)
    a, b = hb.add_request(np.arange(20), 9), hb.add_request(np.arange(50) + 3, 9)
    hb.allocate([a, b])
    for r in (a, b):
        r.complete_one()
    hb.release(a)
    table, free = hb.tables.page_table.copy(), list(hb.cache_manager.free_pages)
    with pytest.raises(RuntimeError):
        hb.compact()
    assert np.array_equal(hb.tables.page_table, table) and hb.cache_manager.free_pages == free
