"""Attention over whole prompts where values, scores and masks are odd, in both of its forms: blocks of one query tile (calls of few items) and
of two (all larger ones).  Plain forms and tolerances: tests/prompt_pages_cases.py."""
import math

import numpy as np
import pytest
import torch

from tests.prompt_pages_cases import PromptSetup, assert_prompt

pytestmark = pytest.mark.gpu
bf16 = torch.bfloat16


def in_pairs(s):
    """Whether the call takes blocks of two query tiles: where these may be more than three quarters of the SMs."""
    span = 2 * (128 // (s.heads // s.kv_heads))
    items = (s.rows.shape[0] // span + len(s.lens)) * s.kv_heads
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    return 2 * items > sms + sms // 2


def of_form(form, lens, heads, kv_heads, dim, **more):
    """The lengths as they are, or as often as it takes for blocks of two query tiles."""
    s = PromptSetup(lens, heads, kv_heads, dim, **more)
    times = 1
    while form == "two tiles" and not in_pairs(s):
        times += 1
        s = PromptSetup(list(lens) * times, heads, kv_heads, dim, **more)
    assert in_pairs(s) == (form == "two tiles")
    return s


FORMS = ["one tile", "two tiles"]


@pytest.mark.parametrize("form", FORMS)
def test_rows_of_scores_that_are_no_numbers(L, form):
    """The first key of a sequence and head is NaN: every row sees it, the first one nothing else; a value behind it is NaN as well."""
    s = of_form(form, [130, 60], 8, 4, 128, seed=1)
    want = s.want("cuda")
    _, k, v = s.parts(s.rows)
    a = s.indptr[0]
    k[a, 1] = float("nan")
    v[a + 1, 1, 3] = float("nan")
    out, lse = s.run(L)
    got, n = out.reshape(-1, 8, 128), s.lens[0]
    assert bool(torch.isnan(got[a:a + n, 2:4]).all()) and bool(torch.isnan(lse[a:a + n, 2:4]).all())
    hit = torch.zeros_like(got, dtype=torch.bool)
    hit[a:a + n, 2:4] = True
    assert_prompt((torch.where(hit, want[0].to(bf16), got), torch.where(hit.any(-1), want[2].float(), lse)), want)
    assert L.read_device_status() == (0, 0)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("dim", [128, 64, 72])
@pytest.mark.parametrize("size", [2.0 ** 90, 2.0 ** 101, 2.0 ** 120, 2.0 ** 127])
def test_large_values(L, form, dim, size):
    """Numbers up to the type's largest, where a score per tile of keys behind the first one is larger by 16 (its weight e^16 < 2^24 of the first
    ones'): the weighted sums of up to 16 tiles pass 2^128 where the means do not."""
    s = of_form(form, [2100, 140, 1] if form == "two tiles" else [2100, 7], 8, 4, dim, seed=2)
    q, k, v = s.parts(s.rows)
    q[:], k[:] = 0.0, 0.0
    q[:, :, 0] = 16.0
    for a, n in zip(s.indptr[:-1], s.lens):
        k[a + 130:a + n:131, :, 0] = math.sqrt(dim)
        k[a + 100:a + n:57, :, 0] = -math.sqrt(dim)
    x = v.float().clamp(-1.99, 1.99)
    v[:] = torch.where(x.abs() < 1.0, torch.sign(x) + x * 0.5, x).to(bf16) * size
    v[:, 0] = v[:, 0].abs()
    assert bool(torch.isfinite(v).all())
    assert_prompt(s.run(L), s.want("cuda"))
    assert L.read_device_status() == (0, 0)


@pytest.mark.parametrize("form", FORMS)
def test_mean_of_the_largest_value(L, form):
    """Equal weights of the type's largest numbers; one column has a NaN besides, from its row on."""
    s = of_form(form, [200, 90], 8, 4, 128, seed=3, q_scale=0.0)
    _, _, v = s.parts(s.rows)
    most = torch.finfo(bf16).max
    v[:] = torch.where(v.float() < 0, -most, most).to(bf16)
    v[:, 1] = most
    want = s.want("cuda")
    v[150, 1, 9] = float("nan")
    out, lse = s.run(L)
    got = out.reshape(-1, 8, 128)
    assert bool(torch.isnan(got[150:200, 2:4, 9]).all()) and bool((got[:150, 2:4] == most).all()) and bool((got[200:, 2:4] == most).all())
    hit = torch.zeros_like(got, dtype=torch.bool)
    hit[150:200, 2:4, 9] = True
    assert_prompt((torch.where(hit, want[0].to(bf16), got), lse), want)


@pytest.mark.parametrize("bad", [float("nan")])
def test_values_that_are_all_no_numbers_cost_little(L, bad):
    """Where every row is no number by its own keys, nothing is summed up again."""
    s = PromptSetup([3000, 2900], 8, 4, 128, seed=4)
    indptr = torch.from_numpy(s.indptr).cuda()

    def time(rows):
        s.run(L, rows, indptr)
        a, b = torch.cuda.Event(True), torch.cuda.Event(True)
        a.record()
        for _ in range(3):
            out, _ = s.run(L, rows, indptr)
        b.record()
        b.synchronize()
        return a.elapsed_time(b) / 3, out

    plain, _ = time(s.rows.cuda())
    for part in (2, 1):   # the values, the keys as well
        s.parts(s.rows)[part][:] = bad
        took, out = time(s.rows.cuda())
        assert bool(torch.isnan(out).all())
        assert took < 10 * plain + 1.0, (took, plain)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 4, 128), (6, 2, 64)])
@pytest.mark.parametrize("where", ["throughout", "behind the first tile", "by their scale"])
def test_scores_beyond_2_to_the_31(L, form, heads, kv_heads, dim, where):
    """Scores are exact products here, far apart or equal: a row is the mean of the values of its largest ones.  Weights are 1 or nothing: what
    is off is their sum's quotient (two roundings of 2^-24) and the output's rounding."""
    s = of_form(form, [300, 140, 60], heads, kv_heads, dim, seed=5)
    q, k, _ = s.parts(s.rows)
    gen = torch.Generator().manual_seed(6)
    size = 1.0 if where == "by their scale" else 2.0 ** 20
    q[:], k[:] = 0.0, 0.0
    q[:, :, 1] = torch.where(torch.rand(q.shape[:2], generator=gen) < 0.5, -size, size).to(bf16)
    k[:, :, 1] = (torch.randint(-3, 4, k.shape[:2], generator=gen) * size).to(bf16)
    if where == "behind the first tile":
        for a in s.indptr[:-1]:
            k[a:a + 140] = 0.0
    s.scale = 1e30 if where == "by their scale" else s.scale
    out, lse = s.run(L, sm_scale=s.scale)
    want, size, want_lse, terms = s.want("cuda")
    assert bool(torch.isfinite(out).all()) and bool(torch.isfinite(lse).all())
    assert_prompt((out, want_lse), (want, size, want_lse, torch.zeros_like(terms)))
    assert_prompt((want.to(bf16), lse), (want, size, want_lse, terms))


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("heads,kv_heads,dim", [(16, 8, 128), (8, 8, 128), (6, 2, 128), (8, 2, 64), (8, 4, 96), (8, 4, 72), (14, 2, 80)])
@pytest.mark.parametrize("bad", [float("nan"), float("-inf")])
def test_odd_values_reach_only_what_sees_them(L, form, heads, kv_heads, dim, bad):
    """An infinity or NaN among keys and values at many places, both query tiles' among them."""
    s = of_form(form, [200, 131, 60, 300], heads, kv_heads, dim, seed=7)
    want = list(s.want("cuda"))
    _, k, v = s.parts(s.rows)
    rng, group = np.random.default_rng(8), heads // kv_heads
    hit = torch.zeros(sum(s.lens), heads, dim, dtype=torch.bool, device="cuda")
    keys = torch.zeros_like(hit)
    for i, (a, n) in enumerate(zip(s.indptr[:-1], s.lens)):
        if i % 4 == 2:
            continue
        for at in sorted(rng.integers(0, n, size=3).tolist() + [n - 1, min(n - 1, 100)]):
            g, c = int(rng.integers(kv_heads)), int(rng.integers(dim))
            v[a + at, g, c] = bad
            hit[a + at:a + n, g * group:(g + 1) * group, c] = True
        if i % 3 == 0:
            at, g = int(rng.integers(n)), int(rng.integers(kv_heads))
            k[a + at, g] = bad
            keys[a + at:a + n, g * group:(g + 1) * group] = True
    out, lse = s.run(L)
    got = out.reshape(hit.shape)
    any_hit = hit | keys
    assert_prompt((torch.where(any_hit, want[0].to(bf16), got), torch.where(keys.any(-1), want[2].float(), lse)), want)
    assert not bool(torch.isfinite(got[keys]).reshape(-1, dim).all(-1).any())
    only = got[hit & ~keys]
    assert bool((torch.isnan(only) if bad != bad else only == bad).all())
    assert L.read_device_status() == (0, 0)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 4, 128), (12, 2, 128), (8, 4, 64), (10, 2, 80), (8, 8, 72), (6, 2, 96), (4, 4, 8)])
def test_neighbours_of_no_numbers(L, form, heads, kv_heads, dim):
    """Every other sequence, and the rows around all of them, are NaN throughout: the rest is as if they were not there."""
    lens = [130, 3, 77, 64, 257, 19, 128, 1, 200, 40]
    s = of_form(form, lens, heads, kv_heads, dim, seed=9, before=5, behind=9, pad=24)
    want = s.want("cuda")
    odd = torch.zeros(sum(s.lens), dtype=torch.bool)
    for i, (a, n) in enumerate(zip(s.indptr[:-1], s.lens)):
        if i % 2:
            s.rows[a:a + n] = float("nan")
            odd[a - 5:a - 5 + n] = True
    out = torch.full((s.rows.shape[0], heads * dim), 7.0, dtype=bf16, device="cuda")
    _, lse = s.run(L, out=out)
    n = sum(s.lens)
    assert bool((out[:5] == 7).all()) and bool((out[5 + n:] == 7).all())
    got, got_lse, odd = out[5:5 + n], lse[5:5 + n], odd.cuda()
    assert bool(torch.isnan(got[odd]).all()) and bool(torch.isnan(got_lse[odd]).all())
    assert_prompt((torch.where(odd[:, None], want[0].to(bf16).reshape(got.shape), got), torch.where(odd[:, None], want[2].float(), got_lse)), want)
    assert L.read_device_status() == (0, 0)


@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 4, 128), (6, 2, 64), (10, 2, 96)])
def test_large_small_and_growing_scores_of_two_tiles(L, heads, kv_heads, dim):
    lens = [300, 140, 700]
    for q_scale in (60.0, 0.0):
        s = of_form("two tiles", lens, heads, kv_heads, dim, seed=10, q_scale=q_scale)
        assert_prompt(s.run(L), s.want("cuda"))
    s = of_form("two tiles", lens, heads, kv_heads, dim, seed=11)
    q, k, _ = s.parts(s.rows)
    q[:] = 1.0
    rise = torch.cat([torch.arange(n) for n in s.lens])[:, None, None] / 64.0
    for sign in (1.0, -1.0):
        k[:] = (sign * rise).to(bf16)
        assert_prompt(s.run(L), s.want("cuda"))
    jumps = torch.cat([torch.arange(n) // 40 % 3 for n in s.lens])[:, None, None] * 4.0   # (the reference moves in the middle of rows)
    k[:] = jumps.to(bf16)
    assert_prompt(s.run(L), s.want("cuda"))


@pytest.mark.parametrize("heads,kv_heads,dim", [(16, 8, 128), (24, 8, 64), (8, 4, 96)])
def test_captured_calls_of_two_tiles(L, heads, kv_heads, dim):
    """One graph, replayed for other lengths: as many rows, from one sequence to all of them short."""
    total, batch = 1500, 12
    first = of_form("two tiles", [total // batch] * batch, heads, kv_heads, dim, seed=12)
    rows, indptr = first.rows.cuda(), torch.from_numpy(first.indptr).cuda()
    total, batch = rows.shape[0], len(first.lens)
    out = torch.zeros(total, heads * dim, dtype=bf16, device="cuda")
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        first.run(L, rows, indptr, out=out)
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        _, lse = first.run(L, rows, indptr, out=out)
    rng = np.random.default_rng(13)
    for k in range(5):
        cuts = np.sort(rng.integers(0, total + 1, size=batch - 1)) if k else np.full(batch - 1, total)
        lens = np.diff(np.concatenate([[0], cuts, [total]])).tolist()
        s = PromptSetup(lens, heads, kv_heads, dim, seed=14 + k)
        rows.copy_(s.rows)
        indptr.copy_(torch.from_numpy(s.indptr))
        out.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert_prompt((out, lse), s.want("cuda"))
    assert L.read_device_status() == (0, 0)


def test_more_items_of_a_cta_than_are_noted_one_by_one(L):
    """1024 sequences of two tokens and 192 heads: some 1300 items per CTA, of which 1024 are noted; the last value of each
    sequence from the 700th on is NaN."""
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    s = PromptSetup([2] * 1024, 192, 192, 8, seed=15)
    assert in_pairs(s) and 1024 * 192 > 1024 * sms
    want = s.want("cuda")
    _, _, v = s.parts(s.rows)
    hit = torch.zeros(2048, 192, 8, dtype=torch.bool, device="cuda")
    v[1401::2, :, 5] = float("nan")
    hit[1401::2, :, 5] = True
    out, lse = s.run(L)
    got = out.reshape(hit.shape)
    assert bool(torch.isnan(got[hit]).all())
    assert_prompt((torch.where(hit, want[0].to(bf16), got), lse), want)
    assert L.read_device_status() == (0, 0)


@pytest.mark.parametrize("form", FORMS)
def test_a_call_repeats_itself(L, form):
    s = of_form(form, [300, 131, 60], 16, 4, 128, seed=16)
    rows, indptr = s.rows.cuda(), torch.from_numpy(s.indptr).cuda()
    out, lse = s.run(L, rows, indptr)
    for _ in range(20):
        again, lse2 = s.run(L, rows, indptr)
        assert torch.equal(out, again) and torch.equal(lse, lse2)
