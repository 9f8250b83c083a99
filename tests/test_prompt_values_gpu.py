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
