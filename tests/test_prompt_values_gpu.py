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
