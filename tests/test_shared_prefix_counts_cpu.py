"""That the comparison of tests/shared_prefix_counts.py sees one key, or the keys of a warp's part of a stage, left out or weighed twice."""
import pytest
import torch

from tests.shared_prefix_cases import assert_attention, bf16
from tests.shared_prefix_counts import STRETCH, CountedSetup


@pytest.mark.parametrize("groups,prefixes,heads,kv_heads", [([[(1, 1), (2, 1)]], [32768], 8, 1), ([[(1, 1), (20, 2)], [(12000, 1)]], [3001, 0], 16, 8)])
@pytest.mark.parametrize("factor", [0.0, 2.0])
@pytest.mark.parametrize("count", [1, 16])
def test_a_key_that_is_lost_or_doubled_shows(groups, prefixes, heads, kv_heads, factor, count):
    s = CountedSetup(groups, prefixes, 16, heads, kv_heads, seed=1, device="cpu")
    weights = s.weights()
    r = len(weights) - 1
    n = weights[r].shape[1]
    for turn in range(s.passes):
        want = s.shares(weights, turn)
        assert_attention(want.to(bf16), want, want)
    for first in {0, 1, 15, 16, 127, 128, 255, 256, prefixes[0] - 1, prefixes[0], n // 2, n // 3, n - count}:
        if not 0 <= first <= n - count:
            continue
        for head in (0, heads - 1):
            wrong = [w.clone() for w in weights]
            wrong[r][head, first:first + count] *= factor
            wrong[r][head] /= wrong[r][head].sum()
            seen = 0
            for turn in range(s.passes):
                if (turn + head * kv_heads // heads) % s.passes != first // STRETCH:
                    continue
                want = s.shares(weights, turn)
                with pytest.raises(AssertionError):
                    assert_attention(s.shares(wrong, turn).to(bf16), want, want)
                seen += 1
            assert seen == 1
