"""Attention over a shared prefix with values that show a single key that is left out or weighed twice, in however long a row.

Every key is one of 8 neighbours whose values are 1 in one output dimension of a KV head and 0 in all others, so that an output is these
keys' share of the row.  128 dimensions hold 1024 keys; a pass looks at one such stretch per KV head, another one in each, and as
many passes as there are stretches look at all keys of all heads.  Scores go up and down by some units along the keys, so that running
maxima move and parts of a row differ; among 8 neighbours of a long row they are alike, a key is no less than 2 percent of its output.

Nothing here is collected by pytest.
"""
from __future__ import annotations

import math

import numpy as np
import torch

from tests.shared_prefix_cases import D, SharedSetup, bf16

EACH = 8                  # keys per output dimension
STRETCH = EACH * D        # keys per KV head and pass


class CountedSetup(SharedSetup):
    def __init__(self, groups, prefixes, page, heads, kv_heads, seed=0, device="cuda"):
        super().__init__(groups, prefixes, page, heads, kv_heads, seed=seed, device=device, q_scale=0.25)
        self.passes = -(-max(self.lens) // STRETCH)
        longest = max(self.lens)
        # one dimension of the keys that all queries see alike: the row's swings, 6 units up and down, three times
        swing = torch.sin(torch.arange(longest, dtype=torch.float64) / longest * 6 * math.pi + 1.0) * 6
        self.q[:, :, 0] = math.sqrt(D)
        self.slots = [torch.from_numpy(self.table[self.table_idx[b], :n].astype(np.int64) - self.low) for b, n in enumerate(self.lens)]
        for b, n in enumerate(self.lens):
            self.k[self.slots[b], :, 0] = swing[:n, None].to(bf16)
        self.unused = self.k[:, 0, 0].isnan()
        self.weights_ = None

    def values(self, turn):
        """The pool's values in pass `turn`."""
        self.v.zero_()
        for h in range(self.kv_heads):
            lo = (turn + h) % self.passes * STRETCH
            for b, n in enumerate(self.lens):
                at = torch.arange(lo, max(min(lo + STRETCH, n), lo))
                if len(at):
                    self.v[self.slots[b][at], h, (at - lo) // EACH] = 1.0
        self.v[self.unused] = float("nan")
        return self.v

    def weights(self):
        """Of every query row, [heads, keys that it sees], in 64 bits."""
        if self.weights_ is None:
            self.weights_ = []
            for b, n in enumerate(self.lens):
                k = self.k[self.slots[b]].double()
                for i in range(self.rows[b]):
                    see = max(n - self.rows[b] + 1 + i, 0)
                    q = self.q[int(self.qo[b]) + i].double().reshape(self.kv_heads, -1, D)
                    s = torch.einsum("hgd,khd->hgk", q, k[:see]) / math.sqrt(D)
                    self.weights_.append(torch.softmax(s, -1).reshape(self.heads, see))
        return self.weights_

    def shares(self, weights, turn):
        """What the outputs of pass `turn` are with these weights: [rows, heads * 128]."""
        group = self.heads // self.kv_heads
        out = torch.zeros(len(weights), self.heads, STRETCH, dtype=torch.float64)
        for h in range(self.kv_heads):
            lo = (turn + h) % self.passes * STRETCH
            for r, w in enumerate(weights):
                part = w[h * group:(h + 1) * group, lo:lo + STRETCH]
                out[r, h * group:(h + 1) * group, :part.shape[1]] = part
        return out.reshape(len(weights), self.heads * D, EACH).sum(-1)


def parts_of_rows(attn, tokens, batch, groups, sms):
    """How many parts the rows of each token were joined from in the last call of `attn`: its plan, as the kernels left it."""
    heads, kv_heads = attn.num_qo_heads_, attn.num_kv_heads_
    group, key_groups = heads // kv_heads, 8 // kv_heads
    rows = -(-tokens * group // batch)
    if groups and tokens * group <= 16 * groups:
        rows = -(-tokens * group // groups)
    eights = 1 if max(rows, group) <= 8 else 2
    slots = 4 * sms + 2 * (tokens // (8 * eights // group)) + batch + groups
    tc_groups = min(groups, tokens * group // 17)
    tc_slots = sms + kv_heads * (tokens // (2 * (128 // group)) + tc_groups) if tokens * group > 16 and groups else 0
    up = lambda n: -(-n // 256) * 256
    at = 256 + up(sms * 8) + up(slots * 48) + up(tc_slots * 32)   # head, tc_of, rows_items, tc_items
    base = -attn.workspace.data_ptr() % 256
    head = attn.workspace[base:base + 32].view(torch.int32).tolist()
    join = attn.workspace[base + at:base + at + tokens * 64].view(torch.int32).reshape(tokens, 16).cpu().tolist()
    fits, per, chunked = head[0], head[2], head[3]
    assert fits == 1
    out = []
    for owned, _, _, own, _, _, pre, _, blocks, _, tiles, _, *_ in join:
        chunks = -(-tiles // per) if blocks and chunked else 1 if blocks else 0
        out.append((own + pre) * key_groups + chunks if owned else 0)
    return out
