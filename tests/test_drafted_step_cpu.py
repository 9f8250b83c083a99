"""What attention over a shared prefix, sampling probabilities and draft verification refuse (checked before any CUDA call)."""
import ctypes

import pytest
import torch

P = ctypes.c_void_p(256)   # never dereferenced: the calls below are refused


def _attention(pkg, **change):
    from sglang_cpp_b200 import _lib
    a = dict(out=256, q=256, q_stride_token=2048, q_stride_head=128, k_cache=256, v_cache=256, num_slots=1024, page_table=256,
             page_table_stride=64, table_idx=256, seq_lens=256, qo_indptr=256, group_indptr=256, prefix_lens=256, tokens=4, batch=4, groups=1,
             q_heads=16, kv_heads=8, head_dim=128, page_size=16, sm_scale=0.1, workspace=256, workspace_bytes=1 << 30)
    a.update(change)
    lib = pkg.load_library()
    rc = lib.b200_attention_shared_prefix(ctypes.byref(_lib.SharedPrefixArgs(**a)), None)
    return rc, lib.b200_last_error().decode()


@pytest.mark.parametrize("change,text", [
    (dict(head_dim=64), "head_dim"), (dict(batch=1025), "batch"), (dict(batch=-1), "batch"), (dict(tokens=-1), "batch"),
    (dict(groups=5), "groups"), (dict(groups=-1), "groups"), (dict(kv_heads=3), "kv_heads"), (dict(kv_heads=16, q_heads=16), "kv_heads"),
    (dict(kv_heads=0), "kv_heads"), (dict(q_heads=20), "q_heads"), (dict(q_heads=0), "q_heads"), (dict(q_heads=136), "q_heads"),
    (dict(page_size=12), "page_size"), (dict(page_size=0), "page_size"), (dict(q_stride_token=2052), "strides"),
    (dict(q_stride_head=132), "strides"), (dict(q_stride_head=0), "strides"), (dict(q_stride_token=-2048), "strides"), (dict(num_slots=0), "num_slots"), (dict(num_slots=1 << 31), "num_slots"),
    (dict(page_table_stride=0), "page_table_stride"), (dict(tokens=1 << 27), "too many"), (dict(out=None), "NULL"), (dict(q=None), "NULL"),
    (dict(group_indptr=None), "NULL"), (dict(prefix_lens=None), "NULL"), (dict(workspace=None), "NULL"), (dict(qo_indptr=None), "NULL"),
    (dict(sm_scale=0.0), "sm_scale"), (dict(sm_scale=-1.0), "sm_scale"), (dict(sm_scale=float("nan")), "sm_scale"),
    (dict(sm_scale=float("inf")), "sm_scale"), (dict(out=260), "aligned"), (dict(q=264), "aligned"),
])
def test_attention_refusals(pkg, change, text):
    rc, said = _attention(pkg, **change)
    assert rc == 1 and text in said, (rc, said)


def test_attention_null_arguments_and_nothing_to_do(pkg):
    lib = pkg.load_library()
    assert lib.b200_attention_shared_prefix(None, None) == 1
    assert _attention(pkg, batch=0, groups=0)[0] == 0
    assert _attention(pkg, tokens=0)[0] == 0


def test_attention_workspace_sizes(pkg):
    size = pkg.load_library().b200_attention_shared_prefix_workspace_bytes
    assert size(64, 64, 16, 8, 128) > 0
    assert size(65, 64, 16, 8, 128) >= size(64, 64, 16, 8, 128) and size(64, 65, 16, 8, 128) > size(64, 64, 16, 8, 128)
    for bad in ((0, 1, 16, 8, 128), (1, 0, 16, 8, 128), (1, 1025, 16, 8, 128), (1, 1, 16, 3, 128), (1, 1, 17, 8, 128), (1, 1, 16, 8, 64),
                (1, 1, 136, 8, 128), (1 << 27, 1, 16, 8, 128)):
        assert size(*bad) == -1


@pytest.mark.parametrize("change,rc,text", [
    (dict(rows=-1), 1, "shape"), (dict(vocab=0), 1, "shape"), (dict(ld=99), 1, "shape"), (dict(vocab=(1 << 24) + 1, ld=1 << 25), 4, "16777216"),
    (dict(out=None), 1, "NULL"), (dict(logits=None), 1, "NULL"), (dict(temperatures=None), 1, "NULL"), (dict(rows=1 << 28), 1, "rows"),
])
def test_sampling_probs_refusals(pkg, change, rc, text):
    a = dict(out=P, logits=P, ld=100, rows=2, vocab=100, temperatures=P, top_k=None, top_p=None)
    a.update(change)
    lib = pkg.load_library()
    assert lib.b200_sampling_probs(*a.values(), None) == rc and text in lib.b200_last_error().decode()


def test_sampling_probs_without_rows(pkg):
    assert pkg.load_library().b200_sampling_probs(None, None, 8, 0, 8, None, None, None, None) == 0


@pytest.mark.parametrize("change,text", [
    (dict(batch=-1), "shape"), (dict(total=-1), "shape"), (dict(most=-1), "shape"), (dict(vocab=0), "shape"), (dict(target_ld=9), "stride"),
    (dict(draft_ld=9), "stride"), (dict(tokens=None), "NULL"), (dict(accepted=None), "NULL"), (dict(target=None), "NULL"),
    (dict(indptr=None), "NULL"), (dict(draw=None), "NULL"), (dict(drafts=None), "NULL"), (dict(accept=None), "NULL"),
    (dict(batch=1 << 25), "large"), (dict(most=1 << 21), "large"),
])
def test_verify_drafts_refusals(pkg, change, text):
    a = dict(tokens=P, accepted=P, target=P, target_ld=10, draft=P, draft_ld=10, drafts=P, indptr=P, accept=P, draw=P, batch=2, total=3, most=2,
             vocab=10)
    a.update(change)
    lib = pkg.load_library()
    assert lib.b200_verify_drafts(*a.values(), None) == 1 and text in lib.b200_last_error().decode()


def test_verify_drafts_of_nobody(pkg):
    assert pkg.load_library().b200_verify_drafts(None, None, None, 8, None, 0, None, None, None, None, 0, 0, 3, 8, None) == 0


def test_oracles_on_known_answers():
    """The plain forms that the GPU tests compare with, on cases worked out by hand."""
    import numpy as np
    import torch

    from tests.shared_prefix_cases import probs_oracle, verify_oracle

    x = torch.tensor([[0.0, np.log(2.0), 0.0, -50.0]])
    assert torch.allclose(probs_oracle(x.double(), [1.0]), torch.tensor([[0.25, 0.5, 0.25, 0.0]], dtype=torch.float64), atol=1e-7)
    assert torch.allclose(probs_oracle(x.double(), [1.0], [2]), torch.tensor([[1 / 3, 2 / 3, 0.0, 0.0]], dtype=torch.float64), atol=1e-7)
    assert torch.equal(probs_oracle(x.double(), [1.0], None, [0.4]), torch.tensor([[0.0, 1.0, 0.0, 0.0]], dtype=torch.float64))
    p = torch.tensor([[0.5, 0.25, 0.25], [0.1, 0.1, 0.8]])
    q = torch.tensor([[0.25, 0.5, 0.25]])
    run = lambda token, u, d: [t.tolist() for t in verify_oracle(p, q, torch.tensor([token]), torch.tensor([0, 1]), torch.tensor([u]),
                                                                 torch.tensor([d]), 1)]
    assert run(0, 0.99, 0.5) == [[[0, 2]], [1]]          # p > q: always accepted
    assert run(1, 0.49, 0.15) == [[[1, 1]], [1]]
    assert run(1, 0.51, 0.7) == [[[0, -1]], [0]]         # refused: the rest is all on token 0


def test_python_calls_take_no_cpu_tensors(pkg):
    """There is no path without the device."""
    from sglang_cpp_b200 import layers as L
    f, i = torch.ones(2), torch.zeros(3, dtype=torch.int32)
    for call in (lambda: L.sampling_probs(torch.zeros(2, 8, dtype=torch.bfloat16), f),
                 lambda: L.verify_drafts(torch.ones(2, 8), i[:0], i, f[:0], f, 0)):
        with pytest.raises(L.B200Error, match="CUDA"):
            call()
