"""Counts that the library takes in 32 bits: a tensor with more is refused, not taken modulo 2^32."""

import pytest
import torch

from diff_gpt_b200 import ops
from test_drafts_cpu import layout

MANY = 2**32 + 3
meta = dict(device="meta")
i32 = dict(dtype=torch.int32, **meta)


@pytest.fixture(autouse=True)
def no_gpu(monkeypatch):
    class Fake:
        def __getattr__(self, name):
            raise AssertionError(f"{name} was called")

    for name, fake in (("_here", lambda *ts: None), ("_cuda", lambda *ts: None), ("_stream", lambda: 0), ("lib", Fake())):
        monkeypatch.setattr(ops, name, fake)


def test_packed_rows():
    one = torch.empty(2, **i32)
    q, k = torch.empty(MANY, 1, 8, **meta), torch.empty(5, 1, 8, **meta)
    for a, b, starts in ((q, q, one), (k, q, one), (k, k, torch.empty(MANY, **i32))):
        with pytest.raises(ValueError, match="32 bits"):
            ops.fmha_packed(a, b, b, starts, a, key_starts=starts)


def test_rows_of_logits():
    for R, V in ((MANY, 1), (1, MANY)):
        with pytest.raises(ValueError, match="32 bits"):
            ops.token_logprobs(torch.empty(R, V, **meta), torch.empty(R, **i32))


def test_sequences_of_trees_and_paths():
    n = torch.empty(MANY, **i32)
    q = torch.empty(MANY, 8, **meta)
    with pytest.raises(ValueError, match="32 bits"):
        ops.tree_attn(q, layout(), n, torch.empty(MANY, 1, dtype=torch.int64, **meta), q, H=1, G=1, D=8)
    with pytest.raises(ValueError, match="32 bits"):
        ops.kv_keep(layout(), n, n, torch.empty(MANY, 1, **i32), n, n_layer=1, layer_stride=0, H=1, D=8, dtype=torch.float32)


def test_shares_of_caches_with_more_slots_than_32_bits_count(monkeypatch):
    """(They are chosen for as many keys as a sequence can have.)"""
    asked = []
    monkeypatch.setattr(ops, "_tree_plan", lambda *a: asked.append(a) or (1, 0))

    class Fake:
        def dgpt_tree_attn(self, *a):
            return 0

    monkeypatch.setattr(ops, "lib", Fake())
    q, n = torch.zeros(1, 8), torch.zeros(1, dtype=torch.int32)
    for keys in (0, 2**33):
        ops.tree_attn(q, layout(page_tokens=2**30, max_pages=8), n, torch.zeros(1, 1, dtype=torch.int64), q, H=1, G=1, D=8, max_keys=keys)
    assert [a[5] for a in asked] == [2**31 - 1] * 2
