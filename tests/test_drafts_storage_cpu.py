"""Caches that do not hold what a call of ops.tree_attn or ops.kv_keep asks of them are refused before anything is launched."""

import pytest
import torch

from diff_gpt_b200 import KVCache, PagedKVCache, _lib, ops
from test_drafts_cpu import ARG, keep, layout, tree

L, PAGES, G, PAGE, D = 2, 9, 2, 64, 64


@pytest.fixture(autouse=True)
def no_gpu(monkeypatch):
    """Tensors pass as they are; what would be launched is noted instead."""
    calls = []

    class Fake:
        dgpt_tree_attn_splits = _lib.lib.dgpt_tree_attn_splits
        dgpt_tree_attn_workspace_bytes = _lib.lib.dgpt_tree_attn_workspace_bytes

        def dgpt_tree_attn(self, *a):
            calls.append("tree_attn")
            return 0

        def dgpt_kv_keep(self, *a):
            calls.append("kv_keep")
            return 0

    for name, fake in (("_here", lambda *ts: None), ("_cuda", lambda *ts: None), ("_stream", lambda: 0), ("lib", Fake())):
        monkeypatch.setattr(ops, name, fake)
    return calls


def paged(table, n_pages=PAGES, layer=0):
    pool = torch.zeros(L, PAGES, 2, G, PAGE, D)
    return ops.kv_layout(pool[layer, 0, 0], pool[layer, 0, 1], pool.stride(1), pool.stride(3), PAGE, table, n_pages=n_pages)


def call_tree(kv, B, H=4, G=G, D=D, token_stride=0):
    q = torch.zeros(B * 3, H * D)
    ops.tree_attn(q, kv, torch.zeros(B, dtype=torch.int32), torch.zeros(B, 3, 1, dtype=torch.int64), q, H=H, G=G, D=D, token_stride=token_stride)


def call_keep(kv, B, H=G, D=D, token_stride=0, n_layer=L, layer_stride=PAGES * 2 * G * PAGE * D):
    i = torch.zeros(B, dtype=torch.int32)
    ops.kv_keep(kv, i, i, torch.zeros(B, 3, dtype=torch.int32), i, n_layer=n_layer, layer_stride=layer_stride, H=H, D=D, dtype=torch.float32,
                token_stride=token_stride)


def table(rows, dtype=torch.int32):
    return torch.zeros(rows, 4, dtype=dtype)


@pytest.mark.parametrize("call", [call_tree, call_keep])
def test_as_many_sequences_as_the_table_has(call, no_gpu):
    call(paged(table(3)), 3)
    call(paged(table(5)), 3)
    call(paged(table(1)[0]), 1)  # one row as a plain list of pages
    assert len(no_gpu) == 3
    for t in (table(2), table(1)[0], table(0)):
        with pytest.raises(ValueError, match="page table"):
            call(paged(t), 3)
    assert len(no_gpu) == 3


@pytest.mark.parametrize("call", [call_tree, call_keep])
def test_tables_that_would_be_read_as_other_numbers(call, no_gpu):
    for t in (table(3, torch.int64), table(8)[::2], torch.zeros(3, 8, dtype=torch.int32)[:, :4], torch.zeros(4, 3, dtype=torch.int32).t()):
        with pytest.raises(ValueError, match="page table"):
            call(paged(t), 3)
    assert not no_gpu


@pytest.mark.parametrize("call", [call_tree, call_keep])
def test_a_dense_cache_has_as_many_sequences_as_it_says(call, no_gpu):
    c = KVCache(batch_size=3, num_heads=G, seq_len=PAGE, head_dim=D, num_layers=L)
    c.ensure(PAGE, torch.float32, torch.device("cpu"))
    kw = {} if call is call_tree else dict(layer_stride=c.kv_cache.stride(0))
    for layer in range(1 if call is call_keep else L):
        assert c.layer_layout(layer).n_pages == 3
        call(c.layer_layout(layer), 3, **kw)
    n = len(no_gpu)
    with pytest.raises(ValueError, match="sequences"):
        call(c.layer_layout(0), 4, **kw)
    assert len(no_gpu) == n


def test_the_library_refuses_more_sequences_than_a_dense_cache_states():
    dense = layout(page_table=None, max_pages=0, n_pages=1)
    assert tree(kv=dense) == ARG and "sequences" in _lib.last_error()
    assert keep(kv=dense) == ARG and "sequences" in _lib.last_error()


@pytest.mark.parametrize("call", [call_tree, call_keep])
def test_nothing_outside_the_storage(call, no_gpu):
    kv = paged(table(3), layer=0 if call is call_keep else L - 1)  # what lies behind is nobody's
    dense = ops.kv_layout(torch.zeros(3, 2, G, PAGE, D)[0, 0], torch.zeros(3, 2, G, PAGE, D)[0, 0], 2 * G * PAGE * D, PAGE * D, PAGE)
    wrong = [(kv, 3, dict(D=2 * D)), (kv, 3, dict(token_stride=2 * D)), (paged(table(3), n_pages=2 * PAGES + 1), 3, {}), (dense, 4, {})]
    wrong.append((kv, 3, dict(G=4) if call is call_tree else dict(H=3)))  # (the last page's values end with the last head)
    if call is call_keep:
        wrong += [(kv, 3, dict(n_layer=L + 1)), (kv, 3, dict(layer_stride=PAGES * 2 * G * PAGE * D + 8)), (kv, 3, dict(layer_stride=-8))]
    for lay, B, kw in wrong:
        if call is call_keep and lay is dense:
            kw = dict(kw, n_layer=1)
        with pytest.raises(ValueError, match="storage"):
            call(lay, B, **kw)
    assert not no_gpu
    call(dense, 3, **(dict(n_layer=1) if call is call_keep else {}))
    assert len(no_gpu) == 1


def test_a_layout_without_its_tensors_is_taken_at_its_word(no_gpu):
    call_tree(layout(), 3)
    call_keep(layout(), 3)
    assert no_gpu == ["tree_attn", "kv_keep"]


def test_paged_caches_keep_as_many_rows_as_they_have(no_gpu):
    c = PagedKVCache(L, G, D, n_series=2, rows_per_series=2, prefix_len=70, max_new=30, dtype=torch.float32, device="cpu")
    i = torch.zeros(5, dtype=torch.int32)
    c.keep_drafts(i[:4], i[:4], torch.zeros(4, 3, dtype=torch.int32), i[:4])
    with pytest.raises(ValueError, match="page table"):
        c.keep_drafts(i, i, torch.zeros(5, 3, dtype=torch.int32), i)
    with pytest.raises(ValueError, match="page table"):
        call_tree(c.prefix_layout(0), 4)  # one row a series
    assert no_gpu == ["kv_keep"]


def test_the_pages_that_kept_drafts_may_move_between():
    """A row's own alone where a prompt is shared; all of them where the prompt is the row's."""
    for rows in (1, 3):
        c = PagedKVCache(L, G, D, n_series=2, rows_per_series=rows, prefix_len=70, max_new=130, dtype=torch.float32, device="cpu")
        assert c.keep_table.dtype == torch.int32 and c.keep_table.is_contiguous() and c.row_table.is_contiguous()
        assert torch.equal(c.keep_table[:, 2:], c.row_table[:, 2:])
        assert torch.equal(c.keep_table[:, :2], c.row_table[:, :2] if rows == 1 else torch.full((6, 2), -1, dtype=torch.int32))
