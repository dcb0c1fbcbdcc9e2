"""What the operators behind serving with drafted tokens refuse, without a GPU, and the host's choices."""

import ctypes as C

import pytest
import torch

from diff_gpt_b200 import _lib, ops
from diff_gpt_b200._lib import lib

P = 1 << 20  # an aligned address that no call below gets to use
ARG, UNSUPPORTED, WORKSPACE = -1, -2, -4


def packed(q=P, qr=256, qh=64, k=P, kr=128, kh=64, v=P, o=P, orow=256, starts=P, key_starts=None, S=2, N=10, M=10, H=4, G=2, D=64, scale=0.1, dtype=1, impl=0):
    return lib.dgpt_fmha_packed(q, qr, qh, k, kr, kh, v, kr, kh, o, orow, 64, None, starts, key_starts, S, N, M, H, G, D, scale, dtype, impl, None, None)


@pytest.mark.parametrize("wrong,code,word", [
    (dict(q=None), ARG, "NULL"), (dict(starts=None), ARG, "NULL"), (dict(k=None), ARG, "NULL"), (dict(q=P + 8), ARG, "aligned"), (dict(v=P + 2), ARG, "aligned"),
    (dict(qr=252), ARG, "strides"), (dict(qh=-64), ARG, "strides"), (dict(kh=32), ARG, "strides"), (dict(H=3), ARG, "sizes"), (dict(G=0), ARG, "sizes"),
    (dict(N=-1), ARG, "sizes"), (dict(N=2**31 - 1, M=2**31 - 1), ARG, "rows"), (dict(M=11), ARG, "starts of their own"), (dict(scale=0.0), ARG, "scale"), (dict(scale=float("nan")), ARG, "scale"),
    (dict(impl=3), ARG, "impl"), (dict(dtype=2), UNSUPPORTED, "dtype"), (dict(D=48), UNSUPPORTED, "head_dim"), (dict(impl=2, dtype=0), UNSUPPORTED, "tensor"),
])
def test_packed_refuses(wrong, code, word):
    assert packed(**wrong) == code and word in _lib.last_error()


def layout(**wrong):
    lay = _lib.KvLayout()
    for name, value in dict(dict(k_base=P, v_base=P, page_stride=16384, head_stride=4096, page_table=P, page_tokens=64, max_pages=4, n_pages=9), **wrong).items():
        setattr(lay, name, value)
    return lay


def tree(kv=None, q=P, qr=256, ts=64, ctx=P, gap=(None, None), anc=P, words=1, out=P, ws=None, ws_bytes=0, splits=1, B=2, T=8, H=4, G=2, D=64, scale=0.1, dtype=1, impl=0):
    return lib.dgpt_tree_attn(q, qr, C.byref(kv or layout()), ts, ctx, *gap, None, anc, words, out, 256, ws, ws_bytes, splits, B, T, H, G, D, scale, dtype, impl, None, None)


@pytest.mark.parametrize("wrong,code,word", [
    (dict(q=None), ARG, "NULL"), (dict(anc=None), ARG, "NULL"), (dict(ctx=None), ARG, "NULL"), (dict(gap=(P, None)), ARG, "gap"), (dict(T=257, words=5), ARG, "256"), (dict(T=65), ARG, "words"),
    (dict(words=5), ARG, "words"), (dict(H=5), ARG, "sizes"), (dict(scale=-1.0), ARG, "scale"), (dict(impl=-1), ARG, "impl"), (dict(splits=0), ARG, "n_splits"),
    (dict(splits=257), ARG, "n_splits"), (dict(splits=2), WORKSPACE, "workspace"), (dict(splits=2, ws=P, ws_bytes=100), WORKSPACE, "workspace"),
    (dict(splits=2, ws=P + 4, ws_bytes=10**9), ARG, "aligned"), (dict(qr=250), ARG, "strides"), (dict(qr=128), ARG, "strides"), (dict(ts=60), ARG, "token stride"), (dict(ts=32), ARG, "token stride"),
    (dict(dtype=7), UNSUPPORTED, "dtype"), (dict(D=40), UNSUPPORTED, "head_dim"), (dict(kv=layout(k_base=None)), ARG, "NULL"), (dict(kv=layout(k_base=P + 8)), ARG, "aligned"),
    (dict(kv=layout(page_tokens=0)), ARG, "page_tokens"), (dict(kv=layout(max_pages=0)), ARG, "max_pages"), (dict(kv=layout(head_stride=100)), ARG, "strides"),
    (dict(kv=layout(page_stride=-8)), ARG, "negative"), (dict(impl=2, dtype=0), UNSUPPORTED, "tensor"),
])
def test_tree_refuses(wrong, code, word):
    assert tree(**wrong) == code and word in _lib.last_error()


def logprobs(logits=P, stride=100, targets=P, T=1.0, out=P, ids=P, k=3, R=2, V=100, dtype=1):
    return lib.dgpt_token_logprobs(logits, stride, targets, T, out, out, ids, ids, k, R, V, dtype, None, None)


@pytest.mark.parametrize("wrong,code,word", [
    (dict(logits=None), ARG, "NULL"), (dict(targets=None), ARG, "NULL"), (dict(ids=None), ARG, "NULL"), (dict(k=33), ARG, "top_k"), (dict(k=-1), ARG, "top_k"),
    (dict(V=2, k=3), ARG, "top_k"), (dict(V=0), ARG, "sizes"), (dict(R=-1), ARG, "sizes"), (dict(T=0.0), ARG, "temperature"), (dict(T=1e-39), ARG, "temperature"), (dict(T=float("inf")), ARG, "temperature"),
    (dict(T=float("nan")), ARG, "temperature"), (dict(stride=99), ARG, "overlap"), (dict(logits=P + 1), ARG, "aligned"), (dict(dtype=3), UNSUPPORTED, "dtype"),
])
def test_logprobs_refuses(wrong, code, word):
    assert logprobs(**wrong) == code and word in _lib.last_error()


def keep(kv=None, ts=64, src=P, path=P, L=2, stride=1024, B=2, T=8, H=4, D=64, dtype=1):
    return lib.dgpt_kv_keep(C.byref(kv or layout()), ts, src, P, path, P, L, stride, B, T, H, D, dtype, None, None)


@pytest.mark.parametrize("wrong,code,word", [
    (dict(src=None), ARG, "NULL"), (dict(path=None), ARG, "NULL"), (dict(T=257), ARG, "256"), (dict(L=0), ARG, "sizes"), (dict(D=4), ARG, "16 bytes"),
    (dict(ts=32), ARG, "strides"), (dict(stride=1001), ARG, "strides"), (dict(dtype=5), UNSUPPORTED, "dtype"), (dict(kv=layout(n_pages=-1)), ARG, "negative"),
    (dict(kv=layout(head_stride=0)), ARG, "apart"), (dict(stride=0), ARG, "apart"),
])
def test_keep_refuses(wrong, code, word):
    assert keep(**wrong) == code and word in _lib.last_error()


def test_nothing_to_do_is_no_error():
    assert packed(S=0, starts=None, q=None) == 0 and packed(N=0, M=0, q=None, k=None, v=None, o=None) == 0
    assert tree(B=0, q=None) == 0 and tree(T=0, anc=None) == 0
    assert logprobs(R=0, logits=None) == 0
    assert keep(B=0, src=None) == 0 and keep(T=0) == 0


def test_workspace_and_splits():
    assert ops.tree_attn_workspace_bytes(3, 5, 4, 64, 1) == 0
    assert ops.tree_attn_workspace_bytes(3, 5, 4, 64, 7) >= 3 * 5 * 4 * 7 * 65 * 4
    assert ops.tree_attn_workspace_bytes(3, 5, 4, 64, 7) % 16 == 0
    for dtype in (torch.float32, torch.bfloat16):
        assert ops.tree_attn_splits(1, 8, 4, 4, 64, 100, dtype) == 1  # short: not worth a second pass
        assert ops.tree_attn_splits(1, 8, 4, 4, 64, 60000, dtype) > 8
        assert 1 <= ops.tree_attn_splits(64, 256, 64, 8, 128, 10**9, dtype) <= 256
        assert ops.tree_attn_splits(0, 8, 4, 4, 64, 100, dtype) == 1


def test_the_wrappers_refuse_cpu_tensors():
    q = torch.zeros(4, 2, 64)
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        ops.fmha_packed(q, q, q, i, q)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        ops.tree_attn(q.view(4, 128), layout(), i, torch.zeros(2, 2, dtype=torch.int64), q.view(4, 128), H=2, G=2, D=64)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        ops.token_logprobs(q.view(4, 128), torch.zeros(4, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        ops.kv_keep(layout(), i, i, torch.zeros(2, 2, dtype=torch.int32), i, n_layer=1, layer_stride=0, H=1, D=8, dtype=torch.float32)


def test_a_cache_of_another_type_or_place_is_refused(monkeypatch):
    lay = layout()
    lay._keep = (torch.zeros(8), torch.zeros(8), None)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        ops._stored("tree_attn", lay, torch.float32)
    monkeypatch.setattr(ops, "_here", lambda *ts: None)
    ops._stored("tree_attn", lay, torch.float32)
    with pytest.raises(TypeError, match="cache of torch.float32"):
        ops._stored("tree_attn", lay, torch.bfloat16)


def test_slots_of_packed_prompts_never_collide():
    """The tensor's rows in tiles of bm: prompt s takes the slots from starts[s] // bm + s on.  Every row lies in one slot, no slot in two prompts, and
    the slots fit rows // bm + prompts: the arithmetic that the kernels repeat."""
    import random

    rng = random.Random(0)
    for _ in range(300):
        bm = rng.choice((64, 128))
        at, lens = rng.randint(0, 300), [rng.choice((0, 1, rng.randint(0, 700), bm, bm - 1, bm + 1)) for _ in range(rng.randint(1, 12))]
        starts = [at]
        for n in lens:
            starts.append(starts[-1] + n)
        rows = starts[-1] + rng.randint(0, 200)
        used = set()
        for s, n in enumerate(lens):
            for tile in range(-(-n // bm)):
                slot = starts[s] // bm + s + tile
                assert slot not in used and slot < rows // bm + len(lens)
                used.add(slot)
                found = max(x for x in range(len(lens)) if starts[x] // bm + x <= slot)
                assert found == s
