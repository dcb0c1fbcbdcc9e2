"""ops.tree_attn: trees of drafted tokens behind paged caches, against float64."""

import random

import pytest
import torch

from drafts_cases import check_rows, rows, scale_of, tree_bits, words

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32


def run(ctx, nodes, T, H, G, D, dtype, impl=0, page=64, layout="heads", n_splits=0, seed=0, bits=None, hole=False, ragged=True, scale=None, gaps=None):
    """layout: "heads" as PagedKVCache ([page][kv][head][token][D]), "rows" as PagedRowCache ([page][token][keys | values]),
    "dense" without a page table; hole: a page number outside the pool (its keys and values count as zeros)."""
    from diff_gpt_b200 import ops

    g = torch.Generator().manual_seed(seed + D + T)
    rng = random.Random(seed)
    B = len(ctx)
    need = [c + n for c, n in zip(ctx, nodes)]
    cap = max(1, -(-max(need) // page)) * page
    pages = cap // page
    keys, vals = (torch.randn(B, G, cap, D, generator=g).to(dtype) for _ in range(2))
    nan = float("nan")
    for b in range(B):
        keys[b, :, need[b] :] = nan  # behind the last draft anything may lie
        vals[b, :, need[b] :] = nan
        if gaps:  # and in the gap
            keys[b, :, gaps[b][0] : gaps[b][1]] = nan
            vals[b, :, gaps[b][0] : gaps[b][1]] = float("inf")
    tokens = 0
    if layout == "dense":
        store = torch.stack([keys, vals], dim=1).cuda()  # [B][kv][G][cap][D]
        kv = ops.kv_layout(store[0, 0], store[0, 1], store.stride(0), store.stride(2), cap)
    else:
        perm = torch.randperm(B * pages, generator=g).to(torch.int32).view(B, pages)
        kp, vp = (x.view(B, G, pages, page, D).permute(0, 2, 1, 3, 4).reshape(B * pages, G, page, D) for x in (keys, vals))
        if layout == "heads":
            pool = torch.full((B * pages, 2, G, page, D), nan, dtype=dtype)
            pool[perm.flatten().long()] = torch.stack([kp, vp], dim=1)
            store = pool.cuda()
            table = perm.clone()
            kv_args = (store[0, 0], store[0, 1], store.stride(0), store.stride(2), page)
        else:
            width = 2 * G * D + 8
            pool = torch.full((B * pages, page, width), nan, dtype=dtype)
            r = torch.cat([kp.permute(0, 2, 1, 3).flatten(2), vp.permute(0, 2, 1, 3).flatten(2)], dim=2)
            pool[perm.flatten().long(), :, : 2 * G * D] = r
            store = pool.cuda()
            table = perm.clone()
            kv_args = (store[0], store[0, :, G * D :], store.stride(0), D, page)
            tokens = width
        if hole:
            table[0, 0], table[-1, 0] = -3, B * pages
            keys[0, :, :page], vals[0, :, :page], keys[-1, :, :page], vals[-1, :, :page] = 0, 0, 0, 0
        table_d = table.cuda()
        kv = ops.kv_layout(*kv_args, table_d, n_pages=B * pages)
    if bits is None:
        bits = [tree_bits([rng.randint(max(-1, t - 5), t - 1) for t in range(T)]) for _ in range(B)]
    W = -(-T // 64)
    anc = torch.stack([words(b, W) for b in bits])
    q = torch.randn(B * T, H * D, generator=g).to(dtype)
    out = torch.full((B * T, H * D), -7.0, dtype=dtype, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    i32 = dict(dtype=torch.int32, device="cuda")
    ops.tree_attn(q.cuda(), kv, torch.tensor(ctx, **i32), anc.cuda(), out, H=H, G=G, D=D, max_keys=max(need),
                  n_nodes=torch.tensor(nodes, **i32) if ragged else None, token_stride=tokens, n_splits=n_splits, impl=impl, status=status, scale=scale,
                  gap_start=torch.tensor([a for a, _ in gaps], **i32) if gaps else None, gap_end=torch.tensor([e for _, e in gaps], **i32) if gaps else None)
    torch.cuda.synchronize()
    assert status.item() == 0
    got = out.cpu().view(B, T, H, D)
    qh = q.view(B, T, H, D)
    for b in range(B):
        c, n = ctx[b], nodes[b]
        assert bool((got[b, n:] == -7).all())
        if n == 0:
            continue
        see = torch.ones(n, c + n, dtype=torch.bool)
        see[:, c:] = torch.tensor([[(bits[b][t] >> j) & 1 for j in range(n)] for t in range(n)], dtype=torch.bool).view(n, n)
        held = torch.ones(c + n, dtype=torch.bool)
        if gaps:
            held[gaps[b][0] : gaps[b][1]] = False
        for h in range(H):
            kvh = h // (H // G)
            want = rows(qh[b, :n, h], keys[b, kvh, : c + n][held], vals[b, kvh, : c + n][held], see[:, held], scale or scale_of(D))
            check_rows(got[b, :n, h], None, want, D, c + n, dtype, dtype == BF and impl != 1)
    return out


TYPES = [(8, F32), (16, F32), (64, F32), (128, F32), (16, BF), (32, BF), (64, BF), (128, BF)]


@pytest.mark.parametrize("impl", [0, 1])
@pytest.mark.parametrize("D,dtype", TYPES)
def test_trees(D, dtype, impl):
    run([300, 0, 63, 64, 129], [9, 9, 1, 5, 0], 9, 4, 2, D, dtype, impl)


@pytest.mark.parametrize("impl", [0, 1])
@pytest.mark.parametrize("T", [1, 2, 16, 63, 64, 65, 130, 256])
@pytest.mark.parametrize("D,dtype", [(64, BF), (128, BF), (16, F32)])
def test_sizes_of_trees(T, D, dtype, impl):
    run([200, 3, 1000], [T, max(1, T // 2), T], T, 4, 2, D, dtype, impl, seed=1)


@pytest.mark.parametrize("impl", [0, 1])
@pytest.mark.parametrize("H,G", [(1, 1), (8, 8), (6, 2), (7, 1), (20, 4), (32, 1)])
@pytest.mark.parametrize("D,dtype", [(64, BF), (128, BF), (16, F32)])
def test_heads(H, G, D, dtype, impl):
    run([333, 90], [21, 30], 30, H, G, D, dtype, impl, seed=2)


@pytest.mark.parametrize("impl", [0, 1])
@pytest.mark.parametrize("page,layout", [(8, "heads"), (16, "rows"), (64, "rows"), (128, "heads"), (256, "rows"), (24, "heads"), (7, "rows"), (1000, "dense"), (64, "dense")])
@pytest.mark.parametrize("D,dtype", [(64, BF), (128, BF), (32, F32)])
def test_layouts(page, layout, D, dtype, impl):
    run([500, 130, 0], [17, 3, 17], 17, 4, 2, D, dtype, impl, page=page, layout=layout, seed=3)


@pytest.mark.parametrize("impl", [0, 1])
@pytest.mark.parametrize("n_splits", [1, 2, 3, 7, 40])
@pytest.mark.parametrize("D,dtype", [(64, BF), (128, BF), (16, F32)])
def test_splits(n_splits, D, dtype, impl):
    """More shares than tiles among them."""
    run([1500, 40, 0, 700], [12, 12, 2, 5], 12, 4, 1, D, dtype, impl, n_splits=n_splits, seed=4)


@pytest.mark.parametrize("impl", [0, 1])
@pytest.mark.parametrize("n_splits", [5, 16, 64])
@pytest.mark.parametrize("D,dtype", [(64, BF), (128, BF), (16, F32)])
def test_many_shares_without_keys(n_splits, D, dtype, impl):
    """More items than the GPU holds at a time, most of them without a key, between ones with up to nine tiles."""
    run([100, 0, 1100, 300, 5, 130] * 7, [3, 1, 2, 3, 1, 3] * 7, 3, 4, 2, D, dtype, impl, n_splits=n_splits, seed=11)


@pytest.mark.parametrize("impl", [0, 1])
@pytest.mark.parametrize("n_splits", [1, 3])
@pytest.mark.parametrize("D,dtype", [(64, BF), (128, BF), (16, F32)])
def test_masks(D, dtype, n_splits, impl):
    """Rows that see nothing (no cache, empty masks), every draft, only drafts behind them, and bits of drafts that are not there."""
    T = 70
    every = (1 << T) - 1
    bits = [[0] * T, [every] * T, [(every >> (t + 1)) << (t + 1) for t in range(T)], [every if t % 3 == 0 else 0 for t in range(T)]]
    run([0, 0, 130, 0], [70, 33, 70, 64], T, 4, 4, D, dtype, impl, n_splits=n_splits, bits=bits, seed=5)


@pytest.mark.parametrize("impl", [0, 1])
@pytest.mark.parametrize("D,dtype", [(64, BF), (128, BF), (16, F32)])
def test_pages_outside_the_pool_are_zeros(D, dtype, impl):
    run([300, 100, 200], [5, 5, 5], 5, 4, 2, D, dtype, impl, hole=True, seed=6)


@pytest.mark.parametrize("impl", [0, 1])
@pytest.mark.parametrize("n_splits", [1, 3])
@pytest.mark.parametrize("D,dtype", [(32, BF), (64, BF), (128, BF), (16, F32)])
def test_gaps(D, dtype, n_splits, impl):
    """What a prompt leaves free of its last page: inside a tile, over tiles, whole tiles, at either end, none, and with nothing before it."""
    gaps = [(100, 128), (120, 400), (128, 384), (0, 70), (300, 300), (299, 300), (0, 300), (64, 65)]
    run([500, 500, 500, 200, 300, 300, 300, 66], [9, 5, 9, 9, 1, 9, 9, 9], 9, 4, 2, D, dtype, impl, n_splits=n_splits, seed=12, gaps=gaps)


@pytest.mark.parametrize("impl", [0, 1])
@pytest.mark.parametrize("scale", [1e-3, 2.0])
@pytest.mark.parametrize("D,dtype", [(64, BF), (16, F32)])
def test_scales(D, dtype, scale, impl):
    run([900, 300], [6, 6], 6, 4, 2, D, dtype, impl, scale=scale, seed=7, ragged=False)


@pytest.mark.parametrize("D,dtype", [(128, BF), (16, F32)])
def test_one_draft_is_a_decode_step(D, dtype):
    """A tree of one node is what ops.decode_attn computes."""
    from diff_gpt_b200 import ops

    H, B, n, page = 4, 3, [200, 65, 1], 64
    g = torch.Generator(device="cuda").manual_seed(9)
    pool = torch.randn(B * 4, 2, H, page, D, generator=g, device="cuda").to(dtype)
    table = torch.arange(B * 4, dtype=torch.int32, device="cuda").view(B, 4)
    kv = ops.kv_layout(pool[0, 0], pool[0, 1], pool.stride(0), pool.stride(2), page, table, n_pages=B * 4)
    q = torch.randn(B, H * D, generator=g, device="cuda").to(dtype)
    lens = torch.tensor(n, dtype=torch.int32, device="cuda")
    zero = torch.zeros_like(lens)
    a, b = torch.empty_like(q), torch.empty_like(q)
    ops.decode_attn(q, kv, zero, zero, lens, None, a, H=H, D=D)
    ops.tree_attn(q, kv, lens - 1, torch.ones(B, 1, dtype=torch.int64, device="cuda"), b, H=H, G=H, D=D)
    # Both lie within u |o| + (tensor cores) 2^-8 A of the exact row; A <= the largest value of the row's keys.
    tol = (2 * 2.0**-8 * a.float().abs() + 2.0**-8 * pool.float().abs().max()) if dtype == BF else 1e-5 * pool.abs().max()
    assert bool(((a.float() - b.float()).abs() <= tol).all())


@pytest.mark.parametrize("D,dtype", [(128, BF), (16, F32)])
def test_repeats_graphs_and_streams(D, dtype):
    from diff_gpt_b200 import ops

    H, G, B, T, page, pages = 8, 2, 5, 11, 64, 30
    g = torch.Generator(device="cuda").manual_seed(10)
    pool = torch.randn(B * pages, 2, G, page, D, generator=g, device="cuda").to(dtype)
    table = torch.randperm(B * pages, generator=g, device="cuda").to(torch.int32).view(B, pages)
    kv = ops.kv_layout(pool[0, 0], pool[0, 1], pool.stride(0), pool.stride(2), page, table, n_pages=B * pages)
    ctx = torch.tensor([1800, 3, 700, 64, 0], dtype=torch.int32, device="cuda")
    anc = words(tree_bits([t // 2 - 1 for t in range(T)]), 1).expand(B, T, 1).contiguous().cuda()
    q = torch.randn(B * T, H * D, generator=g, device="cuda").to(dtype)
    out = torch.empty_like(q)

    def call(to=None):
        ops.tree_attn(q, kv, ctx, anc, out if to is None else to, H=H, G=G, D=D, max_keys=1900)

    call()
    first = out.clone()
    for _ in range(5):
        out.zero_()
        call()
        assert torch.equal(out, first)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out.zero_()
        call()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(out, first)
    # two graphs, each with the workspace of its own capture, replayed in turn over a cache that has grown meanwhile
    other = torch.empty_like(out)
    graphs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()]
    for gr, to in zip(graphs, (out, other)):
        with torch.cuda.graph(gr):
            call(to)
    ctx += 40
    want = torch.empty_like(out)
    call(want)
    for gr in graphs + graphs:
        gr.replay()
    assert torch.equal(out, want) and torch.equal(other, want)


@pytest.mark.parametrize("impl", [0, 1])
def test_wrong_lengths_are_reported(impl):
    from diff_gpt_b200 import ops

    H, D, page, pages, T = 2, 64, 64, 3, 4
    pool = torch.randn(2 * pages, 2, H, page, D, device="cuda").to(BF)
    table = torch.arange(2 * pages, dtype=torch.int32, device="cuda").view(2, pages)
    kv = ops.kv_layout(pool[0, 0], pool[0, 1], pool.stride(0), pool.stride(2), page, table, n_pages=2 * pages)
    q = torch.randn(2 * T, H * D, device="cuda").to(BF)
    anc = torch.full((2, T, 1), -1, dtype=torch.int64, device="cuda")
    i32 = dict(dtype=torch.int32, device="cuda")
    for ctx, n in (([190, 0], [4, 4]), ([-1, 5], [4, 4]), ([10, 10], [5, 4]), ([10, 10], [-1, 4]), ([2**31 - 1, 3], [4, 4])):
        status = torch.zeros(1, **i32)
        out = torch.zeros_like(q)
        ops.tree_attn(q, kv, torch.tensor(ctx, **i32), anc, out, H=H, G=H, D=D, n_nodes=torch.tensor(n, **i32), impl=impl, status=status)
        assert status.item() == 1, (ctx, n)
        assert bool(torch.isfinite(out).all())
    for a, e in ((-1, 3), (5, 4), (3, 11)):
        status = torch.zeros(1, **i32)
        ops.tree_attn(q, kv, torch.tensor([10, 10], **i32), anc, out, H=H, G=H, D=D, gap_start=torch.tensor([0, a], **i32),
                      gap_end=torch.tensor([0, e], **i32), impl=impl, status=status)
        assert status.item() == 1, (a, e)
        assert bool(torch.isfinite(out).all())
