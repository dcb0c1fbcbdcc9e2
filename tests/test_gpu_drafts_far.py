"""The operators behind serving with drafted tokens where lengths, strides and groups are large, and where calls run at the same time; against float64."""

import pytest
import torch

from drafts_cases import check_rows, rows, scale_of, tree_bits, words
from test_gpu_logprobs import keep_plain
from test_gpu_logprobs_bounds import check as check_logprobs
from test_gpu_tree import run as run_tree

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32
i32 = dict(dtype=torch.int32, device="cuda")


def randn(*shape, seed, dtype):
    return torch.randn(*shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").to(dtype)


@pytest.mark.parametrize("D,dtype,impl", [(64, BF, 0), (128, BF, 0), (64, BF, 1), (16, F32, 0), (64, F32, 0)])
@pytest.mark.parametrize("ctx,T", [([70000, 33000], 5), ([20001], 70)])
def test_trees_behind_long_caches(ctx, T, D, dtype, impl):
    from diff_gpt_b200 import ops

    H, G, page, B = 4, 2, 64, len(ctx)
    pages = -(-(max(ctx) + T) // page)
    pool = randn(B * pages, 2, G, page, D, seed=D + T, dtype=dtype)
    table = torch.randperm(B * pages, generator=torch.Generator().manual_seed(1)).to(torch.int32).view(B, pages).cuda()
    bits = tree_bits([(t - 1) // 2 if t else -1 for t in range(T)])
    anc = words(bits, 2).expand(B, T, 2).contiguous().cuda()
    q = randn(B * T, H * D, seed=2, dtype=dtype)
    out, status = torch.empty_like(q), torch.zeros(1, **i32)
    kv = ops.kv_layout(pool[0, 0], pool[0, 1], pool.stride(0), pool.stride(2), page, table, n_pages=B * pages)
    for n_splits in (0, 3):
        out.fill_(float("nan"))
        ops.tree_attn(q, kv, torch.tensor(ctx, **i32), anc, out, H=H, G=G, D=D, max_keys=max(ctx) + T, n_splits=n_splits, impl=impl, status=status)
        assert status.item() == 0
        for b, c in enumerate(ctx):
            k, v = (pool[table[b].long(), kind].transpose(0, 1).reshape(G, -1, D)[:, : c + T] for kind in (0, 1))
            see = torch.ones(T, c + T, dtype=torch.bool, device="cuda")
            see[:, c:] = torch.tensor([[(x >> j) & 1 for j in range(T)] for x in bits], dtype=torch.bool)
            for h in range(H):
                got = out.view(B, T, H, D)[b, :, h]
                check_rows(got, None, rows(q.view(B, T, H, D)[b, :, h], k[h // 2], v[h // 2], see, scale_of(D)), D, c + T, dtype, dtype == BF and impl != 1)


@pytest.mark.parametrize("D,dtype,impl", [(64, BF, 0), (128, BF, 0), (64, BF, 1), (16, F32, 0)])
def test_long_prompts(D, dtype, impl):
    from diff_gpt_b200 import ops

    lens, past, H, G = [5000, 130, 900], [0, 9000, 64], 2, 1
    N, M = sum(lens), sum(lens) + sum(past)
    q, k, v = (randn(n, h, D, seed=s, dtype=dtype) for n, h, s in ((N, H, 1), (M, G, 2), (M, G, 3)))
    qs, ks = [0, *torch.tensor(lens).cumsum(0).tolist()], [0, *(torch.tensor(lens) + torch.tensor(past)).cumsum(0).tolist()]
    out, lse, status = torch.empty_like(q), torch.empty(N, H, device="cuda"), torch.zeros(1, **i32)
    ops.fmha_packed(q, k, v, torch.tensor(qs, **i32), out, key_starts=torch.tensor(ks, **i32), lse=lse, impl=impl, status=status)
    assert status.item() == 0
    for s, (n, p) in enumerate(zip(lens, past)):
        a, b = slice(qs[s], qs[s + 1]), slice(ks[s], ks[s + 1])
        see = torch.ones(n, n + p, dtype=torch.bool, device="cuda").tril(p)
        for h in range(H):
            check_rows(out[a, h], lse[a, h], rows(q[a, h], k[b, 0], v[b, 0], see, scale_of(D)), D, n + p, dtype, dtype == BF and impl != 1)


@pytest.mark.parametrize("D,dtype,impl", [(64, BF, 0), (128, BF, 1), (16, F32, 0)])
def test_thousands_of_short_prompts(D, dtype, impl):
    from diff_gpt_b200 import ops

    lens = torch.randint(0, 3, (5000,), generator=torch.Generator().manual_seed(4))
    starts = torch.cat([torch.zeros(1, dtype=torch.long), lens.cumsum(0)])
    N, H = int(starts[-1]), 2
    q, k, v = (randn(N, H, D, seed=s, dtype=dtype) for s in (5, 6, 7))
    out, status = torch.empty_like(q), torch.zeros(1, **i32)
    ops.fmha_packed(q, k, v, starts.to(**i32), out, impl=impl, status=status)
    # a first token is its own value's; a second's row has two keys
    first = starts[:-1][lens > 0].cuda()
    assert torch.equal(out[first], v[first]) and status.item() == 0
    second = starts[:-1][lens > 1].cuda() + 1
    pair = torch.stack([second - 1, second], dim=1)
    s = (q[second].double()[:, None] * k[pair].double()).sum(-1) * scale_of(D)
    p = s.softmax(dim=1)[..., None]
    want, A = (p * v[pair].double()).sum(1), (p * v[pair].double().abs()).sum(1)
    S = (q[second].double()[:, None] * k[pair].double()).abs().sum(-1).amax(1)[..., None] * scale_of(D)
    u = 2.0**-8 if dtype == BF else 2.0**-24
    tol = u * want.abs() + A * (4 * (D + 4) * 2.0**-24 * (S + 1) + 2.0**-20 + (2.0**-8 if dtype == BF and impl != 1 else 0.0))
    assert bool(((out[second].double() - want).abs() <= tol).all())


@pytest.mark.parametrize("H,G", [(144, 1), (130, 1), (260, 2)])
@pytest.mark.parametrize("D,dtype", [(64, BF), (128, BF), (16, F32)])
def test_more_query_heads_a_group_than_a_tile_has_rows(H, G, D, dtype):
    run_tree([333, 90], [3, 2], 3, H, G, D, dtype, seed=21)


@pytest.mark.parametrize("impl", [0, 1])
@pytest.mark.parametrize("D,dtype", [(64, BF), (128, BF), (16, F32)])
def test_wider_masks_and_rows_than_a_tree_needs(D, dtype, impl):
    """More words of ancestors than T asks for, their other bits set; q and out as columns of wider rows."""
    from diff_gpt_b200 import ops

    H, G, B, T, cap = 4, 2, 2, 9, 200
    store = randn(B, 2, G, cap, D, seed=8, dtype=dtype)
    kv = ops.kv_layout(store[0, 0], store[0, 1], store.stride(0), store.stride(2), cap, n_pages=B)
    q = randn(B * T, H * D, seed=9, dtype=dtype)
    ctx, bits = torch.tensor([150, 0], **i32), tree_bits([t // 2 - 1 for t in range(T)])
    narrow = words(bits, 1).expand(B, T, 1).contiguous().cuda()
    wide = words([b | (2**256 - 2**T) for b in bits], 4).expand(B, T, 4).contiguous().cuda()
    want = torch.empty_like(q)
    ops.tree_attn(q, kv, ctx, narrow, want, H=H, G=G, D=D, impl=impl)
    big_q, big_o = torch.full((2, B * T, H * D + 40), float("nan"), dtype=dtype, device="cuda").unbind()
    big_q[:, 16 : 16 + H * D] = q
    out = big_o[:, 24 : 24 + H * D]
    ops.tree_attn(big_q[:, 16 : 16 + H * D], kv, ctx, wide, out, H=H, G=G, D=D, impl=impl)
    assert torch.equal(out, want)
    assert bool(torch.isnan(big_o[:, :24]).all()) and bool(torch.isnan(big_o[:, 24 + H * D :]).all())
    for b, c in enumerate(ctx.tolist()):
        see = torch.ones(T, c + T, dtype=torch.bool, device="cuda")
        see[:, c:] = torch.tensor([[(x >> j) & 1 for j in range(T)] for x in bits], dtype=torch.bool)
        for h in range(H):
            check_rows(want.view(B, T, H, D)[b, :, h], None, rows(q.view(B, T, H, D)[b, :, h], store[b, 0, h // 2, : c + T], store[b, 1, h // 2, : c + T], see, scale_of(D)),
                       D, c + T, dtype, dtype == BF and impl != 1)


# ---- more than 2^31 elements between a tensor's ends -------------------------------------------------------------
FAR = 2**23 + 64  # elements between rows, 300 of them


@pytest.mark.parametrize("D,dtype,impl", [(64, BF, 0), (64, BF, 1), (16, F32, 0)])
def test_packed_rows_far_apart(D, dtype, impl):
    from diff_gpt_b200 import ops

    N, H, G = 300, 2, 1
    room = torch.empty(N, FAR, dtype=dtype, device="cuda")
    q, k, v = (randn(N, h, D, seed=s, dtype=dtype) for h, s in ((H, 1), (G, 2), (G, 3)))
    starts = torch.tensor([0, 100, 290], **i32)
    want, want_lse, lse = torch.zeros_like(q), torch.zeros(N, H, device="cuda"), torch.zeros(N, H, device="cuda")
    ops.fmha_packed(q, k, v, starts, want, lse=want_lse, impl=impl)
    at, views = 0, []
    for x in (q, k, v, want):
        w = x.shape[1] * D
        views.append(room[:, at : at + w].unflatten(1, (-1, D)))
        at = FAR // 2 if at == 0 else at + w  # (the others' last rows lie further back still)
    for view, x in zip(views, (q, k, v, torch.zeros_like(want))):
        view.copy_(x)
    ops.fmha_packed(views[0], views[1], views[2], starts, views[3], lse=lse, impl=impl)
    assert torch.equal(views[3], want) and torch.equal(lse, want_lse)


@pytest.mark.parametrize("layout", ["pages", "dense"])
@pytest.mark.parametrize("D,dtype,impl", [(64, BF, 0), (64, BF, 1), (16, F32, 0)])
def test_caches_with_far_pages(D, dtype, impl, layout):
    """Trees, and accepted rows' move, in pages (or whole sequences) that lie 2^26 elements apart."""
    from diff_gpt_b200 import ops

    H, G, B, T, page, per = 4, 2, 2, 5, 64, 20
    apart, n = (2**26, B * per) if layout == "pages" else (2**31 + 64, B)
    tokens = page if layout == "pages" else page * 4
    small = randn(n, 2, G, tokens, D, seed=4, dtype=dtype)
    room = torch.empty((n - 1) * apart + small[0].numel(), dtype=dtype, device="cuda")
    far = room.as_strided(small.shape, (apart, *small.stride()[1:]))
    far.copy_(small)
    table = torch.randperm(n, generator=torch.Generator().manual_seed(2)).to(torch.int32).view(B, per).cuda() if layout == "pages" else None
    near_kv, far_kv = (ops.kv_layout(x[0, 0], x[0, 1], x.stride(0), x.stride(2), tokens, table, n_pages=n) for x in (small, far))
    slots = per * page if layout == "pages" else tokens
    ctx = torch.tensor([slots - T, slots // 2], **i32)
    anc = words(tree_bits([t - 1 for t in range(T)]), 1).expand(B, T, 1).contiguous().cuda()
    q = randn(B * T, H * D, seed=5, dtype=dtype)
    a, b, status = torch.empty_like(q), torch.empty_like(q), torch.zeros(1, **i32)
    ops.tree_attn(q, near_kv, ctx, anc, a, H=H, G=G, D=D, impl=impl, status=status)
    ops.tree_attn(q, far_kv, ctx, anc, b, H=H, G=G, D=D, impl=impl, status=status)
    assert torch.equal(a, b) and status.item() == 0 and bool(torch.isfinite(a).all())
    path, count = torch.tensor([[1, 3, 4], [0, 2, 3]], **i32), torch.tensor([3, 2], **i32)
    for kv in (near_kv, far_kv):
        ops.kv_keep(kv, ctx, ctx - 70, path, count, n_layer=1, layer_stride=0, H=G, D=D, dtype=dtype, status=status)
    assert torch.equal(far, small) and status.item() == 0


@pytest.mark.parametrize("dtype", [BF, F32])
def test_accepted_rows_of_far_layers(dtype):
    """Layers 2^31 elements apart."""
    from diff_gpt_b200 import ops

    L, pages, H, page, D, apart = 2, 4, 2, 16, 16, 2**31 + 8
    small = randn(L, pages, 2, H, page, D, seed=6, dtype=dtype)
    room = torch.empty(apart + small[0].numel(), dtype=dtype, device="cuda")
    far = room.as_strided(small.shape, (apart, *small.stride()[1:]))
    far.copy_(small)
    table, path = torch.tensor([[3, 1], [0, 2]]), [[1, 2], [0, 3]]
    kv = ops.kv_layout(far[0, 0, 0], far[0, 0, 1], far.stride(1), far.stride(3), page, table.to(**i32), n_pages=pages)
    ops.kv_keep(kv, torch.tensor([14, 20], **i32), torch.tensor([3, 20], **i32), torch.tensor(path, **i32), torch.tensor([2, 2], **i32), n_layer=L,
                layer_stride=apart, H=H, D=D, dtype=dtype)
    assert torch.equal(far.cpu(), keep_plain(small.cpu(), table.tolist(), [14, 20], [3, 20], path, [2, 2], page))


@pytest.mark.parametrize("dtype", [BF, F32])
def test_rows_of_logits_far_apart(dtype):
    R, V = 300, 1001
    far = torch.empty(R, FAR, dtype=dtype, device="cuda")[:, 3 : 3 + V]
    far.copy_(randn(R, V, seed=7, dtype=dtype))
    check_logprobs(far, torch.arange(R, **i32), 1.0, 5)


# ---- at the same time --------------------------------------------------------------------------------------------
@pytest.mark.parametrize("D,dtype", [(64, BF), (16, F32)])
def test_calls_on_two_streams_at_once(D, dtype):
    """Trees whose shares need a workspace, prompts and log probabilities, each on either stream while the other's are at work."""
    from diff_gpt_b200 import ops

    H, G, B, T, cap = 4, 2, 3, 7, 6000
    store = randn(B, 2, G, cap, D, seed=10, dtype=dtype)
    kv = ops.kv_layout(store[0, 0], store[0, 1], store.stride(0), store.stride(2), cap, n_pages=B)
    ctx, anc = torch.tensor([5900, 300, 4000], **i32), words(tree_bits([t - 1 for t in range(T)]), 1).expand(B, T, 1).contiguous().cuda()
    starts = torch.tensor([0, 400, 700], **i32)

    def job(seed):
        q, x = randn(B * T, H * D, seed=seed, dtype=dtype), randn(700, H, D, seed=seed + 1, dtype=dtype)
        z, t = randn(50, 9001, seed=seed + 2, dtype=dtype), torch.arange(50, **i32)

        def go():
            o, p = torch.empty_like(q), torch.empty_like(x)
            ops.tree_attn(q, kv, ctx, anc, o, H=H, G=G, D=D)
            ops.fmha_packed(x, x, x, starts, p)
            return [o, p, *ops.token_logprobs(z, t, top_k=4)]

        return go

    jobs = [job(20), job(30)]
    want = [go() for go in jobs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(20):
        for i in (0, 1):
            with torch.cuda.stream(streams[i]):
                got[i].append(jobs[i]())
    torch.cuda.synchronize()
    for i in (0, 1):
        assert all(torch.equal(a, b) for r in got[i] for a, b in zip(r, want[i]))
