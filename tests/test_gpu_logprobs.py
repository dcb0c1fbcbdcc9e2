"""ops.token_logprobs against float64, and ops.kv_keep against indexing."""

import math

import pytest
import torch

from drafts_cases import logprobs

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32


def check(logits, targets, T, k, r):
    """Within bounds that follow from the formula.  x = (z - m) log2(e) has three roundings, 2^-22 |x|; 2^x adds 2^-21 relative, its sum, in chains
    of at most V / 256 numbers a thread and 40 steps between threads, (V / 256 + 40) 2^-24 (2^-23 with the joins' factors); a log probability is the difference of
    x and the sum's logarithm.  entropy = sum p (-log p): every term's factor p is off by that relative, on terms of which the largest -log p that counts is below 40."""
    V = logits.shape[1]
    lp, ent, ids, top = logprobs(logits.cpu(), targets.cpu(), T, k)
    tol = 2.0**-20 + (V / 256 + 40) * 2.0**-23
    for got, want, t in ((r.logprob, lp, tol), (r.entropy, ent, tol * 40), (r.top_logprobs, top, tol)):
        got = got.cpu().double()
        inf = torch.isneginf(want.float())  # the answer is fp32: beyond its range it is -inf
        assert torch.equal(torch.isneginf(got), inf)
        off = torch.where(inf, 0.0, (got - want).abs())
        assert bool((off <= t + 2.0**-22 * torch.where(inf, 0.0, want.abs())).all()), (off - t).max().item()
    assert torch.equal(r.top_ids.cpu().long(), ids)


def make(R, V, dtype, seed, kind="normal"):
    g = torch.Generator(device="cuda").manual_seed(seed)
    z = torch.randn(R, V, generator=g, device="cuda") * 3
    if kind == "ties":
        z = z.round()
    elif kind == "level":
        z = torch.full_like(z, 1.5)
    elif kind == "rising":
        z = torch.arange(V, device="cuda").float().expand(R, V) / V * 9
    elif kind == "falling":
        z = -torch.arange(V, device="cuda").float().expand(R, V) / V * 9
    elif kind == "peaked":
        z[:, V // 2] = 60.0
    elif kind == "masked":
        z[torch.rand(R, V, generator=g, device="cuda") < 0.99] = float("-inf")
        z[:, min(V - 1, 3)] = 0.25
    elif kind == "three":  # fewer tokens left than are asked for
        z[:, : max(1, V - 3)] = float("-inf")
    elif kind == "comb":  # the largest lie where one group of threads reads them
        z[:, ::256] += 50.0
    elif kind == "zeros":
        z = torch.where(torch.rand(R, V, generator=g, device="cuda") < 0.5, 0.0, -0.0)
    elif kind == "lowest":
        z[:, V // 3 :] = torch.finfo(dtype).min
    return z.to(dtype), torch.randint(0, V, (R,), generator=g, device="cuda").to(torch.int32)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("R,V", [(1, 1), (3, 2), (2, 31), (5, 257), (1, 4096), (7, 5000), (2, 32001), (1, 128255), (33, 16384), (400, 777), (1000, 64)])
def test_sizes(R, V, dtype):
    from diff_gpt_b200 import ops

    logits, targets = make(R, V, dtype, V)
    for k in sorted({0, 1, min(5, V), min(32, V)}):
        check(logits, targets, 1.0, k, ops.token_logprobs(logits, targets, top_k=k))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("R,V,kind", [(200, 70001, "normal"), (200, 70001, "ties"), (160, 70001, "rising"), (160, 70001, "falling"), (160, 70001, "masked"), (700, 40003, "normal")])
def test_rows_of_many_rounds(R, V, kind, dtype):
    """Rows too many for clusters and too long for four rounds of loads, and several of them to a CTA."""
    from diff_gpt_b200 import ops

    logits, targets = make(R, V, dtype, 6, kind)
    check(logits, targets, 1.0, 20, ops.token_logprobs(logits, targets, top_k=20))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("kind", ["ties", "level", "rising", "falling", "peaked", "masked", "three", "comb", "zeros", "lowest"])
@pytest.mark.parametrize("R,V", [(2, 40), (3, 20000), (320, 6001), (1, 100000)])
def test_distributions(R, V, kind, dtype):
    from diff_gpt_b200 import ops

    logits, targets = make(R, V, dtype, 3, kind)
    for k, T in ((20, 1.0), (32, 0.6)):
        check(logits, targets, T, k, ops.token_logprobs(logits, targets, top_k=k, temperature=T))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("off", [0, 1, 2, 3, 5, 7])
def test_rows_on_any_boundary(off, dtype):
    """Columns of a wider tensor whose neighbours are not numbers."""
    from diff_gpt_b200 import ops

    for R, V in ((3, 9), (4, 1001), (300, 515)):
        wide = torch.full((R, V + 13), float("nan"), dtype=dtype, device="cuda")
        logits, targets = make(R, V, dtype, off + V)
        view = wide[:, off : off + V]
        view.copy_(logits)
        check(logits, targets, 1.3, 5, ops.token_logprobs(view, targets, top_k=5, temperature=1.3))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("V", [50, 9000, 70000])
def test_rows_without_a_distribution(V, dtype):
    """NaN, +inf, nothing but -inf: NaN for them, in their rows alone; ids stay tokens."""
    from diff_gpt_b200 import ops

    logits, targets = make(6, V, dtype, 1)
    logits[1, V // 2] = float("nan")
    logits[2, V - 1] = float("inf")
    logits[3] = float("-inf")
    logits[4] = float("nan")
    r = ops.token_logprobs(logits, targets, top_k=8)
    bad = torch.tensor([0, 1, 1, 1, 1, 0], dtype=torch.bool, device="cuda")
    assert torch.equal(torch.isnan(r.logprob), bad) and torch.equal(torch.isnan(r.entropy), bad)
    assert torch.equal(torch.isnan(r.top_logprobs), bad[:, None].expand(6, 8))
    assert bool(((r.top_ids >= 0) & (r.top_ids < V)).all())
    assert r.top_ids[2, 0].item() == V - 1 and r.top_ids[3].tolist() == list(range(8)) == r.top_ids[4].tolist()
    ok = [0, 5]
    part = ops.token_logprobs(logits[ok].contiguous(), targets[ok].contiguous(), top_k=8)
    check(logits[ok], targets[ok], 1.0, 8, part)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("V", [11, 40, 5001])
def test_ids_of_rows_with_nans_at_the_ends(V, dtype):
    """NaN where a row's first and last vectors are partly another row's, -inf and nothing else between: ids are tokens, NaN behind -inf."""
    from diff_gpt_b200 import ops

    logits = torch.full((9, V), float("-inf"), dtype=dtype, device="cuda")
    logits[:, :3] = float("nan")
    logits[:, -2:] = float("nan")
    r = ops.token_logprobs(logits, torch.zeros(9, dtype=torch.int32, device="cuda"), top_k=8)
    want = (list(range(3, V - 2)) + [0, 1, 2, V - 2, V - 1])[:8]
    assert r.top_ids.tolist() == [want] * 9 and bool(torch.isnan(r.top_logprobs).all())


@pytest.mark.parametrize("dtype", [BF, F32])
def test_rows_beyond_the_range_of_one_exponent(dtype):
    """Nothing but the type's lowest value, huge logits of either sign, temperatures next to zero."""
    from diff_gpt_b200 import ops

    low = torch.finfo(dtype).min
    for V in (100, 40000):
        logits, targets = make(4, V, dtype, 8)
        logits[0] = low
        logits[1, :] = low / 2
        logits[1, 7] = low / 4
        logits[2] = logits[2] * 1e30
        logits[3, 5] = -low
        r = ops.token_logprobs(logits, targets, top_k=3)
        lp, ent, ids, top = logprobs(logits.cpu(), targets.cpu(), 1.0, 3)
        assert torch.equal(r.top_ids.cpu().long(), ids) and bool(torch.isfinite(r.entropy).all())
        assert torch.allclose(r.entropy.cpu().double(), ent, atol=1e-5, rtol=1e-5)  # log V, 0, 0, 0: see check()
        assert torch.allclose(r.top_logprobs.cpu().double(), top.float().double(), atol=1e-5, rtol=2.0**-21)
        cold = ops.token_logprobs(logits[:1] * 0 + 1.0, targets[:1], top_k=1, temperature=1e-30)
        assert abs(cold.entropy.item() - math.log(V)) < 1e-5


def test_targets_outside_the_vocabulary():
    from diff_gpt_b200 import ops

    logits, targets = make(4, 100, F32, 2)
    targets[1], targets[2] = -1, 100
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    r = ops.token_logprobs(logits, targets, top_k=2, status=status)
    assert status.item() == 4 and torch.isnan(r.logprob).tolist() == [False, True, True, False]
    assert bool(torch.isfinite(r.entropy).all()) and bool(torch.isfinite(r.top_logprobs).all())
    assert ops.token_logprobs(logits[:0], targets[:0], top_k=2).top_ids.shape == (0, 2)


@pytest.mark.parametrize("R,V", [(1, 50000), (500, 5000)])
def test_agrees_with_token_nll_repeats_and_graphs(R, V):
    from diff_gpt_b200 import ops

    logits, targets = make(R, V, F32, 4)
    r = ops.token_logprobs(logits, targets, top_k=4)
    assert (r.logprob + ops.token_nll(logits, targets)).abs().max().item() < 1e-4
    again = ops.token_logprobs(logits, targets, top_k=4)
    assert all(torch.equal(a, b) for a, b in zip(r, again))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = ops.token_logprobs(logits, targets, top_k=4)
    fresh, _ = make(R, V, F32, 5)
    logits.copy_(fresh)
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(kept, ops.token_logprobs(fresh, targets, top_k=4)))


# ---- kv_keep ----------------------------------------------------------------------------------------------------
def keep_plain(pool, table, src, dst, path, count, page):
    """pool [L, pages, kinds, H, page, D] after the move."""
    new = pool.clone()
    for s, n in enumerate(count):
        for i in range(n):
            a, b = src[s] + path[s][i], dst[s] + i
            new[:, table[s][b // page], :, :, b % page] = pool[:, table[s][a // page], :, :, a % page]
    return new


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("T,page,D", [(1, 64, 64), (8, 64, 16), (16, 8, 128), (17, 64, 8), (64, 16, 64), (65, 64, 32), (256, 24, 24)])
def test_accepted_rows_move(T, page, D, dtype):
    from diff_gpt_b200 import ops

    L, H, B = 3, 2, 4
    g = torch.Generator().manual_seed(T)
    pages = (2 * T + 150) // page + 2
    pool = torch.randn(L, B * pages, 2, H, page, D, generator=g).to(dtype)
    table = torch.randperm(B * pages, generator=g).view(B, pages)
    src = [70, 0, 100, T + 3]
    dst = [70, 5, 0, 20]  # in place, behind the source (overlapping), in front of it, in front (overlapping)
    count = [T, T, max(1, T // 2), T]
    path = [torch.randperm(T, generator=g).tolist(), list(range(T)), torch.randint(0, T, (T,), generator=g).tolist(), sorted(torch.randint(0, T, (T,), generator=g).tolist())]
    i32 = dict(dtype=torch.int32, device="cuda")
    status = torch.zeros(1, **i32)
    dev = pool.cuda()
    kv = ops.kv_layout(dev[0, 0, 0], dev[0, 0, 1], dev.stride(1), dev.stride(3), page, table.to(torch.int32).cuda(), n_pages=B * pages)
    ops.kv_keep(kv, torch.tensor(src, **i32), torch.tensor(dst, **i32), torch.tensor(path, **i32), torch.tensor(count, **i32), n_layer=L,
                layer_stride=dev.stride(0), H=H, D=D, dtype=dtype, status=status)
    assert status.item() == 0
    assert torch.equal(dev.cpu(), keep_plain(pool, table.tolist(), src, dst, path, count, page))


@pytest.mark.parametrize("dtype", [BF, F32])
def test_rows_of_one_storage_and_a_dense_cache(dtype):
    """A row cache (k_base == v_base, one head as wide as a row) and the reference's dense tensor."""
    from diff_gpt_b200 import KVCache, ops

    i32 = dict(dtype=torch.int32, device="cuda")
    rows = torch.randn(5, 16, 40).to(dtype)
    table = torch.tensor([[4, 1], [0, 2]])
    dev = rows.cuda()
    kv = ops.kv_layout(dev, dev, dev.stride(0), 0, 16, table.to(torch.int32).cuda(), n_pages=5)
    path = [[1, 3, 6], [0, 2, 2]]
    ops.kv_keep(kv, torch.tensor([10, 20], **i32), torch.tensor([10, 19], **i32), torch.tensor(path, **i32), torch.tensor([3, 2], **i32),
                n_layer=1, layer_stride=0, H=1, D=40, dtype=dtype)
    want = keep_plain(rows[None, :, None, None], table.tolist(), [10, 20], [10, 19], path, [3, 2], 16)
    assert torch.equal(dev.cpu(), want[0, :, 0, 0])
    c = KVCache(batch_size=2, num_heads=3, seq_len=32, head_dim=16, num_layers=2)
    c.ensure(32, dtype, torch.device("cuda"))
    c.kv_cache.copy_(torch.randn(c.kv_shape).to(dtype))
    old = c.kv_cache.clone()
    ops.kv_keep(c.layer_layout(0), torch.tensor([8, 12], **i32), torch.tensor([8, 12], **i32), torch.tensor([[1, 4], [2, 0]], **i32),
                torch.tensor([2, 1], **i32), n_layer=2, layer_stride=c.kv_cache.stride(0), H=3, D=16, dtype=dtype)
    old[:, :, 0, :, 8], old[:, :, 0, :, 9], old[:, :, 1, :, 12] = old[:, :, 0, :, 9].clone(), old[:, :, 0, :, 12].clone(), old[:, :, 1, :, 14].clone()
    assert torch.equal(c.kv_cache, old)


def test_rows_that_do_not_exist_stay_and_are_reported():
    from diff_gpt_b200 import ops

    i32 = dict(dtype=torch.int32, device="cuda")
    for src, dst, path, count, table in (
        ([30], [0], [[5, 0]], [1], [[0, 1]]), ([0], [31], [[5, 6]], [2], [[0, 1]]), ([0], [0], [[-1, 3]], [1], [[0, 1]]), ([-9], [0], [[1, 2]], [1], [[0, 1]]),
        ([0], [0], [[1, 1]], [3], [[5, 1]]), ([0], [0], [[1, 1]], [-1], [[0, 1]]), ([0], [17], [[1, 1]], [1], [[0, -1]]), ([2**31 - 1], [0], [[2**31 - 1, 0]], [1], [[0, 1]]),
    ):
        pool = torch.randn(1, 2, 2, 1, 16, 8, device="cuda")
        old = pool.clone()
        kv = ops.kv_layout(pool[0, 0, 0], pool[0, 0, 1], pool.stride(1), pool.stride(3), 16, torch.tensor(table, **i32), n_pages=2)
        status = torch.zeros(1, **i32)
        ops.kv_keep(kv, torch.tensor(src, **i32), torch.tensor(dst, **i32), torch.tensor(path, **i32), torch.tensor(count, **i32), n_layer=1,
                    layer_stride=0, H=1, D=8, dtype=torch.float32, status=status)
        assert status.item() == 1, (src, dst)
        if dst != [31]:
            assert torch.equal(pool, old)
