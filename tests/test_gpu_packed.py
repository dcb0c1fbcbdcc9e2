"""ops.fmha_packed: prompts of different lengths one behind another, against attention of each in float64."""

import pytest
import torch

from drafts_cases import check_rows, rows, scale_of, starts

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32
LENS = {
    "one": [1], "edges": [127, 128, 129], "ragged": [0, 5, 0, 1, 130, 300, 0], "many": [3, 17, 64, 1, 33, 2, 90, 250, 7, 128, 256, 65],
    "long": [1100, 77], "none": [0, 0],
}


def run(lens, H, G, D, dtype, impl, past=None, first=0, tail=0, scale=None, seed=0, fused=False, spoil=None, base=0.0):
    """past: keys that each prompt has before its own (negative: fewer keys than queries); first, tail: rows before and behind the
    prompts; fused: views of one wide tensor; spoil: a prompt whose numbers are not numbers."""
    from diff_gpt_b200 import ops

    g = torch.Generator().manual_seed(seed + 31 * D + H)
    past = past or [0] * len(lens)
    own_keys = any(past)
    qs = starts(lens, first)
    klens = [max(0, n + p) for n, p in zip(lens, past)]
    ks = starts(klens, first if not own_keys else 3) if own_keys else qs
    N, M = qs[-1] + tail, ks[-1] + (tail if not own_keys else 2)
    if not own_keys:
        M = N
    if fused:
        wide = torch.randn(N, (H + 2 * G) * D + 24, generator=g).to(dtype)
        q, k, v = (x.reshape(N, -1, D) for x in (wide[:, : H * D], wide[:, H * D : (H + G) * D], wide[:, (H + G) * D : (H + 2 * G) * D]))
    else:
        q, k, v = (torch.randn(n, h, D, generator=g).to(dtype) + base for n, h in ((N, H), (M, G), (M, G)))
        q, k, v = q.to(dtype), k.to(dtype), v.to(dtype)
    inside_q = torch.zeros(N, dtype=torch.bool)
    inside_k = torch.zeros(M, dtype=torch.bool)
    inside_q[qs[0] : qs[-1]] = True
    inside_k[ks[0] : ks[-1]] = True
    bad = torch.tensor([float("nan"), float("inf"), -float("inf")]).to(dtype)
    outside_q, outside_k = torch.nonzero(~inside_q)[:, 0], torch.nonzero(~inside_k)[:, 0]
    q, k, v = q.clone(), k.clone(), v.clone()
    q[outside_q] = bad[outside_q % 3][:, None, None]
    k[outside_k] = bad[outside_k % 3][:, None, None]
    v[outside_k] = bad[outside_k % 3][:, None, None]
    if spoil is not None:
        for t, s in ((q, qs), (k, ks), (v, ks)):
            t[s[spoil] : s[spoil + 1]] = float("nan")
    if fused:
        wide[:, : H * D], wide[:, H * D : (H + G) * D], wide[:, (H + G) * D : (H + 2 * G) * D] = q.flatten(1), k.flatten(1), v.flatten(1)
        w = wide.cuda()
        dq, dk, dv = (x.view(N, -1, D) if x.is_contiguous() else x.unflatten(1, (-1, D)) for x in
                      (w[:, : H * D], w[:, H * D : (H + G) * D], w[:, (H + G) * D : (H + 2 * G) * D]))
    else:
        dq, dk, dv = q.cuda(), k.cuda(), v.cuda()
    out = torch.full((N, H, D), -7.0, dtype=dtype, device="cuda")
    lse = torch.full((N, H), -7.0, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    i32 = dict(dtype=torch.int32, device="cuda")
    ops.fmha_packed(dq, dk, dv, torch.tensor(qs, **i32), out, key_starts=torch.tensor(ks, **i32) if own_keys else None, lse=lse, impl=impl,
                    status=status, scale=scale)
    torch.cuda.synchronize()
    assert status.item() == 0
    got, got_lse = out.cpu(), lse.cpu()
    assert bool((got[outside_q] == -7).all()) and bool((got_lse[outside_q] == -7).all())  # rows of no prompt stay
    for s, (n, m) in enumerate(zip(lens, klens)):
        if s == spoil or n == 0:
            continue
        see = torch.ones(n, m, dtype=torch.bool).tril(m - n)
        for h in range(H):
            kv = h // (H // G)
            a, b = slice(qs[s], qs[s] + n), slice(ks[s], ks[s] + m)
            want = rows(q[a, h], k[b, kv], v[b, kv], see, scale or scale_of(D))
            check_rows(got[a, h], got_lse[a, h], want, D, m, dtype, dtype == BF and impl != 1)
    return out


@pytest.mark.parametrize("impl", [0, 1])
@pytest.mark.parametrize("lens", list(LENS))
@pytest.mark.parametrize("D,dtype", [(8, F32), (16, F32), (32, F32), (64, F32), (128, F32), (8, BF), (16, BF), (32, BF), (64, BF), (128, BF)])
def test_lengths(lens, D, dtype, impl):
    run(LENS[lens], 4, 2, D, dtype, impl)


@pytest.mark.parametrize("impl", [0, 1])
@pytest.mark.parametrize("H,G", [(1, 1), (3, 3), (6, 2), (5, 1), (16, 4)])
@pytest.mark.parametrize("D,dtype", [(64, BF), (128, BF), (16, F32)])
def test_heads(H, G, D, dtype, impl):
    run([200, 31, 140], H, G, D, dtype, impl, seed=1)


@pytest.mark.parametrize("impl", [0, 1])
@pytest.mark.parametrize("past", [[40, 0, 300, 129], [-5, -130, 60, -1000], [1, -1, 0, -64]])
@pytest.mark.parametrize("D,dtype", [(64, BF), (128, BF), (32, F32)])
def test_keys_of_their_own(past, D, dtype, impl):
    """Keys that were there before, and queries that see no key: zeros and -inf."""
    run([130, 140, 1, 64], 4, 2, D, dtype, impl, past=past, seed=2)


@pytest.mark.parametrize("impl", [0, 1])
@pytest.mark.parametrize("D,dtype", [(32, BF), (64, BF), (128, BF), (16, F32)])
def test_rows_of_no_prompt(D, dtype, impl):
    """Numbers that are none before, between (an empty prompt) and behind the prompts reach no output."""
    run([100, 0, 150], 4, 4, D, dtype, impl, first=5, tail=70, seed=3)
    run([100, 3, 150], 4, 4, D, dtype, impl, first=5, tail=3, seed=4, fused=True)


@pytest.mark.parametrize("impl", [0, 1])
@pytest.mark.parametrize("spoil", [0, 1, 2])
@pytest.mark.parametrize("D,dtype", [(64, BF), (128, BF), (16, F32)])
def test_a_prompt_of_nans_spoils_no_other(spoil, D, dtype, impl):
    run([100, 29, 200], 2, 1, D, dtype, impl, spoil=spoil, seed=5)


@pytest.mark.parametrize("impl", [0, 1])
@pytest.mark.parametrize("D,dtype", [(64, BF), (128, BF), (16, F32)])
@pytest.mark.parametrize("scale", [1e-3, 0.5, 3.0])
def test_scales(scale, D, dtype, impl):
    """From nearly level probabilities to one key that takes everything, with maxima that move from tile to tile."""
    run([500, 260], 2, 2, D, dtype, impl, scale=scale, seed=6)


@pytest.mark.parametrize("impl", [0, 1])
@pytest.mark.parametrize("D,dtype", [(32, BF), (64, BF), (128, BF), (16, F32)])
def test_heads_before_rows(D, dtype, impl):
    """A head's rows side by side, as a cache lays them out: the same numbers as with a row's heads side by side."""
    from diff_gpt_b200 import ops

    H, G, starts = 4, 2, torch.tensor([0, 130, 131, 131, 300], dtype=torch.int32, device="cuda")
    q, k, v = (torch.randn(h, 300, D, device="cuda").to(dtype) for h in (H, G, G))
    o, want, lse, want_lse = torch.empty_like(q), q.new_empty(300, H, D), torch.empty(300, H, device="cuda"), torch.empty(300, H, device="cuda")
    ops.fmha_packed(*(x.transpose(0, 1) for x in (q, k, v)), starts, o.transpose(0, 1), lse=lse, impl=impl)
    ops.fmha_packed(*(x.transpose(0, 1).contiguous() for x in (q, k, v)), starts, want, lse=want_lse, impl=impl)
    assert torch.equal(o.transpose(0, 1), want) and torch.equal(lse, want_lse)


@pytest.mark.parametrize("D,dtype", [(64, BF), (128, BF), (16, F32)])
def test_rising_scores(D, dtype):
    """Scores that grow along the prompt: the running maximum moves in every tile."""
    from diff_gpt_b200 import ops

    n, g = 900, torch.Generator().manual_seed(7)
    q, k, v = (torch.randn(n, 1, D, generator=g).abs() for _ in range(3))
    k = k * torch.linspace(0.1, 12, n)[:, None, None]
    q, k, v = q.to(dtype), k.to(dtype), v.to(dtype)
    out = torch.empty(n, 1, D, dtype=dtype, device="cuda")
    lse = torch.empty(n, 1, device="cuda")
    ops.fmha_packed(q.cuda(), k.cuda(), v.cuda(), torch.tensor([0, n], dtype=torch.int32, device="cuda"), out, lse=lse)
    want = rows(q[:, 0], k[:, 0], v[:, 0], torch.ones(n, n, dtype=torch.bool).tril(), scale_of(D))
    check_rows(out[:, 0].cpu(), lse[:, 0].cpu(), want, D, n, dtype, dtype == BF)


@pytest.mark.parametrize("impl", [0, 1])
@pytest.mark.parametrize("D,dtype", [(64, BF), (128, BF), (16, F32)])
def test_many_prompts_without_keys(D, dtype, impl):
    """More tiles than the GPU holds at a time, most of whose queries see no key, between ones with up to nine tiles of them."""
    lens = [130, 5, 1, 260, 64] * 40
    run(lens, 2, 2, D, dtype, impl, past=[-200, -5, 1100, -300, 0] * 40, seed=9)


@pytest.mark.parametrize("D,dtype", [(128, BF), (16, F32)])
def test_repeats_graphs_and_streams(D, dtype):
    """The same bits from call to call, from a graph that is replayed over new numbers, and on another stream."""
    from diff_gpt_b200 import ops

    H, G, lens = 8, 2, [300, 5, 777, 0, 64]
    st = torch.tensor(starts(lens), dtype=torch.int32, device="cuda")
    N = sum(lens)
    g = torch.Generator(device="cuda").manual_seed(8)
    q, k, v = (torch.randn(N, h, D, generator=g, device="cuda").to(dtype) for h in (H, G, G))
    out = torch.empty_like(q)
    ops.fmha_packed(q, k, v, st, out)
    first = out.clone()
    for _ in range(5):
        out.zero_()
        ops.fmha_packed(q, k, v, st, out)
        assert torch.equal(out, first)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out.zero_()
        ops.fmha_packed(q, k, v, st, out)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(out, first)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.fmha_packed(q, k, v, st, out)
    q2 = torch.randn(N, H, D, generator=g, device="cuda").to(dtype)
    want = torch.empty_like(q)
    ops.fmha_packed(q2, k, v, st, want)
    q.copy_(q2)
    out.zero_()
    graph.replay()
    assert torch.equal(out, want)


@pytest.mark.parametrize("impl", [0, 1])
@pytest.mark.parametrize("bad", [[0, 90, 50, 300], [-4, 20, 100, 200], [0, 100, 200, 400], [0, 100, 100, 2**31 - 1], [-2**31, -1, -1, 5]])
def test_wrong_starts_are_reported(bad, impl):
    from diff_gpt_b200 import ops

    q, k, v = (torch.randn(300, 2, 64, device="cuda").to(BF) for _ in range(3))
    out = torch.zeros_like(q)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    ops.fmha_packed(q, k, v, torch.tensor(bad, dtype=torch.int32, device="cuda"), out, impl=impl, status=status)
    assert status.item() & 1


def test_no_rows_and_no_prompts():
    from diff_gpt_b200 import ops

    q = torch.zeros(0, 2, 64, dtype=BF, device="cuda")
    one = torch.zeros(1, dtype=torch.int32, device="cuda")
    ops.fmha_packed(q, q, q, one, q)
    x = torch.ones(5, 2, 64, dtype=BF, device="cuda")
    out = torch.full_like(x, 3)
    ops.fmha_packed(x, x, x, one, out)
    seen = out.clone()
    ops.fmha_packed(x, x[:0], x[:0], torch.tensor([0, 5], dtype=torch.int32, device="cuda"), seen,
                    key_starts=torch.zeros(2, dtype=torch.int32, device="cuda"))
    assert bool((out == 3).all()) and not bool(seen.any())  # no keys: zeros
