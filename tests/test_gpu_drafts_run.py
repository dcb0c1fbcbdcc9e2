"""The operators together, as a server with drafted tokens uses them: prompts of different lengths in one launch, drafts appended to a paged
cache, attention of the tree, probabilities, the accepted path kept, and on from there."""

import pytest
import torch

from drafts_cases import check_rows, logprobs, rows, scale_of, starts, tree_bits, words

pytestmark = pytest.mark.gpu

PARENTS = [-1, 0, 0, 1, 2, 2, 4]
DEPTH = [0, 1, 1, 2, 2, 2, 3]
PATHS = [[0, 2, 4, 6], [0, 1]]  # what is accepted of either sequence


@pytest.mark.parametrize("dtype,D", [(torch.bfloat16, 64), (torch.bfloat16, 128), (torch.float32, 16)])
def test_prompts_drafts_and_what_follows(dtype, D):
    from diff_gpt_b200 import PagedKVCache, ops
    from diff_gpt_b200.model.rope import precompute_freqs_cis

    L, H, V, T, lens = 2, 4, 500, len(PARENTS), [70, 131]
    S, C, N = len(lens), H * D, sum(lens)
    g = torch.Generator(device="cuda").manual_seed(D)
    dev = dict(device="cuda")
    i32 = dict(dtype=torch.int32, device="cuda")
    table = torch.randn(L, V, 3 * C, generator=g, **dev).to(dtype)  # q, k and v of a token, before rotation and norm
    head = (torch.randn(V, C, generator=g, **dev) / C**0.5).to(dtype)
    cs = precompute_freqs_cis(D, 400, 10000.0).to(dtype).cuda()
    cache = PagedKVCache(L, H, D, n_series=S, rows_per_series=1, prefix_len=max(lens), max_new=100, dtype=dtype, device="cuda")
    cache.pool.fill_(float("nan"))
    status = torch.zeros(1, **i32)

    def append(layer, ids, seq, pos, slot):
        """Tokens anywhere in any sequence: each a sequence of one token with its row's pages."""
        x = table[layer][ids]
        lay = cache._layout(layer, cache.row_table[seq].contiguous())
        q = torch.empty(len(ids), C, dtype=dtype, **dev)
        ops.rope_qknorm_kvappend(x[:, :C], x[:, C : 2 * C], x[:, 2 * C :], q, cs, lay, pos, slot, None, len(ids), 1, H, D, status)
        return q

    def held(layer, seq, slots):
        """Keys and values [slots, H, D] of a sequence."""
        page, at = cache.row_table[seq].long()[slots // cache.page_tokens], slots % cache.page_tokens
        return cache.pool[layer, page, 0, :, at], cache.pool[layer, page, 1, :, at]

    # ---- prompts ----
    st = torch.tensor(starts(lens), **i32)
    seq = torch.repeat_interleave(torch.arange(S, **dev), torch.tensor(lens, **dev))
    pos = torch.cat([torch.arange(n, **i32) for n in lens])
    ids = torch.randint(0, V, (N,), generator=g, **dev)
    for layer in range(L):
        q = append(layer, ids, seq, pos, pos)
        kv = [held(layer, s, torch.arange(n, **dev)) for s, n in enumerate(lens)]
        k, v = torch.cat([a for a, _ in kv]), torch.cat([b for _, b in kv])
        out = torch.empty(N, H, D, dtype=dtype, **dev)
        ops.fmha_packed(q.view(N, H, D), k, v, st, out, status=status)
        for s, n in enumerate(lens):
            a = starts(lens)[s]
            see = torch.ones(n, n, dtype=torch.bool).tril()
            for h in range(H):
                want = rows(q.view(N, H, D)[a : a + n, h].cpu(), k[a : a + n, h].cpu(), v[a : a + n, h].cpu(), see, scale_of(D))
                check_rows(out[a : a + n, h].cpu(), None, want, D, n, dtype, dtype == torch.bfloat16)
    # ---- drafts ----
    prompt, first = torch.tensor(lens, **i32), torch.full((S,), cache.suffix_slot0, **i32)
    masks = words(tree_bits(PARENTS), 1).expand(S, T, 1).contiguous().cuda()
    drafts = torch.randint(0, V, (S * T,), generator=g, **dev)
    d_seq = torch.arange(S, **dev).repeat_interleave(T)
    d_pos = (prompt.repeat_interleave(T) + torch.tensor(DEPTH * S, **i32)).contiguous()
    d_slot = (first.repeat_interleave(T) + torch.arange(T, **i32).repeat(S)).contiguous()
    path = torch.tensor([p + [0] * (T - len(p)) for p in PATHS], **i32)
    count = torch.tensor([len(p) for p in PATHS], **i32)
    new = torch.randint(0, V, (S,), generator=g, **dev)
    n_pos, n_slot = prompt + count, first + count
    one = torch.ones(S, 1, dtype=torch.int64, **dev)

    def step():
        """Drafts, their attention and probabilities, the accepted ones kept, one more token behind them."""
        seen, after = [], []
        for layer in range(L):
            q = append(layer, drafts, d_seq, d_pos, d_slot)
            o = torch.empty(S * T, C, dtype=dtype, **dev)
            ops.tree_attn(q, cache.row_layout(layer), first, masks, o, H=H, G=H, D=D, gap_start=prompt, gap_end=first, status=status)
            seen.append((q, o))
        scores = ops.token_logprobs((seen[0][1] + seen[1][1]) @ head.T, drafts.to(torch.int32), top_k=3, status=status)
        cache.keep_drafts(first, first, path, count, status)
        for layer in range(L):
            q = append(layer, new, torch.arange(S, **dev), n_pos, n_slot)
            a, b = torch.empty(S, C, dtype=dtype, **dev), torch.empty(S, C, dtype=dtype, **dev)
            ops.tree_attn(q, cache.row_layout(layer), n_slot, one, a, H=H, G=H, D=D, gap_start=prompt, gap_end=first, status=status)
            ops.decode_attn(q, cache.row_layout(layer), prompt, first, count + 1, None, b, H=H, D=D)
            after.append((q, a, b))
        return seen, scores, after

    seen, scores, after = step()
    assert status.item() == 0
    lp, ent, top_ids, _ = logprobs(((seen[0][1] + seen[1][1]) @ head.T).cpu(), drafts.cpu(), 1.0, 3)
    assert (scores.logprob.cpu() - lp).abs().max() < 1e-5 and torch.equal(scores.top_ids.cpu().long(), top_ids)
    for layer in range(L):
        for s, n in enumerate(lens):
            # the drafts' keys before the move: append them once more elsewhere, in a cache of their own
            q, o = seen[layer]
            kept, values = held(layer, s, torch.arange(n, **dev))
            x = table[layer][drafts.view(S, T)[s]]
            fresh = torch.zeros(1, 2, H, T, D, dtype=dtype, **dev)
            lay = ops.kv_layout(fresh[0, 0], fresh[0, 1], 2 * H * T * D, T * D, T)
            for t in range(T):  # each at its own depth's position
                ops.rope_qknorm_kvappend(x[t : t + 1, :C], x[t : t + 1, C : 2 * C], x[t : t + 1, 2 * C :], torch.empty(1, C, dtype=dtype, **dev), cs, lay,
                                         d_pos.view(S, T)[s, t : t + 1].contiguous(), torch.tensor([t], **i32), None, 1, 1, H, D, status)
            dk, dv = fresh[0, 0].transpose(0, 1), fresh[0, 1].transpose(0, 1)
            k, v = torch.cat([kept, dk]).cpu(), torch.cat([values, dv]).cpu()
            bits = tree_bits(PARENTS)
            see = torch.tensor([[True] * n + [bool((bits[t] >> j) & 1) for j in range(T)] for t in range(T)])
            for h in range(H):
                want = rows(q.view(S, T, H, D)[s, :, h].cpu(), k[:, h], v[:, h], see, scale_of(D))
                check_rows(o.view(S, T, H, D)[s, :, h].cpu(), None, want, D, n + T, dtype, dtype == torch.bfloat16)
            # what was kept is the path's, in its order
            a, b = held(layer, s, cache.suffix_slot0 + torch.arange(len(PATHS[s]), **dev))
            assert torch.equal(a, dk[PATHS[s]]) and torch.equal(b, dv[PATHS[s]])
        q, a, b = after[layer]
        # both lie within u |o| + (tensor cores) 2^-8 A of the exact row, A at most the largest value
        tol = (2 * 2.0**-8 * b.float().abs() + 2.0**-8 * table[layer][:, 2 * C :].float().abs().max()) if dtype == torch.bfloat16 else 1e-5
        assert bool(((a.float() - b.float()).abs() <= tol).all())
    # ---- the same from a graph ----
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        again = step()
    for _ in range(2):
        graph.replay()
    assert status.item() == 0
    assert all(torch.equal(x, y) for x, y in zip(scores, again[1]))
    for p, r in zip(seen + after, again[0] + again[2]):
        assert all(torch.equal(x, y) for x, y in zip(p, r))
