"""The operators behind serving with drafted tokens: what is measured, their plain forms, and their values in 64 bits.

    packed      ops.fmha_packed: causal attention over prompts of different lengths that lie one behind another, grouped heads;
                also portions of prompts whose earlier keys are there already (more keys than queries)
    tree        ops.tree_attn: a tree of drafted tokens behind every sequence of a paged cache; a draft sees the cached tokens and
                its own ancestors
    logprobs    ops.token_logprobs: log probability of a given token per row of logits, entropy, top alternatives
    keep        PagedKVCache's accepted drafts, ops.kv_keep: rows of an accepted path move to the cache's end, in every layer

Sizes are those of the reference configurations (heads of 16, 64 and 128, 4 to 16 of them) and of the design runs (16 query heads
on 4 key/value heads, vocabulary 16384), lengths from one token up.
"""

import math
import random

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
PAGE = 64  # the caches' default


def listed():
    return [
        # the smallest call: one short prompt, all latency
        dict(name="packed_one", kind="packed", lens=1, low=61, high=61, past=0, heads=16, groups=4, dim=64, dtype="bf16", shape=1),
        # a batch of questions of every length between one line and a page (12 heads of 64, reference configuration 4)
        dict(name="packed_mixed", kind="packed", lens=40, low=17, high=1000, past=0, heads=12, groups=12, dim=64, dtype="bf16", shape=2),
        # long documents, grouped heads (the design runs' 16 on 4 heads of 128)
        dict(name="packed_long", kind="packed", lens=4, low=2500, high=4096, past=0, heads=16, groups=4, dim=128, dtype="bf16", shape=3),
        # small fp32 models (reference configuration 1), portions behind keys that are there already
        dict(name="packed_f32", kind="packed", lens=32, low=20, high=140, past=90, heads=4, groups=4, dim=16, dtype="f32", shape=4),
        # one request, eight drafts: latency
        dict(name="tree_one", kind="tree", batch=1, nodes=8, low=777, high=777, heads=16, groups=4, dim=128, dtype="bf16", shape=5),
        # a serving batch, trees of up to 32 drafts behind caches of very different lengths
        dict(name="tree_batch", kind="tree", batch=48, nodes=32, low=300, high=4000, heads=16, groups=4, dim=128, dtype="bf16", shape=6),
        # few requests with long caches, wide trees
        dict(name="tree_long", kind="tree", batch=3, nodes=64, low=40000, high=65000, heads=16, groups=4, dim=128, dtype="bf16", shape=7),
        # small fp32 models
        dict(name="tree_f32", kind="tree", batch=24, nodes=13, low=30, high=500, heads=4, groups=4, dim=16, dtype="f32", shape=8),
        # a step's drafts of a small batch under the sampling temperature: few rows
        dict(name="logprobs_step", kind="logprobs", rows=13, vocab=16384, top=5, temperature=0.8, masked=0.0, dtype="bf16"),
        # scoring whole prompts: rows of an odd vocabulary, so that hardly a row starts on a vector's boundary
        dict(name="logprobs_prompt", kind="logprobs", rows=4096, vocab=32001, top=20, temperature=1.0, masked=0.0, dtype="bf16"),
        # three of eight drafts accepted of one request
        dict(name="keep_one", kind="keep", batch=1, nodes=8, most=3, layers=12, heads=12, dim=64, low=777, high=777, dtype="bf16", shape=9),
        # a serving batch, up to a dozen accepted
        dict(name="keep_batch", kind="keep", batch=192, nodes=64, most=12, layers=12, heads=12, dim=64, low=100, high=900, dtype="bf16", shape=10),
    ]


def _log(rng, low, high):
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    kind = rng.choice(("packed", "packed", "tree", "tree", "logprobs", "keep"))
    shape = rng.randint(100, 10**6)
    dtype = rng.choice(("bf16", "bf16", "bf16", "f32"))
    if kind == "packed":
        dim = rng.choice((32, 64, 128, 128)) if dtype == "bf16" else rng.choice((8, 16, 32, 64))
        groups = rng.choice((1, 2, 4, 8))
        heads = groups * rng.choice((1, 1, 2, 3, 4))
        high = _log(rng, 1, 4096 if dtype == "bf16" else 700)
        room = (4 * 16 * 4096**2 * 128 if dtype == "bf16" else 32 * 4 * 700**2 * 16) // (heads * dim * max(high, 64) ** 2)
        return dict(kind=kind, lens=_log(rng, 1, max(1, min(96, room, 16384 // high))), low=max(1, high // rng.choice((1, 3, 20))), high=high,
                    past=rng.choice((0, 0, high // 2)), heads=heads, groups=groups, dim=dim, dtype=dtype, shape=shape)
    if kind == "tree":
        dim = rng.choice((32, 64, 128, 128)) if dtype == "bf16" else rng.choice((8, 16, 32, 64))
        groups = rng.choice((1, 2, 4, 8))
        heads = groups * rng.choice((1, 2, 3, 4, 8))
        high, nodes = _log(rng, 1, 30000 if dtype == "bf16" else 2000), _log(rng, 1, 150)
        room = (3 * 40000 * 4 * 128 if dtype == "bf16" else 24 * 2000 * 4 * 16) // (groups * dim * (high + nodes))
        room = min(room, 3 * 65000 * 64 * 16 // ((high + nodes) * nodes * heads))
        return dict(kind=kind, batch=_log(rng, 1, max(1, min(64, room))), nodes=nodes, low=max(0, high // rng.choice((1, 3, 20)) - 1), high=high,
                    heads=heads, groups=groups, dim=dim, dtype=dtype, shape=shape)
    if kind == "logprobs":
        vocab = _log(rng, 40, 130000)
        return dict(kind=kind, rows=_log(rng, 1, max(1, min(4096, 4096 * 16000 // vocab))), vocab=vocab, top=rng.choice((0, 1, 5, 8, 20, 32)),
                    temperature=rng.choice((1.0, 0.7, 1.3)), masked=rng.choice((0.0, 0.0, 0.95)), dtype=dtype)
    nodes = _log(rng, 1, 150)
    return dict(kind=kind, batch=_log(rng, 1, 160), nodes=nodes, most=rng.randint(1, min(nodes, 12)), layers=rng.randint(2, 12),
                heads=rng.choice((4, 8, 12)), dim=rng.choice((16, 32, 64)), low=rng.randint(1, 300), high=rng.randint(300, 900), dtype=dtype, shape=shape)


# ---- shapes: a case's lengths follow from the case alone --------------------------------------------------------
def _lens(case, n, salt=0):
    rng = random.Random(case["shape"] * 64 + salt)
    return [rng.randint(case["low"], case["high"]) for _ in range(n)]


def _packed_lens(case):
    q = _lens(case, case["lens"])
    rng = random.Random(case["shape"] * 64 + 1)
    return q, [n + (rng.randint(0, case["past"]) if case["past"] else 0) for n in q]


def _tree_lens(case):
    """Cached tokens and drafts of every sequence; the first has the largest tree."""
    rng = random.Random(case["shape"] * 64 + 2)
    n = [case["nodes"]] + [rng.randint(max(1, case["nodes"] // 2), case["nodes"]) for _ in range(case["batch"] - 1)]
    return _lens(case, case["batch"]), n


def _keep_lens(case):
    rng = random.Random(case["shape"] * 64 + 3)
    return _lens(case, case["batch"]), [rng.randint(0 if case["batch"] > 1 else case["most"], case["most"]) for _ in range(case["batch"])]


def _visible(lq, lk):
    """Pairs of query and key of one prompt."""
    return sum(max(0, min(lk, i + 1 + lk - lq)) for i in range(lq))


def work(case):
    size = 2 if case["dtype"] == "bf16" else 4
    if case["kind"] == "packed":
        lq, lk = _packed_lens(case)
        H, G, D = case["heads"], case["groups"], case["dim"]
        return {"bytes": (2 * sum(lq) * H * D + 2 * sum(lk) * G * D) * size + sum(lq) * H * 4,
                "flops": 4 * D * H * sum(_visible(a, b) for a, b in zip(lq, lk))}
    if case["kind"] == "tree":
        ctx, n = _tree_lens(case)
        H, G, D = case["heads"], case["groups"], case["dim"]
        return {"bytes": (2 * sum(n) * H * D + 2 * (sum(ctx) + sum(n)) * G * D) * size, "flops": 4 * D * H * sum(b * (a + b / 2) for a, b in zip(ctx, n))}
    if case["kind"] == "logprobs":
        R, V = case["rows"], case["vocab"]
        return {"bytes": R * V * size + R * (12 + 8 * min(case["top"], V)), "flops": 5 * R * V}
    _, count = _keep_lens(case)
    return {"bytes": 2 * sum(count) * case["layers"] * 2 * case["heads"] * case["dim"] * size, "flops": 0}


# ---- what a user's program has in hand --------------------------------------------------------------------------
def _starts(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return torch.tensor(out, dtype=torch.int32, device="cuda")


def _tree_masks(case, n, seed):
    """int64 [B, T, words]: bit j of a draft's words says whether it sees draft j: its ancestors and itself.  A draft's parent is one
    of those before it, or the last cached token."""
    B, T = case["batch"], case["nodes"]
    rng = random.Random(seed * 1000003 + case["shape"])
    words = -(-T // 64)
    rows = []
    for s in range(B):
        bits = []
        for t in range(T):
            parent = rng.randint(max(-1, t - 6), t - 1)
            bits.append((1 << t) | (bits[parent] if parent >= 0 else 0))
        rows.append([[((b >> (64 * w)) & (2**64 - 1)) for w in range(words)] for b in bits])
    signed = [[[x - 2**64 if x >= 2**63 else x for x in w] for w in r] for r in rows]
    return torch.tensor(signed, dtype=torch.int64, device="cuda")


def _table(B, pages, g):
    """Pages of the sequences, scattered over the pool as a server's are after a while."""
    return torch.randperm(B * pages, generator=g, device="cuda").to(torch.int32).view(B, pages)


def prepare(case, seed):
    dt = DTYPES[case["dtype"]]
    g = torch.Generator(device="cuda").manual_seed(9176 * seed + 3)

    def n(*shape):
        return torch.randn(shape, generator=g, device="cuda").to(dt)

    s = {"kind": case["kind"], "case": case}
    if case["kind"] == "packed":
        lq, lk = _packed_lens(case)
        H, G, D, N, M = case["heads"], case["groups"], case["dim"], sum(lq), sum(lk)
        if case["past"]:
            q, k, v = n(N, H, D), n(M, G, D), n(M, G, D)
        else:  # one projection's output
            qkv = n(N, (H + 2 * G) * D)
            q, k, v = (x.view(N, -1, D) for x in qkv.split([H * D, G * D, G * D], dim=1))
        return dict(s, q=q, k=k, v=v, seq_starts=_starts(lq), key_starts=_starts(lk) if case["past"] else None, longest=(max(lq), max(lk)),
                    out=torch.zeros((N, H, D), dtype=dt, device="cuda"), lse=torch.zeros((N, H), dtype=torch.float32, device="cuda"),
                    status=torch.zeros(1, dtype=torch.int32, device="cuda"))
    if case["kind"] == "tree":
        ctx, nodes = _tree_lens(case)
        H, G, D, B, T = case["heads"], case["groups"], case["dim"], case["batch"], case["nodes"]
        pages = -(-(max(ctx) + T) // PAGE)
        pool = n(B * pages, 2, G, PAGE, D)
        i32 = dict(dtype=torch.int32, device="cuda")
        return dict(s, q=n(B * T, H * D), pool=pool, table=_table(B, pages, g), ctx=torch.tensor(ctx, **i32), nodes=torch.tensor(nodes, **i32),
                    masks=_tree_masks(case, nodes, seed), longest=max(ctx) + T, out=torch.zeros((B * T, H * D), dtype=dt, device="cuda"),
                    status=torch.zeros(1, **i32))
    if case["kind"] == "logprobs":
        R, V = case["rows"], case["vocab"]
        logits = (torch.randn((R, V), generator=g, device="cuda") * 3).to(dt)
        targets = torch.randint(0, V, (R,), generator=g, device="cuda")
        if case["masked"]:  # behind a top-p filter: most tokens are out, the given one is in
            out = torch.rand((R, V), generator=g, device="cuda") < case["masked"]
            out.scatter_(1, targets[:, None], False)
            logits.masked_fill_(out, float("-inf"))
        return dict(s, logits=logits, targets=targets.to(torch.int32), status=torch.zeros(1, dtype=torch.int32, device="cuda"))
    ctx, count = _keep_lens(case)
    B, T, L, H, D = case["batch"], case["nodes"], case["layers"], case["heads"], case["dim"]
    pages = -(-(max(ctx) + case["most"]) // PAGE)
    drafts = -(-T // PAGE)  # the drafts' own pages lie behind the others
    rng = random.Random(seed * 1000003 + case["shape"])
    path = [sorted(rng.sample(range(T), case["most"])) + [0] * (T - case["most"]) for _ in range(B)]
    i32 = dict(dtype=torch.int32, device="cuda")
    return dict(s, pool=n(L, B * (pages + drafts), 2, H, PAGE, D), table=_table(B, pages + drafts, g), ctx=torch.tensor(ctx, **i32),
                drafts=torch.full((B,), pages * PAGE, **i32), path=torch.tensor(path, **i32), count=torch.tensor(count, **i32), status=torch.zeros(1, **i32))


# ---- one pass ---------------------------------------------------------------------------------------------------
def run(s):
    kind, c = s["kind"], s["case"]
    if not own:
        return {"packed": _packed, "tree": _tree, "logprobs": _logprobs, "keep": _keep}[kind](s)
    from diff_gpt_b200 import ops

    if kind == "packed":
        ops.fmha_packed(s["q"], s["k"], s["v"], s["seq_starts"], s["out"], key_starts=s["key_starts"], lse=s["lse"], status=s["status"])
        return {"out": s["out"], "lse": s["lse"]}
    if kind == "tree":
        pool, G, D = s["pool"], c["groups"], c["dim"]
        kv = ops.kv_layout(pool[0, 0], pool[0, 1], pool.stride(0), pool.stride(2), PAGE, s["table"], n_pages=pool.shape[0])
        ops.tree_attn(s["q"], kv, s["ctx"], s["masks"], s["out"], H=c["heads"], G=G, D=D, n_nodes=s["nodes"], max_keys=s["longest"], status=s["status"])
        return s["out"]
    if kind == "logprobs":
        r = ops.token_logprobs(s["logits"], s["targets"], top_k=c["top"], temperature=c["temperature"], status=s["status"])
        return {"logprob": r.logprob, "entropy": r.entropy, "top_ids": r.top_ids, "top_logprobs": r.top_logprobs}
    pool = s["pool"]
    kv = ops.kv_layout(pool[0, 0, 0], pool[0, 0, 1], pool.stride(1), pool.stride(3), PAGE, s["table"], n_pages=pool.shape[1])
    ops.kv_keep(kv, s["drafts"], s["ctx"], s["path"], s["count"], n_layer=c["layers"], layer_stride=pool.stride(0), H=c["heads"], D=c["dim"],
                dtype=pool.dtype, status=s["status"])
    return pool


def _packed(s):
    q, k, v, starts = s["q"], s["k"], s["v"], s["seq_starts"].long()
    kst = starts if s["key_starts"] is None else s["key_starts"].long()
    (N, H, D), G, (Lq, Lk), dev = q.shape, k.shape[1], s["longest"], q.device
    lq, lk = starts.diff(), kst.diff()
    i, j = torch.arange(Lq, device=dev), torch.arange(Lk, device=dev)
    rows, cols = (starts[:-1, None] + i).clamp(max=N - 1), (kst[:-1, None] + j).clamp(max=k.shape[0] - 1)
    qf = q[rows].float().view(-1, Lq, G, H // G, D).permute(0, 2, 3, 1, 4)
    kf, vf = (x[cols].float().permute(0, 2, 3, 1)[:, :, None] for x in (k, v))
    see = (j <= (i[:, None] + (lk - lq)[:, None, None])) & (j < lk[:, None, None])
    score = (qf @ kf * (1.0 / math.sqrt(D))).masked_fill_(~see[:, None, None], float("-inf"))
    top = score.amax(dim=-1, keepdim=True).clamp(min=-1e30)
    p = score.sub_(top).exp_()
    total = p.sum(dim=-1, keepdim=True)
    o = (p @ vf.transpose(-1, -2)) / total.clamp(min=1e-30)
    lse = (top + total.log()).squeeze(-1)
    real = i < lq[:, None]
    s["out"][rows[real]] = o.permute(0, 3, 1, 2, 4).reshape(-1, Lq, H, D)[real].to(q.dtype)
    s["lse"][rows[real]] = lse.permute(0, 3, 1, 2).reshape(-1, Lq, H)[real]
    return {"out": s["out"], "lse": s["lse"]}


def _tree(s):
    c, pool, dev = s["case"], s["pool"], s["q"].device
    B, T, H, G, D, L = c["batch"], c["nodes"], c["heads"], c["groups"], c["dim"], s["longest"]
    ctx, nodes, j, t = s["ctx"].long()[:, None], s["nodes"].long()[:, None], torch.arange(L, device=dev), torch.arange(T, device=dev)
    page = s["table"].long()[:, j // PAGE]
    kf, vf = (pool[page, x, :, j % PAGE].float().permute(0, 2, 3, 1)[:, :, None] for x in (0, 1))
    qf = s["q"].view(B, T, G, H // G, D).permute(0, 2, 3, 1, 4).float()
    d = (j - ctx).clamp(0, T - 1)  # which draft a slot holds
    bit = (s["masks"].gather(2, (d // 64)[:, None].expand(B, T, L)) >> (d % 64)[:, None]) & 1
    see = (j < ctx)[:, None] | (((j >= ctx) & (j < ctx + nodes))[:, None] & (bit == 1))
    score = (qf @ kf * (1.0 / math.sqrt(D))).masked_fill_(~see[:, None, None], float("-inf"))
    p = score.sub_(score.amax(dim=-1, keepdim=True).clamp(min=-1e30)).exp_()
    o = (p @ vf.transpose(-1, -2)) / p.sum(dim=-1, keepdim=True).clamp(min=1e-30)
    real = (t < nodes).view(-1)
    s["out"][real] = o.permute(0, 3, 1, 2, 4).reshape(B * T, H * D)[real].to(s["out"].dtype)
    return s["out"]


def _logprobs(s):
    z = s["logits"].float() / s["case"]["temperature"]
    top = z.amax(dim=-1, keepdim=True)
    e = (z - top).exp()
    total = e.sum(dim=-1, keepdim=True)
    logp = z - top - total.log()
    entropy = -torch.where(e > 0, e / total * logp, torch.zeros_like(e)).sum(dim=-1)
    ids = s["logits"].float().sort(dim=-1, descending=True, stable=True).indices[:, : s["case"]["top"]]
    return {"logprob": logp.gather(1, s["targets"].long()[:, None])[:, 0], "entropy": entropy, "top_ids": ids.to(torch.int32), "top_logprobs": logp.gather(1, ids)}


def _keep(s):
    pool, T = s["pool"], s["path"].shape[1]
    i = torch.arange(T, device=pool.device)
    src, dst = s["drafts"].long()[:, None] + s["path"].long(), s["ctx"].long()[:, None] + i
    seq, at = torch.nonzero(i < s["count"].long()[:, None], as_tuple=True)
    src, dst, table = src[seq, at], dst[seq, at], s["table"].long()
    pool[:, table[seq, dst // PAGE], :, :, dst % PAGE] = pool[:, table[seq, src // PAGE], :, :, src % PAGE]
    return pool


# ---- the definitions in 64 bits ---------------------------------------------------------------------------------
def _softmax_rows(score, v):
    """softmax(score) v and the log of the sum for rows of one head, nothing where nothing is seen."""
    lse = torch.logsumexp(score, dim=-1, keepdim=True)
    w = torch.where(torch.isneginf(score) | torch.isneginf(lse), 0.0, (score - lse).exp())
    return w @ v, lse[..., 0]


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "packed":
        lq, lk = _packed_lens(case)
        out, lse = s["out"].double(), s["lse"].double()
        a = b = 0
        for n, m in zip(lq, lk):
            see = torch.ones((n, m), dtype=torch.bool, device="cuda").tril(m - n)
            for h in range(case["heads"]):
                kv = h * case["groups"] // case["heads"]
                score = s["q"][a : a + n, h].double() @ s["k"][b : b + m, kv].double().T / math.sqrt(case["dim"])
                out[a : a + n, h], lse[a : a + n, h] = _softmax_rows(score.masked_fill(~see, float("-inf")), s["v"][b : b + m, kv].double())
            a, b = a + n, b + m
        return {"out": out, "lse": lse}
    if case["kind"] == "tree":
        ctx, nodes = _tree_lens(case)
        T, H, G, D = case["nodes"], case["heads"], case["groups"], case["dim"]
        out = s["out"].double().view(case["batch"], T, H, D)
        masks = s["masks"].tolist()
        for b, (c, n) in enumerate(zip(ctx, nodes)):
            rows = s["pool"][s["table"][b].long()].permute(1, 2, 0, 3, 4).reshape(2, G, -1, D)[:, :, : c + n].double()
            see = torch.tensor([[(masks[b][t][x // 64] >> (x % 64)) & 1 for x in range(n)] for t in range(n)], dtype=torch.bool, device="cuda")
            see = torch.cat([torch.ones((n, c), dtype=torch.bool, device="cuda"), see], dim=1)
            for h in range(H):
                kv = h * G // H
                score = s["q"].view(-1, T, H, D)[b, :n, h].double() @ rows[0, kv].T / math.sqrt(D)
                out[b, :n, h] = _softmax_rows(score.masked_fill(~see, float("-inf")), rows[1, kv])[0]
        return out.view(-1, H * D)
    if case["kind"] == "logprobs":
        names = ("logprob", "entropy", "top_ids", "top_logprobs")
        parts = []
        for z, target in zip(s["logits"].split(256), s["targets"].split(256)):
            order = torch.argsort(z.double(), dim=-1, descending=True, stable=True)[:, : case["top"]]
            logp = torch.log_softmax(z.double() / case["temperature"], dim=-1)
            p = logp.exp()
            parts.append((logp.gather(1, target.long()[:, None])[:, 0], -(p * logp.masked_fill(p == 0, 0.0)).sum(dim=-1), order.to(torch.int32), logp.gather(1, order)))
        return {k: torch.cat(x) for k, x in zip(names, zip(*parts))}
    ctx, count = _keep_lens(case)
    pool, old, table, path = s["pool"], s["pool"].clone(), s["table"].tolist(), s["path"].tolist()
    first = s["drafts"].tolist()
    for b, (c, n) in enumerate(zip(ctx, count)):
        for i in range(n):
            src, dst = first[b] + path[b][i], c + i
            pool[:, table[b][dst // PAGE], :, :, dst % PAGE] = old[:, table[b][src // PAGE], :, :, src % PAGE]
    return pool.double()
