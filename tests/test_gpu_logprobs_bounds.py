"""ops.token_logprobs against float64 within bounds that follow from the chains of its sums, at every temperature that it takes.

u = 2^-24 (a rounding of fp32), 2^x (ex2.approx) is within 2^-22 of itself.  With y_j = (z_j - max z), in nats and never positive, p = e^y / s, s = sum e^y:
  a term     y is off by 4 u |y| (a product or a difference, the factor log2(e) / temperature and its own two roundings; the factor is rounded in
             2^-149 where it is below the normal numbers, which is 2 u there), so e^y is off by 2^-22 + 4 u |y| relative
  the sum    one thread adds `in_round` numbers a round and a round to its sum; whenever its maximum moves the sum is multiplied by a power: 2^-22 + 3 u; lanes,
             warps and CTAs are joined by at most 18 additions and 3 such products.  One warp by itself (rows beyond the usual range): V / 32 + VEC additions and 5.
             r: all of that relative
  log s      is off by r + 4 u A and 2^-22 of itself, A = sum p |y|
  w = sum p y  every term and every addition as before, and no two terms cancel (y <= 0): r A + 4 u B, B = sum p y^2, beside what its division by s brings
so |logprob - exact| <= r + 4 u (A + |y_t| + log s + |logprob|) + 2^-22 and |entropy - exact| <= r (1 + 2 A) + 4 u (A + 2 B + log s + H) + 2^-22."""

import pytest
import torch

from test_gpu_logprobs import make

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32
U = 2.0**-24


def single(x):
    return torch.tensor(x, dtype=F32).item()


def check(logits, targets, T, k, alone=False):
    """alone: rows that one warp sums by itself, or some of them."""
    from diff_gpt_b200 import ops

    T = single(T)
    got = ops.token_logprobs(logits, targets, top_k=k, temperature=T)
    V, vec = logits.shape[1], 8 if logits.dtype == BF else 4
    rounds = 10 + V // (1024 * vec)
    r = 2.0**-22 + (16 + 2 + rounds + 18) * U + (rounds + 3) * (2.0**-22 + 3 * U)
    if alone:
        r = max(r, 2.0**-22 + (V / 32 + vec + 5) * U)
    x = logits.cpu().double()
    y = (x - x.amax(dim=1, keepdim=True)) / T
    e = y.exp()
    s = e.sum(dim=1, keepdim=True)
    p, y0 = e / s, torch.where(e > 0, y, torch.zeros_like(y))
    A, B, log_s = -(p * y0).sum(dim=1), (p * y0 * y0).sum(dim=1), s.log()[:, 0]
    H = log_s + A
    off = (got.entropy.cpu().double() - H).abs()
    bound = r * (1 + 2 * A) + 4 * U * (A + 2 * B + log_s + H) + 2.0**-22
    assert bool((off <= bound).all()), ((off - bound).max().item(), off.max().item())
    ids = torch.argsort(x, dim=1, descending=True, stable=True)[:, :k]
    assert torch.equal(got.top_ids.cpu().long(), ids)
    for mine, at in ((got.logprob[:, None], targets.cpu().long()[:, None]), (got.top_logprobs, ids)):
        yt = y.gather(1, at)
        want = yt - log_s[:, None]
        none = torch.isneginf(want.float())  # the answer is fp32: beyond its range it is -inf
        mine = mine.cpu().double()
        assert torch.equal(torch.isneginf(mine), none)
        bound = r + 4 * U * (A[:, None] + yt.abs() + log_s[:, None] + want.abs()) + 2.0**-22
        assert bool(((mine - want).abs()[~none] <= bound[~none]).all())


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("kind", ["normal", "ties", "level", "rising", "falling", "peaked", "masked", "three"])
@pytest.mark.parametrize("R,V", [(3, 5), (2, 40), (5, 777), (3, 20000), (320, 6001), (2, 128255), (200, 70001)])
def test_within_the_bounds(R, V, kind, dtype):
    logits, targets = make(R, V, dtype, 11, kind)
    check(logits, targets, 1.0, min(V, 9))
    check(logits, targets, 0.7, 0)


HOT = [1e4, 1e19, 1.4e20, 1.5e20, 1e21, 1.3e21, 5e21, 1e25, 1e28, 1e30, 1e35, 2e38, torch.finfo(F32).max]


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("T", HOT)
@pytest.mark.parametrize("kind", ["normal", "masked", "three", "prefix", "lowest", "low_or_none", "huge"])
@pytest.mark.parametrize("R,V", [(2, 40), (3, 9001), (400, 1003), (1, 100000)])
def test_high_temperatures(R, V, kind, T, dtype):
    """What is masked (-inf, or the type's lowest value) counts for what it is, however high the temperature: nothing, or e^(lowest / T)."""
    low = torch.finfo(dtype).min
    logits, targets = make(R, V, dtype, 12, kind if kind in ("normal", "masked", "three", "lowest") else "normal")
    if kind == "prefix":  # whole threads, and CTAs, see nothing but -inf
        logits[:, : V - V // 8] = float("-inf")
    elif kind == "low_or_none":  # nothing but the lowest value and -inf
        logits = torch.where(torch.arange(V, device="cuda") % 3 == 0, torch.full_like(logits, low), torch.full_like(logits, float("-inf")))
    elif kind == "huge":  # both ends of the type: their difference has no fp32 number
        logits[:, V // 2 :] = low
        logits[:, V // 3] = -low
    check(logits, targets, T, 7, alone=True)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("T", [1.0, 1e21, 1e30, torch.finfo(F32).max])
def test_rows_without_a_distribution_at_high_temperatures(T, dtype):
    from diff_gpt_b200 import ops

    for V in (50, 9000, 70000):
        logits, targets = make(6, V, dtype, 13)
        logits[1, V // 2] = float("nan")
        logits[2, V - 1] = float("inf")
        logits[3] = float("-inf")
        logits[4] = float("nan")
        r = ops.token_logprobs(logits, targets, top_k=4, temperature=T)
        bad = torch.tensor([0, 1, 1, 1, 1, 0], dtype=torch.bool, device="cuda")
        assert torch.equal(torch.isnan(r.logprob), bad) and torch.equal(torch.isnan(r.entropy), bad)
        assert torch.equal(torch.isnan(r.top_logprobs), bad[:, None].expand(6, 4))
