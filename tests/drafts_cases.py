"""Plain float64 forms of the operators behind serving with drafted tokens, and the bounds that follow from the formulas.

Bounds of attention.  u is the rounding of the stored type (half a step, relative: bf16 2^-8, fp32 2^-24), e = 2^-24.
  scores     products of stored numbers summed in fp32, D of them: off by at most (D + 2) e S, S = scale * sum_d |q_d k_d|; the kernels
             take them to base 2 by one more rounding, e |s|, and 2^x is within 2^-21 of itself relative, so a probability is off by
             r = 2 (D + 4) e S + 2^-21 relative (S at its largest over the row's keys), twice that once it is divided by the sum
  P V        bf16 on the tensor cores: each probability rounded to bf16, relative 2^-8; n products and one sum in fp32, (n + 2) e relative;
             all against A = sum_j p_j |v_j|
  the output one rounding, u |o|
so |o - exact| <= u |o| + A (2 r + (n + 8) e + [tensor cores] 2^-8), and |lse - exact| <= r + (n + 8) e + 2^-21 |lse| + 2^-21.
(A row's running maximum may lag behind the true one by 2^8: probabilities are then up to 2^8 instead of 1, which no relative bound sees.)
"""

import math

import torch

U = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-8}
E = 2.0**-24


def rows(q, k, v, see, scale):
    """q [n, D], k [m, D], v [m, D], see [n, m] -> o, A, lse, S in float64; a row that sees nothing: zeros and -inf."""
    q, k, v = q.double(), k.double(), v.double()
    neg = float("-inf")
    s = (q @ k.T * scale).masked_fill(~see, neg)
    lse = torch.logsumexp(s, dim=1) if s.shape[1] else torch.full((q.shape[0],), neg, dtype=torch.float64)
    p = torch.where(see, (s - lse.clamp(min=-1e300)[:, None]).exp(), torch.zeros_like(s)) if s.shape[1] else s
    size = (q.abs() @ k.abs().T * scale).masked_fill(~see, 0.0)
    return p @ v, p @ v.abs(), lse, size.amax(dim=1) if s.shape[1] else torch.zeros(q.shape[0], dtype=torch.float64)


def check_rows(got, got_lse, want, D, n, dtype, tensor_cores):
    """got [rows, D] against rows()'s answer within the bounds above."""
    o, A, lse, S = want
    r = 2 * (D + 4) * E * S + 2.0**-21
    tol = U[dtype] * o.abs() + A * (2 * r + (n + 8) * E + (2.0**-8 if tensor_cores else 0.0))[:, None]
    err = (got.double() - o).abs()
    assert bool((err <= tol).all()), (err - tol).max().item()
    if got_lse is not None:
        none = torch.isneginf(lse)
        assert torch.equal(torch.isneginf(got_lse), none)
        off = (got_lse.double() - lse)[~none].abs()
        assert bool((off <= (r + (n + 8) * E + 2.0**-21 * (1 + lse.abs()))[~none]).all()), off.max().item()


def starts(lens, first=0):
    out = [first]
    for n in lens:
        out.append(out[-1] + n)
    return out


def tree_bits(parents):
    """Each draft's own bit and its ancestors', as whole numbers."""
    bits = []
    for t, p in enumerate(parents):
        bits.append((1 << t) | (bits[p] if p >= 0 else 0))
    return bits


def words(bits, n_words):
    """Whole numbers -> int64 [len, n_words]."""
    out = [[(b >> (64 * w)) & (2**64 - 1) for w in range(n_words)] for b in bits]
    return torch.tensor([[x - 2**64 if x >= 2**63 else x for x in r] for r in out], dtype=torch.int64).reshape(len(bits), n_words)


def logprobs(logits, targets, temperature, k):
    """float64: logprob, entropy, ids and log probabilities of the top k (ties by index)."""
    z = logits.double() / temperature
    logp = torch.log_softmax(z, dim=1)
    p = logp.exp()
    entropy = -(torch.where(p > 0, p * logp, torch.zeros_like(p))).sum(dim=1)
    ids = torch.argsort(logits.double(), dim=1, descending=True, stable=True)[:, :k]
    return logp.gather(1, targets.long()[:, None])[:, 0], entropy, ids, logp.gather(1, ids)


def scale_of(D):
    return 1.0 / math.sqrt(D)
