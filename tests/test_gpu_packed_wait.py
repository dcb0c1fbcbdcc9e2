"""Waits of the tensor-core kernel of packed prompts that run out while copies and products are in flight.

The limit is made too short for a prompt of many tiles; nothing waits for what cannot come, nothing faults.  The kernel has to report it, return, and leave the
GPU as it was: calls behind it on the same SMs get their TMEM and the same numbers as before."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_the_probe_refuses():
    from diff_gpt_b200._lib import lib

    P = 1 << 20
    for wrong in (dict(limit=0), dict(limit=2 * 10**9 + 1), dict(x=None), dict(status=None), dict(rows=2**20 + 1), dict(x=P + 8)):
        a = dict(dict(limit=5, x=P, rows=100, status=P), **wrong)
        assert lib.dgpt_packed_wait_probe(a["limit"], a["x"], P, P, 1, a["rows"], 2, 64, a["status"], None) == -1
    assert lib.dgpt_packed_wait_probe(5, P, P, P, 1, 100, 2, 16, P, None) == -2


@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("limit", [1, 300, 1000, 3000])
def test_a_wait_that_runs_out_is_reported_and_leaves_nothing_behind(limit, D):
    from diff_gpt_b200 import _lib, ops

    lens, H = [6000, 1500], 4
    g = torch.Generator(device="cuda").manual_seed(D)
    x = torch.randn(sum(lens), H, D, generator=g, device="cuda").bfloat16()
    starts = torch.tensor([0, lens[0], sum(lens)], dtype=torch.int32, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    want, out, lost = torch.empty_like(x), torch.empty_like(x), torch.empty_like(x)
    ops.fmha_packed(x, x, x, starts, want, status=status)
    torch.cuda.synchronize()
    assert status.item() == 0
    stream = torch.cuda.current_stream().cuda_stream
    for _ in range(3):
        # sixteen limits pass before the first item's 47 tiles of more than 1000 cycles each do
        _lib.check(_lib.lib.dgpt_packed_wait_probe(limit, x.data_ptr(), lost.data_ptr(), starts.data_ptr(), 2, sum(lens), H, D, status.data_ptr(), stream))
        torch.cuda.synchronize()
        assert status.item() == 2
        status.zero_()
        out.zero_()
        ops.fmha_packed(x, x, x, starts, out, status=status)
        assert torch.equal(out, want) and status.item() == 0


@pytest.mark.parametrize("D", [64, 128])
def test_waits_that_suffice(D):
    """The same kernel with a limit that is long enough: an ordinary result."""
    from diff_gpt_b200 import _lib, ops

    x = torch.randn(700, 2, D, device="cuda").bfloat16()
    starts = torch.tensor([0, 500, 700], dtype=torch.int32, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    want, out = torch.empty_like(x), torch.empty_like(x)
    ops.fmha_packed(x, x, x, starts, want, scale=1.0 / D)
    _lib.check(_lib.lib.dgpt_packed_wait_probe(10**8, x.data_ptr(), out.data_ptr(), starts.data_ptr(), 2, 700, 2, D, status.data_ptr(),
                                               torch.cuda.current_stream().cuda_stream))
    assert torch.equal(out, want) and status.item() == 0
