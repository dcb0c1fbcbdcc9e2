"""PagedKVCache.keep_drafts where several rows share a prompt's pages."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows", [1, 2])
def test_a_shared_prompt_is_not_written(rows, dtype):
    """A target in the prompt's last page (its end, where the drafts would go if the page were the row's) is refused where others read that page:
    nothing of that path moves there, the status says so, the rest moves."""
    from diff_gpt_b200 import PagedKVCache

    L, H, D, T = 2, 3, 16, 4
    c = PagedKVCache(L, H, D, n_series=2, rows_per_series=rows, prefix_len=70, max_new=60, dtype=dtype, device="cuda")
    c.pool.copy_(torch.randn(c.pool.shape))
    old, first = c.pool.clone(), c.suffix_slot0
    i32 = dict(dtype=torch.int32, device="cuda")
    status = torch.zeros(1, **i32)
    n = c.n_rows
    src, count = torch.full((n,), first, **i32), torch.full((n,), 3, **i32)
    dst = torch.full((n,), first, **i32)
    dst[0], dst[n - 1] = 70, first - 2  # the latter reaches into the row's own pages
    path = torch.tensor([[0, 2, 3, 1]] * n, **i32)
    c.keep_drafts(src, dst, path, count, status)
    want = old.clone()
    for r in range(n):
        for i in range(3):
            a, b = first + path[r, i].item(), dst[r].item() + i
            if b >= first or rows == 1:
                want[:, c.row_table[r, b // 64].item(), :, :, b % 64] = old[:, c.row_table[r, a // 64].item(), :, :, a % 64]
    assert torch.equal(c.pool, want)
    assert status.item() == (0 if rows == 1 else 1)
    if rows > 1:
        prompts = 2 * c.prefix_pages
        assert torch.equal(c.pool[:, :prompts], old[:, :prompts])
    status.zero_()
    c.keep_drafts(src, src, path, torch.zeros_like(count), status)
    assert torch.equal(c.pool, want) and status.item() == 0
