"""Calls of the 8-bit cache and the rotation at the borders of what their
documentation allows: numbers near 31 bits, outputs that share memory,
derivatives, growth."""
import pytest
import torch

from wnw_b200.kv8 import KV8Store

gpu = pytest.mark.gpu
BF16 = torch.bfloat16


@gpu
@pytest.mark.parametrize("left", [1, 40])
def test_append_behind_two_billion_rows(left):
    """A token behind almost 2^31 others: the blocks that a longer append
    would fill begin beyond 31 bits and are left alone."""
    width = (1 << 20) - 1  # pages of 2,048 rows
    table = torch.full((1, width), -1, dtype=torch.int32, device="cuda")
    pool = torch.full((1, 64, 64 * 64 + 128), 7, dtype=torch.uint8, device="cuda")
    tk = torch.zeros(1, 2, 32, 64, dtype=BF16, device="cuda")
    s = KV8Store.wrap(pool, table, tk, torch.zeros(1, 2, 64, 32, dtype=BF16, device="cuda"))
    rows = width * 2048 - left
    k = torch.ones(1, 1, 5000, 64, dtype=BF16, device="cuda")
    s.append(k, k, torch.tensor([rows], dtype=torch.int32, device="cuda"),
             counts=torch.ones(1, dtype=torch.int32, device="cuda"))
    if left == 1:  # it fills a block whose page is none
        with pytest.raises(RuntimeError, match="out of range"):
            s.check()
    else:
        s.check()
        at = rows // 32 % 2
        want = torch.zeros_like(tk)
        want[0, at, rows % 32] = 1
        assert torch.equal(s.tail_k, want) and torch.equal(s.tail_v, want.transpose(2, 3))
    assert bool((s.pool == 7).all())
