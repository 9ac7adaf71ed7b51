"""Rotary positions at the largest numbers of heads and rows: as many pairs as an int counts, against the same pairs in calls of their own."""
import pytest
import torch

from mx230_b200 import llm_attention as la

pytestmark = pytest.mark.gpu

MOST = 2 ** 31 - 1


@pytest.mark.parametrize("by_heads", [True, False])
def test_as_many_pairs_as_an_int_counts(handle, by_heads):
    if torch.cuda.mem_get_info()[0] < 20 << 30:
        pytest.skip("not enough memory")
    plan = la.Rotary(2, 1e4)
    x = torch.empty(MOST, 2, dtype=torch.float16, device="cuda").fill_(0.5)
    shape = lambda t: t[None] if by_heads else t[:, None]  # noqa: E731
    at = [0, 1 << 20, (1 << 30) - 500, MOST - 1000]
    before = []
    for a in at:
        x[a:a + 1000] = torch.randn(1000, 2, generator=torch.Generator().manual_seed(a % 1000)).half().cuda()
        before.append(x[a:a + 1000].clone())
    first = 3 if by_heads else -MOST // 2   # (positions are ints: rows from one to the other end of them)
    la.rotary(handle, shape(x), shape(x), first, plan)
    for a, b in zip(at, before):
        la.rotary(handle, shape(b), shape(b), first if by_heads else first + a, plan)
        assert torch.equal(x[a:a + 1000], b), a
    handle.check_status()
