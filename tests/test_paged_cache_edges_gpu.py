"""The paged 8-bit KV cache where its calls are easily wrong: guesses of no rows, workspaces that serve several calls, pages without a
scale or with very unlike ones, wrong offsets. Against float64 definitions (paged_pool.py)."""

import pytest
import torch

from paged_pool import Pool, attention
from test_paged_cache_gpu import _attend, _check, _context, _done

pytestmark = pytest.mark.gpu

GUARD = 1 << 20


def _guarded(need):
    """A workspace with bytes behind it that nobody may write."""
    ws = torch.empty(need + GUARD, dtype=torch.uint8, device="cuda").random_(0, 256)
    return ws, ws[need:].clone()


@pytest.mark.parametrize("d,keys", [(64, 2340), (128, 3120)])
def test_attention_with_a_guess_of_no_rows_keeps_to_its_workspace(d, keys):
    """Sixteen heads a KV head, so that one row is more than the eight pairs of the smaller kernel. 48 segments of 37 and of 49 steps
    of 64 keys: one and two a warp of 148 SMs with 12 and 8 warps, so that the last warps leave parts too."""
    ctx = _context()
    n_seq = 12
    pool = Pool(ctx, n_pages=n_seq * 50, n_kv=4, d=d, page=64, n_seq=n_seq, max_pages=50)
    start, counts = [keys - 1 - 2 * i for i in range(n_seq)], [1] * n_seq
    pool.give([s + 1 for s in start])
    handle = pool.handle()
    need = [ctx.kv_block_attention_workspace(handle, 64, n_seq + 2, most) for most in (0, 1)]
    assert need[0] == need[1]
    ws, guard = _guarded(need[0])
    q = torch.randn(n_seq, 64, d, device="cuda", generator=pool.g)
    got, live = _attend(ctx, pool, q, counts, start, most=0, ws=ws)
    _done(ctx)
    _check(got, live, *attention(pool, q, start, counts))
    assert torch.equal(ws[need[0]:], guard)
    ctx.close()
