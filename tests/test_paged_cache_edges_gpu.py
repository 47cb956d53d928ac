"""The paged 8-bit KV cache where its calls are easily wrong: guesses of no rows, workspaces that serve several calls, pages without a
scale or with very unlike ones, wrong offsets. Against float64 definitions (paged_pool.py)."""
import math

import pytest
import torch

from paged_pool import Pool, attention, i32
from test_paged_cache_gpu import Book, _append, _attend, _check, _context, _done, _expect_append, _extend, _positions, _refused, _same

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


@pytest.mark.parametrize("most", [2, 80])
@pytest.mark.parametrize("causal,window", [(True, 0), (False, 0), (True, 37), (False, 20)])
def test_attention_across_pages_whose_key_scales_are_zero(most, causal, window):
    """Such a page's keys count with a score of 0 where a row sees them and not at all where it does not: a diagonal, a window's
    border and a last page that is not full run through them."""
    ctx = _context()
    pool = Pool(ctx, n_pages=60, n_kv=2, d=64, page=16, n_seq=2, max_pages=30)
    start, counts = [0, 130], [150, 70]
    pool.give([150, 200])
    for i in range(2):
        pool.ks[:, pool.table[i, [0, 3, 4, 8, 9, 12]].clamp(min=0).long()] = 0.0
    q = torch.randn(220, 8, 64, device="cuda", generator=pool.g)
    got, live = _attend(ctx, pool, q, counts, start, causal, window, most=most)
    assert ("tcgen05" in ctx.last_kernel()) == (most == 80)
    _done(ctx)
    _check(got, live, *attention(pool, q, start, counts, causal, window))
    ctx.close()


@pytest.mark.parametrize("most", [2, 80])
@pytest.mark.parametrize("size,scale", [(1e-9, 0.0), (1e-30, 0.0), (1.0, 1e-42)])
def test_attention_of_zero_keys_as_append_holds_them(most, size, scale):
    """Small queries, or a small scale, over keys of 0 and others: scores below what fp32 holds are 0, what is hidden stays hidden."""
    ctx = _context()
    pool = Pool(ctx, n_pages=30, n_kv=1, d=128, page=32, n_seq=1, max_pages=10)
    pool.give([200])
    k, v = (torch.randn(200, 1, 128, device="cuda", generator=pool.g) for _ in range(2))
    k[:90] = 0.0
    k[170:] = 0.0
    _append(ctx, pool, k, v, [200], [0])
    q = torch.randn(200, 4, 128, device="cuda", generator=pool.g) * size
    got, live = _attend(ctx, pool, q, [200], [0], scale=scale, most=most)
    _done(ctx)
    _check(got, live, *attention(pool, q, [0], [200], scale=scale))
    ctx.close()


def _by_what_a_row_sees(pool, q, start, counts, causal, window):
    """float64 result, and a bound that goes by the values a row sees: A, its weighted mean of |scale| * 127, and not by the largest
    value of all. As in paged_pool.attention() a weight is off relatively by its score's error (twice) and 2^-21; what is less is the error
    of a weight that is rounded to whole numbers: half a unit, of which the largest weight times scale of a row's 64 keys has 2^22 at least,
    so that 64 of them are off by 64 * 2^-23 A. Two fp16 terms (the other kernel) are off by less. Sums over steps as there."""
    n_q, d, n_kv = q.shape[1], q.shape[2], pool.n_kv
    out, tol, row = torch.zeros(q.shape, dtype=torch.float64, device="cuda"), torch.zeros(q.shape, dtype=torch.float64, device="cuda"), 0
    for i, (s0, m) in enumerate(zip(start, counts)):
        if m == 0:
            continue
        k, v = pool.rows(i, s0 + m)
        here, key = torch.arange(s0, s0 + m, device="cuda")[:, None], torch.arange(s0 + m, device="cuda")[None, :]
        hidden = (key > here) if causal else torch.zeros_like(key > here)
        if window:
            hidden = hidden | (key <= here - window)
        vs = pool.vs[0][pool.table[i].long()[torch.arange(s0 + m, device="cuda") // pool.page]].double()
        for h in range(n_q):
            g = h // (n_q // n_kv)
            x = q[row:row + m, h].double()
            score = (x @ k[:, g].T / math.sqrt(d)).masked_fill(hidden, -math.inf)
            p = torch.softmax(score, -1)
            out[row:row + m, h] = p @ v[:, g]
            off = x.abs().amax(-1, keepdim=True) * k[:, g].abs().sum(-1).max() / math.sqrt(d) * 2.0 ** -24
            size = score.masked_fill(hidden, 0.0).abs().amax(-1, keepdim=True)
            tol[row:row + m, h] = (2 * (off + size * 2.0 ** -21) + 2.0 ** -17 + 2.0 ** -21 + ((s0 + m) / 64 + 5) * 2.0 ** -23) * (p @ vs[:, g, None]) * 127
        row += m
    return out, tol


@pytest.mark.parametrize("d,most", [(64, 2), (128, 2), (256, 2), (64, 4), (128, 4), (64, 80), (128, 80)])
@pytest.mark.parametrize("causal,window", [(True, 0), (True, 1), (True, 23), (False, 40)])
@pytest.mark.parametrize("octaves", [12, 36, 70])
def test_attention_over_pages_of_very_unlike_values(d, most, causal, window, octaves):
    """A row whose keys have small values keeps its bits beside pages with large ones, which it does not see or hardly weighs."""
    ctx = _context()
    pool = Pool(ctx, n_pages=60, n_kv=2, d=d, page=16, n_seq=2, max_pages=30)
    start, counts = [0, 330], [150, 6]
    pool.give([150, 336])
    for i in range(2):
        for c in range(22):
            p = int(pool.table[i, c])
            if p >= 0:
                pool.vs[:, p] *= 2.0 ** -(octaves * ((c * 5) % 4) / 3.0)
    q = torch.randn(156, 8, d, device="cuda", generator=pool.g)
    got, live = _attend(ctx, pool, q, counts, start, causal, window, most=most)
    _done(ctx)
    _check(got, live, *_by_what_a_row_sees(pool, q, start, counts, causal, window))
    ctx.close()


# offsets of three sequences, and whether the operands' six rows have to be told
WRONG_OFFSETS = [
    ([0, 2, 4, 7], True), ([0, 2, 4, 0x7FFFFFFF], True), ([9, 9, 9, 9], True), ([-4, 2, 4, 6], False), ([0, 2, 9, 6], False), ([0, 2, 1, 6], False),
    ([0x7FFFFFFF, -(1 << 31), 4, 6], False), ([0, 2, 4, -1], False),
]


@pytest.mark.parametrize("off,told", WRONG_OFFSETS)
@pytest.mark.parametrize("most", [0, 2, 300])
def test_append_and_read_leave_sequences_out_whose_offsets_are_wrong(off, told, most):
    """Falling offsets and ones outside the rows: status 4, the pages and the rows of the others as they should be, nothing else touched."""
    ctx = _context()
    pool = Pool(ctx, n_pages=40, n_kv=2, d=64, page=16, n_seq=3, max_pages=12)
    start = [97, 47, 147]
    pool.give([110, 60, 160])
    x = torch.randn(2, 6 + 4, 128, device="cuda", generator=pool.g)
    x[:, 6:] = 1e6                                      # rows that would make every scale grow
    handle, o, st = pool.handle(), i32(off), i32(start)
    for rows in (6,) if told else (6, None):
        room = off[3] if rows is None else rows
        served = [i for i in range(3) if 0 <= off[i] <= off[i + 1] <= room]
        counts = [off[i + 1] - off[i] if i in served else 0 for i in range(3)]
        before = pool.state()
        torch.cuda.synchronize()
        ctx.kv_block_append_dev(handle, 0, x[0].data_ptr(), x[1].data_ptr(), 128, o.data_ptr(), st.data_ptr(), most, rows=rows)
        _done(ctx, 4)
        k, v = (torch.cat([t[off[i]:off[i] + counts[i]] for i in served] + [t[:0]]).view(-1, 2, 64) for t in x)
        _same(pool, _expect_append(before, pool, k, v, counts, start))
        out = torch.full((2, 6 + 4, 128), 5.0, device="cuda")
        want = out.clone()
        torch.cuda.synchronize()
        ctx.kv_block_read_dev(handle, 0, o.data_ptr(), st.data_ptr(), most, out[0].data_ptr(), out[1].data_ptr(), 128, rows=rows)
        _done(ctx, 4)
        for i in served:
            for w, c in zip(want, pool.rows(i, start[i] + counts[i])):
                w[off[i]:off[i] + counts[i]] = c[start[i]:].float().reshape(-1, 128)
        # (a row that two sequences claim, as [0, 2, 1, 6] has it, holds what one of them has there)
        once = [sum(off[i] <= r < off[i] + counts[i] for i in served) < 2 for r in range(10)]
        assert torch.equal(out[:, once], want[:, once])
        pool.restore(before)
    ctx.close()


def test_append_and_read_refuse_rows_beyond_counting():
    ctx = _context()
    pool = Pool(ctx)
    handle, x, n = pool.handle(), torch.zeros(4096, device="cuda"), i32([0] * 8)
    p, i = x.data_ptr(), n.data_ptr()
    torch.cuda.synchronize()
    for rows in (1 << 31, (1 << 64) - 1):
        _refused(lambda: ctx.kv_block_append_dev(handle, 0, p, p, 128, i, i, 1, rows=rows), -3)
        _refused(lambda: ctx.kv_block_read_dev(handle, 0, i, i, 1, p, p, 128, rows=rows), -3)
    ctx.kv_block_append_dev(handle, 0, p, p, 128, i, i, 1, rows=0)
    ctx.kv_block_read_dev(handle, 0, i, i, 1, p, p, 128, rows=0)
    _done(ctx)
    ctx.close()


@pytest.mark.parametrize("off", [off for off, _ in WRONG_OFFSETS] + [[0, 2, 100, 4], [0, 2, 4, 3]])
def test_pages_grow_for_sequences_whose_offsets_are_right(off):
    """Falling offsets and ones outside the rows: status 4, -1 and no pages for those, the others' pages and positions as they should be."""
    ctx = _context()
    pool = Pool(ctx, n_pages=20, n_kv=1, d=16, page=16, n_seq=4, max_pages=8)
    pool.give([31, 16, 0, 40])
    off = off + [6]
    book = Book(pool)
    inside = [0 <= a <= b <= 6 for a, b in zip(off, off[1:])]
    new = [off[i + 1] - off[i] if inside[i] else 0 for i in range(4)]
    before = pool.state()
    start, pos = torch.full((4,), 77, dtype=torch.int32, device="cuda"), torch.full((6,), 77, dtype=torch.int32, device="cuda")
    handle, o = pool.handle(), i32(off)
    ws = torch.empty(ctx.kv_pages_workspace(handle), dtype=torch.uint8, device="cuda").random_(0, 256)
    torch.cuda.synchronize()
    ctx.kv_pages_extend_dev(handle, o.data_ptr(), 6, start.data_ptr(), pos.data_ptr(), ws.data_ptr(), ws.numel())
    _done(ctx, 0 if all(inside) else 4)
    want, status = book.extend(new)
    assert status == 0 and start.tolist() == want
    book.same(pool, before)
    for r in range(6):
        here = [i for i in range(4) if want[i] >= 0 and off[i] <= r < off[i + 1]]
        assert pos[r] == (want[here[0]] + r - off[here[0]] if here else -1)
    ctx.close()


def test_pages_grow_without_positions():
    ctx = _context()
    pool = Pool(ctx, n_pages=20, n_kv=1, d=16, page=16, n_seq=3, max_pages=8)
    pool.give([31, 16, 0])
    book, before = Book(pool), pool.state()
    handle, o, start = pool.handle(), i32([0, 2, 40, 41]), i32([77] * 3)
    ws = torch.empty(ctx.kv_pages_workspace(handle), dtype=torch.uint8, device="cuda").random_(0, 256)
    torch.cuda.synchronize()
    ctx.kv_pages_extend_dev(handle, o.data_ptr(), 0, start.data_ptr(), None, ws.data_ptr(), ws.numel())
    _done(ctx)
    assert book.extend([2, 38, 1]) == (start.tolist(), 0)
    book.same(pool, before)
    ctx.close()


@pytest.mark.parametrize("d,n_seq", [(64, 2), (128, 2), (256, 2), (64, 400), (128, 400)])
@pytest.mark.parametrize("group", [1, 3, 8, 16, 40])
def test_a_workspace_for_many_rows_serves_fewer(d, n_seq, group):
    """A server has one workspace, sized for its longest prompt, for every call with as many heads: nothing behind it is written."""
    ctx = _context()
    pool = Pool(ctx, n_pages=60, n_kv=2, d=d, page=16, n_seq=n_seq, max_pages=30)
    handle, rows = pool.handle(), 700
    most = [0, 1, 2, 3, 5, 9, 17, 32, 33, 65, 600]
    need = [ctx.kv_block_attention_workspace(handle, 2 * group, rows, m) for m in most]
    assert need == sorted(need)
    assert all(ctx.kv_block_attention_workspace(handle, 2 * group, r, most[-1]) <= need[-1] for r in (0, 1, 40, 699))
    ws, guard = _guarded(need[-1])
    pool.give([400] + [0] * (n_seq - 2) + [300])
    q = torch.randn(40, 2 * group, d, device="cuda", generator=pool.g)
    for m in (1, 2, 5, 20):
        counts = [m] + [0] * (n_seq - 2) + [m // 2]
        start = [400 - m] + [-1] * (n_seq - 2) + [290]
        got, live = _attend(ctx, pool, q[:sum(counts)], counts, start, ws=ws[:need[-1]])
        _done(ctx)
        _check(got, live, *attention(pool, q[:sum(counts)], start, counts))
        assert torch.equal(ws[need[-1]:], guard)
    ctx.close()


@pytest.mark.parametrize("most", [1, 40])
def test_a_window_of_two_to_the_thirty(most):
    """A billion keys, which one page holds again and again; the first ones, in front of the window, would take all the weight."""
    ctx = _context()
    window = 1 << 30
    start = window + 200
    pool = Pool(ctx, n_pages=2, n_kv=1, d=64, page=128, n_seq=1, max_pages=(1 << 23) + 2)
    q = torch.randn(1, 1, 64, device="cuda", generator=pool.g)
    pool.table.fill_(1)
    pool.table[0, 0] = 0                                # keys 0 .. 127: along the query
    flat = (127.0 * torch.sign(q[0, 0])).to(torch.int8).expand(128, 64)
    pool.k[0, 0, 0] = flat.reshape(8, 16, 4, 16).permute(0, 2, 1, 3)
    pool.v[0, 0] = 127
    pool.ks[0, 0], pool.ks[0, 1] = 0.05, 0.01
    got, _ = _attend(ctx, pool, q, [1], [start], window=window, most=most)
    assert ("tcgen05" in ctx.last_kernel()) == (most == 40)
    _done(ctx)
    k, v = pool.rows(0, 256)
    p = torch.softmax(k[128:, 0] @ q[0, 0].double() / 8.0, 0)
    # every key of the page 2^23 times, give or take one; sums over the steps of a warp, 2^24 / (148 * 12), or the tiles of an SM, 2^23 / 148
    tol = (2.0 ** -22 + 2.0 ** -18 + 2.0 ** 16 * 2.0 ** -23) * float(v[128:].abs().max())
    assert float((got[0, 0].double() - p @ v[128:, 0]).abs().max()) < tol
    ctx.close()


def test_pages_of_a_pool_that_shared_memory_has_no_bits_for():
    """More than 131072 pages: those behind are looked up again, for the free ones and for what moves."""
    ctx = _context()
    pool = Pool(ctx, n_pages=150000, n_kv=1, d=16, page=16, n_seq=40, max_pages=3800)
    tokens = [60000 - 7 * i for i in range(36)] + [0] * 4
    pool.give(tokens)
    book, handle = Book(pool), pool.handle()
    ws = torch.empty(ctx.kv_pages_workspace(handle), dtype=torch.uint8, device="cuda").random_(0, 256)
    new = [17] * 36 + [40000, 9, 0, 1]
    for turn in range(2):
        before = pool.state()
        start, pos = _extend(ctx, pool, new)
        want, status = book.extend(new)
        assert status == 0 and start == want and pos == _positions(want, new)
        _done(ctx)
        book.same(pool, before)
        gone = [1, 5, 36]
        seqs = i32(gone)
        before = pool.state()
        torch.cuda.synchronize()
        ctx.kv_pages_trim_dev(handle, seqs.data_ptr(), None, 3)
        ctx.kv_pages_compact_dev(handle, ws.data_ptr(), ws.numel())
        _done(ctx)
        book.trim(gone, [0] * 3)
        book.compact()
        book.same(pool, before)
    ctx.close()
