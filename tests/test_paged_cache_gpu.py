"""The paged 8-bit KV cache: append and read, attention, pages; and rotary positions. Against float64 definitions (paged_pool.py)."""
import math

import numpy as np
import pytest
import torch

import yscv_b200
from paged_pool import LEAST, Pool, appended, attention, i32, offsets

pytestmark = pytest.mark.gpu


def _context():
    stream = torch.cuda.Stream()
    return yscv_b200.Context(0, stream=stream.cuda_stream)


def _done(ctx, status=0):
    ctx.synchronize()
    assert ctx.device_status() == status


# ---- rotary positions -------------------------------------------------------------------------------

def _frequencies(rot, scaling, factor, theta=10000.0, original=4096.0):
    w = theta ** (-2.0 * np.arange(rot // 2) / rot)
    kept = np.zeros(rot // 2)
    if scaling == "none":
        return w, 1.0
    if scaling == "banded":
        kept = np.clip((original * w / (2 * math.pi) - 1.0) / 3.0, 0, 1)
    if scaling == "yarn":
        lo, hi = (rot * math.log(original / (b * 2 * math.pi)) / (2 * math.log(theta)) for b in (32.0, 1.0))
        lo, hi = max(math.floor(lo), 0), min(math.ceil(hi), rot - 1)
        kept = 1 - np.clip((np.arange(rot // 2) - lo) / max(hi - lo, 0.001), 0, 1)
    return w * kept + w / factor * (1 - kept), (0.1 * math.log(factor) + 1 if scaling == "yarn" else 1.0)


@pytest.mark.parametrize("d,rot", [(64, 64), (128, 96), (128, 128), (256, 64), (80, 80), (64, 62), (34, 6), (7, 2), (512, 512)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("rows,heads,scaling,pad,shift,place", [
    (1, 5, "none", 0, 0, "out"), (3, 40, "yarn", 8, 0, "in"), (700, 3, "linear", 4, 4, "out"), (5, 2, "banded", 1, 1, "in"),
])
def test_rope(d, rot, interleaved, rows, heads, scaling, pad, shift, place):
    ctx = _context()
    g = torch.Generator(device="cuda").manual_seed(d + rows)
    stride = heads * d + pad
    buf = torch.randn(rows * stride + shift + 8, device="cuda", generator=g)
    x = buf[shift:shift + rows * stride].view(rows, stride)
    pos = torch.randint(0, 1 << 20, (rows,), dtype=torch.int32, device="cuda", generator=g)
    pos[0] = 0x7FFFFFFF if rows > 1 else 131071
    if rows > 2:
        pos[1], pos[2] = -1, 0
    before = buf.clone()
    out_buf = buf if place == "in" else torch.full_like(buf, 7.0)
    start = out_buf.clone()
    torch.cuda.synchronize()
    factor = 1.0 if scaling == "none" else 8.0
    rope = yscv_b200.Rope(rotary_dim=rot, interleaved=interleaved, scaling=scaling, factor=factor, original_positions=4096.0)
    ctx.rope_dev(x.data_ptr(), stride, rows, heads, d, pos.data_ptr(), rope, out_buf[shift:].data_ptr(), stride)
    _done(ctx)
    w, f = _frequencies(rot, scaling, factor)
    # (an angle at position p is off by p w 2^-52 or so in any fp64 form: 1e-6 at 2^31)
    angle = pos.double()[:, None] * torch.tensor(w, device="cuda")
    c, s = (torch.cos(angle) * f)[:, None], (torch.sin(angle) * f)[:, None]
    src = before[shift:shift + rows * stride].view(rows, stride)[:, :heads * d].double().view(rows, heads, d)
    want, size = src.clone(), src.abs()
    i = torch.arange(rot // 2, device="cuda")
    ia, ib = (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)
    a, b = src[..., ia], src[..., ib]
    want[..., ia], want[..., ib] = a * c - b * s, b * c + a * s
    size[..., ia] = size[..., ib] = (a.abs() + b.abs()) * f
    got = out_buf[shift:shift + rows * stride].view(rows, stride)[:, :heads * d].double().view(rows, heads, d)
    # sine and cosine to 2 ulp (2^-22), their angle to 2^-25 of a quarter turn, the factor, two products and a sum: 2^-24 each
    tol = size * (2.0 ** -22 + 2.0 ** -24 + 4 * 2.0 ** -24 + (pos.double().abs() * 2.0 ** -51)[:, None, None])
    live = pos >= 0
    assert torch.all(((got - want).abs() <= tol)[live])
    if rot < d:
        assert torch.equal(got[live][..., rot:], src[live][..., rot:])
    # rows that belong to nobody, the gaps between rows and what lies around them are as they were
    keep = torch.ones_like(out_buf, dtype=torch.bool)
    keep[shift:shift + rows * stride].view(rows, stride)[live, :heads * d] = False
    assert torch.equal(out_buf[keep], start[keep])
    ctx.close()


# ---- append and read --------------------------------------------------------------------------------

def _append(ctx, pool, k, v, counts, start, most=None, layer=0, pad=0, shift=0):
    n = pool.n_kv * pool.d
    rows = k.shape[0]
    buf = torch.full((2, rows * (n + pad) + shift + 4), 9.0, device="cuda")
    for t, x in zip(buf, (k, v)):
        t[shift:shift + rows * (n + pad)].view(rows, n + pad)[:, :n] = x.reshape(rows, n)
    off, st = offsets(counts), i32(start)
    torch.cuda.synchronize()
    ctx.kv_block_append_dev(pool.handle(), layer, buf[0, shift:].data_ptr(), buf[1, shift:].data_ptr(), n + pad, off.data_ptr(), st.data_ptr(),
                            most if most is not None else max(counts))
    ctx.synchronize()


def _expect_append(before, pool, k, v, counts, start, layer=0):
    """The pool's arrays after the append, block by block on the CPU."""
    arrays = [t.cpu().numpy().copy() for t in before[:4]]
    table = before[5].cpu().numpy()
    row = 0
    for i, (m, s0) in enumerate(zip(counts, start)):
        t = 0
        while s0 >= 0 and t < m:
            p, at = divmod(s0 + t, pool.page)
            n = min(m - t, pool.page - at)
            if p < pool.max_pages and 0 <= table[i, p] < pool.n_pages:
                for name, x, q8, sc in (("k", k, arrays[0], arrays[2]), ("v", v, arrays[1], arrays[3])):
                    for h in range(pool.n_kv):
                        block = q8[layer, table[i, p], h]
                        flat = (block.transpose(0, 2, 1, 3) if name == "k" else block.transpose(0, 2, 1)).reshape(pool.page, pool.d)
                        new, s = appended(flat[:at], sc[layer, table[i, p], h], at, x[row + t:row + t + n, h].cpu().numpy())
                        flat = flat.copy()
                        flat[:at + n] = new
                        sc[layer, table[i, p], h] = s
                        if name == "k":
                            q8[layer, table[i, p], h] = flat.reshape(-1, 16, pool.d // 16, 16).transpose(0, 2, 1, 3)
                        else:
                            q8[layer, table[i, p], h] = flat.reshape(-1, 16, pool.d).transpose(0, 2, 1)
            t += n
        row += m
    return arrays


def _same(pool, arrays):
    for t, want in zip((pool.k, pool.v, pool.ks, pool.vs), arrays):
        assert np.array_equal(t.cpu().numpy(), want)


@pytest.mark.parametrize("d,page,n_kv,start,counts", [
    (64, 16, 2, [0, 15, 31], [1, 1, 1]),              # an empty page, the last place of one, the first of the next
    (128, 64, 1, [5, 63, 0], [3, 130, 64]),           # into a begun group, over two borders, a whole page
    (16, 32, 3, [1, 0, 17], [0, 95, 33]),             # a sequence without rows
    (256, 128, 1, [100, -1, 0], [29, 4, 200]),        # one that takes no part
    (48, 128, 2, [17, 3, 128], [1, 250, 2]),
])
@pytest.mark.parametrize("size", [1.0, 1e-3])         # larger and smaller than what the begun pages hold
def test_append_holds_the_nearest_number(d, page, n_kv, start, counts, size):
    ctx = _context()
    pool = Pool(ctx, layers=2, n_pages=24, n_kv=n_kv, d=d, page=page, n_seq=3, max_pages=-(-300 // page), seed=d)
    pool.n_pages, pool.k, pool.v, pool.ks, pool.vs = _grown(pool, 3 * pool.max_pages + 2)
    pool.refs = torch.zeros(pool.n_pages, dtype=torch.int32, device="cuda")
    pool.give([max(0, s) + m for s, m in zip(start, counts)])
    rows = sum(counts)
    k, v = (torch.randn(rows, n_kv, d, device="cuda", generator=pool.g) * 8.0 * size for _ in range(2))
    k[0, 0, 0] = 0.5
    before = pool.state()
    _append(ctx, pool, k, v, counts, start, layer=1, pad=d % 3, shift=d // 16 % 2)
    _done(ctx)
    _same(pool, _expect_append(before, pool, k, v, counts, start, layer=1))
    ctx.close()


def _grown(pool, n_pages):
    p = Pool(pool.ctx, pool.layers, n_pages, pool.n_kv, pool.d, pool.page, pool.n_seq, pool.max_pages, seed=pool.d)
    return n_pages, p.k, p.v, p.ks, p.vs


@pytest.mark.parametrize("most", [1, 3, 400])
def test_append_of_more_or_fewer_rows_than_expected(most):
    ctx = _context()
    pool = Pool(ctx, n_pages=40, page=16, n_seq=3, max_pages=13)
    start, counts = [7, 0, 130], [150, 1, 40]
    pool.give([s + m for s, m in zip(start, counts)])
    k, v = (torch.randn(sum(counts), 2, 64, device="cuda", generator=pool.g) for _ in range(2))
    before = pool.state()
    _append(ctx, pool, k, v, counts, start, most=most)
    _done(ctx)
    _same(pool, _expect_append(before, pool, k, v, counts, start))
    ctx.close()


def test_append_borders_and_values_that_are_no_numbers():
    """Values half way between two whole numbers go to the even one; NaN and infinities do not touch the other tokens' scale."""
    ctx = _context()
    pool = Pool(ctx, n_pages=4, n_kv=4, page=16, n_seq=1, max_pages=2)
    pool.give([32])
    k = torch.zeros(17, 4, 64, device="cuda")
    k[:, 0] = torch.arange(64, device="cuda") - 31.5           # scale: 127 / 127 = 1 with the next line
    k[0, 0, 0] = 127.0
    k[:, 1] = 3.0
    k[3, 1, 5], k[4, 1, 6], k[5, 1, 7] = float("nan"), float("inf"), -float("inf")
    k[:, 2] = 1e-38                                             # below the smallest scale: 0
    k[:, 3] = 3.0e38
    k[7, 3, :32] = -3.0e38
    v = k.flip(1).contiguous()
    before = pool.state()
    _append(ctx, pool, k, v, [17], [2])
    _done(ctx)
    _same(pool, _expect_append(before, pool, k, v, [17], [2]))
    ks = pool.ks[0, pool.table[0, 0].item()]
    assert ks[1].item() >= float(np.float32(3.0) / np.float32(127)) and ks[2].item() >= float(np.float32(LEAST) / np.float32(127))
    ctx.close()


@pytest.mark.parametrize("d,page,n_kv", [(64, 16, 2), (256, 128, 1), (16, 32, 5)])
def test_read_is_number_times_scale(d, page, n_kv):
    ctx = _context()
    pool = Pool(ctx, n_pages=30, n_kv=n_kv, d=d, page=page, n_seq=4, max_pages=9)
    start, counts = [0, 5, -1, page - 1], [page * 2 + 3, 1, 4, 2]
    pool.give([max(0, s) + m for s, m in zip(start, counts)])
    n, rows = n_kv * d, sum(counts) + 2
    out = torch.full((2, rows, n + 3), 5.0, device="cuda")
    torch.cuda.synchronize()
    off, st = offsets(counts), i32(start)
    ctx.kv_block_read_dev(pool.handle(), 0, off.data_ptr(), st.data_ptr(), max(counts), out[0].data_ptr(), out[1].data_ptr(), n + 3)
    _done(ctx)
    row = 0
    for i, (s, m) in enumerate(zip(start, counts)):
        for t, got in enumerate(out[:, row:row + m]):
            want = torch.full((m, n), 5.0, device="cuda") if s < 0 else pool.rows(i, s + m)[t][s:].float().reshape(m, n)
            assert torch.equal(got[:, :n], want)
        row += m
    assert torch.all(out[:, row:] == 5.0) and torch.all(out[:, :, n:] == 5.0)
    ctx.close()


# ---- attention --------------------------------------------------------------------------------------

def _attend(ctx, pool, q, counts, start, causal=True, window=0, scale=0.0, most=None, pad=0, shift=0, layer=0, extra=2, ws=None):
    rows, n_q, d = q.shape
    stride = n_q * d + pad
    buf = torch.full(((rows + extra) * stride + shift + 4,), 2.0, device="cuda")
    buf[shift:shift + rows * stride].view(rows, stride)[:, :n_q * d] = q.reshape(rows, n_q * d)
    out = torch.full_like(buf, 3.0)
    off, st = offsets(counts), i32(start)
    most = max(counts) if most is None else most
    handle = pool.handle()
    need = ctx.kv_block_attention_workspace(handle, n_q, rows + extra, most)
    ws = torch.empty(need, dtype=torch.uint8, device="cuda").random_(0, 256) if ws is None else ws
    torch.cuda.synchronize()
    ctx.kv_block_attention_dev(handle, layer, buf[shift:].data_ptr(), stride, n_q, off.data_ptr(), st.data_ptr(), rows + extra, most, causal, window,
                               scale, out[shift:].data_ptr(), stride, ws.data_ptr(), need)
    ctx.synchronize()
    used = out[shift:shift + rows * stride].view(rows, stride)
    keep = torch.ones_like(out, dtype=torch.bool)
    live = torch.repeat_interleave(torch.tensor([s >= 0 for s in start], device="cuda"), torch.tensor(counts, device="cuda"))
    keep[shift:shift + rows * stride].view(rows, stride)[live, :n_q * d] = False
    assert torch.all(out[keep] == 3.0)
    return used[:, :n_q * d].reshape(rows, n_q, d), live


def _check(got, live, want, tol):
    assert torch.all(((got.double() - want).abs() <= tol)[live]), float(((got.double() - want).abs() / tol)[live].max())


SHAPES = [
    # d, page, n_kv, group, start, counts
    (64, 16, 1, 1, [0, 1, 62, 63, 64], [1, 1, 1, 1, 1]),             # lengths around a step's border, one key
    (128, 64, 2, 8, [200, 0, -1, 5000, 77], [1, 1, 3, 1, 0]),        # long beside short, one that takes no part, one without rows
    (128, 16, 3, 5, [19, 300, 7], [2, 3, 5]),                        # drafts, groups that are no power of two
    (256, 32, 1, 12, [131, 1000], [1, 4]),
    (64, 128, 2, 16, [4000, 3], [1, 1]),
    (64, 32, 8, 3, [90, 1500, 2], [8, 7, 1]),
]


@pytest.mark.parametrize("d,page,n_kv,group,start,counts", SHAPES)
@pytest.mark.parametrize("causal,window", [(True, 0), (False, 0), (True, 37), (True, 1), (False, 100)])
def test_attention_of_a_few_rows(d, page, n_kv, group, start, counts, causal, window):
    ctx = _context()
    most = max(max(0, s) + m for s, m in zip(start, counts))
    max_pages = -(-most // page) + 1
    pool = Pool(ctx, layers=2, n_pages=sum(-(-(max(0, s) + m) // page) for s, m in zip(start, counts)) + 3, n_kv=n_kv, d=d, page=page,
                n_seq=len(start), max_pages=max_pages, seed=page)
    pool.give([max(0, s) + m for s, m in zip(start, counts)])
    q = torch.randn(sum(counts), n_kv * group, d, device="cuda", generator=pool.g)
    got, live = _attend(ctx, pool, q, counts, start, causal, window, layer=1, pad=(group % 2) * 3, shift=group % 3)
    _done(ctx)
    _check(got, live, *attention(pool, q, start, counts, causal, window, layer=1))
    ctx.close()


PROMPTS = [
    # d, page, n_kv, group, start, counts
    (128, 64, 2, 8, [0], [300]),                       # whole tiles and a part of one
    (64, 16, 1, 4, [0, 130, -1], [129, 33, 40]),       # positions around the tiles' borders
    (128, 128, 1, 1, [5, 0], [257, 1]),                # one head a KV head: 256 positions to a tile
    (64, 32, 2, 48, [700], [5]),                       # two positions of 48 heads to a half
    (128, 16, 1, 128, [3, 1000], [3, 2]),              # one position to a half
    (128, 32, 8, 6, [0, 2000, 17, 5], [31, 90, 0, 11]),
    (64, 64, 4, 3, [64, 63], [200, 350]),
    (128, 64, 1, 16, [9000], [20]),                    # a short piece over a long cache: every SM has a part of it
]


@pytest.mark.parametrize("d,page,n_kv,group,start,counts", PROMPTS)
@pytest.mark.parametrize("causal,window", [(True, 0), (False, 0), (True, 100), (False, 33)])
def test_attention_of_prompts(d, page, n_kv, group, start, counts, causal, window):
    ctx = _context()
    total = [max(0, s) + m for s, m in zip(start, counts)]
    pool = Pool(ctx, layers=2, n_pages=sum(-(-t // page) for t in total) + 3, n_kv=n_kv, d=d, page=page, n_seq=len(start),
                max_pages=-(-max(total) // page) + 1, seed=page)
    pool.give(total)
    q = torch.randn(sum(counts), n_kv * group, d, device="cuda", generator=pool.g)
    got, live = _attend(ctx, pool, q, counts, start, causal, window, layer=1, pad=(n_kv % 2) * 3, shift=n_kv % 3)
    assert "tcgen05" in ctx.last_kernel()
    _done(ctx)
    _check(got, live, *attention(pool, q, start, counts, causal, window, layer=1))
    ctx.close()


@pytest.mark.parametrize("size,scale", [(0.0, 0.0), (1e-30, 0.0), (30.0, 0.0), (1.0, 0.02), (1e30, 1e-30)])
def test_attention_of_queries_of_any_size(size, scale):
    """Flat and peaked weights, rows whose size differs by 10^3, scales of pages that differ by 10^4."""
    ctx = _context()
    pool = Pool(ctx, n_pages=60, n_kv=2, d=128, page=32, n_seq=2, max_pages=40)
    pool.ks *= torch.exp(1.5 * torch.randn(pool.ks.shape, device="cuda", generator=pool.g))
    pool.vs *= torch.exp(3.0 * torch.randn(pool.vs.shape, device="cuda", generator=pool.g))
    start, counts = [1000, 333], [1, 2]
    pool.give([s + m for s, m in zip(start, counts)])
    q = torch.randn(3, 8, 128, device="cuda", generator=pool.g) * size
    q[1:] *= torch.logspace(-3, 0, 8, device="cuda")[None, :, None]
    for most in (2, 100):   # the kernel for a few rows, and the one for prompts
        got, live = _attend(ctx, pool, q, counts, start, scale=scale, most=most)
        assert ("tcgen05" in ctx.last_kernel()) == (most == 100)
        _done(ctx)
        _check(got, live, *attention(pool, q, start, counts, scale=scale))
    ctx.close()


@pytest.mark.parametrize("d,most", [(64, 3), (128, 3), (256, 3), (64, 90), (128, 90)])
def test_attention_keeps_rows_apart_that_are_no_numbers(d, most):
    ctx = _context()
    pool = Pool(ctx, n_pages=40, n_kv=2, d=d, page=32, n_seq=2, max_pages=30)
    pool.give([501, 303])
    q = torch.randn(4, 8, d, device="cuda", generator=pool.g)
    clean = q.clone()
    q[0, 3, 5], q[2, 1, 0], q[2, 7, d - 1] = float("nan"), float("inf"), -float("inf")
    got, live = _attend(ctx, pool, q, [1, 3], [500, 300], most=most)
    _done(ctx)
    want, tol = attention(pool, clean, [500, 300], [1, 3])
    bad = torch.zeros(4, 8, dtype=torch.bool, device="cuda")
    bad[0, 3] = bad[2, 1] = bad[2, 7] = True
    assert torch.all(torch.isnan(got[bad])) and not torch.any(torch.isnan(got[~bad]))
    assert torch.all(((got.double() - want).abs() <= tol)[~bad])
    ctx.close()


@pytest.mark.parametrize("most", [1, 80])
def test_attention_leaves_pages_out_that_are_not_there(most):
    """A page number outside the pool hides its keys and is told; so are positions behind the table."""
    ctx = _context()
    pool = Pool(ctx, n_pages=30, n_kv=1, d=64, page=16, n_seq=2, max_pages=8)
    pool.give([100, 90])
    q = torch.randn(2, 4, 64, device="cuda", generator=pool.g)
    good, _ = _attend(ctx, pool, q, [1, 1], [99, 89], most=most)
    _done(ctx)
    for number in (-1, 30, 1 << 30, -(1 << 31)):
        pool.table[0, 2] = number
        got, _ = _attend(ctx, pool, q, [1, 1], [99, 89], most=most)
        _done(ctx, 4)
        assert torch.equal(got[1], good[1])
        k, v = (torch.cat([x[:32], x[48:100]]) for x in _rows_without(pool))
        want = torch.softmax(torch.einsum("hd,kd->hk", q[0].double(), k[:, 0]) / 8.0, -1) @ v[:, 0]
        assert float((got[0].double() - want).abs().max()) < 1e-5 * float(v.abs().max())   # (100 keys: 2^-18 + scores of 6)
    pool.table[0, 2] = 0
    got, _ = _attend(ctx, pool, q, [1, 1], [8 * 16 + 40, 89], most=most)
    assert ctx.device_status() in (3, 4)   # behind the table, and its last place has no page: the word holds either
    assert torch.equal(got[1], good[1])
    pool.table.fill_(-1)
    got, _ = _attend(ctx, pool, q, [1, 1], [99, 89], most=most)
    _done(ctx, 4)
    assert torch.all(got == 0)
    ctx.close()


def _rows_without(pool):
    saved = pool.table.clone()
    pool.table[0].clamp_(0, pool.n_pages - 1)
    rows = pool.rows(0, 100)
    pool.table.copy_(saved)
    return rows


def test_attention_of_many_sequences_and_of_none():
    ctx = _context()
    n = 300
    pool = Pool(ctx, n_pages=2 * n, n_kv=1, d=64, page=16, n_seq=n, max_pages=3)
    counts = [(i * 7) % 3 for i in range(n)]
    start = [-1 if i % 11 == 0 else (i * 5) % 30 for i in range(n)]
    pool.give([max(0, s) + m if m else 0 for s, m in zip(start, counts)])
    q = torch.randn(sum(counts), 4, 64, device="cuda", generator=pool.g)
    got, live = _attend(ctx, pool, q, counts, start)
    _done(ctx)
    _check(got, live, *attention(pool, q, start, counts))
    _attend(ctx, pool, q, [0] * (n - 1) + [len(q)], [-1] * n)
    _done(ctx)
    ctx.close()


# ---- pages ------------------------------------------------------------------------------------------

class Book:
    """The pages of a pool as a list of sequences would keep them, one after another."""

    def __init__(self, pool):
        self.page, self.n_pages, self.max_pages = pool.page, pool.n_pages, pool.max_pages
        self.table = [[p for p in row if p >= 0] for row in pool.table.tolist()]
        self.length, self.refs = pool.length.tolist(), pool.refs.tolist()
        self.copies = []

    def extend(self, new):
        free = [p for p in range(self.n_pages) if self.refs[p] == 0]
        refs0, start, used, failed, status = list(self.refs), [], 0, False, 0
        self.copies = []
        for i, m in enumerate(new):
            wanted, held = -(-(self.length[i] + m) // self.page), len(self.table[i])
            if m == 0 or wanted > self.max_pages:
                start.append(-1)
                status = 3 if m else status
                continue
            share = self.length[i] % self.page != 0 and refs0[self.table[i][-1]] > 1
            need = wanted - held + share
            if need and (failed or used + need > len(free)):
                failed = True
                start.append(-1)
                continue
            mine, used = free[used:used + need], used + need
            start.append(self.length[i])
            if share:
                old, p = self.table[i][-1], mine.pop(0)
                self.table[i][-1], self.refs[p] = p, 1
                self.refs[old] -= 1
                self.copies.append((old, p))
            for p in mine:
                self.table[i].append(p)
                self.refs[p] = 1
            self.length[i] += m
        return start, 5 if failed else status

    def trim(self, seqs, keep):
        for i, k in zip(seqs, keep):
            self.length[i] = min(self.length[i], max(0, k))
            held = -(-self.length[i] // self.page)
            for p in self.table[i][held:]:
                self.refs[p] -= 1
            del self.table[i][held:]

    def fork(self, src, dst):
        for s, d in zip(src, dst):
            self.table[d], self.length[d] = list(self.table[s]), self.length[s]
            for p in self.table[d]:
                self.refs[p] += 1

    def compact(self):
        used = [p for p in range(self.n_pages) if self.refs[p]]
        gaps = [p for p in range(len(used)) if not self.refs[p]]
        self.copies = list(zip([p for p in used if p >= len(used)], gaps))
        to = dict(self.copies)
        self.table = [[to.get(p, p) for p in row] for row in self.table]
        for s, d in self.copies:
            self.refs[s], self.refs[d] = 0, self.refs[s]

    def same(self, pool, before):
        want = torch.full((pool.n_seq, pool.max_pages), -1, dtype=torch.int32)
        for i, row in enumerate(self.table):
            want[i, :len(row)] = torch.tensor(row, dtype=torch.int32)
        assert torch.equal(pool.table.cpu(), want)
        assert pool.length.tolist() == self.length and pool.refs.tolist() == self.refs
        for t, b in zip((pool.k, pool.v, pool.ks, pool.vs), before[:4]):
            b = b.clone()
            for s, d in self.copies:
                b[:, d] = b[:, s]
            assert torch.equal(t, b)


def _extend(ctx, pool, new, extra=3):
    rows = sum(new) + extra
    start, pos = torch.full((pool.n_seq,), 77, dtype=torch.int32, device="cuda"), torch.full((rows,), 77, dtype=torch.int32, device="cuda")
    off = offsets(new)
    handle = pool.handle()
    need = ctx.kv_pages_workspace(handle)
    ws = torch.empty(need, dtype=torch.uint8, device="cuda").random_(0, 256)
    torch.cuda.synchronize()
    ctx.kv_pages_extend_dev(handle, off.data_ptr(), rows, start.data_ptr(), pos.data_ptr(), ws.data_ptr(), need)
    ctx.synchronize()
    return start.tolist(), pos.tolist()


def _positions(start, new, extra=3):
    return [s + j if s >= 0 else -1 for s, m in zip(start, new) for j in range(m)] + [-1] * extra


@pytest.mark.parametrize("page,n_kv,d,layers", [(16, 1, 16, 3), (64, 4, 128, 2), (128, 8, 256, 1)])
def test_pages_of_sequences_that_grow_fork_and_end(page, n_kv, d, layers):
    ctx = _context()
    pool = Pool(ctx, layers=layers, n_pages=40, n_kv=n_kv, d=d, page=page, n_seq=9, max_pages=7)
    book = Book(pool)
    rng = np.random.default_rng(page)
    handle = pool.handle()
    for turn in range(25):
        new = [int(rng.integers(0, page + 3)) if rng.random() < 0.7 else 0 for _ in range(9)]
        before = pool.state()
        start, pos = _extend(ctx, pool, new)
        want, status = book.extend(new)
        assert start == want and pos == _positions(want, new)
        seen = ctx.device_status()
        assert seen == 0 if status == 0 else seen in (3, 5)
        book.same(pool, before)
        ends = [int(i) for i in rng.choice(9, int(rng.integers(0, 4)), replace=False)]
        keep = [int(rng.integers(-2, 2 * page)) if rng.random() < 0.5 else 0 for _ in ends]
        if ends:
            e, k = i32(ends), i32(keep)
            before = pool.state()
            torch.cuda.synchronize()
            ctx.kv_pages_trim_dev(handle, e.data_ptr(), k.data_ptr(), len(ends))
            ctx.synchronize()
            book.trim(ends, keep)
            book.copies = []
            book.same(pool, before)
        empty = [i for i in range(9) if book.length[i] == 0]
        full = [i for i in range(9) if book.length[i]]
        pairs = [(int(rng.choice(full)), d_) for d_ in empty[:2]] if full else []
        if pairs:
            s, t = i32(p[0] for p in pairs), i32(p[1] for p in pairs)
            before = pool.state()
            torch.cuda.synchronize()
            ctx.kv_pages_fork_dev(handle, s.data_ptr(), t.data_ptr(), len(pairs))
            _done(ctx)
            book.fork(*zip(*pairs))
            book.copies = []
            book.same(pool, before)
        if turn % 4 == 3:
            ws = torch.empty(ctx.kv_pages_workspace(handle), dtype=torch.uint8, device="cuda").random_(0, 256)
            before = pool.state()
            torch.cuda.synchronize()
            ctx.kv_pages_compact_dev(handle, ws.data_ptr(), ws.numel())
            _done(ctx)
            book.compact()
            book.same(pool, before)
    ctx.close()


def test_pages_of_a_large_pool():
    """More sequences than threads, more pages than a pass of the block over them."""
    ctx = _context()
    n = 2500
    pool = Pool(ctx, n_pages=9000, n_kv=1, d=16, page=16, n_seq=n, max_pages=5)
    book = Book(pool)
    new = [(i * 37) % 70 for i in range(n)]
    before = pool.state()
    start, pos = _extend(ctx, pool, new)
    want, status = book.extend(new)
    assert status == 0 and start == want and pos == _positions(want, new)
    book.same(pool, before)
    gone = i32(range(0, n, 3))
    handle = pool.handle()
    ctx.kv_pages_trim_dev(handle, gone.data_ptr(), None, len(gone))
    ws = torch.empty(ctx.kv_pages_workspace(handle), dtype=torch.uint8, device="cuda")
    before = pool.state()
    torch.cuda.synchronize()
    ctx.kv_pages_compact_dev(handle, ws.data_ptr(), ws.numel())
    _done(ctx)
    book.trim(range(0, n, 3), [0] * n)
    book.compact()
    book.same(pool, before)
    src = i32(i for i in range(1, n, 3))
    dst = i32(i - 1 for i in range(1, n, 3))
    torch.cuda.synchronize()
    ctx.kv_pages_fork_dev(handle, src.data_ptr(), dst.data_ptr(), len(src))
    _done(ctx)
    book.fork(src.tolist(), dst.tolist())
    book.copies = []
    new = [i % 2 for i in range(n)]
    before = pool.state()
    start, pos = _extend(ctx, pool, new)
    want, status = book.extend(new)
    assert start == want and pos == _positions(want, new) and ctx.device_status() == status
    book.same(pool, before)
    ctx.close()


def test_numbers_that_pages_cannot_use_are_left_out():
    ctx = _context()
    pool = Pool(ctx, n_pages=20, n_seq=6, max_pages=4)
    pool.give([20, 0, 30, 0, 0, 5])
    book = Book(pool)
    handle = pool.handle()
    before = pool.state()
    # a destination twice, one that is not empty, a source that is a destination, numbers that are no sequence
    src, dst = i32([0, 2, 2, 3, 6, 0, -1, 2]), i32([1, 1, 5, 4, 3, -1, 3, 6])
    torch.cuda.synchronize()
    ctx.kv_pages_fork_dev(handle, src.data_ptr(), dst.data_ptr(), 8)
    _done(ctx, 4)
    book.fork([0], [1])
    book.same(pool, before)
    # the same sequence twice, numbers that are no sequence
    seqs, keep = i32([0, 0, 0, 77, -3]), i32([17, 3, 40, 0, 0])
    torch.cuda.synchronize()
    ctx.kv_pages_trim_dev(handle, seqs.data_ptr(), keep.data_ptr(), 5)
    _done(ctx, 4)
    book.trim([0], [3])
    book.same(pool, before)
    for _ in range(2):
        ctx.kv_pages_trim_dev(handle, seqs.data_ptr(), None, 2)
        _done(ctx)
        book.trim([0], [0])
        book.same(pool, before)
    ctx.close()


def test_copy_of_pages():
    ctx = _context()
    pool = Pool(ctx, layers=3, n_pages=20, n_kv=3, d=48, page=32, n_seq=1, max_pages=1)
    before = pool.state()
    src, dst = i32([3, -1, 5, 4, 19, 2, 20]), i32([7, 2, 5, -1, 0, 1 << 20, 6])
    torch.cuda.synchronize()
    ctx.kv_pages_copy_dev(pool.handle(), src.data_ptr(), dst.data_ptr(), 7)
    _done(ctx, 4)
    for t, b in zip((pool.k, pool.v, pool.ks, pool.vs), before):
        b[:, 7], b[:, 0] = b[:, 3].clone(), b[:, 19].clone()
        assert torch.equal(t, b)
    ctx.close()


# ---- the calls that go wrong, and the ones that are easily forgotten --------------------------------

@pytest.mark.parametrize("most", [0, 1, 80])
def test_attention_serves_the_others_where_a_sequence_s_numbers_are_wrong(most):
    """Offsets outside the call's rows or falling ones, starts behind the table: told, and nothing beside them changes."""
    ctx = _context()
    pool = Pool(ctx, n_pages=40, n_kv=1, d=64, page=16, n_seq=3, max_pages=12)
    pool.give([100, 50, 150])
    q = torch.randn(6, 4, 64, device="cuda", generator=pool.g)
    want, tol = attention(pool, q, [98, 48, 148], [2, 2, 2])
    handle = pool.handle()
    ws = torch.zeros(ctx.kv_block_attention_workspace(handle, 4, 6, most), dtype=torch.uint8, device="cuda")

    def run(off, start):
        out = torch.full((8, 4, 64), 3.0, device="cuda")
        off, start = i32(off), i32(start)
        torch.cuda.synchronize()
        ctx.kv_block_attention_dev(handle, 0, q.data_ptr(), 256, 4, off.data_ptr(), start.data_ptr(), 6, most, True, 0, 0.0, out.data_ptr(), 256,
                                   ws.data_ptr(), ws.numel())
        ctx.synchronize()
        assert torch.all(out[6:] == 3.0)
        return out[:6], ctx.device_status()

    whole, status = run([0, 2, 4, 6], [98, 48, 148])
    assert status == 0 and torch.all((whole.double() - want).abs() <= tol)
    # rows that belong to a served sequence alone (the fourth case's last sequence has row 1 too)
    for off, here in [([0, 2, 4, 7], [0, 1, 2, 3]), ([0, 2, 4, 0x7FFFFFFF], [0, 1, 2, 3]), ([-4, 2, 4, 6], [2, 3, 4, 5]), ([0, 2, 1, 6], [0]),
                      ([0x7FFFFFFF, -(1 << 31), 4, 6], [4, 5])]:
        got, status = run(off, [98, 48, 148])
        assert status == 4
        assert torch.equal(got[here], whole[here])
    for start in (0x7FFFFFFF, 0x7FFFFFFE, 12 * 16 - 1, 1 << 24):
        got, status = run([0, 2, 4, 6], [98, start, 148])
        assert status in (3, 4) and torch.equal(got[:2], whole[:2]) and torch.equal(got[4:], whole[4:])
    ctx.close()


@pytest.mark.parametrize("d,page,counts,start", [
    (256, 64, [130, 1, 40], [0, 500, 70]),             # heads of 256 have one kernel for all lengths
    (128, 128, [129, 256, 3], [127, 0, 128]),          # pages of a tile's size, positions around them
    (64, 128, [400], [40000]),                         # a piece of a prompt over a long cache, one sequence
])
def test_attention_of_longer_rows(d, page, counts, start):
    ctx = _context()
    total = [s + m for s, m in zip(start, counts)]
    pool = Pool(ctx, n_pages=sum(-(-t // page) for t in total) + 2, n_kv=2, d=d, page=page, n_seq=len(start), max_pages=-(-max(total) // page) + 3)
    pool.give(total)
    q = torch.randn(sum(counts), 8, d, device="cuda", generator=pool.g)
    for window in (0, 200):
        got, live = _attend(ctx, pool, q, counts, start, True, window, scale=0.11)
        _done(ctx)
        _check(got, live, *attention(pool, q, start, counts, True, window, 0.11))
    ctx.close()


def test_attention_of_sequences_that_overlap_without_end():
    """Falling offsets can let sequences claim the same rows, so many times that their work is beyond counting: told, and left alone."""
    ctx = _context()
    rows, n_seq = 4096, 80
    pool = Pool(ctx, n_pages=2, n_kv=1, d=64, page=128, n_seq=n_seq, max_pages=8192)
    q = torch.zeros(rows, 128, 64, device="cuda")
    out = torch.full_like(q, 3.0)
    off, start = i32([rows * (i % 2) for i in range(n_seq + 1)]), i32([8192 * 128 - rows] * n_seq)
    handle = pool.handle()
    ws = torch.empty(ctx.kv_block_attention_workspace(handle, 128, rows, 100), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    ctx.kv_block_attention_dev(handle, 0, q.data_ptr(), 128 * 64, 128, off.data_ptr(), start.data_ptr(), rows, 100, True, 0, 0.0, out.data_ptr(), 128 * 64,
                               ws.data_ptr(), ws.numel())
    assert "tcgen05" in ctx.last_kernel()
    _done(ctx, 4)
    assert torch.all(out == 3.0)
    ctx.close()


@pytest.mark.parametrize("d", [64, 128, 256])
def test_attention_of_as_many_sequences_as_there_may_be(d):
    """The largest n_seq that is not refused, of which the first, the last and one between take part."""
    ctx = _context()

    def takes(n):
        pool = Pool(ctx, n_pages=2, n_kv=1, d=d, page=16, n_seq=1, max_pages=4)
        try:
            ctx.kv_block_attention_workspace(pool.handle(n_seq=n), 2, 8, 1)
        except yscv_b200.YscvCudaError:
            return False
        return True

    lo, hi = 1, 1 << 17
    while hi - lo > 1:
        lo, hi = ((lo + hi) // 2, hi) if takes((lo + hi) // 2) else (lo, (lo + hi) // 2)
    assert lo > 1000
    pool = Pool(ctx, n_pages=20, n_kv=1, d=d, page=16, n_seq=lo, max_pages=4)
    counts, start = [0] * lo, [-1] * lo
    for i, m, s in ((0, 3, 20), (lo // 2, 1, 63), (lo - 1, 4, 0)):
        counts[i], start[i] = m, s
    pool.give([max(0, s) + m if m else 0 for s, m in zip(start, counts)])
    q = torch.randn(8, 2, d, device="cuda", generator=pool.g)
    for most in (1, 100):
        got, live = _attend(ctx, pool, q, counts, start, most=most)
        _done(ctx)
        _check(got, live, *attention(pool, q, start, counts))
    ctx.close()


@pytest.mark.parametrize("most", [1, 70])
def test_attention_of_pages_whose_scales_are_zero(most):
    """Keys of 0 take part with a score of 0, values of 0 with their weight: beside others, and alone."""
    ctx = _context()
    pool = Pool(ctx, n_pages=40, n_kv=1, d=64, page=16, n_seq=2, max_pages=20)
    pool.give([200, 150])
    pages = pool.table[0].long()
    pool.vs[:, pages[2:5]] = 0.0
    pool.ks[:, pages[4:7]] = 0.0
    pool.vs[:, pool.table[1, :10].long()] = 0.0
    q = torch.randn(2, 4, 64, device="cuda", generator=pool.g)
    got, live = _attend(ctx, pool, q, [1, 1], [199, 149], most=most)
    _done(ctx)
    _check(got, live, *attention(pool, q, [199, 149], [1, 1]))
    assert torch.all(got[1] == 0)
    ctx.close()


@pytest.mark.parametrize("rows", [31, 32, 33, 64, 65])
@pytest.mark.parametrize("n_seq", [1, 40])
def test_attention_on_both_sides_of_the_choice_of_a_kernel(rows, n_seq):
    ctx = _context()
    pool = Pool(ctx, n_pages=n_seq * 7, n_kv=1, d=64, page=32, n_seq=n_seq, max_pages=7)
    counts, start = [rows] + [i % 3 for i in range(1, n_seq)], [100 + 3 * (i % 5) for i in range(n_seq)]
    pool.give([s + m for s, m in zip(start, counts)])
    q = torch.randn(sum(counts), 1, 64, device="cuda", generator=pool.g)
    got, live = _attend(ctx, pool, q, counts, start)
    _done(ctx)
    assert ("tcgen05" in ctx.last_kernel()) == (rows > 32)
    _check(got, live, *attention(pool, q, start, counts))
    ctx.close()


def test_pages_behind_two_gigabytes_of_a_layer():
    """32-bit byte offsets end at page 32768 of these, 32-bit signed ones at 16384."""
    ctx = _context()
    page, n_kv, d, n = 64, 8, 128, 33000
    pool = Pool.__new__(Pool)
    pool.__dict__.update(ctx=ctx, layers=2, n_pages=n, n_kv=n_kv, d=d, page=page, n_seq=2, max_pages=4, dev="cuda")
    pool.k = torch.empty(2, n, n_kv, page // 16, d // 16, 16, 16, dtype=torch.int8, device="cuda")
    pool.v = torch.empty(2, n, n_kv, page // 16, d, 16, dtype=torch.int8, device="cuda")
    pool.ks, pool.vs = (torch.zeros(2, n, n_kv, device="cuda") for _ in range(2))
    pool.refs, pool.length = torch.zeros(n, dtype=torch.int32, device="cuda"), i32([0, 0])
    pool.table = torch.tensor([[n - 1, 7, -1, -1], [16384, n - 2, 16383, -1]], dtype=torch.int32, device="cuda")
    for p in pool.table.flatten().tolist():
        if p >= 0:
            pool.refs[p] = 1
    g = torch.Generator(device="cuda").manual_seed(3)
    counts, start = [100, 140], [0, 0]
    kv = torch.randn(240, 2 * n_kv * d, device="cuda", generator=g)
    handle, off, st = pool.handle(), offsets(counts), i32(start)
    torch.cuda.synchronize()
    for layer in (0, 1):
        ctx.kv_block_append_dev(handle, layer, kv.data_ptr(), kv[:, n_kv * d:].data_ptr(), 2 * n_kv * d, off.data_ptr(), st.data_ptr(), 140)
    # another page of the last ones, by a copy
    src, dst = i32([n - 1]), i32([n - 3])
    torch.cuda.synchronize()
    ctx.kv_pages_copy_dev(handle, src.data_ptr(), dst.data_ptr(), 1)
    _done(ctx)
    pool.table[0, 0] = n - 3
    x = kv.view(240, 2, n_kv, d).double()
    row = 0
    for i, m in enumerate(counts):
        for got, want in zip(pool.rows(i, m, 1), (x[row:row + m, 0], x[row:row + m, 1])):
            # half a step of the scale, which is a 127th of the largest value of a page's head: at most 5.5 / 127
            assert float((got - want).abs().max()) < 0.5 * 5.5 / 127
        row += m
    q = torch.randn(240, 2 * n_kv, d, device="cuda", generator=g)
    got, live = _attend(ctx, pool, q, counts, start, layer=1)
    _check(got, live, *attention(pool, q, start, counts, layer=1))
    got, live = _attend(ctx, pool, q[:2], [1, 1], [99, 139], layer=1)
    _check(got, live, *attention(pool, q[:2], [99, 139], [1, 1], layer=1))
    _done(ctx)
    ctx.close()


def test_two_contexts_attend_at_once():
    """Two streams over one pool, a workspace each, prompts and single tokens, again and again."""
    ctxs = [_context(), _context()]
    pool = Pool(ctxs[0], n_pages=80, n_kv=4, d=128, page=32, n_seq=2, max_pages=40)
    start, counts = [[1000, 700], [400, 100]], [[1, 1], [90, 300]]
    pool.give([1001, 800])
    qs = [torch.randn(sum(c), 16, 128, device="cuda", generator=pool.g) for c in counts]
    offs, sts = [offsets(c) for c in counts], [i32(s) for s in start]
    outs = [[torch.zeros_like(q) for _ in range(20)] for q in qs]
    handle = pool.handle()
    need = [ctxs[0].kv_block_attention_workspace(handle, 16, len(q), max(c)) for q, c in zip(qs, counts)]
    ws = [torch.empty(n, dtype=torch.uint8, device="cuda") for n in need]
    torch.cuda.synchronize()
    for j in range(20):
        for i, ctx in enumerate(ctxs):
            ctx.kv_block_attention_dev(handle, 0, qs[i].data_ptr(), 2048, 16, offs[i].data_ptr(), sts[i].data_ptr(), len(qs[i]), max(counts[i]), True, 0,
                                       0.0, outs[i][j].data_ptr(), 2048, ws[i].data_ptr(), need[i])
    for i, ctx in enumerate(ctxs):
        _done(ctx)
        want, tol = attention(pool, qs[i], start[i], counts[i])
        assert torch.all((outs[i][0].double() - want).abs() <= tol)
        for o in outs[i][1:]:
            assert torch.equal(o, outs[i][0])
        ctx.close()


class Server:
    """What a server runs for a step of its sequences, in all layers: pages for the new tokens, then for every layer rotary positions,
    the cache, attention. The next layer's rows are this one's output, so that a wrong layer shows in all behind it."""

    def __init__(self, stream, n_seq, most, layers=3, n_q=8, n_kv=2, d=64, page=16, n_pages=120, max_pages=30):
        self.ctx = yscv_b200.Context(0, stream=stream.cuda_stream)
        self.pool = Pool(self.ctx, layers, n_pages, n_kv, d, page, n_seq, max_pages)
        self.n_q, self.n_kv, self.d, self.most = n_q, n_kv, d, most
        self.rows = n_seq * most
        self.width = (n_q + 2 * n_kv) * d
        self.rope = yscv_b200.Rope(rotary_dim=d)
        self.handle = self.pool.handle()
        self.off, self.start, self.pos = (torch.zeros(n, dtype=torch.int32, device="cuda") for n in (n_seq + 1, n_seq, self.rows))
        self.qkv = torch.zeros(layers, self.rows, self.width, device="cuda")
        self.turned, self.out = torch.zeros_like(self.qkv), torch.zeros(layers, self.rows, n_q * d, device="cuda")
        self.work = torch.empty(self.ctx.kv_pages_workspace(self.handle), dtype=torch.uint8, device="cuda")
        self.ws = torch.empty(self.ctx.kv_block_attention_workspace(self.handle, n_q, self.rows, most), dtype=torch.uint8, device="cuda")
        torch.cuda.synchronize()

    def step(self):
        ctx, pool, d = self.ctx, self.pool, self.d
        ctx.kv_pages_extend_dev(self.handle, self.off.data_ptr(), self.rows, self.start.data_ptr(), self.pos.data_ptr(), self.work.data_ptr(),
                                self.work.numel())
        for layer in range(pool.layers):
            x, t = self.qkv[layer], self.turned[layer]
            ctx.rope_dev(x.data_ptr(), self.width, self.rows, self.n_q + self.n_kv, d, self.pos.data_ptr(), self.rope, t.data_ptr(), self.width)
            ctx.kv_block_append_dev(self.handle, layer, t[:, self.n_q * d:].data_ptr(), x[:, (self.n_q + self.n_kv) * d:].data_ptr(), self.width,
                                    self.off.data_ptr(), self.start.data_ptr(), self.most)
            ctx.kv_block_attention_dev(self.handle, layer, t.data_ptr(), self.width, self.n_q, self.off.data_ptr(), self.start.data_ptr(), self.rows,
                                       self.most, True, 0, 0.0, self.out[layer].data_ptr(), self.n_q * d, self.ws.data_ptr(), self.ws.numel())

    def check(self, counts, start):
        """This step's results against the definitions: rotary positions from fp64, the cache as it is now."""
        n_q, n_kv, d, n = self.n_q, self.n_kv, self.d, sum(counts)
        pos = np.concatenate([np.arange(s, s + m) if s >= 0 else np.full(m, -1) for s, m in zip(start, counts)]).astype(int)
        assert self.pos[:n].tolist() == pos.tolist() and torch.all(self.pos[n:] == -1) and self.start.tolist() == [s if m else -1 for s, m in zip(start, counts)]
        angle = torch.tensor(pos, device="cuda").double()[:, None, None] * torch.tensor(_frequencies(d, "none", 1.0)[0], device="cuda")
        for layer in range(self.pool.layers):
            x = self.qkv[layer, :n].double().view(n, -1, d)
            a, b = x[:, :n_q + n_kv, :d // 2], x[:, :n_q + n_kv, d // 2:]
            turned = torch.cat([a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin()], -1)
            got = self.turned[layer, :n].double().view(n, -1, d)[:, :n_q + n_kv]
            live = torch.tensor(pos >= 0, device="cuda")
            # two products, a sum and a sine to 2^-22 of values below 6
            assert float((got - turned)[live].abs().max()) < 12 * 2.0 ** -22
            row = 0
            for i, (s, m) in enumerate(zip(start, counts)):
                if s >= 0 and m:
                    for c, w in zip(self.pool.rows(i, s + m, layer), (got[row:row + m, n_q:], x[row:row + m, n_q + n_kv:])):
                        # a page's scale may grow once per later token of the page, half a step each time, of values below 6
                        assert float((c[s:] - w).abs().max()) < 16 * 0.5 * 6 / 127
                row += m
            want, tol = attention(self.pool, self.turned[layer, :n].view(n, -1, d)[:, :n_q], start, counts, layer=layer)
            out = self.out[layer, :n].view(n, n_q, d).double()
            assert torch.all(((out - want).abs() <= tol)[live])


def _plan(server, counts, g):
    """Lays out a step's rows; what runs next on another stream waits for it."""
    server.off.copy_(offsets(counts))
    server.qkv.copy_(torch.randn(server.qkv.shape, device="cuda", generator=g))
    torch.cuda.synchronize()


def test_a_server_s_steps():
    """Prompts, single tokens, drafts and their rejection, branches that share pages, an end, compaction, a prompt in the place that is free."""
    stream = torch.cuda.Stream()
    s = Server(stream, n_seq=4, most=70)
    g = torch.Generator(device="cuda").manual_seed(5)
    length = [0, 0, 0, 0]

    def go(counts):
        _plan(s, counts, g)
        s.step()
        _done(s.ctx)
        start = [n if m else -1 for n, m in zip(length, counts)]
        s.check(counts, start)
        for i, m in enumerate(counts):
            length[i] += m
        assert s.pool.length.tolist() == length

    def lists(call, *rows):
        rows = [i32(r) for r in rows]
        torch.cuda.synchronize()
        call(s.handle, *(r.data_ptr() for r in rows), len(rows[0]))
        _done(s.ctx)

    go([70, 33, 0, 1])
    for _ in range(3):
        go([1, 1, 0, 1])
    go([5, 4, 0, 70])                                  # drafts beside a piece of a prompt
    lists(s.ctx.kv_pages_trim_dev, [0, 1], [75, 36])   # of which some were wrong
    length[0], length[1] = 75, 36
    lists(s.ctx.kv_pages_fork_dev, [0], [2])           # another branch
    length[2] = 75
    for _ in range(18):
        go([1, 0, 1, 1])
    lists(s.ctx.kv_pages_trim_dev, [0], [0])           # the first one's end
    length[0] = 0
    s.ctx.kv_pages_compact_dev(s.handle, s.work.data_ptr(), s.work.numel())
    _done(s.ctx)
    used = int((s.pool.refs > 0).sum())
    assert torch.all(s.pool.refs[:used] > 0) and int(s.pool.table.max()) == used - 1
    go([64, 1, 1, 1])
    go([1, 1, 1, 1])
    s.ctx.close()


@pytest.mark.parametrize("most", [1, 40])
def test_a_captured_step_serves_sequences_as_they_grow(most):
    """One graph, replayed with other offsets and rows while an eager server does the same: bit for bit. Two graphs of one context, with
    the same workspaces, take turns."""
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    eager, captured = (Server(s, n_seq=3, most=most) for s in streams)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=streams[1], capture_error_mode="thread_local"):
            captured.step()
    g = torch.Generator(device="cuda").manual_seed(6)
    for t in range(24):
        counts = [1 + (t * 7 + i * 5) % most if (t + i) % 4 else 0 for i in range(3)]
        _plan(eager, counts, g)
        captured.off.copy_(eager.off)
        captured.qkv.copy_(eager.qkv)
        torch.cuda.synchronize()
        eager.step()
        with torch.cuda.stream(streams[1]):
            graphs[t % 2].replay()
        for s in (eager, captured):
            s.ctx.synchronize()
        assert eager.ctx.device_status() == captured.ctx.device_status()
        n = sum(counts)
        assert torch.equal(eager.start, captured.start) and torch.equal(eager.pos, captured.pos)
        assert torch.equal(eager.out[:, :n], captured.out[:, :n])
        for a, b in zip(eager.pool.state()[4:], captured.pool.state()[4:]):
            assert torch.equal(a, b)
    del graphs
    for s in (eager, captured):
        s.ctx.close()


def _refused(call, *codes):
    with pytest.raises(yscv_b200.YscvCudaError) as e:
        call()
    assert e.value.status in (codes or (-1, -3))


def refusals(ctx, dev="cuda"):
    """Every call that has to be refused, and nothing that is not."""
    pool = Pool(ctx, layers=2, n_pages=8, n_kv=2, d=64, page=16, n_seq=2, max_pages=4, dev=dev)
    good = pool.handle()
    f = torch.zeros(4096, device=dev)
    n = torch.zeros(64, dtype=torch.int32, device=dev)
    ws = torch.zeros(1 << 24, dtype=torch.uint8, device=dev)
    p, i, w = f.data_ptr(), n.data_ptr(), ws.data_ptr()
    big = 1 << 31

    def calls(h, layer=0, stride=512, k=p, v=p, off=i, start=i, most=1, n_q=4, q=p, out=p + 4096, rows=2, scale=0.0, space=w, size=1 << 24, pos=i, src=i,
              count=2, seqs=i):
        return dict(
            append=lambda: ctx.kv_block_append_dev(h, layer, k, v, stride, off, start, most),
            read=lambda: ctx.kv_block_read_dev(h, layer, off, start, most, k, v, stride),
            attend=lambda: ctx.kv_block_attention_dev(h, layer, q, stride, n_q, off, start, rows, most, True, 0, scale, out, stride, space, size),
            room=lambda: ctx.kv_block_attention_workspace(h, n_q, rows, most),
            work=lambda: ctx.kv_pages_workspace(h),
            extend=lambda: ctx.kv_pages_extend_dev(h, off, rows, start, pos, space, size),
            trim=lambda: ctx.kv_pages_trim_dev(h, seqs, None, count),
            fork=lambda: ctx.kv_pages_fork_dev(h, src, seqs, count),
            compact=lambda: ctx.kv_pages_compact_dev(h, space, size),
            copy=lambda: ctx.kv_pages_copy_dev(h, src, seqs, count))

    def refuse(names, *codes, **change):
        for name in names.split():
            _refused(calls(good, **change)[name], *codes)

    every = "append read attend room work extend trim fork compact copy"
    for change in (dict(d_k=None), dict(d_v=None), dict(d_kscale=None), dict(d_vscale=None), dict(d_refs=None), dict(d_table=None), dict(d_length=None),
                   dict(layers=0), dict(n_pages=0), dict(n_kv=0), dict(d_head=0), dict(n_seq=0), dict(max_pages=0), dict(page=8), dict(page=48), dict(page=256),
                   dict(d_head=40), dict(d_head=272), dict(n_pages=1 << 30), dict(n_seq=1 << 20), dict(max_pages=1 << 24), dict(n_kv=1 << 16),
                   dict(d_k=pool.k.data_ptr() + 8), dict(d_v=pool.v.data_ptr() + 1), dict(d_kscale=pool.ks.data_ptr() + 2), dict(d_refs=pool.refs.data_ptr() + 1),
                   dict(d_table=pool.table.data_ptr() + 3), dict(d_length=pool.length.data_ptr() + 2)):
        bad = calls(pool.handle(**change))
        for name in every.split():
            _refused(bad[name])
    refuse("append read attend", -1, layer=2)
    refuse("append read attend", -1, stride=127)
    refuse("append read", k=None)
    refuse("append read", v=None)
    refuse("append read", -3, k=p + 2)
    refuse("append read", -3, v=p + 1)
    refuse("append read attend extend", -1, off=None)
    refuse("append read attend extend", -1, start=None)
    refuse("append read attend extend", -3, off=i + 2)
    refuse("append read attend extend", -3, start=i + 1)
    refuse("append read attend room", most=big)
    refuse("attend room", -1, n_q=0)
    refuse("attend room", -1, n_q=3)
    refuse("attend room", -3, n_q=65536)
    refuse("attend room", -3, rows=big // 4)
    refuse("extend", -3, rows=big)
    refuse("attend", -1, q=None)
    refuse("attend", -1, out=None)
    refuse("attend", -1, out=p)
    refuse("attend", -3, q=p + 1)
    refuse("attend", -3, out=p + 4098)
    for scale in (-1.0, math.inf, math.nan):
        refuse("attend", -1, scale=scale)
    refuse("attend extend compact", -1, space=None)
    refuse("attend extend compact", -1, size=8)
    refuse("attend", -3, space=w + 8)
    refuse("extend compact", -3, space=w + 2)
    refuse("extend", -1, pos=None)
    refuse("extend", -3, pos=i + 1)
    refuse("trim fork copy", -1, seqs=None)
    refuse("trim fork copy", -3, seqs=i + 2)
    refuse("fork copy", -1, src=None)
    refuse("fork copy", -3, src=i + 2)
    refuse("trim fork copy", -3, count=1 << 30)
    for change in (dict(d_head=48), dict(d_head=16), dict(d_head=192)):
        for name in ("attend", "room"):
            _refused(calls(pool.handle(**change))[name], -3)
    _refused(calls(pool.handle(n_seq=100000, max_pages=16), n_q=2)["room"], -3)

    def rope(x=p, stride=512, rows=2, heads=4, d=64, pos=i, out=p, out_stride=512, **fields):
        r = yscv_b200.Rope(**{"rotary_dim": 64, **fields})
        return lambda: ctx.rope_dev(x, stride, rows, heads, d, pos, r, out, out_stride)

    for change in (dict(x=None), dict(pos=None), dict(out=None), dict(x=p + 2), dict(pos=i + 1), dict(out=p + 4098), dict(stride=255), dict(out_stride=255),
                   dict(out_stride=516), dict(rows=big), dict(heads=0), dict(d=0), dict(rotary_dim=0), dict(rotary_dim=63), dict(rotary_dim=66),
                   dict(heads=1, d=600, stride=600, out_stride=600, rotary_dim=600), dict(theta=1.0), dict(theta=math.nan), dict(theta=math.inf),
                   dict(scaling="linear", factor=0.5), dict(scaling="linear", factor=math.nan), dict(scaling="banded", factor=8.0, original_positions=0.0),
                   dict(scaling="banded", factor=8.0, original_positions=64.0, low_band=4.0, high_band=1.0),
                   dict(scaling="yarn", factor=8.0, original_positions=64.0, beta_fast=1.0, beta_slow=32.0), dict(attention_factor=-1.0),
                   dict(attention_factor=math.inf)):
        _refused(rope(**change))
    return pool, calls, rope


def test_refusals():
    ctx = _context()
    torch.cuda.synchronize()
    pool, calls, rope = refusals(ctx)
    before = pool.state()
    # nothing to do is no error, whatever else is missing
    rope(rows=0, x=None, pos=None, out=None)()
    for name in ("trim", "fork", "copy"):
        calls(pool.handle(), count=0, seqs=None, src=None)[name]()
    calls(pool.handle(), rows=0)["attend"]()
    _done(ctx)
    for a, b in zip(pool.state(), before):
        assert torch.equal(a, b)
    ctx.close()
