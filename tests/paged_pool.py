"""A paged int8 KV cache for the tests: its arrays, what they hold, and the operators' definitions in 64 bits."""
import math

import numpy as np
import torch

import yscv_b200

LEAST = 2.0 ** -100


class Pool:
    def __init__(self, ctx, layers=1, n_pages=12, n_kv=2, d=64, page=16, n_seq=3, max_pages=6, seed=0, dev="cuda"):
        self.ctx, self.layers, self.n_pages, self.n_kv, self.d, self.page = ctx, layers, n_pages, n_kv, d, page
        self.n_seq, self.max_pages, self.dev = n_seq, max_pages, dev
        g = torch.Generator(device=dev)
        g.manual_seed(seed)
        self.g = g
        self.k = torch.randint(-127, 128, (layers, n_pages, n_kv, page // 16, d // 16, 16, 16), dtype=torch.int8, device=dev, generator=g)
        self.v = torch.randint(-127, 128, (layers, n_pages, n_kv, page // 16, d, 16), dtype=torch.int8, device=dev, generator=g)
        self.ks, self.vs = (0.01 + 0.02 * torch.rand(layers, n_pages, n_kv, device=dev, generator=g) for _ in range(2))
        self.refs = torch.zeros(n_pages, dtype=torch.int32, device=dev)
        self.table = torch.full((n_seq, max_pages), -1, dtype=torch.int32, device=dev)
        self.length = torch.zeros(n_seq, dtype=torch.int32, device=dev)

    def handle(self, **change):
        f = dict(d_k=self.k.data_ptr(), d_v=self.v.data_ptr(), d_kscale=self.ks.data_ptr(), d_vscale=self.vs.data_ptr(), layers=self.layers,
                 n_pages=self.n_pages, n_kv=self.n_kv, d_head=self.d, page=self.page, d_refs=self.refs.data_ptr(),
                 d_table=self.table.data_ptr(), d_length=self.length.data_ptr(), n_seq=self.n_seq, max_pages=self.max_pages)
        f.update(change)
        return yscv_b200.KvPool(**f)

    def give(self, tokens, seed=1):
        """Pages in no order for so many tokens of every sequence."""
        order = torch.randperm(self.n_pages, generator=torch.Generator().manual_seed(seed)).tolist()
        table = torch.full((self.n_seq, self.max_pages), -1, dtype=torch.int32)
        refs = torch.zeros(self.n_pages, dtype=torch.int32)
        for i, n in enumerate(tokens):
            for c in range(-(-n // self.page)):
                p = order.pop()
                table[i, c], refs[p] = p, 1
        self.table.copy_(table)
        self.refs.copy_(refs)
        self.length.copy_(torch.tensor(tokens, dtype=torch.int32))

    def rows(self, seq, count, layer=0):
        """The first `count` cached rows of a sequence: keys and values, float64 [count][n_kv][d]."""
        t = torch.arange(count, device=self.dev)
        pages, at = self.table[seq].long()[t // self.page], t % self.page
        h, j = torch.arange(self.n_kv, device=self.dev)[None, :, None], torch.arange(self.d, device=self.dev)[None, None, :]
        p3, g3, a3 = pages[:, None, None], (at // 16)[:, None, None], (at % 16)[:, None, None]
        k = self.k[layer][p3, h, g3, j // 16, a3, j % 16].double() * self.ks[layer][pages][..., None].double()
        v = self.v[layer][p3, h, g3, j, a3].double() * self.vs[layer][pages][..., None].double()
        return k, v

    def state(self):
        return [t.clone() for t in (self.k, self.v, self.ks, self.vs, self.refs, self.table, self.length)]

    def restore(self, state):
        for t, s in zip((self.k, self.v, self.ks, self.vs, self.refs, self.table, self.length), state):
            t.copy_(s)


def i32(values, dev="cuda"):
    return torch.tensor(list(values), dtype=torch.int32, device=dev)


def offsets(counts, dev="cuda"):
    return i32(np.concatenate([[0], np.cumsum(counts)]).tolist(), dev)


def attention(pool, q, start, counts, causal=True, window=0, scale=0.0, layer=0):
    """float64 result [rows][n_q][d] and a bound on every value's error, from q [rows][n_q][d].

    The bound: a query is off by at most 2^-24 of its row's largest magnitude (24-bit whole numbers), a score by that times the
    keys plus 4 fp32 roundings and the rounding of its place in the exponent, a weight by its score's error, 2^-22 of the
    exponential and 2^-24 of the largest weight of its 64 keys (64 of them: 2^-18), sums over n steps of 64 keys by n + 4 roundings.
    A weight's relative error reaches the result once through the weighted sum and once through the normalisation."""
    n_q, d, n_kv = q.shape[1], q.shape[2], pool.n_kv
    scale = scale or 1.0 / math.sqrt(d)
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    tol = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    row = 0
    for i, (s0, m) in enumerate(zip(start, counts)):
        if s0 < 0 or m == 0:
            row += m
            continue
        k, v = pool.rows(i, s0 + m, layer)
        here, key = torch.arange(s0, s0 + m, device=q.device)[:, None], torch.arange(s0 + m, device=q.device)[None, :]
        hidden = (key > here) if causal else torch.zeros_like(key > here)
        if window:
            hidden = hidden | (key <= here - window)
        for h in range(n_q):
            x, kh, vh = q[row:row + m, h].double(), k[:, h // (n_q // n_kv)], v[:, h // (n_q // n_kv)]
            score = (x @ kh.T * scale).masked_fill(hidden, -math.inf)
            p = torch.softmax(score, -1)
            out[row:row + m, h] = p @ vh
            off = x.abs().amax(-1, keepdim=True) * kh.abs().sum(-1).max() * scale * 2.0 ** -24
            size = score.masked_fill(hidden, 0.0).abs().amax(-1, keepdim=True)
            steps = (s0 + m) / 64 + 1
            tol[row:row + m, h] = (2 * (off + size * 2.0 ** -21) + 2.0 ** -18 + 2.0 ** -21 + (steps + 4) * 2.0 ** -23) * vh.abs().max()
        row += m
    return out, tol


def appended(old_q, old_s, held, rows):
    """One block (a page's head): whole numbers [tokens][d] and scale after `rows` [n][d] float32 are put behind `held` tokens."""
    rows = rows.astype(np.float32)
    finite = np.where(np.isfinite(rows), np.abs(rows), np.float32(0))
    s = np.float32(max(np.float32(finite.max()), np.float32(LEAST)) / np.float32(127))
    old = old_q.astype(np.float64)
    if held:
        if s > old_s:
            old = np.rint(old * float(old_s) / float(s))
        else:
            s = np.float32(old_s)
    with np.errstate(invalid="ignore"):
        new = np.clip(np.rint(rows.astype(np.float64) / float(s)), -127, 127)
    new[np.isnan(rows)] = 0
    return np.concatenate([old[:held], new]).astype(np.int8), s
