"""Operators of a server that decodes many conversations at once, over a paged 8-bit KV cache, with their plain forms.

The cache holds int8 in pages. A page is a block of ``page`` consecutive tokens of one conversation, and every page has one
fp32 scale for each KV head, keys and values apart. Tokens lie in groups of 16, the way the tensor cores take them:

    keys    [layers][n_pages][n_kv][page / 16][d / 16][16 tokens][16 d]
    values  [layers][n_pages][n_kv][page / 16][d][16 tokens]
    scales  [layers][n_pages][n_kv]

A scale is the fp32 number nearest to the block's largest magnitude / 127, a value is held as the whole number nearest to its
quotient by the scale (the even one of two). Where new tokens make a block's scale grow, what it holds is rounded again.
``table`` [n_seq][max_pages] says which pages a conversation has (-1: none), ``length`` [n_seq] how many tokens,
``refs`` [n_pages] how many conversations share a page (0: free). The rows of a call are ragged: conversation i has the rows
offsets[i] .. offsets[i + 1] - 1, at positions start[i], start[i] + 1, ...

Kinds of case:

- ``rope``: rotary positions of the query and key heads of fused [q | k | v] rows.
- ``append``: new keys and values into the pages, read back as the values the touched pages then stand for.
- ``attend``: attention of the new rows over everything cached so far.
- ``beam``: drop the old branches of every search, fork its parent, give every branch room for a token.
- ``turnover``: half of the conversations end, what is left moves together, as many new ones begin.
"""
from __future__ import annotations

import math

import torch

own = False

LEAST = 2.0 ** -100          # the smallest magnitude a block is scaled to
BETA_FAST, BETA_SLOW, LOW_BAND, HIGH_BAND = 32.0, 1.0, 1.0, 4.0


def listed():
    return [
        # a decode step of eight conversations with a 1B decoder: launch latency
        {"name": "rope_step_8", "kind": "rope", "rows": 8, "n_q": 32, "n_kv": 4, "d": 64, "rot": 64, "interleaved": False,
         "scaling": "none", "factor": 1.0, "far": 2048},
        # a prompt at the 70B head shape: pairs side by side, part of the head, stretched to a million positions
        {"name": "rope_prompt_4099", "kind": "rope", "rows": 4099, "n_q": 64, "n_kv": 8, "d": 128, "rot": 96,
         "interleaved": True, "scaling": "yarn", "factor": 32.0, "far": 1 << 20},
        # a decode step of a full server batch at the 70B head shape
        {"name": "append_step_64", "kind": "append", "n_seq": 64, "n_kv": 8, "d": 128, "page": 64, "cached_lo": 1000,
         "cached_hi": 8000, "new_lo": 1, "new_hi": 1},
        # prompts of four conversations, most of them behind earlier turns
        {"name": "append_prompt_4", "kind": "append", "n_seq": 4, "n_kv": 8, "d": 128, "page": 32, "cached_lo": 0,
         "cached_hi": 99, "new_lo": 501, "new_hi": 1500},
        # one conversation with a 1B decoder, shortly after its prompt
        {"name": "attend_step_1x200", "kind": "attend", "n_seq": 1, "n_q": 32, "n_kv": 4, "d": 64, "page": 16,
         "cached_lo": 200, "cached_hi": 200, "new_lo": 1, "new_hi": 1, "causal": True, "window": 0},
        # a full server batch at the 70B head shape, conversations of very different lengths
        {"name": "attend_step_64", "kind": "attend", "n_seq": 64, "n_q": 64, "n_kv": 8, "d": 128, "page": 64,
         "cached_lo": 1000, "cached_hi": 8000, "new_lo": 1, "new_hi": 1, "causal": True, "window": 0},
        # one conversation over a very long document
        {"name": "attend_step_131k", "kind": "attend", "n_seq": 1, "n_q": 64, "n_kv": 8, "d": 128, "page": 128,
         "cached_lo": 131000, "cached_hi": 131000, "new_lo": 1, "new_hi": 1, "causal": True, "window": 0},
        # a drafted continuation is checked: five tokens at once
        {"name": "attend_draft_8x5", "kind": "attend", "n_seq": 8, "n_q": 32, "n_kv": 4, "d": 64, "page": 32,
         "cached_lo": 3001, "cached_hi": 4003, "new_lo": 5, "new_hi": 5, "causal": True, "window": 0},
        # a prompt on an empty cache
        {"name": "attend_prompt_2047", "kind": "attend", "n_seq": 1, "n_q": 64, "n_kv": 8, "d": 128, "page": 64,
         "cached_lo": 0, "cached_hi": 0, "new_lo": 2047, "new_hi": 2047, "causal": True, "window": 0},
        # pieces of three prompts over what is cached of them, each token sees the last 4096
        {"name": "attend_chunk_3", "kind": "attend", "n_seq": 3, "n_q": 32, "n_kv": 4, "d": 128, "page": 64,
         "cached_lo": 2000, "cached_hi": 8000, "new_lo": 17, "new_hi": 511, "causal": True, "window": 4096},
        # sixteen searches with four branches each, one step
        {"name": "beam_16x4", "kind": "beam", "n_seq": 64, "width": 4, "layers": 22, "n_kv": 4, "d": 64, "page": 16,
         "lo": 100, "hi": 2000},
        # a full server: half of its conversations end
        {"name": "turnover_128", "kind": "turnover", "n_seq": 128, "width": 1, "layers": 16, "n_kv": 8, "d": 128, "page": 64,
         "lo": 100, "hi": 1000},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rope", "append", "append", "attend", "attend", "attend", "attend", "beam", "turnover"])
    d = rng.choice([64, 64, 128, 128, 128, 256])
    n_kv, group = rng.choice([1, 2, 4, 8, 8]), rng.choice([1, 3, 4, 6, 8, 8, 16])
    page = rng.choice([16, 32, 64, 64, 128])
    if kind == "rope":
        scaling = rng.choice(["none", "none", "linear", "banded", "yarn"])
        return {"kind": kind, "rows": _log(rng, 1, 4099 * 9216 // ((n_kv * group + n_kv) * d) // 2), "n_q": n_kv * group,
                "n_kv": n_kv, "d": d, "rot": rng.choice([d, d, d // 2, d // 4, d - 2]), "interleaved": rng.random() < 0.5,
                "scaling": scaling, "factor": 1.0 if scaling == "none" else rng.choice([2.0, 8.0, 32.0]),
                "far": _log(rng, 64, 1 << 20)}
    if kind in ("append", "attend"):
        base = {"kind": kind, "n_kv": n_kv, "d": d, "page": page}
        if kind == "attend":
            base["n_q"] = n_kv * group
        form = rng.choice(["step", "step", "draft", "prompt"])
        if form == "prompt":
            new = _log(rng, 6, 2047)
            n_seq = _log(rng, 1, max(1, min(16, 2047 // new)))
            cached = 0 if rng.random() < 0.4 else _log(rng, 16, 6000)
            if kind == "attend":  # no more than the largest listed work
                while n_seq * new * (cached + new) * n_kv * group * d > 2047 * 1000 * 64 * 128:
                    cached, new = cached // 2, max(1, new * 3 // 4)
            lens = (cached // 2, cached, (new + 1) // 2, new)
        else:
            new = 1 if form == "step" else rng.randint(2, 8)
            n_seq, hi = _log(rng, 1, 128), _log(rng, 16, 65536)
            while n_seq * (hi + new) * n_kv * d > 64 * 4500 * 8 * 128 or n_seq * hi * new * n_kv * group > 64 * 4500 * 64 * 2:
                n_seq, hi = max(1, n_seq * 3 // 4), max(1, hi * 3 // 4)
            lens = (rng.choice([hi, max(1, hi // 8)]), hi, new, new)
        base.update(n_seq=n_seq, cached_lo=lens[0], cached_hi=lens[1], new_lo=lens[2], new_hi=lens[3])
        if kind == "attend":
            base.update(causal=rng.random() < 0.85, window=rng.choice([0, 0, 0, _log(rng, 8, 4096)]))
        return base
    n_seq, hi, layers = 2 * _log(rng, 2, 64), _log(rng, 8, 2000), rng.randint(1, 22)
    width = rng.choice([2, 4]) if kind == "beam" else 1
    n_seq = max(width, n_seq // width * width)
    while n_seq * (hi + 2 * page) * layers * n_kv * d > 128 * 600 * 16 * 8 * 128:
        hi, layers = max(2, hi // 2), max(1, layers * 3 // 4)
    return {"kind": kind, "n_seq": n_seq, "width": width, "layers": layers, "n_kv": n_kv, "d": d, "page": page,
            "lo": max(1, hi // 10), "hi": hi}


# ---- inputs ------------------------------------------------------------------------------------------

def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _spread(lo, hi, n):
    """n lengths from lo to hi in no order."""
    return [hi if n == 1 else lo + int((hi - lo) * ((0.5 + 0.6180339887 * i) % 1.0) + 0.5) for i in range(n)]


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _ceil(a, b):
    return -(-a // b)


def _offsets(counts):
    at = [0]
    for c in counts:
        at.append(at[-1] + c)
    return at


def _pool(case, g, layers, n_pages, n_seq, max_pages):
    n_kv, d, page = case["n_kv"], case["d"], case["page"]
    k = torch.empty(layers, n_pages, n_kv, page // 16, d // 16, 16, 16, dtype=torch.int8, device="cuda")
    v = torch.empty(layers, n_pages, n_kv, page // 16, d, 16, dtype=torch.int8, device="cuda")
    for t in (k, v):
        for layer in range(layers):  # what rows of normal values quantise to, the largest of a block at 127
            t[layer] = torch.empty(t.shape[1:], device="cuda").normal_(0.0, 36.0, generator=g).round_().clamp_(-127, 127).to(torch.int8)
    ks, vs = (torch.exp(torch.randn(layers, n_pages, n_kv, device="cuda", generator=g) * 0.3) / 36.0 for _ in range(2))
    return {"k": k, "v": v, "ks": ks, "vs": vs, "refs": torch.zeros(n_pages, dtype=torch.int32, device="cuda"),
            "table": torch.full((n_seq, max_pages), -1, dtype=torch.int32, device="cuda"),
            "length": torch.zeros(n_seq, dtype=torch.int32, device="cuda"), "page": page}


def _give(pool, pages, owners):
    """owners[i] gets the next counts of the list `pages`."""
    table = pool["table"].cpu()
    at = 0
    for slot, count in owners:
        table[slot, :count] = pages[at:at + count]
        at += count
    pool["table"].copy_(table)
    pool["refs"][pages[:at].long().cuda()] = 1


def prepare(case, seed):
    g = _generator(seed)
    state = {"rope": _prepare_rope, "append": _prepare_rows, "attend": _prepare_rows, "beam": _prepare_beam,
             "turnover": _prepare_turnover}[case["kind"]](case, g, seed)
    state["case"] = case
    if own:  # the handle and the workspace that a program keeps
        _bind(state)
    return state


def _prepare_rope(case, g, _):
    heads, d, rows = case["n_q"] + 2 * case["n_kv"], case["d"], case["rows"]
    return {"qkv": torch.randn(rows, heads * d, device="cuda", generator=g),
            "pos": torch.randint(0, case["far"], (rows,), dtype=torch.int32, device="cuda", generator=g),
            "out": torch.empty(rows, (case["n_q"] + case["n_kv"]) * d, device="cuda")}


def _counts(case):
    n = case["n_seq"]
    return _spread(case["cached_lo"], case["cached_hi"], n), _spread(case["new_lo"], case["new_hi"], n)


def _prepare_rows(case, g, seed):
    n_seq, n_kv, d, page = case["n_seq"], case["n_kv"], case["d"], case["page"]
    cached, new = _counts(case)
    held = [_ceil(c + m, page) for c, m in zip(cached, new)]
    order = torch.randperm(sum(held) + 3, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    pool = _pool(case, g, 1, len(order), n_seq, max(held) + 1)
    _give(pool, order, list(enumerate(held)))
    pool["length"].copy_(_i32([c + m for c, m in zip(cached, new)]))
    rows = sum(new)
    s = {"pool": pool, "offsets": _i32(_offsets(new)), "start": _i32(cached), "rows": rows, "most": max(new)}
    if case["kind"] == "append":
        kv = torch.randn(rows, 2 * n_kv * d, device="cuda", generator=g)
        kv *= torch.exp(0.3 * torch.randn(rows, 1, device="cuda", generator=g))
        touched = [c % page + m for c, m in zip(cached, new)]  # from the first token of the first page
        s.update(kv=kv, read_offsets=_i32(_offsets(touched)), read_start=_i32([c - c % page for c in cached]),
                 read_most=max(touched), k_out=torch.empty(sum(touched), n_kv * d, device="cuda"),
                 v_out=torch.empty(sum(touched), n_kv * d, device="cuda"))
    else:
        q = torch.randn(rows, (case["n_q"] + 2 * n_kv) * d, device="cuda", generator=g)
        s.update(q=q * torch.exp(0.5 * torch.randn(rows, 1, device="cuda", generator=g)),
                 out=torch.empty(rows, case["n_q"] * d, device="cuda"))
    return s


def _prepare_beam(case, g, seed):
    n_seq, width, page = case["n_seq"], case["width"], case["page"]
    lens = _spread(case["lo"], case["hi"], n_seq // width)
    held = [_ceil(n, page) for n in lens]
    n_pages = sum(held) + 2 * n_seq + 8
    order = torch.randperm(n_pages, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    pool = _pool(case, g, case["layers"], n_pages, n_seq, max(held) + 2)
    _give(pool, order, [(i * width, h) for i, h in enumerate(held)])
    keep = [lens[i // width] if i % width == 0 else 0 for i in range(n_seq)]
    pool["length"].copy_(_i32(keep))
    children = [i for i in range(n_seq) if i % width]
    return {"pool": pool, "slots": _i32(list(range(n_seq))), "keep": _i32(keep), "parents": _i32([i // width * width for i in children]),
            "children": _i32(children), "offsets": _i32(list(range(n_seq + 1))), "rows": n_seq,
            "start": torch.empty(n_seq, dtype=torch.int32, device="cuda"), "pos": torch.empty(n_seq, dtype=torch.int32, device="cuda")}


def _prepare_turnover(case, g, _):
    n_seq, page = case["n_seq"], case["page"]
    lens = _spread(case["lo"], case["hi"], n_seq)
    held = [_ceil(n, page) for n in lens]
    n_pages = sum(held) + 5
    pool = _pool(case, g, case["layers"], n_pages, n_seq, max(held) + 1)
    _give(pool, torch.arange(n_pages, dtype=torch.int32), list(enumerate(held)))
    pool["length"].copy_(_i32(lens))
    turns = []
    for half in (range(n_seq // 2), range(n_seq // 2, n_seq)):  # the half that lies lowest ends first
        new = [lens[i] if i in half else 0 for i in range(n_seq)]
        turns.append({"slots": _i32(list(half)), "offsets": _i32(_offsets(new)), "rows": sum(new),
                      "pos": torch.empty(sum(new), dtype=torch.int32, device="cuda")})
    return {"pool": pool, "turns": turns, "turn": 0, "start": torch.empty(n_seq, dtype=torch.int32, device="cuda")}


# ---- the framework's calls ----------------------------------------------------------------------------

_PROGRAM = {}


def _context():
    if not _PROGRAM:
        from yscv_b200 import Context
        _PROGRAM["stream"] = torch.cuda.Stream()
        _PROGRAM["ctx"] = Context(0, stream=_PROGRAM["stream"].cuda_stream)
    return _PROGRAM["ctx"]


def _bind(s):
    import yscv_b200
    ctx, case = _context(), s["case"]
    s["ctx"] = ctx
    if case["kind"] == "rope":
        s["rope"] = yscv_b200.Rope(theta=10000.0, rotary_dim=case["rot"], interleaved=case["interleaved"], scaling=case["scaling"],
                                   factor=case["factor"], original_positions=4096, beta_fast=BETA_FAST, beta_slow=BETA_SLOW,
                                   low_band=LOW_BAND, high_band=HIGH_BAND)
        return
    p = s["pool"]
    layers, n_pages, n_kv = p["ks"].shape
    n_seq, max_pages = p["table"].shape
    s["handle"] = yscv_b200.KvPool(
        d_k=p["k"].data_ptr(), d_v=p["v"].data_ptr(), d_kscale=p["ks"].data_ptr(), d_vscale=p["vs"].data_ptr(), layers=layers,
        n_pages=n_pages, n_kv=n_kv, d_head=case["d"], page=case["page"], d_refs=p["refs"].data_ptr(),
        d_table=p["table"].data_ptr(), d_length=p["length"].data_ptr(), n_seq=n_seq, max_pages=max_pages)
    if case["kind"] == "attend":
        s["bytes"] = ctx.kv_block_attention_workspace(s["handle"], case["n_q"], s["rows"], s["most"])
    elif case["kind"] != "append":
        s["bytes"] = ctx.kv_pages_workspace(s["handle"])
    if "bytes" in s:
        s["workspace"] = torch.empty(max(16, s["bytes"]), dtype=torch.uint8, device="cuda")


# ---- one pass -----------------------------------------------------------------------------------------

def run(state):
    kind = state["case"]["kind"]
    return {"rope": _rope, "append": _append, "attend": _attend, "beam": _beam, "turnover": _turnover}[kind](state)


def _frequencies(case):
    """Radians per position of every pair, and the factor on cosine and sine, in 64 bits."""
    rot, factor, theta, original = case["rot"], case["factor"], 10000.0, 4096.0
    i = torch.arange(rot // 2, dtype=torch.float64, device="cuda")
    freq = theta ** (-2.0 * i / rot)
    if case["scaling"] == "linear":
        return freq / factor, 1.0
    if case["scaling"] == "banded":  # long waves are stretched, short ones kept, those between blended
        turns = original * freq / (2.0 * math.pi)
        part = ((turns - LOW_BAND) / (HIGH_BAND - LOW_BAND)).clamp(0.0, 1.0)
        return freq * (part + (1.0 - part) / factor), 1.0
    if case["scaling"] == "yarn":
        low, high = (rot * math.log(original / (2.0 * math.pi * beta)) / (2.0 * math.log(theta)) for beta in (BETA_FAST, BETA_SLOW))
        low, high = max(math.floor(low), 0), min(math.ceil(high), rot - 1)
        part = 1.0 - ((i - low) / max(high - low, 0.001)).clamp(0.0, 1.0)
        return freq * (part + (1.0 - part) / factor), 0.1 * math.log(factor) + 1.0
    return freq, 1.0


def _rope(s):
    case = s["case"]
    heads, d, rot, rows = case["n_q"] + case["n_kv"], case["d"], case["rot"], case["rows"]
    if own:
        s["ctx"].rope_dev(s["qkv"].data_ptr(), s["qkv"].shape[1], rows, heads, d, s["pos"].data_ptr(), s["rope"], s["out"].data_ptr(),
                          heads * d)
        return s["out"]
    freq, factor = _frequencies(case)
    angle = s["pos"].double()[:, None] * freq
    cos, sin = ((f(angle) * factor).float()[:, None, :] for f in (torch.cos, torch.sin))
    x = s["qkv"][:, :heads * d].view(rows, heads, d)
    out = s["out"].view(rows, heads, d)
    if case["interleaved"]:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        out[..., 0:rot:2], out[..., 1:rot:2] = a * cos - b * sin, b * cos + a * sin
    else:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        out[..., :rot // 2], out[..., rot // 2:rot] = a * cos - b * sin, b * cos + a * sin
    out[..., rot:] = x[..., rot:]
    return s["out"]


def _places(pool, offsets, start, rows):
    """Sequence, position, page and place in the page of every row of a ragged call."""
    counts = (offsets[1:] - offsets[:-1]).long()
    seq = torch.repeat_interleave(torch.arange(len(counts), device="cuda"), counts, output_size=rows)
    pos = start.long()[seq] + torch.arange(rows, device="cuda") - offsets.long()[seq]
    return seq, pos, pool["table"][seq, pos // pool["page"]].long(), pos % pool["page"]


def _append(s):
    case, pool = s["case"], s["pool"]
    n_kv, d, page, rows = case["n_kv"], case["d"], case["page"], s["rows"]
    if own:
        at = s["kv"].data_ptr()
        s["ctx"].kv_block_append_dev(s["handle"], 0, at, at + 4 * n_kv * d, 2 * n_kv * d, s["offsets"].data_ptr(), s["start"].data_ptr(),
                                     s["most"])
        s["ctx"].kv_block_read_dev(s["handle"], 0, s["read_offsets"].data_ptr(), s["read_start"].data_ptr(), s["read_most"],
                                   s["k_out"].data_ptr(), s["v_out"].data_ptr(), n_kv * d)
        return s["k_out"], s["v_out"]
    seq, pos, pages, at = _places(pool, s["offsets"], s["start"], rows)
    head = torch.arange(n_kv, device="cuda")[None, :]
    first = s["start"].long()
    begun = (first % page != 0)[:, None]  # the page of the first new token holds older ones
    page0 = torch.gather(pool["table"].long(), 1, (first // page)[:, None])[:, 0].clamp_(min=0)
    for name, x in (("k", s["kv"][:, :n_kv * d]), ("v", s["kv"][:, n_kv * d:])):
        q8, scale = pool[name][0], pool[name + "s"][0]
        x = x.reshape(rows, n_kv, d)
        most = torch.zeros_like(scale).index_reduce_(0, pages, x.abs().amax(-1), "amax")
        step = (most.clamp_(min=LEAST).double() / 127.0).float()  # quotients in 64 bits: many lie next to a border
        old = scale[page0]
        now = torch.where(begun, torch.maximum(step[page0], old), step[page0])
        shape = (-1, n_kv) + (1,) * (q8.dim() - 2)
        held = q8[page0].double()
        q8[page0] = torch.where(begun.view((-1,) + shape[2:] + (1,)), torch.round(held * old.double().view(shape) / now.double().view(shape)), held).to(torch.int8)
        step[page0] = now
        scale[pages] = step[pages]
        values = torch.round(x.double() / step[pages].double()[..., None]).clamp_(-127, 127).to(torch.int8)
        if name == "k":
            q8[pages[:, None], head, (at // 16)[:, None], :, (at % 16)[:, None], :] = values.view(rows, n_kv, d // 16, 16)
        else:
            q8[pages[:, None], head, (at // 16)[:, None], :, (at % 16)[:, None]] = values
    rows = s["k_out"].shape[0]
    seq, pos, pages, at = _places(pool, s["read_offsets"], s["read_start"], rows)
    where = (pages[:, None], head, (at // 16)[:, None], slice(None), (at % 16)[:, None])
    s["k_out"].view(rows, n_kv, d).copy_(pool["k"][0][where].reshape(rows, n_kv, d) * pool["ks"][0][pages][..., None])
    s["v_out"].view(rows, n_kv, d).copy_(pool["v"][0][where] * pool["vs"][0][pages][..., None])
    return s["k_out"], s["v_out"]


def _attend(s):
    case, pool = s["case"], s["pool"]
    n_q, n_kv, d, page, rows = case["n_q"], case["n_kv"], case["d"], case["page"], s["rows"]
    if own:
        s["ctx"].kv_block_attention_dev(s["handle"], 0, s["q"].data_ptr(), s["q"].shape[1], n_q, s["offsets"].data_ptr(),
                                        s["start"].data_ptr(), rows, s["most"], case["causal"], case["window"], 0.0, s["out"].data_ptr(), n_q * d,
                                        s["workspace"].data_ptr(), s["bytes"])
        return s["out"]
    n_seq, most = case["n_seq"], s["most"]
    table = pool["table"].long().clamp_(min=0)
    keys = table.shape[1] * page
    k = pool["k"][0][table].permute(0, 1, 3, 5, 2, 4, 6).reshape(n_seq, -1, page, n_kv, d) * pool["ks"][0][table][:, :, None, :, None]
    v = pool["v"][0][table].permute(0, 1, 3, 5, 2, 4).reshape(n_seq, -1, page, n_kv, d) * pool["vs"][0][table][:, :, None, :, None]
    k, v = (t.reshape(n_seq, keys, n_kv, d) for t in (k, v))
    seq, pos, _, _ = _places(pool, s["offsets"], s["start"], rows)
    at = pos - s["start"].long()[seq]
    q = torch.zeros(n_seq, most, n_q, d, device="cuda")
    q[seq, at] = s["q"][:, :n_q * d].reshape(rows, n_q, d)
    score = torch.einsum("bshgd,bkhd->bhgsk", q.view(n_seq, most, n_kv, n_q // n_kv, d), k) * (1.0 / math.sqrt(d))
    new = (s["offsets"][1:] - s["offsets"][:-1]).long()
    here = s["start"].long()[:, None] + torch.arange(most, device="cuda")                     # position of every row
    last = here if case["causal"] else (s["start"].long() + new - 1)[:, None].expand_as(here)
    key = torch.arange(keys, device="cuda")
    seen = key <= last[..., None]
    if case["window"]:
        seen &= key > here[..., None] - case["window"]
    score.masked_fill_(~seen[:, None, None], -math.inf)
    weight = torch.exp(score - score.amax(-1, keepdim=True).clamp_(min=-3.0e38))
    total = weight.sum(-1, keepdim=True)
    weight /= torch.where(total > 0, total, torch.ones_like(total))
    out = torch.einsum("bhgsk,bkhd->bshgd", weight, v).reshape(n_seq, most, n_q * d)
    s["out"].copy_(out[seq, at])
    return s["out"]


def _pool_state(pool):
    """The whole of a pool; cached bytes and scales as whole numbers, since pages move as they are."""
    words = {n: pool[n].view(torch.int64) for n in ("k", "v")} | {n: pool[n].view(torch.int32) for n in ("ks", "vs")}
    return words | {n: pool[n] for n in ("refs", "table", "length")}


def _plain_trim(pool, slots, keep):
    slots = slots.long()
    column = torch.arange(pool["table"].shape[1], device="cuda")
    table = pool["table"][slots]
    length = torch.minimum(pool["length"][slots], keep)
    gone = (column >= ((length + pool["page"] - 1) // pool["page"])[:, None]) & (table >= 0)
    pool["refs"].index_add_(0, table[gone].long(), torch.full((1,), -1, dtype=torch.int32, device="cuda").expand(int(gone.sum())))
    pool["table"][slots] = table.masked_fill(gone, -1)
    pool["length"][slots] = length


def _plain_copy(pool, src, dst):
    for name in ("k", "v", "ks", "vs"):
        pool[name][:, dst] = pool[name][:, src]


def _plain_extend(pool, offsets, start, pos):
    page, refs, table, length = pool["page"], pool["refs"], pool["table"], pool["length"]
    n_seq, max_pages = table.shape
    new = offsets[1:] - offsets[:-1]
    held, wanted = (length + page - 1) // page, (length + new + page - 1) // page
    last = torch.gather(table.long(), 1, ((length - 1).clamp(min=0) // page).long()[:, None])[:, 0].clamp_(min=0)
    shared = (new > 0) & (length % page != 0) & (refs[last] > 1)
    need = torch.where((new > 0) & (wanted <= max_pages), wanted - held + shared, torch.zeros_like(new)).long()
    free = (refs == 0).nonzero()[:, 0]
    upto = need.cumsum(0)
    ok = (new > 0) & (wanted <= max_pages) & ((need == 0) | (upto <= len(free)))
    shared &= ok
    first = upto - need
    column = torch.arange(max_pages, device="cuda")
    fresh = (column >= held[:, None]) & (column < wanted[:, None]) & ok[:, None]
    index = first[:, None] + shared[:, None].long() + column - held[:, None]
    copy_src, copy_dst = last[shared], free[first[shared]]
    _plain_copy(pool, copy_src, copy_dst)
    given = torch.cat([free[index[fresh]], copy_dst])
    table[fresh] = free[index[fresh]].to(torch.int32)
    table[shared, (held[shared] - 1).long()] = copy_dst.to(torch.int32)
    refs.index_add_(0, copy_src, torch.full_like(copy_src, -1, dtype=torch.int32))
    refs[given] = 1
    start.copy_(torch.where(ok, length, torch.full_like(length, -1)))
    counts = new.long()
    seq = torch.repeat_interleave(torch.arange(n_seq, device="cuda"), counts, output_size=len(pos))
    at = start[seq] + (torch.arange(len(pos), device="cuda") - offsets.long()[seq]).to(torch.int32)
    pos.copy_(torch.where(ok[seq], at, torch.full_like(at, -1)))
    length += torch.where(ok, new, torch.zeros_like(new))


def _beam(s):
    pool = s["pool"]
    if own:
        ctx, handle, count = s["ctx"], s["handle"], len(s["children"])
        ctx.kv_pages_trim_dev(handle, s["slots"].data_ptr(), s["keep"].data_ptr(), len(s["slots"]))
        ctx.kv_pages_fork_dev(handle, s["parents"].data_ptr(), s["children"].data_ptr(), count)
        ctx.kv_pages_extend_dev(handle, s["offsets"].data_ptr(), s["rows"], s["start"].data_ptr(), s["pos"].data_ptr(),
                                s["workspace"].data_ptr(), s["bytes"])
        return _pool_state(pool) | {"start": s["start"], "pos": s["pos"]}
    _plain_trim(pool, s["slots"], s["keep"])
    parents, children = s["parents"].long(), s["children"].long()
    table = pool["table"][parents]
    pool["table"][children] = table
    pool["length"][children] = pool["length"][parents]
    held = table[table >= 0].long()
    pool["refs"].index_add_(0, held, torch.ones_like(held, dtype=torch.int32))
    _plain_extend(pool, s["offsets"], s["start"], s["pos"])
    return _pool_state(pool) | {"start": s["start"], "pos": s["pos"]}


def _turnover(s):
    pool, turn = s["pool"], s["turns"][s["turn"]]
    s["turn"] ^= 1
    if own:
        ctx, handle = s["ctx"], s["handle"]
        ctx.kv_pages_trim_dev(handle, turn["slots"].data_ptr(), None, len(turn["slots"]))
        ctx.kv_pages_compact_dev(handle, s["workspace"].data_ptr(), s["bytes"])
        ctx.kv_pages_extend_dev(handle, turn["offsets"].data_ptr(), turn["rows"], s["start"].data_ptr(), turn["pos"].data_ptr(),
                                s["workspace"].data_ptr(), s["bytes"])
        return _pool_state(pool) | {"start": s["start"], "pos": turn["pos"]}
    _plain_trim(pool, turn["slots"], torch.zeros_like(turn["slots"]))
    used = pool["refs"] > 0
    count = used.sum()
    page = torch.arange(len(used), device="cuda")
    src, dst = (used & (page >= count)).nonzero()[:, 0], (~used & (page < count)).nonzero()[:, 0]
    _plain_copy(pool, src, dst)
    moved = page.to(torch.int32)
    moved[src] = dst.to(torch.int32)
    pool["table"].copy_(torch.where(pool["table"] >= 0, moved[pool["table"].long().clamp_(min=0)], pool["table"]))
    pool["refs"][dst] = pool["refs"][src]
    pool["refs"][src] = 0
    _plain_extend(pool, turn["offsets"], s["start"], turn["pos"])
    return _pool_state(pool) | {"start": s["start"], "pos": turn["pos"]}


# ---- what a pass cannot do without ----------------------------------------------------------------------

def work(case):
    kind, n_kv, d = case["kind"], case["n_kv"], case["d"]
    if kind == "rope":
        heads = case["n_q"] + n_kv
        return {"bytes": case["rows"] * (8 * heads * d + 4), "flops": 3.0 * case["rows"] * heads * case["rot"]}
    page = case["page"]
    if kind == "append":
        cached, new = _counts(case)
        touched = [c % page + m for c, m in zip(cached, new)]
        return {"bytes": 2 * n_kv * d * (5 * sum(new) + 5 * sum(touched)), "flops": 6.0 * n_kv * d * sum(new)}
    if kind == "attend":
        cached, new = _counts(case)
        keys = pairs = 0
        for c, m in zip(cached, new):
            w = case["window"]
            spans = [((p + 1 if case["causal"] else c + m), max(0, p + 1 - w) if w else 0) for p in (c, c + m - 1)]
            keys += spans[1][0] - spans[0][1]
            pairs += sum((p + 1 if case["causal"] else c + m) - (max(0, p + 1 - w) if w else 0) for p in range(c, c + m))
        return {"bytes": 2 * n_kv * keys * (d + 4 / page) + 8 * case["n_q"] * d * sum(new), "flops": 4.0 * case["n_q"] * d * pairs}
    content = case["layers"] * n_kv * (2 * page * d + 8)  # bytes of a page
    if kind == "beam":
        lens = _spread(case["lo"], case["hi"], case["n_seq"] // case["width"])
        copies = sum(1 + case["width"] for n in lens if n % page)
        return {"bytes": copies * content + 8 * case["n_seq"], "flops": 0.0}
    held = [_ceil(n, page) for n in _spread(case["lo"], case["hi"], case["n_seq"])]
    half = case["n_seq"] // 2
    return {"bytes": 2 * min(sum(held[:half]), sum(held[half:])) * content + 8 * sum(held), "flops": 0.0}


# ---- the definitions in 64 bits --------------------------------------------------------------------------

def exact(case, seed):
    """Loops over rows' owners and heads, from the definitions; pages as such have nothing to compute."""
    if case["kind"] == "rope":
        s = prepare(case, seed)
        return _exact_rope(case, s)
    if case["kind"] == "append":
        return _exact_append(case, prepare(case, seed))
    if case["kind"] == "attend":
        return _exact_attend(case, prepare(case, seed))
    return None


def _exact_rope(case, s):
    heads, d, rot = case["n_q"] + case["n_kv"], case["d"], case["rot"]
    out = s["qkv"][:, :heads * d].double().view(-1, heads, d).clone()
    scale = 1.0
    for i in range(rot // 2):
        w = 1.0 / 10000.0 ** (2.0 * i / rot)
        if case["scaling"] == "linear":
            w = w / case["factor"]
        elif case["scaling"] == "banded":
            wave = 2.0 * math.pi / w
            if wave > 4096.0 / LOW_BAND:
                w = w / case["factor"]
            elif wave > 4096.0 / HIGH_BAND:
                smooth = (4096.0 / wave - LOW_BAND) / (HIGH_BAND - LOW_BAND)
                w = (1.0 - smooth) * w / case["factor"] + smooth * w
        elif case["scaling"] == "yarn":
            scale = 0.1 * math.log(case["factor"]) + 1.0
            low = max(0, math.floor(rot / 2.0 * math.log(4096.0 / (BETA_FAST * 2.0 * math.pi)) / math.log(10000.0)))
            high = min(rot - 1, math.ceil(rot / 2.0 * math.log(4096.0 / (BETA_SLOW * 2.0 * math.pi)) / math.log(10000.0)))
            ramp = min(1.0, max(0.0, (i - low) / (high - low if high > low else 0.001)))
            w = ramp * w / case["factor"] + (1.0 - ramp) * w
        a, b = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + rot // 2)
        turn = torch.polar(torch.full_like(s["pos"], 1, dtype=torch.float64) * scale, s["pos"].double() * w)
        z = torch.complex(out[..., a], out[..., b]) * turn[:, None]
        out[..., a], out[..., b] = z.real, z.imag
    return out.view(-1, heads * d)


def _rows_of(pool, name, i, count):
    """The first `count` cached rows of conversation i in 64 bits, [count][n_kv][d]."""
    x, scale, page = pool[name][0], pool[name + "s"][0], pool["page"]
    d = x.shape[3] * 16 if name == "k" else x.shape[3]
    t = torch.arange(count, device="cuda")
    pages = pool["table"][i].long()[t // page]
    at, j, h = t % page, torch.arange(d, device="cuda"), torch.arange(x.shape[1], device="cuda")
    group, place = (at // 16)[:, None, None], (at % 16)[:, None, None]
    if name == "k":
        v = x[pages[:, None, None], h[None, :, None], group, j // 16, place, j % 16]
    else:
        v = x[pages[:, None, None], h[None, :, None], group, j, place]
    return v.double() * scale[pages][..., None].double()


def _exact_append(case, s):
    """Every touched page from its own rows: the step that holds them all, older rows rounded to it once more."""
    n_kv, d, page, pool = case["n_kv"], case["d"], case["page"], s["pool"]
    cached, new = _counts(case)
    at = _offsets(new)
    result = []
    for name, lo in (("k", 0), ("v", n_kv * d)):
        rows = []
        for i, (c, m) in enumerate(zip(cached, new)):
            x = s["kv"][at[i]:at[i + 1], lo:lo + n_kv * d].double().view(m, n_kv, d)
            c0 = c - c % page
            old = _rows_of(pool, name, i, c)[c0:] if c > c0 else x[:0]
            every = torch.cat([old, x])
            for p in range(0, len(every), page):
                block = every[p:p + page]
                fresh = block[max(0, c - c0 - p):]
                step = (fresh.abs().amax((0, 2)).clamp(min=LEAST) / 127.0).float().double()  # a scale is an fp32 number
                if p == 0 and c > c0:
                    step = torch.maximum(step, pool[name + "s"][0][pool["table"][i, c // page].long()].double())
                rows.append((block / step[None, :, None]).round().clamp(-127, 127) * step[None, :, None])
        result.append(torch.cat(rows).view(-1, n_kv * d))
    return tuple(result)


def _exact_attend(case, s):
    n_q, n_kv, d, pool = case["n_q"], case["n_kv"], case["d"], s["pool"]
    group = n_q // n_kv
    cached, new = _counts(case)
    at = _offsets(new)
    out = torch.zeros(at[-1], n_q, d, dtype=torch.float64, device="cuda")
    for i, (c, m) in enumerate(zip(cached, new)):
        k, v = (_rows_of(pool, name, i, c + m) for name in ("k", "v"))
        here = torch.arange(c, c + m, device="cuda")[:, None]
        key = torch.arange(c + m, device="cuda")[None, :]
        hidden = key > here if case["causal"] else torch.zeros_like(key > here)
        if case["window"]:
            hidden = hidden | (key <= here - case["window"])
        for h in range(n_q):
            q = s["q"][at[i]:at[i + 1], h * d:(h + 1) * d].double()
            p = torch.softmax((q @ k[:, h // group].T / math.sqrt(d)).masked_fill(hidden, -math.inf), -1)
            out[at[i]:at[i + 1], h] = p @ v[:, h // group]
    return out.view(-1, n_q * d)
