"""The paged 8-bit cache's operators, as measured: what writes it, what reads it and what moves its pages.

A cache page holds BS tokens of every KV head as 8-bit codes with one fp32 scale per (page, head), for K and for V: an
element is code * scale.  Codes are e4m3 (torch.float8_e4m3fn) or int8; the scales that an append makes are powers of two.
Sizes follow the repository's decode and prefill configurations (10 heads of 128, 64-token pages, a 512-token window with
8 selected blocks, 256 requests) and generic grouped-query ones.

Operators: append (new tokens into the cache), attend (single tokens, a few draft tokens, or prompt rows), beam (beams that
lose are freed and beams that win are forked, with the copy of their part-filled page), compact (live pages to the lowest
page ids).
"""

import math
import os
import sys

import numpy as np
import torch

own = False

QMAX = {"e4m3": 448.0, "int8": 127.0}
CODE = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}
REAL = {"bf16": torch.bfloat16, "f16": torch.float16}
MIN_EXP = -64  # the smallest scale an append makes is 2**-64


def listed():
    return [
        # one new token of each of 256 decoding requests, every layer and step of batched decode
        {"name": "append_decode_batch", "kind": "append", "code": "e4m3", "real": "bf16", "R": 256, "rows": 1,
         "new_min": 1, "new_max": 1, "pre_min": 1, "pre_max": 700, "Hkv": 10, "D": 128, "BS": 64},
        # ragged prompts written in one call, some after a cached prefix that ends inside a page
        {"name": "append_prompts_ragged", "kind": "append", "code": "e4m3", "real": "bf16", "R": 9, "rows": 0,
         "new_min": 1, "new_max": 7001, "pre_min": 0, "pre_max": 300, "Hkv": 10, "D": 128, "BS": 64},
        # the first answers of one short chat: latency
        {"name": "attend_one_short", "kind": "attend", "code": "int8", "real": "bf16", "R": 1, "rows": 1,
         "len_min": 257, "len_max": 257, "H": 10, "Hkv": 10, "D": 128, "BS": 64, "window": -1, "sinks": 0, "K": 0},
        # batched decode at long context: the window and the selected blocks of 256 requests
        {"name": "attend_sparse_batch", "kind": "attend", "code": "e4m3", "real": "bf16", "R": 256, "rows": 1,
         "len_min": 2048, "len_max": 20000, "H": 10, "Hkv": 10, "D": 128, "BS": 64, "window": 512, "sinks": 0, "K": 8},
        # dense decode of a few very long requests, grouped-query heads
        {"name": "attend_dense_long", "kind": "attend", "code": "e4m3", "real": "bf16", "R": 6, "rows": 1,
         "len_min": 30011, "len_max": 131072, "H": 32, "Hkv": 8, "D": 128, "BS": 64, "window": -1, "sinks": 0, "K": 0},
        # three draft tokens per request checked at once, sliding window with sinks, int8, heads of 64
        {"name": "attend_draft_sinks", "kind": "attend", "code": "int8", "real": "f16", "R": 48, "rows": 3,
         "len_min": 5, "len_max": 9000, "H": 14, "Hkv": 2, "D": 64, "BS": 32, "window": 1024, "sinks": 4, "K": 0},
        # ragged prompt chunks after cached prefixes, the sliding window with sinks
        {"name": "prompt_window_ragged", "kind": "prompt", "code": "e4m3", "real": "bf16", "R": 7, "rows": 0,
         "new_min": 1, "new_max": 2600, "pre_min": 0, "pre_max": 5000, "H": 10, "Hkv": 10, "D": 128, "BS": 64,
         "window": 512, "sinks": 64},
        # one long chunk after a long prefix, all of it visible: the tensor-core end of the range
        {"name": "prompt_dense_long", "kind": "prompt", "code": "e4m3", "real": "bf16", "R": 1, "rows": 0,
         "new_min": 8192, "new_max": 8192, "pre_min": 8192, "pre_max": 8192, "H": 16, "Hkv": 4, "D": 128, "BS": 64,
         "window": -1, "sinks": 0},
        # four beams of one request: the step's losers are freed and its winner forked
        {"name": "beam_one_request", "kind": "beam", "code": "e4m3", "R": 8, "forks": 3, "len_min": 150, "len_max": 900,
         "Hkv": 10, "D": 128, "BS": 64},
        # the same for 64 requests in one batch with long contexts
        {"name": "beam_batch", "kind": "beam", "code": "e4m3", "R": 256, "forks": 128, "len_min": 1000, "len_max": 9000,
         "Hkv": 4, "D": 128, "BS": 64},
        # a small pool after a few requests left
        {"name": "compact_small", "kind": "compact", "code": "int8", "R": 12, "len_min": 10, "len_max": 700,
         "leave": 50, "Hkv": 4, "D": 64, "BS": 64},
        # a serving pool after half of its requests left, before their room is handed to another model
        {"name": "compact_large", "kind": "compact", "code": "e4m3", "R": 160, "len_min": 200, "len_max": 6000,
         "leave": 50, "Hkv": 10, "D": 128, "BS": 64},
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    kind = rng.choice(["append", "attend", "attend", "prompt", "prompt", "beam", "compact"])
    H, Hkv = rng.choice([(10, 10), (32, 8), (14, 2), (8, 1), (12, 4), (16, 16), (24, 2), (5, 5)])
    c = {"kind": kind, "code": rng.choice(["e4m3", "int8"]), "Hkv": Hkv, "D": rng.choice([64, 128, 128]),
         "BS": rng.choice([16, 32, 64, 64, 64, 128])}
    if kind in ("append", "attend", "prompt"):
        c["real"] = rng.choice(["bf16", "f16"])
    if kind == "append":
        if rng.random() < 0.5:
            c.update(R=log(1, 256), rows=rng.choice([1, 1, 1, 4]))
            c.update(new_min=c["rows"], new_max=c["rows"], pre_min=0, pre_max=log(1, 900))
        else:
            c.update(R=log(1, 12), rows=0, new_min=rng.choice([0, 1]), new_max=log(2, 5000), pre_min=0, pre_max=log(1, 900))
    elif kind == "attend":
        c["H"] = H
        c["rows"] = rng.choice([1, 1, 1, 2, 4])
        if rng.random() < 0.4:  # dense
            top = log(16, 100000)
            R = min(log(1, 128), max(1, 300000 // top))
            c.update(R=R, len_min=max(c["rows"], top // 4), len_max=top, window=-1, sinks=0, K=0)
        else:
            top = log(16, 16000)
            R = min(log(1, 192), max(1, 1500000 // top))
            c.update(R=R, len_min=max(c["rows"], top // 8), len_max=top, window=rng.choice([0, 1, 128, 333, 512, 1024]),
                     sinks=rng.choice([0, 0, 1, 4, 70]), K=rng.choice([0, 4, 8, 16]))
    elif kind == "prompt":
        c["H"] = H
        new, pre = log(2, 5000), rng.choice([0, log(1, 9000)])
        R = min(log(1, 8), max(1, 40000000 // (new * (new + pre) + 1)))
        c.update(R=R, rows=0, new_min=rng.choice([0, 1]) if R > 1 else new, new_max=new, pre_min=pre // 8, pre_max=pre,
                 window=rng.choice([-1, -1, 100, 512, 1024]), sinks=rng.choice([0, 4, 64]))
    elif kind == "beam":
        c["R"] = log(2, 200)
        c.update(forks=max(1, int(c["R"] * rng.uniform(0.1, 0.5))), len_min=1, len_max=log(10, 6000))
    else:
        c["R"] = log(2, 100)
        c.update(len_min=1, len_max=log(10, 5000), leave=rng.choice([10, 30, 50, 80]))
    return c


# ---------------------------------------------------------------- sizes of a case (the same for every seed)
def _spread(lo, hi, n, tag):
    """n whole numbers from lo to hi, log-spread, fixed by the arguments."""
    r = np.random.default_rng([lo, hi, n, tag])
    v = np.exp(r.uniform(math.log(lo + 1), math.log(hi + 1 + 1e-9), n)) - 1
    v = np.clip(np.round(v).astype(np.int64), lo, hi)
    if n:
        v[0] = hi
    return v


def _lens(c):
    """(prefix, new) per request for rows that come with new tokens, else the lengths."""
    if c["kind"] in ("append", "prompt"):
        return _spread(c["pre_min"], c["pre_max"], c["R"], 1), _spread(c["new_min"], c["new_max"], c["R"], 2)
    return _spread(c["len_min"], c["len_max"], c["R"], 3)


def _page_bytes(c):
    """Bytes of one page over the tensors that are moved with it."""
    return 2 * c["BS"] * c["Hkv"] * c["D"] + 2 * 4 * c["Hkv"] + c["BS"] * 128 * 2 + 128 * 4


def _shape_rows(c, lens):
    """(position, request) of every query row."""
    if c["rows"]:
        pos = (lens[:, None] - c["rows"] + np.arange(c["rows"])).reshape(-1)
        return pos, np.repeat(np.arange(c["R"]), c["rows"])
    pre, new = lens
    req = np.repeat(np.arange(c["R"]), new)
    first = np.concatenate([[0], np.cumsum(new)])
    return pre[req] + np.arange(int(new.sum())) - first[req], req


def _remote(c, pos):
    """[lo, hi) block range of a row's selection: blocks past the sinks that end before the window."""
    w = c["window"]
    ls = np.maximum(pos - w + 1, 0) if w >= 0 else np.zeros_like(pos)
    lo = -(-c["sinks"] // c["BS"])
    return np.full_like(pos, lo), np.maximum(ls // c["BS"], lo)


def _visible(c, pos):
    """Visible keys of each row."""
    w, s = c["window"], c["sinks"]
    ls = np.maximum(pos - w + 1, 0) if w >= 0 else np.zeros_like(pos)
    n = pos + 1 - ls + np.minimum(np.minimum(s, ls), pos + 1)
    if c.get("K", 0):
        lo, hi = _remote(c, pos)
        n = n + np.minimum(hi - lo, c["K"]) * c["BS"]
    return n


def work(c):
    kind, Hkv, D = c["kind"], c["Hkv"], c["D"]
    if kind == "append":
        pre, new = _lens(c)
        pages = np.where(new > 0, (pre + new + c["BS"] - 1) // c["BS"] - pre // c["BS"], 0).sum()
        n = int(new.sum())
        return {"bytes": float(n * Hkv * D * 2 * 3 + pages * (Hkv * 16 + 4)), "flops": float(n * Hkv * D * 2 * 2)}
    if kind in ("attend", "prompt"):
        lens = _lens(c)
        pos, req = _shape_rows(c, lens)
        vis = _visible(c, pos)
        flops = 4.0 * c["H"] * D * float(vis.sum())
        if kind == "attend":  # the rows of one request share their window and sinks
            last = vis.reshape(c["R"], c["rows"])[:, -1]
            extra = (c["rows"] - 1) * (c.get("K", 0) > 0)
            sel = np.minimum(np.diff(np.stack(_remote(c, pos)), axis=0)[0], c.get("K", 0)) * c["BS"]
            keys = float(last.sum()) + (float(sel.sum()) * extra / c["rows"] if extra else 0.0)
        else:
            pre, new = lens
            w, s = c["window"], c["sinks"]
            first = np.maximum(pre - w + 1, 0) if w >= 0 else np.zeros_like(pre)
            keys = float(np.where(new > 0, pre + new - first + np.minimum(s, first), 0).sum())
        rows = len(pos)
        return {"bytes": keys * Hkv * (2 * D + 8.0 / c["BS"]) + rows * c["H"] * (4.0 * D + 4), "flops": flops}
    lens = _lens(c)
    pages = -(-lens // c["BS"])
    if kind == "beam":
        par, kids = _beam_rows(c)
        part = int((lens[par] % c["BS"] > 0).sum())
        touched = int(pages[par].sum())
        return {"bytes": 2.0 * part * _page_bytes(c) + 4.0 * 4 * touched * 2, "flops": 0.0}
    stay = np.ones(c["R"], bool)
    stay[_leavers(c)] = False
    live, P = int(pages[stay].sum()), int(pages.sum())
    moved = live * (1.0 - live / max(P, 1))  # live pages at or past n_live, on average over the page orders
    return {"bytes": 2.0 * moved * _page_bytes(c) + 2 * 4.0 * (P + P), "flops": 0.0}


def _beam_rows(c):
    """(parents, children): rows in the first half of the table win, rows at its end lose."""
    r = np.random.default_rng([c["R"], c["forks"], 4])
    kids = np.arange(c["R"] - c["forks"], c["R"])
    return r.integers(0, c["R"] - c["forks"], c["forks"]), kids


def _leavers(c):
    r = np.random.default_rng([c["R"], c["leave"], 5])
    return r.permutation(c["R"])[: max(1, c["R"] * c["leave"] // 100)]


# ---------------------------------------------------------------- inputs
def _codes(c, shape, g):
    """Codes as an append leaves them: normal values, the largest of a page near the top of the type's range."""
    out = torch.empty(shape, device="cuda", dtype=CODE[c["code"]])
    step = max(1, (1 << 26) // max(1, math.prod(shape[1:])))
    for i in range(0, shape[0], step):
        n = min(step, shape[0] - i)
        x = torch.randn((n, *shape[1:]), device="cuda", dtype=torch.float16, generator=g)
        x = (x * (QMAX[c["code"]] / 5.0)).clamp_(-QMAX[c["code"]], QMAX[c["code"]])
        out[i:i + n] = (x.round_() if c["code"] == "int8" else x).to(out.dtype)
    return out


def _table(lens, BS, P, g, W=None):
    """Block table [R, W] of a random page order, -1 past a request's pages."""
    R = len(lens)
    used = torch.from_numpy(-(-lens // BS)).cuda()
    W = max(1, int(used.max())) if W is None else W
    order = torch.randperm(P, device="cuda", generator=g)
    at = torch.arange(W, device="cuda")[None] < used[:, None]
    table = torch.full((R, W), -1, device="cuda", dtype=torch.int32)
    table[at] = order[: int(used.sum())].to(torch.int32)
    return table


def prepare(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    kind, R, Hkv, D, BS = c["kind"], c["R"], c["Hkv"], c["D"], c["BS"]
    s = {"case": c, "seed": seed}
    lens = _lens(c)
    full = lens[0] + lens[1] if isinstance(lens, tuple) else lens
    total = int((-(-full // BS)).sum())
    P = total + (c["forks"] + 2 if kind == "beam" else 0 if kind == "compact" else 3)
    s["table"] = _table(full, BS, P, g)
    shape = (P, Hkv, BS, D)  # a (page, head) tile is contiguous; the calls see [P, BS, Hkv, D]
    s["k"], s["v"] = (_codes(c, shape, g).transpose(1, 2) for _ in range(2))
    s["ks"], s["vs"] = (torch.exp2(torch.randint(-7, -4, (P, Hkv), device="cuda", generator=g).float())
                        * (5 * 64 / QMAX[c["code"]]) for _ in range(2))
    if kind == "append":
        s["ks"], s["vs"] = (torch.exp2(torch.log2(x).ceil()) for x in (s["ks"], s["vs"]))
    s["lens"] = torch.from_numpy(full.astype(np.int32)).cuda()
    if isinstance(lens, tuple):
        pre, new = lens
        s["pre"] = torch.from_numpy(pre.astype(np.int32)).cuda()
        s["cu"] = torch.from_numpy(np.concatenate([[0], np.cumsum(new)]).astype(np.int32)).cuda()
        N = int(new.sum())
    else:
        N = R * c.get("rows", 0)
    if kind == "append":
        # projections of a layer: heads of different magnitude, a few large features
        mag = torch.exp2(torch.randint(-3, 2, (1, Hkv, 1), device="cuda", generator=g).float())
        s["nk"], s["nv"] = ((torch.randn(N, Hkv, D, device="cuda", generator=g) * mag).to(REAL[c["real"]]) for _ in range(2))
    elif kind in ("attend", "prompt"):
        s["q"] = torch.randn(N, c["H"], D, device="cuda", generator=g).to(REAL[c["real"]])
        s["scale"] = 1.0 / math.sqrt(D)
        s["topk"] = s["bias"] = None
        if c.get("K", 0):
            pos, _ = _shape_rows(c, lens)
            lo, hi = (torch.from_numpy(x).cuda() for x in _remote(c, pos))
            width = max(int((hi - lo).max()), c["K"])
            u = torch.rand(N, width, device="cuda", generator=g)
            u.masked_fill_(torch.arange(width, device="cuda")[None] >= (hi - lo)[:, None], 2.0)
            near, idx = u.topk(c["K"], dim=1, largest=False)
            s["topk"] = torch.where(near < 1.5, idx + lo[:, None], -1).to(torch.int32)
            s["bias"] = torch.randn(N, c["K"], device="cuda", generator=g) * 0.5
    else:
        s["idx"] = torch.randn(P, BS, 128, device="cuda", generator=g).to(torch.bfloat16)
        s["kbar"] = torch.randn(P, 128, device="cuda", generator=g)
        s["refs"] = torch.zeros(P, device="cuda", dtype=torch.int32)
        if kind == "beam":
            par, kids = _beam_rows(c)
            s["refs"][s["table"][s["table"] >= 0].long()] = 1
            s["par"], s["kids"] = (torch.from_numpy(x.astype(np.int32)).cuda() for x in (par, kids))
        else:
            gone = torch.from_numpy(_leavers(c)).cuda()
            s["table"][gone] = -1
            s["lens"][gone] = 0
            s["refs"][s["table"][s["table"] >= 0].long()] = 1
    return s


# ---------------------------------------------------------------- plain forms
def _pages_of(s, req, pos):
    BS = s["case"]["BS"]
    return s["table"][req, torch.div(pos, BS, rounding_mode="floor")].long()


def _plain_scale(amax, qmax):
    """The smallest power of two s with amax <= qmax * s, at least 2**MIN_EXP."""
    m, e = torch.frexp(amax)
    top = {448.0: (9, 0.875), 127.0: (7, 127.0 / 128.0)}[qmax]
    e = (e - top[0] + (m > top[1])).clamp_min(MIN_EXP)
    e = torch.where(amax > 0, e, torch.full_like(e, MIN_EXP))
    return torch.ldexp(torch.ones_like(amax), e)


def _plain_round(y, code):
    if code == "int8":
        return torch.nan_to_num(y, nan=0.0).round().clamp(-127, 127).to(torch.int8)
    return y.clamp(-448, 448).to(torch.float8_e4m3fn)


def _plain_append(s):
    c = s["case"]
    BS, qmax = c["BS"], QMAX[c["code"]]
    R, N = c["R"], s["nk"].shape[0]
    if c["rows"]:
        req = torch.arange(N, device="cuda") // c["rows"]
        pos = s["lens"][req] - c["rows"] + torch.arange(N, device="cuda") % c["rows"]
        start = s["lens"] - c["rows"]
        count = torch.full_like(start, c["rows"])
    else:
        req = torch.searchsorted(s["cu"], torch.arange(N, device="cuda", dtype=torch.int32), right=True) - 1
        pos = s["pre"][req] + torch.arange(N, device="cuda") - s["cu"][req]
        start, count = s["pre"], s["cu"][1:] - s["cu"][:-1]
    page = _pages_of(s, req, pos)
    # the pages that hold earlier tokens: one at most per request, its first
    held = torch.nonzero((count > 0) & (start % BS > 0))[:, 0]
    first = _pages_of(s, held, start[held])
    keep = start[held] % BS
    out = []
    for x, cache, scale in ((s["nk"], s["k"], s["ks"]), (s["nv"], s["v"], s["vs"])):
        x = x.float()
        a = torch.where(torch.isfinite(x), x.abs(), 0.0).amax(-1)
        amax = torch.zeros_like(scale).index_reduce_(0, page, a, "amax")
        new = _plain_scale(amax, qmax)
        old = scale[first]
        new[first] = torch.maximum(new[first], old)
        was = cache[first].float()
        again = _plain_round(was * (old / new[first])[:, None, :, None], c["code"])
        row = torch.arange(BS, device="cuda")
        grown = (row[None, :, None, None] < keep[:, None, None, None]) & (new[first] > old)[:, None, :, None]
        b = cache.view(torch.uint8)
        b[first] = torch.where(grown, again.view(torch.uint8), b[first])
        b[page, pos % BS] = _plain_round(x / new[page][:, :, None], c["code"]).view(torch.uint8)
        scale[page] = new[page]
        out += [cache, scale]
    return {"k": out[0], "k_scale": out[1], "v": out[2], "v_scale": out[3]}


def _plain_rows(s):
    """One gathered key list per row: sinks, window, selected blocks."""
    c = s["case"]
    BS, H, Hkv, D, rows = c["BS"], c["H"], c["Hkv"], c["D"], c["rows"]
    N = s["q"].shape[0]
    n = torch.arange(N, device="cuda")
    req = n // rows
    p = (s["lens"][req] - rows + n % rows).long()
    W = s["table"].shape[1]
    top = int(c["len_max"])
    win = top if c["window"] < 0 else min(c["window"], top)
    ls = (p - win + 1).clamp_min(0)
    sink = torch.arange(min(c["sinks"], top), device="cuda")[None].expand(N, -1)
    near = ls[:, None] + torch.arange(win, device="cuda")[None]
    parts = [(sink, (sink < ls[:, None]) & (sink <= p[:, None]), None), (near, near <= p[:, None], None)]
    if s["topk"] is not None:
        t = s["topk"].long()
        K = t.shape[1]
        again = ((t[:, :, None] == t[:, None, :]) & torch.ones(K, K, device="cuda", dtype=torch.bool).tril(-1)).any(-1)
        j = t[:, :, None] * BS + torch.arange(BS, device="cuda")
        ok = ((t >= 0) & (t < W) & ~again)[:, :, None] & (j < ls[:, None, None]) & (j >= c["sinks"]) & (j <= p[:, None, None])
        parts.append((j.reshape(N, -1), ok.reshape(N, -1), s["bias"][:, :, None].expand(-1, -1, BS).reshape(N, -1)))
    j = torch.cat([x[0] for x in parts], 1)
    ok = torch.cat([x[1] for x in parts], 1)
    b = torch.cat([torch.zeros_like(x[0], dtype=torch.float32) if x[2] is None else x[2] for x in parts], 1)
    j = torch.where(ok, j, 0)
    page = s["table"][req[:, None], torch.div(j, BS, rounding_mode="floor")].long().clamp_min(0)
    k = s["k"].view(torch.uint8)[page, j % BS].view(CODE[c["code"]]).float()      # [N, J, Hkv, D]
    z = torch.einsum("nhgd,njhd->nhgj", s["q"].float().view(N, Hkv, H // Hkv, D), k)
    del k
    z = z * (s["ks"][page].transpose(1, 2)[:, :, None] * s["scale"]) + b[:, None, None]
    z = z.masked_fill(~ok[:, None, None], -math.inf)
    m = z.amax(-1, keepdim=True)
    m = torch.where(torch.isfinite(m), m, 0.0)
    e = torch.exp(z - m)
    total = e.sum(-1, keepdim=True)
    v = s["v"].view(torch.uint8)[page, j % BS].view(CODE[c["code"]]).float().masked_fill_(~ok[:, :, None, None], 0.0)
    o = torch.einsum("nhgj,njhd->nhgd", e * s["vs"][page].transpose(1, 2)[:, :, None], v)
    o = o / torch.where(total > 0, total, 1.0)
    return {"o": o.reshape(N, H, D).to(s["q"].dtype), "lse": (m + torch.log(total)).reshape(N, H)}


def _plain_prompt(s):
    """Dense scores of every request's padded rows and keys."""
    c = s["case"]
    BS, H, Hkv, D, R = c["BS"], c["H"], c["Hkv"], c["D"], c["R"]
    pre, new = _lens(c)
    T, S = max(1, int(new.max())), max(1, int((pre + new).max()))
    N = s["q"].shape[0]
    n = torch.arange(N, device="cuda", dtype=torch.int32)
    req = (torch.searchsorted(s["cu"], n, right=True) - 1).long()
    i = (n - s["cu"][req]).long()
    q = torch.zeros(R, T, H, D, device="cuda")
    q[req, i] = s["q"].float()
    j = torch.arange(S, device="cuda")
    page = s["table"][:, torch.div(j, BS, rounding_mode="floor")].long().clamp_min(0)    # [R, S]
    there = j[None] < s["lens"][:, None]
    p = s["pre"].long()[:, None] + torch.arange(T, device="cuda")                           # [R, T]
    ok = (j <= p[:, :, None]) & there[:, None]
    if c["window"] >= 0:
        ok &= (j > p[:, :, None] - c["window"]) | (j < c["sinks"])
    k = s["k"].view(torch.uint8)[page, j % BS].view(CODE[c["code"]]).float() * s["ks"][page][..., None]
    z = torch.einsum("rthgd,rjhd->rhgtj", q.view(R, T, Hkv, H // Hkv, D), k) * s["scale"]
    z.masked_fill_(~ok[:, None, None], -math.inf)
    m = z.amax(-1, keepdim=True)
    m = torch.where(torch.isfinite(m), m, 0.0)
    e = z.sub_(m).exp_()
    total = e.sum(-1, keepdim=True)
    v = s["v"].view(torch.uint8)[page, j % BS].view(CODE[c["code"]]).float() * s["vs"][page][..., None]
    v.masked_fill_(~there[:, :, None, None], 0.0)
    o = torch.einsum("rhgtj,rjhd->rhgtd", e, v) / torch.where(total > 0, total, 1.0)
    lse = (m + torch.log(total))[..., 0]
    o = o.permute(0, 3, 1, 2, 4).reshape(R, T, H, D)[req, i]
    lse = lse.permute(0, 3, 1, 2).reshape(R, T, H)[req, i]
    return {"o": o.to(s["q"].dtype), "lse": lse}


def _plain_beam(s):
    c = s["case"]
    BS, table, lens, refs = c["BS"], s["table"], s["lens"], s["refs"]
    kids, par = s["kids"].long(), s["par"].long()
    W = table.shape[1]
    blk = torch.arange(W, device="cuda")
    # free the children
    used = (lens[kids] + BS - 1) // BS
    on = blk[None] < used[:, None]
    pages = table[kids][on].long()
    refs.index_add_(0, pages, torch.full_like(pages, -1, dtype=torch.int32))
    table[kids] = torch.where(on, -1, table[kids])
    lens[kids] = 0
    # fork: full pages shared, the part-filled page copied into the lowest free pages, in order
    n = lens[par]
    part = n % BS > 0
    free = torch.nonzero(refs == 0)[:, 0]
    rank = torch.cumsum(part.int(), 0) - 1
    made = ~part | (rank < free.numel())
    dst = free[rank.clamp(0, max(free.numel() - 1, 0))]
    last = torch.div(n, BS, rounding_mode="floor").long().clamp_max(W - 1)
    src = table[par, last].long()
    rows = torch.where(blk[None] < torch.div(n, BS, rounding_mode="floor")[:, None], table[par], -1)
    shared = rows[made]
    shared = shared[shared >= 0].long()
    refs.index_add_(0, shared, torch.ones_like(shared, dtype=torch.int32))
    copy = part & made
    i = torch.nonzero(copy)[:, 0]
    rows[i, last[i]] = dst[i].to(torch.int32)
    refs[dst[i]] = 1
    table[kids] = torch.where(made[:, None], rows, table[kids])
    lens[kids] = torch.where(made, n, 0).to(torch.int32)
    for x in (s["k"].view(torch.uint8), s["v"].view(torch.uint8), s["ks"], s["vs"], s["idx"], s["kbar"]):
        x[dst[i]] = x[src[i]]
    short = (part & ~made).sum().to(torch.int32).reshape(1)
    return {"table": table, "lens": lens, "refs": refs, "short": short, "k": s["k"], "v": s["v"], "k_scale": s["ks"],
            "v_scale": s["vs"], "idx": s["idx"], "kbar": s["kbar"]}


def _plain_compact(s):
    refs, table = s["refs"], s["table"]
    P = refs.shape[0]
    live = refs > 0
    n = live.sum()
    page = torch.arange(P, device="cuda")
    src = torch.nonzero(live & (page >= n))[:, 0]
    dst = torch.nonzero(~live & (page < n))[:, 0]
    to = page.clone()
    to[src] = dst
    for x in (s["k"].view(torch.uint8), s["v"].view(torch.uint8), s["ks"], s["vs"], s["idx"], s["kbar"]):
        x[dst] = x[src]
    out = torch.where(table >= 0, to[table.long().clamp_min(0)].to(torch.int32), table)
    count = refs.clone()
    count[dst] = refs[src]
    count[src] = 0
    return {"table": out, "refs": count, "live": n.to(torch.int32).reshape(1), "k": s["k"], "v": s["v"],
            "k_scale": s["ks"], "v_scale": s["vs"], "idx": s["idx"], "kbar": s["kbar"]}


# ---------------------------------------------------------------- the framework's calls
def _mine():
    here = os.path.join(os.getcwd(), "unlimited-ocr_b200")
    if here not in sys.path:
        sys.path.insert(0, here)
    from srswa import cache8
    return cache8


def _own(s):
    c = s["case"]
    m = _mine()
    kind = c["kind"]
    where = dict(seq_lens=s["lens"]) if c.get("rows") else dict(cu_seqlens=s.get("cu"), prefix_lens=s.get("pre"))
    if kind == "append":
        m.cache8_append(s["nk"], s["nv"], s["k"], s["v"], s["ks"], s["vs"], s["table"], **where)
        return {"k": s["k"], "k_scale": s["ks"], "v": s["v"], "v_scale": s["vs"]}
    if kind in ("attend", "prompt"):
        o, lse = m.cache8_attend(s["q"], s["k"], s["v"], s["ks"], s["vs"], s["table"], **where,
                                 window=None if c["window"] < 0 else c["window"], sinks=c["sinks"],
                                 topk_idx=s["topk"], bias=s["bias"], sm_scale=s["scale"], lse=True)
        return {"o": o, "lse": lse}
    tensors = (s["k"], s["v"], s["ks"], s["vs"], s["idx"], s["kbar"])
    rest = {"k": s["k"], "v": s["v"], "k_scale": s["ks"], "v_scale": s["vs"], "idx": s["idx"], "kbar": s["kbar"]}
    if kind == "beam":
        m.pages_free(s["kids"], s["table"], s["lens"], s["refs"], block_size=c["BS"])
        short = m.pages_fork(s["par"], s["kids"], s["table"], s["lens"], s["refs"], tensors, block_size=c["BS"])
        return {"table": s["table"], "lens": s["lens"], "refs": s["refs"], "short": short, **rest}
    table, refs, live = m.pages_compact(s["table"], s["refs"], tensors)
    return {"table": table, "refs": refs, "live": live, **rest}


def run(s):
    if own:
        return _own(s)
    return {"append": _plain_append, "attend": _plain_rows, "prompt": _plain_prompt, "beam": _plain_beam,
            "compact": _plain_compact}[s["case"]["kind"]](s)


# ---------------------------------------------------------------- the definitions in 64 bits
def _exact_round(y, code):
    if code == "int8":
        return y.round().clamp(-127, 127)
    a = y.abs()
    step = torch.exp2(torch.floor(torch.log2(a.clamp_min(2.0 ** -30))).clamp_min(-6) - 3)
    return ((a / step).round() * step).clamp_max(448.0) * torch.sign(y)


def _exact_append(c, s):
    BS, qmax = c["BS"], QMAX[c["code"]]
    pre, new = _lens(c)
    if c["rows"]:
        pre = (pre + new) - c["rows"]
        new = np.full_like(pre, c["rows"])
    out = {}
    for name, x, cache, scale in (("k", s["nk"], s["k"], s["ks"]), ("v", s["nv"], s["v"], s["vs"])):
        codes, scales = cache.double().clone(), scale.double().clone()
        at = 0
        for r in range(c["R"]):
            a, n = int(pre[r]), int(new[r])
            for b in range(a // BS, -(-(a + n) // BS) if n else 0):
                lo, hi = max(a, b * BS), min(a + n, (b + 1) * BS)
                page = int(s["table"][r, b])
                y = x[at + lo - a: at + hi - a].double()
                amax = y.abs().amax((0, 2)).clamp_min(1e-300)
                e = torch.ceil(torch.log2(amax / qmax))
                e = torch.where(amax <= qmax * torch.exp2(e - 1), e - 1, torch.where(amax > qmax * torch.exp2(e), e + 1, e))
                sc = torch.exp2(e.clamp_min(MIN_EXP))
                if lo > b * BS:
                    old = scales[page].clone()
                    sc = torch.maximum(sc, old)
                    rows = slice(0, lo - b * BS)
                    grown = (sc > old)[None, :, None]
                    codes[page, rows] = torch.where(grown, _exact_round(codes[page, rows] * (old / sc)[None, :, None], c["code"]),
                                                    codes[page, rows])
                codes[page, lo - b * BS: hi - b * BS] = _exact_round(y / sc[None, :, None], c["code"])
                scales[page] = sc
            at += n
        out[name], out[name + "_scale"] = codes if c["code"] == "e4m3" else None, scales
    return out


def _exact_attend(c, s):
    BS, H, Hkv, D = c["BS"], c["H"], c["Hkv"], c["D"]
    lens = _lens(c)
    pos, req = _shape_rows(c, lens)
    full = lens[0] + lens[1] if isinstance(lens, tuple) else lens
    G = H // Hkv
    N = len(pos)
    o = torch.zeros(N, H, D, device="cuda", dtype=torch.float64)
    lse = torch.full((N, H), -math.inf, device="cuda", dtype=torch.float64)
    for r in range(c["R"]):
        mine = np.nonzero(req == r)[0]
        if not len(mine):
            continue
        S = int(full[r])
        table = s["table"][r, : -(-S // BS)].long()
        ks, vs = (x[table].double().repeat_interleave(BS, 0)[:S] for x in (s["ks"], s["vs"]))
        k, v = (x.view(torch.uint8)[table].view(CODE[c["code"]]).reshape(-1, Hkv, D)[:S] for x in (s["k"], s["v"]))
        step = max(1, (1 << 28) // max(1, S * Hkv * G))
        for a in range(0, len(mine), step):
            rows = torch.from_numpy(mine[a: a + step]).cuda()
            p = torch.from_numpy(pos[mine[a: a + step]]).cuda()[:, None]
            j = torch.arange(S, device="cuda")[None]
            seen = j <= p
            bias = torch.zeros(len(rows), S, device="cuda", dtype=torch.float64)
            if c["window"] >= 0:
                plain = seen & ((j > p - c["window"]) | (j < c["sinks"]))
                seen = plain.clone()
                if s["topk"] is not None:
                    for slot in range(c["K"]):
                        t = s["topk"][rows, slot].long()[:, None]
                        add = (t >= 0) & (j // BS == t) & (j <= p) & ~seen
                        bias = torch.where(add, s["bias"][rows, slot].double()[:, None], bias)
                        seen = seen | add
            for h in range(Hkv):
                q = s["q"][rows, h * G: (h + 1) * G].double()
                z = torch.einsum("ngd,jd->ngj", q, k[:, h].double()) * ks[:, h] * s["scale"] + bias[:, None]
                z = z.masked_fill(~seen[:, None], -math.inf)
                l = torch.logsumexp(z, -1)
                e = torch.exp(z - torch.where(torch.isfinite(l), l, 0.0)[..., None])
                o[rows, h * G: (h + 1) * G] = torch.einsum("ngj,jd->ngd", e * vs[:, h], v[:, h].double())
                lse[rows, h * G: (h + 1) * G] = l
    return {"o": o, "lse": lse}


def exact(c, seed):
    if c["kind"] in ("beam", "compact"):
        return None  # whole numbers and copied pages
    s = prepare(c, seed)
    if c["kind"] == "append":
        return _exact_append(c, s) if c["R"] <= 64 or c["rows"] else None
    if 4.0 * c["H"] * c["D"] * float(_visible(dict(c, window=-1, K=0), _shape_rows(c, _lens(c))[0]).sum()) > 3e13:
        return None
    return _exact_attend(c, s)
