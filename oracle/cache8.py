"""Plain 64-bit restatements of the scaled 8-bit cache's operators and of the
page operators (numpy / python loops, no GPU, nothing of the library)."""

from __future__ import annotations

import math

import numpy as np

QMAX = {"e4m3": 448.0, "int8": 127.0}


def e4m3_values():
    """Value of every e4m3 code (NaN for 0x7f / 0xff)."""
    v = np.empty(256)
    for c in range(256):
        e, m = (c >> 3) & 15, c & 7
        x = math.ldexp(m / 8, -6) if e == 0 else math.ldexp(1 + m / 8, e - 7)
        v[c] = (math.nan if c & 127 == 127 else x) * (-1 if c & 128 else 1)
    return v


def codes_to_values(c, code):
    """Values of codes held as uint8 bytes."""
    return e4m3_values()[c] if code == "e4m3" else c.view(np.int8).astype(np.float64)


def round_to_code(y, code):
    """Values y in steps of the code, to nearest even, saturated; int8: NaN -> 0."""
    y = np.asarray(y, np.float64)
    if code == "int8":
        return np.clip(np.round(np.nan_to_num(y, nan=0.0, posinf=1e9, neginf=-1e9)), -127, 127)
    a = np.minimum(np.abs(y), 1e6)
    with np.errstate(divide="ignore", invalid="ignore"):
        e = np.maximum(np.floor(np.log2(np.where(a > 0, a, 1.0))), -6)
        step = np.exp2(e - 3)
        r = np.minimum(np.round(a / step) * step, 448.0)
    return np.where(np.isnan(y), np.nan, np.copysign(r, y))


def pow2_scale(amax, qmax):
    """The smallest power of two s >= 2**-64 with amax <= qmax * s."""
    e = -64
    while amax > qmax * 2.0 ** e:
        e += 1
    return 2.0 ** e


def append(x, values, scale, table, start, count, BS, code):
    """One of K / V: new rows x [N, Hkv, D] (requests in turn, count[r] each)
    from position start[r] into values [P, BS, Hkv, D] (the codes' values) and
    scale [P, Hkv], in place."""
    at = 0
    for r, (a, n) in enumerate(zip(start, count)):
        for b in range(a // BS, -(-(a + n) // BS) if n else 0):
            lo, hi = max(a, b * BS), min(a + n, (b + 1) * BS)
            page = table[r, b] if b < table.shape[1] else -1
            if not 0 <= page < len(values):
                continue
            y = x[at + lo - a: at + hi - a].astype(np.float64)
            for h in range(y.shape[1]):
                v = np.abs(y[:, h])
                v = v[np.isfinite(v)]
                s = pow2_scale(v.max() if v.size else 0.0, QMAX[code])
                if lo > b * BS:
                    old = scale[page, h]
                    if s > old:
                        held = values[page, : lo - b * BS, h]
                        # the ratio is an fp32 number in the library too
                        values[page, : lo - b * BS, h] = round_to_code(held * float(np.float32(old) / np.float32(s)), code)
                    s = max(s, old)
                values[page, lo - b * BS: hi - b * BS, h] = round_to_code(y[:, h] / s, code)
                scale[page, h] = s
        at += n


def visible(p, S, BS, window, sinks, sel, W):
    """(keys, slot of each or -1) that the row at position p sees; sel: its slots."""
    keys, slots = [], []
    first = 0 if window is None else p - window + 1
    picked = {}
    for i, t in enumerate(sel):
        if 0 <= t < W and t not in picked:
            picked[int(t)] = i
    for j in range(0, min(p + 1, W * BS)):
        if j >= first or j < sinks:
            keys.append(j)
            slots.append(-1)
        elif j // BS in picked:
            keys.append(j)
            slots.append(picked[j // BS])
    return np.array(keys, np.int64), np.array(slots, np.int64)


def attend(q, kv, vv, ks, vs, table, req, pos, window, sinks, topk, bias, sm_scale):
    """q [N, H, D], values [P, BS, Hkv, D], scales [P, Hkv], rows at pos[n] of
    request req[n]; topk / bias [Hkv or 1, N, K] or None -> o [N, H, D], lse
    [N, H], and the softmax-weighted mean of |v| (what a relative error of the
    weights can move o by)."""
    N, H, D = q.shape
    P, BS, Hkv, _ = kv.shape
    G = H // Hkv
    o, a, lse = np.zeros((N, H, D)), np.zeros((N, H, D)), np.full((N, H), -np.inf)
    for n in range(N):
        for h in range(Hkv):
            hs = 0 if topk is None or topk.shape[0] == 1 else h
            sel = [] if topk is None else topk[hs, n]
            j, slot = visible(int(pos[n]), None, BS, window, sinks, sel, table.shape[1])
            if len(j):
                page = table[req[n], j // BS]
                ok = (page >= 0) & (page < P)
                j, slot, page = j[ok], slot[ok], page[ok]
            if not len(j):
                continue
            k = kv[page, j % BS, h] * ks[page, h][:, None]
            v = vv[page, j % BS, h] * vs[page, h][:, None]
            b = np.zeros(len(j))
            if bias is not None:
                b = np.where(slot >= 0, bias[hs, n][np.maximum(slot, 0)], 0.0)
            for g in range(G):
                z = (k @ q[n, h * G + g].astype(np.float64)) * sm_scale + b
                m = z.max()
                e = np.exp(z - m)
                lse[n, h * G + g] = m + math.log(e.sum())
                o[n, h * G + g] = e @ v / e.sum()
                a[n, h * G + g] = e @ np.abs(v) / e.sum()
    return o, lse, a


class Pool:
    """Block tables and reference counts, one step at a time."""

    def __init__(self, table, lens, refs, BS, data=()):
        self.table, self.lens, self.refs, self.BS = table.copy(), lens.copy(), refs.copy(), BS
        self.data = [d.copy() for d in data]

    def pages(self, n):
        return -(-int(n) // self.BS)

    def lowest(self, n):
        f = np.nonzero(self.refs == 0)[0]
        return f[:n] if len(f) >= n else None

    def free(self, rows):
        for r in rows:
            if not 0 <= r < len(self.lens):
                continue
            for b in range(min(self.pages(self.lens[r]), self.table.shape[1])):
                if 0 <= self.table[r, b] < len(self.refs):
                    self.refs[self.table[r, b]] -= 1
                self.table[r, b] = -1
            self.lens[r] = 0

    def _serve(self, items):
        """items: (need, act) of the valid ones; pages in order, each item's
        need counted whether or not it is made."""
        free = list(np.nonzero(self.refs == 0)[0])
        at, short = 0, 0
        for need, act in items:
            if need and at + need > len(free):
                short += 1
            else:
                act(free[at: at + need])
            at += need
        return short

    def extend(self, rows, new_lens):
        lens, named, items = self.lens.copy(), set(), []
        for r, n in zip(rows, new_lens):
            if not 0 <= r < len(lens) or n < lens[r] or self.pages(n) > self.table.shape[1] or r in named:
                continue
            named.add(r)

            def act(pages, r=r, n=n):
                a = self.pages(lens[r])
                self.table[r, a: a + len(pages)] = pages
                self.refs[pages] = 1
                self.lens[r] = n
            items.append((self.pages(n) - self.pages(lens[r]), act))
        return self._serve(items)

    def fork(self, parents, children):
        lens, table, named, items = self.lens.copy(), self.table.copy(), set(), []
        for a, c in zip(parents, children):
            R = len(lens)
            if not (0 <= a < R and 0 <= c < R) or lens[c] or not lens[a] or c in named:
                continue
            named.add(c)

            def act(pages, a=a, c=c):
                full = lens[a] // self.BS
                self.table[c, :full] = table[a, :full]
                for p in table[a, :full]:
                    if 0 <= p < len(self.refs):
                        self.refs[p] += 1
                if len(pages):
                    self.table[c, full] = pages[0]
                    self.refs[pages[0]] = 1
                    if 0 <= table[a, full] < len(self.refs):
                        for d in self.data:
                            d[pages[0]] = d[table[a, full]]
                self.lens[c] = lens[a]
            items.append((1 if lens[a] % self.BS else 0, act))
        return self._serve(items)

    def compact(self):
        live = int((self.refs > 0).sum())
        src = [p for p in range(live, len(self.refs)) if self.refs[p] > 0]
        dst = [p for p in range(live) if self.refs[p] <= 0]
        to = dict(zip(src, dst))
        for s, d in to.items():
            for x in self.data:
                x[d] = x[s]
            self.refs[d], self.refs[s] = self.refs[s], 0
        self.table = np.vectorize(lambda p: to.get(int(p), int(p)), otypes=[np.int32])(self.table)
        return live
