"""The scaled 8-bit cache at the limits of its contract: value scales of any
spread, table entries past a request's end, queries and biases at the ends of
their types, requests shorter than their rows, rows of no request.

Tolerance of the attend, from the arithmetic, for rows and tiles alike: softmax
weights are rounded to f16 (2^-11 of each product p v), the rest is fp32 (the
same again allowed, 2^-11 of sum p |v|, as in test_gpu_cache8.py), the output is
rounded to its type.  f16 ends at 2^-24: the weights are kept such that the
row's largest product of a weight and a value scale is at 2^7 or more, so each
key may be off by 2^-25 / 2^7 of that times its code: 2^-32 max(p s) sum |code|.
What lies under fp32's smallest normal, 2^-126, may be lost.  Scores are fp32 sums
of exact products, so lse may be off by (D + 2) 2^-24 of the largest sum |q k|
(1e-4 for the normal queries of test_gpu_cache8.py)."""

import math

import numpy as np
import pytest
import torch

from oracle import cache8 as O8
from srswa import _lib as L
from srswa import cache8, ops, paged
from test_gpu_cache8 import CODE, U, check, make_cache
from test_gpu_cache8_forms import tiles_take

pytestmark = pytest.mark.gpu


def dense(q, vals, sc, table, req, pos, window, sinks, sm):
    """o, lse, sum p |v|, max(p s) sum |code| and the largest sum |q k| of every
    row, in 64 bits."""
    N, H, D = q.shape
    P, BS, Hkv, _ = vals.shape[1:]
    G = H // Hkv
    o, a, f = (np.zeros((N, H, D)) for _ in range(3))
    lse, y = np.full((N, H), -np.inf), np.zeros((N, H))
    for r in np.unique(req):
        n = np.nonzero(req == r)[0]
        S = min(max(int(pos[n].max()) + 1, 0), table.shape[1] * BS)
        j = np.arange(S)
        page = table[r, j // BS]
        there = (page >= 0) & (page < P)
        page = np.where(there, page, 0)
        p = pos[n][:, None]
        seen = there & (j <= p)
        if window is not None:
            seen &= (j > p - window) | (j < sinks)
        with np.errstate(invalid="ignore"):
            for h in range(Hkv):
                k = np.where(there[:, None], vals[0, page, j % BS, h] * sc[0, page, h][:, None], 0.0)
                s = np.where(there, sc[1, page, h], 0.0)
                c = np.where(there[:, None], vals[1, page, j % BS, h], 0.0)
                for g in range(h * G, h * G + G):
                    z = np.where(seen, q[n, g] @ k.T * sm, -np.inf)
                    m = z.max(1, keepdims=True, initial=-np.inf)
                    e = np.where(seen, np.exp(z - np.where(np.isfinite(m), m, 0.0)), 0.0)
                    t = e.sum(1, keepdims=True)
                    e /= np.where(t > 0, t, 1.0)
                    lse[n, g] = np.where(t[:, 0] > 0, m[:, 0] + np.log(np.where(t > 0, t, 1.0))[:, 0], -np.inf)
                    o[n, g] = (e * s) @ c
                    a[n, g] = (e * s) @ np.abs(c)
                    f[n, g] = (e * s).max(1, keepdims=True, initial=0.0) * (seen @ np.abs(c))
                    y[n, g] = np.where(seen, np.abs(q[n, g]) @ np.abs(k.T), 0.0).max(1, initial=0.0) * abs(sm)
    return o, lse, a, f, y


def close(out, lse, ref):
    o, l, a, f, y = ref
    got = out.double().cpu().numpy()
    assert np.isfinite(got).all()
    tol = U[out.dtype] * np.abs(o) + 2.0 ** -10 * a + 2.0 ** -32 * f + 2.0 ** -126
    assert (np.abs(got - o) <= tol).all(), np.nanmax(np.abs(got - o) / np.where(tol > 0, tol, 1e-300))
    g = lse.double().cpu().numpy()
    assert np.array_equal(np.isneginf(g), np.isneginf(l))
    fin = np.isfinite(l)
    assert (np.abs(g[fin] - l[fin]) <= np.maximum(1e-4, (o.shape[2] + 2) * 2.0 ** -24 * y[fin])).all()


def place(dev, form, lens, rows):
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    pos = np.concatenate([n - rows + np.arange(rows) for n in lens])
    req = np.repeat(np.arange(len(lens)), rows)
    if form == "ragged":
        return pos, req, dict(cu_seqlens=i32([rows * i for i in range(len(lens) + 1)]), prefix_lens=i32([n - rows for n in lens]))
    return pos, req, dict(seq_lens=i32(lens))


@pytest.mark.parametrize("code,real,BS", [("e4m3", "bf16", 64), ("int8", "f32", 16)])
@pytest.mark.parametrize("ahead,behind", [(5, 0), (200, 0), (0, 77), (517, 300)])
def test_append_rows_of_no_request(cuda, code, real, BS, ahead, behind):
    """cu_seqlens may begin behind row 0 and end before the last row."""
    rng = np.random.default_rng(66)
    start, count = [0, 70, 3, 0], [65, 1, 0, 130]
    R, Hkv, D, W = len(start), 2, 128, -(-130 // BS) + 1
    real = {"bf16": torch.bfloat16, "f32": torch.float32}[real]
    bt = torch.from_numpy(rng.permutation(R * W).astype(np.int32).reshape(R, W)).to(cuda)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
    x = torch.from_numpy(rng.standard_normal((2, ahead + sum(count) + behind, Hkv, D))).to(cuda).to(real)
    cu = np.array([0, *np.cumsum(count)])
    a, b = (cache8.Cache8(R * W, BS, Hkv, D, dtype=CODE[code], device=cuda) for _ in range(2))
    a.append(*x, bt, cu_seqlens=i32(cu + ahead), prefix_lens=i32(start))
    b.append(*x[:, ahead: ahead + sum(count)], bt, cu_seqlens=i32(cu), prefix_lens=i32(start))
    for s, t in zip(a.tensors(), b.tensors()):
        assert torch.equal(*(y if y.dtype == torch.float32 else y.view(torch.uint8) for y in (s, t)))


@pytest.mark.parametrize("window,sinks", [(None, 0), (100, 4)])
@pytest.mark.parametrize("ahead,behind", [(5, 0), (700, 0), (0, 77), (517, 1300)])
@pytest.mark.parametrize("new", [[300, 1, 0, 469], [3, 1, 0, 4]])
def test_attend_rows_of_no_request(cuda, window, sinks, ahead, behind, new):
    """Such rows give 0 and -inf, and the others what they give without them."""
    rng = np.random.default_rng(67)
    pre, H, Hkv, D, BS = [0, 70, 3, 131], 8, 2, 128, 64
    lens = [p + n for p, n in zip(pre, new)]
    k, v, ks, vs, table, vals, sc = make_cache(rng, cuda, lens, Hkv, D, BS, "e4m3")
    n = sum(new)
    if n > 100:
        assert tiles_take(N=ahead + n + behind, R=4, H=H, Hkv=Hkv, D=D, W=table.shape[1], P=30, block_size=BS,
                          window=window or -1, sinks=sinks)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
    q = torch.from_numpy(rng.standard_normal((ahead + n + behind, H, D))).to(cuda).to(torch.bfloat16)
    cu = np.array([0, *np.cumsum(new)])
    out = torch.full(q.shape, math.nan, device=cuda, dtype=torch.float32)
    o, lse = ops.cache8_attend(q, k, v, ks, vs, torch.from_numpy(table).to(cuda), cu_seqlens=i32(cu + ahead),
                               prefix_lens=i32(pre), window=window, sinks=sinks, lse=True, out=out)
    mine = slice(ahead, ahead + n)
    for part in (slice(0, ahead), slice(ahead + n, None)):
        assert (o[part] == 0).all() and torch.isneginf(lse[part]).all()
    pos, req = np.concatenate([a + np.arange(m) for a, m in zip(pre, new)]), np.repeat(np.arange(4), new)
    close(o[mine], lse[mine], dense(q[mine].double().cpu().numpy(), vals, sc, table, req, pos, window, sinks, D ** -0.5))


@pytest.mark.parametrize("form,rows", [("rows", 270), ("ragged", 270), ("rows", 1), ("rows", 5), ("ragged", 3)])
@pytest.mark.parametrize("scale", [1e30, math.inf, math.nan])
@pytest.mark.parametrize("window", [None, 100])
def test_table_entries_past_the_end(cuda, form, rows, scale, window):
    """Pages that the table names past a request's tokens (room reserved, or left
    over from another request) do not reach its rows."""
    rng = np.random.default_rng(62)
    # 270 rows of 4 heads a KV head end in the first tile of their last pair, a few keys before a page's end
    lens, H, Hkv, D, BS = [701, 318], 8, 2, 128, 64
    k, v, ks, vs, table, vals, sc = make_cache(rng, cuda, lens, Hkv, D, BS, "e4m3")
    unused = np.setdiff1d(np.arange(len(ks)), table[table >= 0])
    assert len(unused) >= 3
    wide = np.full((2, table.shape[1] + 1), -1, np.int32)
    wide[:, : table.shape[1]] = table
    full = wide.copy()
    for r in range(2):
        full[r, -(-lens[r] // BS):] = unused[np.arange(full.shape[1] - -(-lens[r] // BS)) % len(unused)]
    for x in (ks, vs):
        x[torch.from_numpy(unused).to(cuda)] = scale
    pos, req, at = place(cuda, form, lens, rows)
    if rows > 64:
        assert tiles_take(N=2 * rows, R=2, H=H, Hkv=Hkv, D=D, W=12, P=20, block_size=BS, window=window or -1,
                          **({} if form == "ragged" else {"rows_per_req": rows}))
    q = torch.from_numpy(rng.standard_normal((2 * rows, H, D))).to(cuda).to(torch.bfloat16)
    run = lambda t: ops.cache8_attend(q, k, v, ks, vs, torch.from_numpy(t).to(cuda), window=window, lse=True, **at)  # noqa: E731
    a, b = run(wide), run(full)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    close(*b, dense(q.double().cpu().numpy(), vals, sc, table, req, pos, window, 0, D ** -0.5))


SPREADS = {"neighbours": lambda b: 30 * (b % 2) - 15, "steps": lambda b: 70 * (b // 2 % 2) - 50, "up": lambda b: 5 * b - 40,
           "down": lambda b: 10 - 5 * b, "thirds": lambda b: [-110, 0, 90][b % 3], "none": lambda b: [0, None][b % 2],
           "all none": lambda b: None}


@pytest.mark.parametrize("spread", list(SPREADS))
@pytest.mark.parametrize("window,sinks", [(None, 0), (40, 3), (200, 0)])
@pytest.mark.parametrize("rows,form,code,D", [(300, "rows", "e4m3", 128), (270, "ragged", "int8", 64), (1, "rows", "e4m3", 128),
                                              (5, "rows", "int8", 64), (1, "split", "e4m3", 64)])
def test_value_scales_of_any_spread(cuda, spread, window, sinks, rows, form, code, D):
    """Value scales up to 2^200 apart, or 0, from page to page: every row as good
    as its own keys allow, whatever its neighbours see."""
    rng = np.random.default_rng(60)
    lens, H, Hkv, BS = [700, 350], 8, 2, 64
    k, v, ks, vs, table, vals, sc = make_cache(rng, cuda, lens, Hkv, D, BS, code)
    for r in range(2):
        for b in range(-(-lens[r] // BS)):
            e = SPREADS[spread](b)
            sc[1, table[r, b]] = 0.0 if e is None else sc[1, table[r, b]] * 2.0 ** e
    vs = torch.from_numpy(sc[1].astype(np.float32)).to(cuda)
    pos, req, at = place(cuda, form, lens, rows)
    if rows > 64:
        assert tiles_take(N=2 * rows, R=2, H=H, Hkv=Hkv, D=D, W=11, P=20, block_size=BS, window=window or -1, sinks=sinks,
                          **({} if form == "ragged" else {"rows_per_req": rows}))
    q = torch.from_numpy(3 * rng.standard_normal((2 * rows, H, D))).to(cuda).to(torch.bfloat16)
    o, lse = ops.cache8_attend(q, k, v, ks, vs, torch.from_numpy(table).to(cuda), window=window, sinks=sinks, lse=True,
                               nsplit=4 if form == "split" else 0, **at)
    close(o, lse, dense(q.double().cpu().numpy(), vals, sc, table, req, pos, window, sinks, D ** -0.5))


@pytest.mark.parametrize("nsplit", [0, 1, 2])
@pytest.mark.parametrize("rows", [1, 6])
def test_small_weight_on_a_large_scale(cuda, rows, nsplit):
    """Keys of weight 2^-20 to 2^-60 whose page's value scale makes up for it."""
    rng = np.random.default_rng(61)
    lens, H, Hkv, D, BS = [400, 200], 4, 2, 128, 64
    k, v, ks, vs, table, vals, sc = make_cache(rng, cuda, lens, Hkv, D, BS, "int8")
    q = torch.ones(2 * rows, H, D, device=cuda, dtype=torch.bfloat16)
    kb = np.zeros((sc.shape[1], BS, Hkv, D), np.uint8)
    for r in range(2):
        for b in range(-(-lens[r] // BS)):  # every key of block b has the logit -8 b: weight 2^(-11.5 b)
            kb[table[r, b], :, :, 0] = 256 - b if b else 0
            sc[0, table[r, b]] = 1.0
            sc[1, table[r, b]] = 2.0 ** (12 * b)
    k = torch.from_numpy(kb).to(cuda).view(torch.int8)
    v = v.contiguous()
    vals[0] = O8.codes_to_values(kb, "int8")
    pos, req, at = place(cuda, "rows", lens, rows)
    ks, vs = (torch.from_numpy(x.astype(np.float32)).to(cuda) for x in sc)
    o, lse = ops.cache8_attend(q, k, v, ks, vs, torch.from_numpy(table).to(cuda), lse=True, sm_scale=8.0,
                               nsplit=nsplit, **at)
    close(o, lse, dense(q.double().cpu().numpy(), vals, sc, table, req, pos, None, 0, 8.0))


@pytest.mark.parametrize("rows", [4, 70])
@pytest.mark.parametrize("code,real,BS", [("e4m3", "bf16", 64), ("int8", "f32", 16)])
def test_append_requests_shorter_than_their_rows(cuda, rows, code, real, BS):
    """The rows at positions 0 and up are written, as the varlen form writes them."""
    rng = np.random.default_rng(65)
    lens = [0, 1, 2, 3, 4, 5, 17, 64, 69, 70, 71, 200]
    R, Hkv, D, W = len(lens), 2, 128, -(-200 // BS)
    real = {"bf16": torch.bfloat16, "f32": torch.float32}[real]
    bt = torch.from_numpy(rng.permutation(R * W).astype(np.int32).reshape(R, W)).to(cuda)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
    a, b = (cache8.Cache8(R * W, BS, Hkv, D, dtype=CODE[code], device=cuda) for _ in range(2))
    pre = [max(n - rows, 0) for n in lens]
    first = torch.from_numpy(rng.standard_normal((2, sum(pre), Hkv, D))).to(cuda).to(real)
    for c in (a, b):
        c.append(*first, bt, cu_seqlens=i32([0, *np.cumsum(pre)]), prefix_lens=i32([0] * R))
    x = torch.from_numpy(rng.standard_normal((2, R * rows, Hkv, D))).to(cuda).to(real)
    a.append(*x, bt, i32(lens))
    there = [r * rows + i for r, n in enumerate(lens) for i in range(rows) if n - rows + i >= 0]
    new = [min(n, rows) for n in lens]
    b.append(*x[:, there], bt, cu_seqlens=i32([0, *np.cumsum(new)]), prefix_lens=i32(pre))
    for s, t in zip(a.tensors(), b.tensors()):
        assert torch.equal(s.view(torch.uint8) if s.dtype != torch.float32 else s, t.view(torch.uint8) if t.dtype != torch.float32 else t)
    # and both are the definition's
    vals, sc = np.zeros((R * W, BS, Hkv, D)), np.ones((R * W, Hkv))
    O8.append(first[0].double().cpu().numpy(), vals, sc, bt.cpu().numpy(), [0] * R, pre, BS, code)
    O8.append(x[0, there].double().cpu().numpy(), vals, sc, bt.cpu().numpy(), pre, new, BS, code)
    got = O8.codes_to_values(np.ascontiguousarray(a.k.view(torch.uint8).cpu().numpy()), code)
    np.testing.assert_array_equal(a.k_scale.double().cpu().numpy(), sc)
    np.testing.assert_array_equal(got, vals)


@pytest.mark.parametrize("qs", [2.0 ** -100, 2.0 ** -40, 1.0, 2.0 ** 30, 2.0 ** 100])
@pytest.mark.parametrize("code,D", [("e4m3", 128), ("int8", 64)])
@pytest.mark.parametrize("rows", [300, 5])
def test_query_range(cuda, qs, code, D, rows):
    """bf16 queries of any magnitude, and one element 2^20 above the rest on a
    feature that the keys leave at 0."""
    rng = np.random.default_rng(63)
    lens, H, Hkv, BS = [700, 350], 8, 2, 64
    k, v, ks, vs, table, vals, sc = make_cache(rng, cuda, lens, Hkv, D, BS, code)
    k.view(torch.uint8)[..., 5] = 0
    vals[0, ..., 5] = 0
    pos, req, at = place(cuda, "rows", lens, rows)
    q = (torch.from_numpy(rng.standard_normal((2 * rows, H, D))) * qs).to(torch.bfloat16)
    q[..., 5] = 2.0 ** 20 * qs
    q = q.to(cuda)
    sm = D ** -0.5 / qs
    o, lse = ops.cache8_attend(q, k, v, ks, vs, torch.from_numpy(table).to(cuda), lse=True, sm_scale=sm, **at)
    close(o, lse, dense(q.double().cpu().numpy(), vals, sc, table, req, pos, None, 0, sm))


@pytest.mark.parametrize("low", [-3.4028234663852886e38, -3e38, -1e38, 3.4028234663852886e38])
@pytest.mark.parametrize("nsplit", [0, 3])
def test_bias_at_the_end_of_its_type(cuda, low, nsplit):
    """Selected blocks all at the lowest value: the row still weighs them (by the
    bias, which swallows the scores); beside keys of the window they weigh
    nothing.  lse is held in log2 units: a bias past 2^128 ln 2 counts as that."""
    rng = np.random.default_rng(64)
    lens, H, Hkv, D, BS = [512, 700], 4, 2, 128, 64
    k, v, ks, vs, table, vals, sc = make_cache(rng, cuda, lens, Hkv, D, BS, "e4m3")
    q = torch.from_numpy(rng.standard_normal((2, H, D))).to(cuda).to(torch.bfloat16)
    topk = torch.tensor([[0, 2, 3], [1, 4, -1]], dtype=torch.int32, device=cuda)
    bias = torch.full((2, 3), low, device=cuda)
    lens_t, bt = torch.tensor(lens, dtype=torch.int32, device=cuda), torch.from_numpy(table).to(cuda)
    run = lambda w, b: ops.cache8_attend(q, k, v, ks, vs, bt, lens_t, window=w, topk_idx=topk, bias=b, lse=True,  # noqa: E731
                                         nsplit=nsplit)
    o, lse = run(0, bias)
    assert torch.isfinite(o).all()
    g = lse.double().cpu().numpy()
    end = math.copysign(min(abs(low), 3.4028234663852886e38 * math.log(2)), low)
    assert np.abs(g / end - 1).max() <= 1e-6
    for r in range(2):
        pages = table[r, [b for b in topk[r].tolist() if b >= 0]]
        for h in range(H):
            val = (vals[1, pages, :, h // 2] * sc[1, pages, h // 2][:, None, None]).reshape(-1, D)
            got = o[r, h].double().cpu().numpy()
            assert (np.abs(got - val.mean(0)) <= 2.0 ** -8 * np.abs(val.mean(0)) + 2.0 ** -10 * np.abs(val).mean(0)).all()
    if low < 0:
        near = ops.cache8_attend(q, k, v, ks, vs, bt, lens_t, window=100, lse=True, nsplit=nsplit)
        both = run(100, bias)
        ref = dense(q.double().cpu().numpy(), vals, sc, table, np.arange(2), np.array(lens) - 1, 100, 0, D ** -0.5)
        close(*both, ref)
        close(*near, ref)
    masked = run(0, torch.full((2, 3), -math.inf, device=cuda))
    assert (masked[0] == 0).all() and torch.isneginf(masked[1]).all()


@pytest.mark.parametrize("rows,form", [(300, "rows"), (257, "ragged"), (64, "ragged")])
@pytest.mark.parametrize("window", [None, 70])
def test_nan_value_code_of_the_last_key(cuda, rows, form, window):
    """It reaches the request's last row alone, in the last step of its tile."""
    rng = np.random.default_rng(68)
    lens, H, Hkv, D, BS = [700, 350], 8, 2, 128, 64
    lens, R = lens * 4, 8
    k, v, ks, vs, table, vals, sc = make_cache(rng, cuda, lens, Hkv, D, BS, "e4m3")
    pos, req, at = place(cuda, form, lens, rows)
    assert tiles_take(N=R * rows, R=R, H=H, Hkv=Hkv, D=D, W=11, P=80, block_size=BS, window=window or -1,
                      **({} if form == "ragged" else {"rows_per_req": rows}))
    q = torch.from_numpy(rng.standard_normal((R * rows, H, D))).to(cuda).to(torch.bfloat16)
    run = lambda: ops.cache8_attend(q, k, v, ks, vs, torch.from_numpy(table).to(cuda), window=window, **at)  # noqa: E731
    clean = run()
    for r in range(R):
        j = lens[r] - 1
        v.view(torch.uint8)[int(table[r, j // BS]), j % BS, :, 9] = 0xFF
    o = run()
    last = torch.zeros(R * rows, dtype=torch.bool, device=cuda)
    last[rows - 1:: rows] = True
    assert torch.isnan(o[last][:, :, 9]).all()
    assert torch.equal(o[~last], clean[~last])


@pytest.mark.parametrize("rows", [1, 300])
def test_strides_of_single_elements(cuda, rows):
    """One head, one request: strides that are never used may have any value."""
    rng = np.random.default_rng(69)
    n, D, BS = 400, 128, 64
    k, v, ks, vs, table, vals, sc = make_cache(rng, cuda, [n], 1, D, BS, "int8")

    def odd(t, dim, stride):
        s = list(t.stride())
        s[dim] = stride
        return t.as_strided(t.shape, s)
    q = torch.from_numpy(rng.standard_normal((rows, 1, D))).to(cuda).to(torch.bfloat16)
    bt, sl = torch.from_numpy(table).to(cuda), torch.tensor([n], dtype=torch.int32, device=cuda)
    want = ops.cache8_attend(q, k, v, ks, vs, bt, sl)
    q1, k1, v1 = odd(q, 1, 5), odd(k, 2, 7), odd(v, 2, 9)
    if rows == 1:
        q1 = odd(q1, 0, 3)
    assert torch.equal(want, ops.cache8_attend(q1, k1, v1, odd(ks, 1, 3), vs, odd(bt, 0, 1), sl, out=odd(torch.empty_like(q), 1, 3)))
    a, b = k.clone(), k.clone()
    ops.cache8_append(q, q, a, v.clone(), ks.clone(), vs.clone(), bt, sl)
    ops.cache8_append(q1, q1, odd(b, 2, 7), odd(v.clone(), 2, 1), odd(ks.clone(), 1, 3), vs.clone(), odd(bt, 0, 1), sl)
    assert torch.equal(a, b)
    refs = torch.zeros(len(ks), dtype=torch.int32, device=cuda)
    refs[bt[0].long()] = 1
    t1, r1, n1 = ops.pages_compact(bt, refs, [ks])
    t2, r2, n2 = ops.pages_compact(odd(bt, 0, 1), refs, [ks.clone()])
    assert torch.equal(t1, t2) and torch.equal(r1, r2) and torch.equal(n1, n2)


@pytest.mark.parametrize("rows", [1, 3])
@pytest.mark.parametrize("direct", [True, False])
def test_routed_blocks(cuda, rows, direct):
    """The decode router's selection and bias (paged.route_decode), taken as they
    are, next to the local window."""
    rng = np.random.default_rng(70)
    lens, H, Hkv, D, BS, local, topk = [900, 70, 2500, 5], 10, 10, 128, 64, 2, 4
    k, v, ks, vs, table, vals, sc = make_cache(rng, cuda, lens, Hkv, D, BS, "e4m3")
    bt, sl = torch.from_numpy(table).to(cuda), torch.tensor(lens, dtype=torch.int32, device=cuda)
    idx_q = torch.from_numpy(rng.standard_normal((len(lens) * rows, 128))).to(cuda).to(torch.bfloat16)
    k_bar = torch.from_numpy(rng.standard_normal((len(ks), 128)).astype(np.float32)).to(cuda)
    width = topk if direct else topk + 3
    out_idx = torch.full((len(lens) * rows, width), 7, dtype=torch.int32, device=cuda)
    out_bias = torch.full((len(lens) * rows, width), 7.0, device=cuda)
    paged.route_decode(idx_q=idx_q, k_bar=k_bar, block_table=bt, seq_lens=sl, image_allow=None, out_idx=out_idx,
                       out_bias=out_bias, max_block=table.shape[1], block_size=BS, local_blocks=local,
                       decode_query_len=rows, idx_scale=128 ** 0.5, prior_floor=1e-4, sigma=1.0, topm=8, budget=topk)
    assert (out_idx >= 0).any() and (out_bias != 0).any()
    q = torch.from_numpy(rng.standard_normal((len(lens) * rows, H, D))).to(cuda).to(torch.bfloat16)
    o, lse = ops.cache8_attend(q, k, v, ks, vs, bt, sl, window=local * BS, topk_idx=out_idx, bias=out_bias, lse=True)
    pos, req, _ = place(cuda, "rows", lens, rows)
    ref = O8.attend(q.double().cpu().numpy(), vals[0], vals[1], sc[0], sc[1], table, req, pos, local * BS, 0,
                    out_idx.cpu().numpy()[None], out_bias.double().cpu().numpy()[None], D ** -0.5)
    check(o, lse, ref, 2.0 ** -11)


@pytest.mark.parametrize("form", ["rows", "ragged"])
def test_tiles_in_a_graph(cuda, form):
    """The tiles' call inside a CUDA graph: lengths are read on the device, and the
    status word is cleared by each replay."""
    rng = np.random.default_rng(71)
    lens, rows, H, Hkv, D, BS = [700, 350], 300, 8, 2, 128, 64
    k, v, ks, vs, table, vals, sc = make_cache(rng, cuda, lens, Hkv, D, BS, "e4m3")
    _, _, at = place(cuda, form, lens, rows)
    assert tiles_take(N=2 * rows, R=2, H=H, Hkv=Hkv, D=D, W=11, P=20, block_size=BS,
                      **({} if form == "ragged" else {"rows_per_req": rows}))
    q = torch.from_numpy(rng.standard_normal((2 * rows, H, D))).to(cuda).to(torch.bfloat16)
    bt, ws = torch.from_numpy(table).to(cuda), torch.full((16,), 255, dtype=torch.uint8, device=cuda)
    run = lambda: ops.cache8_attend(q, k, v, ks, vs, bt, lse=True, workspace=ws, **at)  # noqa: E731
    run()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        o, lse = run()
    for n in (lens, [512, 301], [300, 17]):
        if form == "ragged":  # the second request's rows: the last of its length
            m = min(n[1], rows)
            at["cu_seqlens"].copy_(torch.tensor([0, rows, rows + m]))
            at["prefix_lens"].copy_(torch.tensor([n[0] - rows, n[1] - m]))
        else:
            at["seq_lens"].copy_(torch.tensor(n))
        ws.fill_(255)
        g.replay()
        assert (ws[:4] == 0).all()
        want = run()
        assert torch.equal(o, want[0]) and torch.equal(lse, want[1])


@pytest.mark.parametrize("R", [8191, 8192, 8193, 20000])
def test_pages_of_many_rows(cuda, R):
    """Claims of table rows on chip and, past 8192 rows, in memory; rows named
    more than once."""
    rng = np.random.default_rng(72)
    P, W, BS, n = 6000, 3, 16, 1700
    lens = np.where(rng.random(R) < 0.1, rng.integers(1, 2 * BS, R), 0).astype(np.int32)
    table, refs, free = np.full((R, W), -1, np.int32), np.zeros(P, np.int32), list(rng.permutation(P))
    for r in np.nonzero(lens)[0]:
        for b in range(-(-int(lens[r]) // BS)):
            table[r, b] = free.pop()
            refs[table[r, b]] = 1
    data = [rng.integers(0, 1 << 30, (P, 4)).astype(np.int32)]
    pool = O8.Pool(table, lens, refs, BS, data)
    i32 = lambda x: torch.tensor(np.asarray(x, np.int32), device=cuda)  # noqa: E731
    bt, sl, rf, t = i32(table), i32(lens), i32(refs), [torch.from_numpy(data[0].copy()).to(cuda)]
    full = np.nonzero(lens)[0]
    par, kid = rng.choice(full, n), rng.integers(R - 900, R, n)  # children named twice on average
    short = ops.pages_fork(i32(par), i32(kid), bt, sl, rf, t, block_size=BS)
    assert int(short) == pool.fork(par, kid)
    rows = rng.integers(0, R, n)
    rows[::3] = R - 1 - rng.integers(0, 40, len(rows[::3]))
    new = pool.lens[rows] + rng.integers(0, 30, n)
    short = ops.pages_extend(i32(rows), i32(new), bt, sl, rf, block_size=BS)
    assert int(short) == pool.extend(rows, new)
    for got, want in ((bt, pool.table), (sl, pool.lens), (rf, pool.refs), (t[0], pool.data[0])):
        np.testing.assert_array_equal(got.cpu().numpy(), want)


@pytest.mark.parametrize("rows", [1, 3, 400])
@pytest.mark.parametrize("W,P", [(0, 0), (0, 5), (3, 0)])
def test_empty_tables_and_pools(cuda, rows, W, P):
    """A table of no blocks, a cache of no pages: nothing is written or seen."""
    R, H, Hkv, D, BS = 2, 4, 2, 128, 64
    c = cache8.Cache8(P, BS, Hkv, D, device=cuda)
    bt = torch.zeros(R, W, dtype=torch.int32, device=cuda)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
    q = torch.randn(R * rows, H, D, device=cuda).to(torch.bfloat16)
    before = c.k.view(torch.uint8).clone()
    for at in (dict(seq_lens=i32([0, rows])), dict(cu_seqlens=i32([0, rows, 2 * rows]), prefix_lens=i32([0, 7]))):
        c.append(q[:, :Hkv], q[:, :Hkv], bt, **at)
        o, lse = c.attend(q, bt, lse=True, **at)
        assert (o == 0).all() and torch.isneginf(lse).all()
    assert torch.equal(before, c.k.view(torch.uint8))
