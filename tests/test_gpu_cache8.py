"""Scaled 8-bit paged cache: append and attend against plain 64-bit
restatements (oracle/cache8.py).

Tolerances, from the arithmetic.  Append: scales are powers of two and every
code is one correctly rounded value, so codes and scales are equal.  Attend:
out is sum(p v) / sum(p).  A relative error u of the weights moves it by at most
u * A, A = the weighted mean of |v|; the logits are fp32 sums of exact products
(|error| <= 130 * 2^-24 * sum |q k| * scale, under 1e-4 here, so 2^-11 * A and
1e-4 on lse); weights are rounded to f16 (u = 2^-11) for single rows, to bf16
(2^-8) for prompt tiles; out is rounded to its type (2^-8 |o| bf16, 2^-11 |o|
f16)."""

import math

import numpy as np
import pytest
import torch

from oracle import cache8 as O8

pytestmark = pytest.mark.gpu

from srswa import cache8, ops  # noqa: E402

CODE = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}
REAL = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def make_cache(rng, dev, lens, Hkv, D, BS, code, layout="heads", extra=3):
    """A cache whose unwritten slots and unused pages hold NaN (e4m3) or -128
    codes and NaN scales, with its block table and its plain values."""
    R = len(lens)
    used = [-(-n // BS) for n in lens]
    W = max(max(used), 1)
    P = sum(used) + extra
    order = rng.permutation(P)
    table = np.full((R, W), -1, np.int32)
    at = 0
    raw = np.full((2, P, BS, Hkv, D), 0x7F if code == "e4m3" else 0x80, np.uint8)
    scale = np.full((2, P, Hkv), np.nan, np.float32)
    for r, n in enumerate(lens):
        table[r, : used[r]] = order[at: at + used[r]]
        at += used[r]
        for b in range(used[r]):
            m = min(BS, n - b * BS)
            c = rng.integers(0, 256, (2, m, Hkv, D)).astype(np.uint8)
            if code == "e4m3":
                c = (c & 0x80) | np.clip(rng.normal(60, 12, c.shape), 0, 126).astype(np.uint8)
            else:
                c = np.clip(rng.normal(0, 35, c.shape), -127, 127).astype(np.int8).view(np.uint8)
            raw[:, table[r, b], :m] = c
            scale[:, table[r, b]] = np.exp2(rng.integers(-3, 3, (2, Hkv))) / (2.0 if code == "e4m3" else 35.0)
    t = torch.from_numpy(raw).to(dev)
    if layout == "heads":  # (page, head) tiles contiguous
        t = t.transpose(2, 3).contiguous().transpose(2, 3)
    k, v = t[0].view(CODE[code]), t[1].view(CODE[code])
    ks, vs = torch.from_numpy(scale[0].copy()).to(dev), torch.from_numpy(scale[1].copy()).to(dev)
    return k, v, ks, vs, table, O8.codes_to_values(raw, code), scale.astype(np.float64)


def check(out, lse, ref, u_weights):
    o, l, a = ref
    got = out.double().cpu().numpy()
    tol = U[out.dtype] * np.abs(o) + (u_weights + 2.0 ** -11) * a + 1e-7
    assert np.isfinite(got).all()
    worst = (np.abs(got - o) / tol).max()
    assert worst <= 1.0, worst
    g = lse.double().cpu().numpy()
    assert np.array_equal(np.isneginf(g), np.isneginf(l))
    fin = np.isfinite(l)
    assert fin.sum() == 0 or np.abs(g[fin] - l[fin]).max() <= 1e-4


def run_rows(dev, rng, lens, rows, H, Hkv, D, BS, code, real, window, sinks, K, layout="heads", idx=torch.int32,
             per_head=False, use_bias=True, out_dtype=None, nsplit=0, scale=None, odd_sel=True):
    k, v, ks, vs, table, vals, sc = make_cache(rng, dev, lens, Hkv, D, BS, code, layout)
    N = len(lens) * rows
    q = torch.from_numpy(rng.standard_normal((N, H, D))).to(dev).to(REAL[real])
    topk = bias = None
    if K:
        nh = Hkv if per_head else 1
        W = table.shape[1]
        topk = rng.integers(-1, W + (2 if odd_sel else 0), (nh, N, K))  # repeats, -1, past the table, in the window
        bias = rng.standard_normal((nh, N, K)).astype(np.float32)
    pos = np.concatenate([n - rows + np.arange(rows) for n in lens])
    req = np.repeat(np.arange(len(lens)), rows)
    sm = 1 / math.sqrt(D) if scale is None else scale
    ref = O8.attend(q.double().cpu().numpy(), vals[0], vals[1], sc[0], sc[1], table, req, pos, window, sinks, topk,
                    bias if use_bias else None, sm)
    out = None if out_dtype is None else torch.empty(N, H, D, device=dev, dtype=out_dtype)
    o, lse = ops.cache8_attend(q, k, v, ks, vs, torch.from_numpy(table).to(dev),
                               torch.tensor(lens, dtype=torch.int32, device=dev), window=window, sinks=sinks,
                               topk_idx=None if topk is None else torch.from_numpy(topk).to(dev).to(idx),
                               bias=None if bias is None or not use_bias else torch.from_numpy(bias).to(dev),
                               sm_scale=scale, out=out, lse=True, nsplit=nsplit)
    check(o, lse, ref, 2.0 ** -11)
    return o


LENS = [1, 15, 16, 17, 63, 64, 65, 200, 511, 777]


@pytest.mark.parametrize("code", ["e4m3", "int8"])
@pytest.mark.parametrize("real", ["bf16", "f16"])
@pytest.mark.parametrize("D,BS,H,Hkv", [(128, 64, 10, 10), (64, 32, 14, 2), (128, 16, 8, 1), (128, 128, 24, 2),
                                        (64, 48, 5, 5)])
def test_rows_dense(cuda, code, real, D, BS, H, Hkv):
    run_rows(cuda, np.random.default_rng(1), LENS, 1, H, Hkv, D, BS, code, real, None, 0, 0)


@pytest.mark.parametrize("window,sinks", [(0, 4), (1, 0), (100, 0), (64, 70), (333, 1), (5000, 3), (128, 64)])
@pytest.mark.parametrize("code,D,BS", [("e4m3", 128, 64), ("int8", 64, 32)])
def test_rows_window_sinks(cuda, window, sinks, code, D, BS):
    run_rows(cuda, np.random.default_rng(2), LENS, 1, 6, 2, D, BS, code, "bf16", window, sinks, 0)


@pytest.mark.parametrize("window,sinks,K", [(128, 0, 8), (0, 0, 4), (70, 5, 3), (200, 100, 40), (None, 0, 4), (64, 0, 1)])
@pytest.mark.parametrize("per_head,idx,use_bias", [(False, torch.int32, True), (True, torch.int64, True),
                                                   (True, torch.int32, False)])
def test_rows_selected(cuda, window, sinks, K, per_head, idx, use_bias):
    run_rows(cuda, np.random.default_rng(3), LENS, 1, 8, 4, 128, 64, "e4m3", "bf16", window, sinks, K, per_head=per_head,
             idx=idx, use_bias=use_bias)


@pytest.mark.parametrize("rows", [2, 3, 5])
@pytest.mark.parametrize("layout", ["heads", "tokens"])
def test_rows_several_per_request(cuda, rows, layout):
    # a request shorter than its rows: the first of them see nothing
    run_rows(cuda, np.random.default_rng(4), [1, 2, 9, 64, 66, 130, 400], rows, 4, 2, 128, 64, "int8", "f16", 90, 2, 4,
             layout=layout)


def test_rows_nothing_visible(cuda):
    o = run_rows(cuda, np.random.default_rng(5), [3, 70, 200], 1, 4, 4, 128, 64, "e4m3", "bf16", 0, 0, 0)
    assert (o == 0).all()
    run_rows(cuda, np.random.default_rng(5), [0, 0, 40], 1, 4, 4, 128, 64, "e4m3", "bf16", None, 0, 0)


@pytest.mark.parametrize("nsplit", [1, 2, 5, 16, 64])
def test_rows_split(cuda, nsplit):
    run_rows(cuda, np.random.default_rng(6), [1, 40, 700, 3000], 1, 8, 2, 128, 64, "e4m3", "bf16", None, 0, 0,
             nsplit=nsplit)
    run_rows(cuda, np.random.default_rng(6), [1, 40, 700, 3000], 1, 4, 4, 64, 64, "int8", "f16", 130, 20, 6,
             nsplit=nsplit)


def test_rows_fp32_out_and_scale(cuda):
    run_rows(cuda, np.random.default_rng(7), LENS, 1, 4, 2, 128, 64, "e4m3", "bf16", 128, 4, 4, out_dtype=torch.float32)
    run_rows(cuda, np.random.default_rng(7), LENS, 1, 4, 2, 128, 64, "e4m3", "bf16", 128, 4, 4, scale=-0.05)


@pytest.mark.parametrize("qs", [2.0 ** -40, 2.0 ** 30])
def test_rows_query_range(cuda, qs):
    """bf16 queries far outside f16's range (the scale brings the logits back)."""
    rng = np.random.default_rng(8)
    k, v, ks, vs, table, vals, sc = make_cache(rng, cuda, [150], 2, 128, 64, "e4m3")
    q = (torch.from_numpy(rng.standard_normal((1, 4, 128))).to(cuda) * qs).to(torch.bfloat16)
    sm = 0.088 / qs
    ref = O8.attend(q.double().cpu().numpy(), vals[0], vals[1], sc[0], sc[1], table, [0], [149], None, 0, None, None, sm)
    o, lse = ops.cache8_attend(q, k, v, ks, vs, torch.from_numpy(table).to(cuda),
                               torch.tensor([150], dtype=torch.int32, device=cuda), sm_scale=sm, lse=True)
    check(o, lse, ref, 2.0 ** -11)


def test_rows_strided_inputs_and_stream(cuda):
    """q and out as slices of wider tensors, a table with a wider row, another stream."""
    rng = np.random.default_rng(9)
    lens = [130, 64, 300]
    k, v, ks, vs, table, vals, sc = make_cache(rng, cuda, lens, 2, 128, 64, "e4m3")
    big = torch.from_numpy(rng.standard_normal((3, 9, 128))).to(cuda).to(torch.bfloat16)
    q = big[:, 2:6]
    wide = torch.full((3, table.shape[1] + 7), -1, dtype=torch.int32, device=cuda)
    wide[:, : table.shape[1]] = torch.from_numpy(table).to(cuda)
    obig = torch.zeros(3, 9, 128, device=cuda, dtype=torch.bfloat16)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        o, lse = ops.cache8_attend(q, k, v, ks, vs, wide[:, : table.shape[1]],
                                   torch.tensor(lens, dtype=torch.int32, device=cuda), window=100, sinks=4,
                                   out=obig[:, 3:7], lse=True)
    st.synchronize()
    ref = O8.attend(q.double().cpu().numpy(), vals[0], vals[1], sc[0], sc[1], table, [0, 1, 2], np.array(lens) - 1, 100, 4,
                    None, None, 128 ** -0.5)
    check(o, lse, ref, 2.0 ** -11)
    assert (obig[:, :3] == 0).all() and (obig[:, 7:] == 0).all()


def test_rows_missing_pages(cuda):
    """Table entries that name no page: their tokens are not seen."""
    rng = np.random.default_rng(10)
    k, v, ks, vs, table, vals, sc = make_cache(rng, cuda, [400, 400], 2, 128, 64, "e4m3")
    table[0, 1], table[1, 3] = -1, 10 ** 6
    q = torch.from_numpy(rng.standard_normal((2, 4, 128))).to(cuda).to(torch.bfloat16)
    ref = O8.attend(q.double().cpu().numpy(), vals[0], vals[1], sc[0], sc[1], table, [0, 1], [399, 399], None, 0, None, None,
                    128 ** -0.5)
    o, lse = ops.cache8_attend(q, k, v, ks, vs, torch.from_numpy(table).to(cuda),
                               torch.tensor([400, 400], dtype=torch.int32, device=cuda), lse=True)
    check(o, lse, ref, 2.0 ** -11)


def test_rows_repeatable(cuda):
    rng = np.random.default_rng(11)
    k, v, ks, vs, table, _, _ = make_cache(rng, cuda, [5000, 900], 2, 128, 64, "e4m3")
    q = torch.from_numpy(rng.standard_normal((2, 8, 128))).to(cuda).to(torch.bfloat16)
    bt, sl = torch.from_numpy(table).to(cuda), torch.tensor([5000, 900], dtype=torch.int32, device=cuda)
    first = ops.cache8_attend(q, k, v, ks, vs, bt, sl, lse=True)
    for _ in range(5):
        again = ops.cache8_attend(q, k, v, ks, vs, bt, sl, lse=True)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


def test_rows_empty_calls(cuda):
    c = cache8.Cache8(4, 64, 2, 128, device=cuda)
    bt = torch.zeros(0, 3, dtype=torch.int32, device=cuda)
    o = c.attend(torch.empty(0, 4, 128, device=cuda, dtype=torch.bfloat16), bt, torch.zeros(0, dtype=torch.int32, device=cuda))
    assert o.shape == (0, 4, 128)
    c.append(*(torch.empty(0, 2, 128, device=cuda, dtype=torch.bfloat16) for _ in range(2)), bt,
             torch.zeros(0, dtype=torch.int32, device=cuda))


# ------------------------------------------------------------------ prompts
def run_prompt(dev, rng, pre, new, H, Hkv, D, BS, code, real, window, sinks, K=0, layout="heads"):
    lens = [a + b for a, b in zip(pre, new)]
    k, v, ks, vs, table, vals, sc = make_cache(rng, dev, lens, Hkv, D, BS, code, layout)
    N = sum(new)
    q = torch.from_numpy(rng.standard_normal((N, H, D))).to(dev).to(REAL[real])
    pos = np.concatenate([a + np.arange(n) for a, n in zip(pre, new)])
    req = np.repeat(np.arange(len(new)), new)
    topk = bias = None
    if K:
        topk = rng.integers(-1, table.shape[1] + 1, (1, N, K))
        bias = rng.standard_normal((1, N, K)).astype(np.float32)
    some = np.unique(np.concatenate([np.arange(N)[:: max(1, N // 60)], np.array([0, N - 1]), np.cumsum(new)[:-1] % N]))
    ref = O8.attend(q.double().cpu().numpy()[some], vals[0], vals[1], sc[0], sc[1], table, req[some], pos[some], window,
                    sinks, None if topk is None else topk[:, some], None if bias is None else bias[:, some],
                    D ** -0.5)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    o, lse = ops.cache8_attend(q, k, v, ks, vs, torch.from_numpy(table).to(dev), cu_seqlens=i32([0, *np.cumsum(new)]),
                               prefix_lens=i32(pre), window=window, sinks=sinks,
                               topk_idx=None if topk is None else torch.from_numpy(topk).to(dev),
                               bias=None if bias is None else torch.from_numpy(bias).to(dev), lse=True)
    assert torch.isfinite(o).all()
    check(o[some], lse[some], ref, 2.0 ** -8)


@pytest.mark.parametrize("code,real", [("e4m3", "bf16"), ("int8", "f16"), ("e4m3", "f16"), ("int8", "bf16")])
@pytest.mark.parametrize("D,BS,H,Hkv", [(128, 64, 4, 4), (64, 32, 14, 2), (128, 16, 8, 1), (128, 128, 24, 2),
                                        (64, 48, 3, 3)])
def test_prompt_dense(cuda, code, real, D, BS, H, Hkv):
    run_prompt(cuda, np.random.default_rng(20), [0, 5, 64, 0, 127, 300], [1, 130, 0, 257, 128, 333], H, Hkv, D, BS, code,
               real, None, 0)


@pytest.mark.parametrize("window,sinks", [(1, 0), (64, 0), (100, 4), (128, 64), (0, 3), (300, 130), (0, 0)])
@pytest.mark.parametrize("D,BS,H,Hkv", [(128, 64, 4, 4), (64, 32, 6, 1)])
def test_prompt_window_sinks(cuda, window, sinks, D, BS, H, Hkv):
    run_prompt(cuda, np.random.default_rng(21), [0, 700, 3], [400, 131, 1], H, Hkv, D, BS, "e4m3", "bf16", window, sinks)


def test_prompt_token_major(cuda):
    run_prompt(cuda, np.random.default_rng(22), [10, 0], [300, 77], 4, 2, 128, 64, "int8", "bf16", 200, 7, layout="tokens")


def test_prompt_selected(cuda):
    run_prompt(cuda, np.random.default_rng(23), [100, 0, 500], [150, 200, 3], 4, 2, 128, 64, "e4m3", "bf16", 100, 4, K=5)


def test_prompt_rows_are_decode_rows(cuda):
    """One new token per request, in the varlen form."""
    run_prompt(cuda, np.random.default_rng(24), [0, 63, 64, 900], [1, 1, 1, 1], 8, 2, 128, 64, "e4m3", "bf16", None, 0)


def test_prompt_longer(cuda):
    run_prompt(cuda, np.random.default_rng(25), [1500], [1000], 2, 2, 128, 64, "e4m3", "bf16", None, 0)


# ------------------------------------------------------------------- append
def run_append(dev, rng, start, count, Hkv, D, BS, code, real, layout="heads", values=None, rows_form=False, scales="pow2"):
    lens = list(start)
    total = [a + n for a, n in zip(start, count)]
    R, W = len(start), max(max(-(-t // BS) for t in total), 1)
    P = R * W + 2
    table = rng.permutation(P)[: R * W].astype(np.int32).reshape(R, W)
    raw = np.full((2, P, BS, Hkv, D), 0x7F if code == "e4m3" else 0x80, np.uint8)
    scale = np.full((2, P, Hkv), np.nan)
    for r, n in enumerate(lens):
        for b in range(-(-n // BS)):
            m = min(BS, n - b * BS)
            c = rng.integers(0, 256, (2, m, Hkv, D)).astype(np.uint8)
            c = np.where(c & 127 == 127, 1, c).astype(np.uint8) if code == "e4m3" else np.where(c == 128, 1, c).astype(np.uint8)
            raw[:, table[r, b], :m] = c
            scale[:, table[r, b]] = np.exp2(rng.integers(-10, 2, (2, Hkv)))
            if scales == "any":
                scale[:, table[r, b]] *= rng.uniform(0.5, 2, (2, Hkv)).astype(np.float32)
    scale = scale.astype(np.float32)
    x = rng.standard_normal((2, sum(count), Hkv, D)) * np.exp2(rng.integers(-4, 4, (2, 1, Hkv, 1)))
    if values is not None:
        x = values(x)
    xt = torch.from_numpy(x).to(dev).to(REAL[real])
    t = torch.from_numpy(raw).to(dev)
    if layout == "heads":
        t = t.transpose(2, 3).contiguous().transpose(2, 3)
    k, v = t[0].view(CODE[code]), t[1].view(CODE[code])
    st = torch.from_numpy(scale).to(dev)
    bt = torch.from_numpy(table).to(dev)
    i32 = lambda y: torch.tensor(y, dtype=torch.int32, device=dev)  # noqa: E731
    if rows_form:
        ops.cache8_append(xt[0], xt[1], k, v, st[0], st[1], bt, i32(total))
    else:
        ops.cache8_append(xt[0], xt[1], k, v, st[0], st[1], bt, cu_seqlens=i32([0, *np.cumsum(count)]), prefix_lens=i32(start))
    for w in range(2):
        vals, sc = O8.codes_to_values(raw[w], code), scale[w].astype(np.float64)
        O8.append(xt[w].double().cpu().numpy(), vals, sc, table, start, count, BS, code)
        got = O8.codes_to_values(np.ascontiguousarray((k, v)[w].view(torch.uint8).cpu().numpy()), code)
        np.testing.assert_array_equal(st[w].double().cpu().numpy(), sc)
        np.testing.assert_array_equal(got, vals)


@pytest.mark.parametrize("code", ["e4m3", "int8"])
@pytest.mark.parametrize("real", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("D,BS,Hkv,layout", [(128, 64, 3, "heads"), (64, 16, 2, "tokens"), (128, 128, 1, "heads"),
                                             (64, 48, 5, "heads"), (128, 32, 10, "tokens")])
def test_append_varlen(cuda, code, real, D, BS, Hkv, layout):
    run_append(cuda, np.random.default_rng(30), [0, 5, 63, 64, 0, 100, 1], [1, 130, 2, 64, 0, 29, 300], Hkv, D, BS, code,
               real, layout)


@pytest.mark.parametrize("code", ["e4m3", "int8"])
@pytest.mark.parametrize("rows", [1, 4])
def test_append_rows(cuda, code, rows):
    start = [0, 1, 15, 62, 63, 64, 127, 200]
    run_append(cuda, np.random.default_rng(31), start, [rows] * len(start), 4, 128, 64, code, "bf16", rows_form=True)


def test_append_many_requests(cuda):
    rng = np.random.default_rng(32)
    run_append(cuda, rng, rng.integers(0, 150, 300).tolist(), [1] * 300, 2, 64, 32, "e4m3", "bf16", rows_form=True)


@pytest.mark.parametrize("code", ["e4m3", "int8"])
def test_append_scale_of_any_value(cuda, code):
    """Earlier scales that are not powers of two (another writer's): kept or outgrown."""
    run_append(cuda, np.random.default_rng(33), [3, 40, 63], [2, 50, 1], 4, 128, 64, code, "f32", scales="any")


@pytest.mark.parametrize("code", ["e4m3", "int8"])
def test_append_special_values(cuda, code):
    def values(x):
        x[:, 0] = 0.0
        x[:, 1, 0] = 0.0
        x[:, 1, 0, 0] = np.nan
        x[:, 2, 0, 1:3] = np.inf, -np.inf
        x[:, 3] = 1e-38
        x[:, 4, 0, 0] = 3e38
        x[:, 5, 0] = 448.0 if code == "e4m3" else 127.0
        x[:, 6, 0] = np.nextafter(np.float32(448.0 if code == "e4m3" else 127.0), np.float32(1e9))
        x[:, 7, 0] = 1e-45
        return x
    # each token a request of its own, so that each sets its own scale
    run_append(cuda, np.random.default_rng(34), [0] * 8, [1] * 8, 2, 64, 32, code, "f32", values=values)


def test_append_growth_keeps_e4m3(cuda):
    """A page written token by token, magnitudes rising: e4m3 codes shift exactly, int8 stays within one step."""
    rng = np.random.default_rng(35)
    x = rng.standard_normal((64, 2, 64)).astype(np.float32) * np.exp2(np.arange(64) / 8).astype(np.float32)[:, None, None]
    xt = torch.from_numpy(x).to(cuda).float()
    for code in ("e4m3", "int8"):
        c = cache8.Cache8(2, 64, 2, 64, dtype=CODE[code], device=cuda)
        bt = torch.tensor([[1]], dtype=torch.int32, device=cuda)
        for i in range(64):
            c.append(xt[i: i + 1], xt[i: i + 1], bt, torch.tensor([i + 1], dtype=torch.int32, device=cuda))
        s = c.k_scale[1].double().cpu().numpy()
        got = c.k[1].float().double().cpu().numpy() * s[:, None]
        if code == "int8":
            assert np.abs(got - x).max() <= s.max()
        else:  # half a step of the value, and one step of the smallest exponents
            assert (np.abs(got - x) <= 2.0 ** -4 * np.abs(x) + s[:, None] * 2.0 ** -9).all()


def test_append_missing_pages(cuda):
    c = cache8.Cache8(3, 64, 2, 128, device=cuda)
    before = c.k.view(torch.uint8).clone()
    x = torch.randn(2, 2, 128, device=cuda).to(torch.bfloat16)
    bt = torch.tensor([[-1], [3]], dtype=torch.int32, device=cuda)
    c.append(x, x, bt, torch.tensor([1, 1], dtype=torch.int32, device=cuda))
    c.append(x, x, bt, torch.tensor([65, 0], dtype=torch.int32, device=cuda))  # past the table; no position
    assert torch.equal(before, c.k.view(torch.uint8))


def test_graph_capture(cuda):
    """Append and attend inside a CUDA graph: positions are read on the device."""
    rng = np.random.default_rng(36)
    c = cache8.Cache8(8, 64, 2, 128, device=cuda)
    bt = torch.arange(8, dtype=torch.int32, device=cuda).view(1, 8)
    sl = torch.tensor([1], dtype=torch.int32, device=cuda)
    kv = torch.zeros(2, 1, 2, 128, device=cuda, dtype=torch.bfloat16)
    q = torch.from_numpy(rng.standard_normal((1, 4, 128))).to(cuda).to(torch.bfloat16)
    c.append(kv[0], kv[1], bt, sl)
    out = c.attend(q, bt, sl, window=100, sinks=4)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        c.append(kv[0], kv[1], bt, sl)
        out = c.attend(q, bt, sl, window=100, sinks=4)
    plain = cache8.Cache8(8, 64, 2, 128, device=cuda)
    for i in range(150):
        x = torch.from_numpy(rng.standard_normal((2, 1, 2, 128))).to(cuda).to(torch.bfloat16)
        kv.copy_(x)
        sl.fill_(i + 1)
        g.replay()
        plain.append(x[0], x[1], bt, sl)
    want = plain.attend(q, bt, sl, window=100, sinks=4)
    assert torch.equal(out, want)
