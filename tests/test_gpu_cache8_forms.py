"""The scaled 8-bit cache's attend in the forms and sizes that change kernels
(tensor-core tiles, a warp or a CTA per item, equal parts), NaN codes that some
rows see and others do not, and the example that runs append, attend and the
pages calls together.

Tolerances as in test_gpu_cache8.py: weights rounded to f16 (2^-11 relative;
2^-8 is allowed for prompt tiles, whose weights carry the value scale too), fp32
sums, the output's own rounding."""

import importlib.util
import os

import numpy as np
import pytest
import torch

from oracle import cache8 as O8
from srswa import _lib as L
from srswa import ops
from test_gpu_cache8 import check, make_cache, run_prompt, run_rows

pytestmark = pytest.mark.gpu


def tiles_take(**sizes):
    """Whether a call of these sizes goes to the tensor-core tiles (their
    workspace is the 16 bytes of the status word)."""
    d = L.Cache8Desc(rows_per_req=1, window=-1)
    for k, v in sizes.items():
        setattr(d, k, v)
    lib = L.lib()
    varlen = 0 if "rows_per_req" in sizes else 1
    lib.srswa_cache8_attend_workspace_size.restype = L.C.c_size_t
    return lib.srswa_cache8_attend_workspace_size(L.C.byref(d), varlen) == 16


@pytest.mark.parametrize("window,sinks", [(1, 0), (64, 0), (100, 4), (0, 3), (300, 130)])
def test_tiles_window_sinks(cuda, window, sinks):
    """64 features, six heads on one, pages of 32."""
    assert tiles_take(N=2477, R=3, H=6, Hkv=1, D=64, W=72, P=300, block_size=32, window=window, sinks=sinks)
    run_prompt(cuda, np.random.default_rng(40), [0, 800, 3], [1500, 900, 77], 6, 1, 64, 32, "e4m3", "bf16", window, sinks)


@pytest.mark.parametrize("code,real,D,BS,H,Hkv", [("int8", "bf16", 128, 64, 4, 2), ("e4m3", "f16", 64, 16, 14, 2)])
def test_tiles_token_major(cuda, code, real, D, BS, H, Hkv):
    assert tiles_take(N=1170, R=3, H=H, Hkv=Hkv, D=D, W=-(-1100 // BS), P=300, block_size=BS)
    run_prompt(cuda, np.random.default_rng(41), [10, 0, 31], [300, 1, 869], H, Hkv, D, BS, code, real, None, 0,
               layout="tokens")


@pytest.mark.parametrize("rows", [33, 70])
@pytest.mark.parametrize("window,sinks", [(None, 0), (90, 5)])
def test_tiles_rows_per_request(cuda, rows, window, sinks):
    """Many rows of each request in the decode form, some before its start."""
    lens = [700, rows, 5, 0, 64, 301] * 6
    assert tiles_take(N=rows * 36, R=36, H=8, Hkv=2, D=128, W=11, P=500, block_size=64, rows_per_req=rows,
                      window=-1 if window is None else window, sinks=sinks)
    run_rows(cuda, np.random.default_rng(42), lens, rows, 8, 2, 128, 64, "e4m3", "bf16", window, sinks, 0)


@pytest.mark.parametrize("rows", [1, 5, 17, 33])
@pytest.mark.parametrize("H,Hkv,D", [(4, 4, 128), (16, 4, 128), (7, 1, 64)])
def test_rows_per_request(cuda, rows, H, Hkv, D):
    """Few requests: rows of one request share passes over the keys, each pass
    with the rows of its own columns."""
    run_rows(cuda, np.random.default_rng(43), [1000, rows + 3], rows, H, Hkv, D, 32, "e4m3", "bf16", 50, 3, 0)
    run_rows(cuda, np.random.default_rng(44), [1000, rows + 3], rows, H, Hkv, D, 32, "int8", "f16", None, 0, 0)


# requests and lengths on both sides of the row kernel's rules
@pytest.mark.parametrize("R,most", [(1, 1024), (1, 1025), (40, 900), (111, 200), (112, 200), (120, 700), (200, 60),
                                    (450, 100), (2049, 40)])
def test_rows_splits(cuda, R, most):
    rng = np.random.default_rng(45)
    lens = [int(n) for n in rng.integers(0, most + 1, R)]
    lens[0] = most
    run_rows(cuda, rng, lens, 1, 8, 4, 128, 64, "e4m3", "bf16", None, 0, 0)


@pytest.mark.parametrize("what", ["k", "v"])
@pytest.mark.parametrize("form", ["draft", "tiles", "ragged tiles"])
@pytest.mark.parametrize("window,sinks", [(None, 0), (40, 2)])
def test_nan_codes(cuda, what, form, window, sinks):
    """A NaN code reaches exactly the rows that see it."""
    rng = np.random.default_rng(46)
    rows = 6 if form == "draft" else 300
    lens, H, Hkv, D, BS = [700, 350], 8, 2, 128, 64
    k, v, ks, vs, table, vals, sc = make_cache(rng, cuda, lens, Hkv, D, BS, "e4m3")
    pos = np.concatenate([n - rows + np.arange(rows) for n in lens])
    req = np.repeat([0, 1], rows)
    sick = [(0, lens[0] - rows + 3, 1, 77), (1, lens[1] - rows + 2, 0, 5)]  # request, position, head, feature
    t = (k if what == "k" else v).view(torch.uint8)
    for r, j, h, d in sick:
        t[int(table[r, j // BS]), j % BS, h, d] = 0x7F
    seen = np.zeros((2 * rows, H), bool)
    for r, j, h, _ in sick:
        sees = (req == r) & (pos >= j) & ((pos - (window or 10 ** 6) < j) | (j < sinks))
        seen[:, h * (H // Hkv):(h + 1) * (H // Hkv)] |= sees[:, None]
    q = torch.from_numpy(rng.standard_normal((2 * rows, H, D))).to(cuda).to(torch.bfloat16)
    bt = torch.from_numpy(table).to(cuda)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
    if form == "ragged tiles":
        at = dict(cu_seqlens=i32([0, rows, 2 * rows]), prefix_lens=i32([n - rows for n in lens]))
    else:
        at = dict(seq_lens=i32(lens))
    if form != "draft":
        assert tiles_take(N=2 * rows, R=2, H=H, Hkv=Hkv, D=D, W=11, P=20, block_size=BS, window=window or -1, sinks=sinks,
                          **({} if form == "ragged tiles" else {"rows_per_req": rows}))
    o, lse = ops.cache8_attend(q, k, v, ks, vs, bt, window=window, sinks=sinks, lse=True, **at)
    some = np.unique(np.concatenate([np.arange(0, 2 * rows, max(1, rows // 40)), np.arange(6), rows - 1 + np.arange(6)]))
    ref = O8.attend(q.double().cpu().numpy()[some], vals[0], vals[1], sc[0], sc[1], table, req[some], pos[some], window,
                    sinks, None, None, D ** -0.5)
    # (vals holds the codes before the NaN was put in: rows that do not see it)
    got = o.double().cpu().numpy()
    assert np.isfinite(got[~seen]).all()
    clean = ~seen[some]
    tol = 2.0 ** -8 * np.abs(ref[0]) + (2.0 ** -8 + 2.0 ** -11) * ref[2] + 1e-7
    assert (np.abs(got[some] - ref[0]) <= tol)[clean].all()
    for r, j, h, d in sick:
        mine = seen.copy()
        mine[req != r] = False
        mine[:, : h * (H // Hkv)] = False
        mine[:, (h + 1) * (H // Hkv):] = False
        assert mine.any()
        sick_part = got[mine] if what == "k" else got[mine][:, d]
        assert np.isnan(sick_part).all()


def test_cache_past_32_bits(cuda):
    """Codes, scales and table entries whose offsets pass 2^32 bytes: the same
    pages at the two ends of one large cache give the same rows."""
    Hkv, D, BS, W = 8, 128, 64, 12
    P = 2 ** 32 // (Hkv * D * BS) + 2 * W + 3
    g = torch.Generator("cuda").manual_seed(47)
    k, v = (torch.empty(P, Hkv, BS, D, dtype=torch.int8, device=cuda).transpose(1, 2) for _ in range(2))
    ks, vs = (torch.ones(P, Hkv, device=cuda) for _ in range(2))
    for t in (k, v):
        t[:W] = torch.randint(-127, 128, (W, BS, Hkv, D), dtype=torch.int8, device=cuda, generator=g)
        t[P - W:] = t[:W]
    low = torch.arange(W, dtype=torch.int32, device=cuda)[None]
    bt = torch.cat([low, P - W + low])
    for rows in (1, 300):
        q = torch.randn(rows, 16, D, device=cuda, generator=g).to(torch.bfloat16).repeat(2, 1, 1)
        sl = torch.tensor([W * BS - 9] * 2, dtype=torch.int32, device=cuda)
        o = ops.cache8_attend(q, k, v, ks, vs, bt, sl, sm_scale=1e-3)
        assert torch.isfinite(o).all() and torch.equal(o[:rows], o[rows:])
    new = torch.randn(80, Hkv, D, device=cuda, generator=g).to(torch.bfloat16).repeat(2, 1, 1)
    for n in (1, 80):
        rows = torch.cat([new[:n], new[:n]])
        ops.cache8_append(rows, rows, k, v, ks, vs, bt, sl)
        assert torch.equal(k[:W], k[P - W:]) and torch.equal(ks[:W], ks[P - W:]) and torch.equal(vs[:W], vs[P - W:])


@pytest.mark.parametrize("code", ["e4m3", "int8"])
def test_example_beams(cuda, code):
    path = os.path.join(os.path.dirname(__file__), "..", "examples", "cache8_beams.py")
    spec = importlib.util.spec_from_file_location("cache8_beams", path)
    ex = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(ex)
    r = ex.run(prompt_lens=(130, 64, 1, 63), beams=3, steps=6, window=48, sinks=2,
               code=torch.int8 if code == "int8" else torch.float8_e4m3fn)
    assert torch.equal(r["before"], r["after"])
    pages, cache, rows = r["pages"], r["cache"], r["rows"]
    lens = pages.seq_lens.cpu().numpy()
    assert [len(t) for t in r["tokens"]] == [int(lens[b]) + 1 for b in rows] == [136, 70, 7, 69]
    assert int(r["live"]) == sum(-(-int(lens[b]) // ex.BLOCK) for b in rows) == int((pages.refs > 0).sum())
    assert int(pages.refs[int(r["live"]):].sum()) == 0
    # the last draft rows against 64-bit attention over the cache's own contents
    raw = torch.stack([cache.k, cache.v]).view(torch.uint8).cpu().numpy()
    vals = O8.codes_to_values(raw, code)
    table = pages.block_table[torch.tensor(rows, device=cuda)].cpu().numpy()
    n = r["draft"]
    pos = np.concatenate([lens[b] - n + np.arange(n) for b in rows])
    o, _, a = O8.attend(r["q"].double().cpu().numpy(), vals[0], vals[1], cache.k_scale.double().cpu().numpy(),
                        cache.v_scale.double().cpu().numpy(), table, np.repeat(np.arange(len(rows)), n), pos,
                        r["window"], r["sinks"], None, None, ex.D ** -0.5)
    assert (np.abs(r["after"].double().cpu().numpy() - o) <= 2.0 ** -8 * np.abs(o) + 2.0 ** -10 * a + 1e-7).all()


@pytest.mark.parametrize("rows", [1, 4])
@pytest.mark.parametrize("lens", [[1], [300], [7, 0, 64, 900]])
def test_rows_see_nothing(cuda, rows, lens):
    """No window, no sinks, no selection: zeros and -inf."""
    o = run_rows(cuda, np.random.default_rng(48), lens, rows, 8, 2, 128, 64, "int8", "bf16", 0, 0, 0)
    assert (o == 0).all()
