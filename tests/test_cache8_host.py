"""Scaled 8-bit cache and page calls: refusals before anything is launched (no
GPU needed: the C entries check before any CUDA call, the wrappers before the
library), and the oracle's own code tables."""

import ctypes as C

import numpy as np
import pytest
import torch

from oracle import cache8 as O8
from srswa import _lib as L
from srswa import ops

X = 1 << 20  # a 16-byte-aligned address that is never read


def desc(**kw):
    d = L.Cache8Desc()
    base = dict(N=4, R=4, H=8, Hkv=2, D=128, P=10, W=5, block_size=64, rows_per_req=1, window=-1, sinks=0, K=0,
                sm_scale=0.1, q_dtype=L.BF16, kv_dtype=L.F8E4M3, out_dtype=L.BF16, idx_is64=0, s_qn=1024, s_qh=128,
                s_on=1024, s_oh=128, s_page=16384, s_pos=128, s_head=8192, s_scale=2, s_bt=5)
    base.update(kw)
    for k, v in base.items():
        setattr(d, k, v)
    return d


def attend(d, q=X, table=X, lens=X, cu=None, pre=None, sel=None, ws=None, n=0, out=X):
    return L.lib().srswa_cache8_attend(C.byref(d), q, X, X, X, X, table, lens, cu, pre, sel, None, out, None, ws, n, None)


def append(d, k=X, lens=X, cu=None, pre=None):
    return L.lib().srswa_cache8_append(C.byref(d), k, X, X, X, X, X, X, lens, cu, pre, None)


@pytest.mark.parametrize("kw,rc", [
    (dict(D=96), L.EUNSUPPORTED), (dict(D=256), L.EUNSUPPORTED), (dict(kv_dtype=L.F8E5M2), L.EUNSUPPORTED),
    (dict(kv_dtype=L.BF16), L.EUNSUPPORTED), (dict(block_size=24), L.EUNSUPPORTED), (dict(block_size=0), L.EINVAL),
    (dict(block_size=2048), L.ETOOLARGE), (dict(N=5), L.EINVAL), (dict(N=-1), L.EINVAL), (dict(R=-1), L.EINVAL),
    (dict(rows_per_req=0), L.EINVAL), (dict(s_page=16392), L.EALIGN), (dict(s_pos=130), L.EALIGN), (dict(Hkv=0), L.EINVAL)])
def test_c_refusals_common(kw, rc):
    assert attend(desc(**kw)) == rc
    assert append(desc(**kw)) == rc


@pytest.mark.parametrize("kw,rc", [
    (dict(H=9), L.EINVAL), (dict(H=0), L.EINVAL), (dict(K=-1), L.EINVAL), (dict(sinks=-1), L.EINVAL),
    (dict(K=3), L.EINVAL), (dict(q_dtype=L.F32), L.EUNSUPPORTED), (dict(out_dtype=L.F16), L.EUNSUPPORTED),
    (dict(s_qh=132), L.EALIGN), (dict(s_on=1028), L.EALIGN), (dict(H=1 << 17, Hkv=2), L.ETOOLARGE)])
def test_c_refusals_attend(kw, rc):
    assert attend(desc(**kw)) == rc


def test_c_refusals_pointers():
    lib = L.lib()
    d = desc()
    assert lib.srswa_cache8_attend(None, *([None] * 14), 0, None) == L.EINVAL
    assert lib.srswa_cache8_append(None, *([None] * 11)) == L.EINVAL
    assert attend(d, q=None) == L.EINVAL and attend(d, q=X + 2) == L.EALIGN and attend(d, table=None) == L.EINVAL
    assert attend(d, lens=None) == L.EINVAL and attend(d, cu=X) == L.EINVAL and attend(d, out=None) == L.EINVAL
    assert append(d, k=None) == L.EINVAL and append(d, k=X + 8) == L.EALIGN and append(desc(s_qn=1025)) == L.EALIGN
    assert attend(desc(N=0, R=0)) == 0


def test_c_refusals_pages():
    lib = L.lib()
    t = (L.PageTensor * 17)()
    for x in t:
        x.base, x.page_bytes, x.stride_bytes = X, 64, 64
    big = 1 << 30
    fork = lambda n=1, R=4, W=4, s_bt=4, P=8, BS=64, nt=1, ws=X, nb=big, par=X, tt=t: lib.srswa_pages_fork(  # noqa: E731
        par, X, n, X, s_bt, R, W, X, X, P, BS, tt, nt, X, ws, nb, None)
    assert fork(n=-1) == L.EINVAL and fork(R=0) == L.EINVAL and fork(s_bt=3) == L.EINVAL and fork(BS=0) == L.EINVAL
    assert fork(nt=17) == L.ETOOLARGE and fork(n=1 << 17) == L.ETOOLARGE and fork(ws=None) == L.EWORKSPACE
    assert fork(nb=8) == L.EWORKSPACE and fork(ws=X + 2) == L.EALIGN and fork(par=None) == L.EINVAL
    t[0].stride_bytes = 32
    assert fork() == L.EINVAL
    assert lib.srswa_pages_free(None, 1, X, 4, 4, 4, X, X, 8, 64, None) == L.EINVAL
    assert lib.srswa_pages_free(X, 0, X, 4, 4, 4, X, X, 8, 64, None) == 0
    assert lib.srswa_pages_extend(X, None, 1, X, 4, 4, 4, X, X, 8, 64, X, X, big, None) == L.EINVAL
    assert lib.srswa_pages_compact(X, 4, 4, 4, X, 8, t, 0, None, 4, X, X, X, big, None) == L.EINVAL
    assert lib.srswa_pages_compact(X, 4, 4, 4, X, 8, t, 0, X, 4, X, X, X, 8, None) == L.EWORKSPACE


def tensors(P=6, BS=64, Hkv=2, D=128, R=3, W=2, H=4, N=3, dt=torch.float8_e4m3fn):
    c = torch.zeros(P, BS, Hkv, D, dtype=torch.uint8).view(dt)
    return dict(q=torch.zeros(N, H, D, dtype=torch.bfloat16), k_cache=c, v_cache=c.clone(), k_scale=torch.ones(P, Hkv),
                v_scale=torch.ones(P, Hkv), block_table=torch.zeros(R, W, dtype=torch.int32),
                seq_lens=torch.ones(R, dtype=torch.int32))


@pytest.mark.parametrize("change,err", [
    (dict(q=torch.zeros(3, 4, 128)), NotImplementedError), (dict(q=torch.zeros(3, 4, 64, dtype=torch.bfloat16)), ValueError),
    (dict(q=torch.zeros(3, 5, 128, dtype=torch.bfloat16)), ValueError),
    (dict(q=torch.zeros(4, 4, 128, dtype=torch.bfloat16)), ValueError),
    (dict(k_cache=torch.zeros(6, 64, 2, 128, dtype=torch.bfloat16)), ValueError),
    (dict(k_cache=torch.zeros(6, 64, 2, 128, dtype=torch.bfloat16), v_cache=torch.zeros(6, 64, 2, 128, dtype=torch.bfloat16)),
     NotImplementedError),
    (dict(k_scale=torch.ones(6, 3)), ValueError), (dict(v_scale=torch.ones(6, 2, dtype=torch.float64)), ValueError),
    (dict(block_table=torch.zeros(3, 2, dtype=torch.int64)), ValueError), (dict(seq_lens=None), ValueError),
    (dict(seq_lens=torch.ones(3, dtype=torch.int64)), ValueError), (dict(seq_lens=torch.ones(2, dtype=torch.int32)), ValueError),
    (dict(cu_seqlens=torch.zeros(4, dtype=torch.int32)), ValueError), (dict(window=-2), ValueError),
    (dict(topk_idx=torch.zeros(3, 2)), NotImplementedError), (dict(topk_idx=torch.zeros(2, 2, dtype=torch.int32)), ValueError),
    (dict(bias=torch.zeros(3, 2)), ValueError),
    (dict(topk_idx=torch.zeros(3, 2, dtype=torch.int32), bias=torch.zeros(3, 3)), ValueError),
    (dict(out=torch.zeros(3, 4, 128, dtype=torch.float16)), ValueError), ({}, L.SrswaError)])
def test_attend_wrapper_refusals(change, err):
    a = tensors()
    a.update(change)
    with pytest.raises(err):  # the last: CPU tensors, no fallback
        ops.cache8_attend(a.pop("q"), a.pop("k_cache"), a.pop("v_cache"), a.pop("k_scale"), a.pop("v_scale"),
                          a.pop("block_table"), a.pop("seq_lens"), **a)


def test_append_wrapper_refusals():
    a = tensors()
    x = torch.zeros(3, 2, 128, dtype=torch.bfloat16)
    rest = (a["k_cache"], a["v_cache"], a["k_scale"], a["v_scale"], a["block_table"], a["seq_lens"])
    with pytest.raises(ValueError):
        ops.cache8_append(x, x.float(), *rest)
    with pytest.raises(ValueError):
        ops.cache8_append(x[:, :1], x[:, :1], *rest)
    with pytest.raises(NotImplementedError):
        ops.cache8_append(x.double(), x.double(), *rest)
    with pytest.raises(L.SrswaError):
        ops.cache8_append(x, x, *rest)


def test_pages_wrapper_refusals():
    i = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    bt, lens, refs = i(3, 2), i(3), i(6)
    with pytest.raises(ValueError):
        ops.pages_free(i(2).long(), bt, lens, refs, block_size=64)
    with pytest.raises(ValueError):
        ops.pages_free(i(2), bt.long(), lens, refs, block_size=64)
    with pytest.raises(ValueError):
        ops.pages_extend(i(2), i(3), bt, lens, refs, block_size=64)
    with pytest.raises(ValueError):
        ops.pages_fork(i(2), i(2), bt, i(4), refs, [], block_size=64)
    with pytest.raises(ValueError):  # not indexed by the pages
        ops.pages_fork(i(2), i(2), bt, lens, refs, [torch.zeros(5, 3)], block_size=64)
    with pytest.raises(ValueError):  # a page with gaps
        ops.pages_compact(bt, refs, [torch.zeros(6, 4, 8)[:, :, :4]])
    with pytest.raises(ValueError):
        ops.pages_compact(bt, refs, [], out_table=i(3, 3))


def test_page_tensor_layouts():
    """Pages may be permuted inside, and lie apart; bytes and strides follow."""
    t = torch.zeros(6, 2, 64, 16, dtype=torch.bfloat16).transpose(1, 2)
    x = torch.zeros(6, 2, 3, 4, 5).permute(0, 3, 1, 4, 2)
    runs = L.bind().page_runs([t, torch.zeros(6, 10)[:, :3], torch.zeros(6), x, torch.zeros(6, 1, 7)], 6)
    assert runs[0] == (t.data_ptr(), 4096, 4096) and runs[1][1:] == (12, 40) and runs[2][1:] == (4, 4)
    assert runs[3][1:] == (480, 480) and runs[4][1:] == (28, 28)
    with pytest.raises(ValueError):
        L.bind().page_runs([torch.zeros(6, 4, 8)[:, :, ::2]], 6)


def test_oracle_codes_match_torch():
    v = O8.e4m3_values()
    t = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    np.testing.assert_array_equal(v, t)
    y = np.concatenate([np.random.default_rng(0).standard_normal(20000) * 50, v[np.isfinite(v)], [2 ** -10, 3 * 2.0 ** -10, 1e-9]])
    y = y.astype(np.float32)
    want = torch.from_numpy(y).clamp(-448, 448).to(torch.float8_e4m3fn).double().numpy()
    np.testing.assert_array_equal(O8.round_to_code(y, "e4m3"), want)
    assert O8.pow2_scale(448.0, 448.0) == 1.0 and O8.pow2_scale(448.1, 448.0) == 2.0 and O8.pow2_scale(0.0, 127.0) == 2.0 ** -64
