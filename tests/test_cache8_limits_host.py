"""Sizes of the scaled 8-bit cache's calls at the limits of their arguments (no
GPU needed: the sizes are computed on the host)."""

import ctypes as C

import pytest

from srswa import _lib as L
from test_cache8_host import desc


def workspace(varlen, **kw):
    return L.lib().srswa_cache8_attend_workspace_size(C.byref(desc(**kw)), varlen)


@pytest.mark.parametrize("kw,some", [(dict(N=900, W=200), True), (dict(N=4, W=500, K=3), True), (dict(N=4), False)])
def test_varlen_workspace_needs_no_rows_per_req(kw, some):
    """rows_per_req is the other row form's; a varlen descriptor may leave it 0."""
    want = workspace(1, **kw)
    assert workspace(1, rows_per_req=0, **kw) == want
    assert workspace(0, rows_per_req=0, **kw) == 0
    assert (want > 0) == some


END = 2 ** 63 - 1


@pytest.mark.parametrize("varlen,kw", [(0, {}), (0, dict(W=4000)), (0, dict(W=4000, K=8)), (1, dict(N=900, W=200))])
def test_plans_at_the_end_of_the_arguments(varlen, kw):
    """Windows, sinks and part counts of any size are as good as all there is."""
    assert workspace(varlen, window=END, **kw) == workspace(varlen, window=-1, **kw)
    assert workspace(varlen, window=END, sinks=END, **kw) == workspace(varlen, window=-1, **kw)
    assert workspace(varlen, window=512, sinks=END, **kw) == workspace(varlen, window=512, sinks=2 ** 30, **kw)
    parts = (kw.get("W", 5) + kw.get("K", 0)) * 2  # units of 32 keys in pages of 64
    for n in (2 ** 62, 2 ** 62 + 1, END):
        assert 0 < workspace(varlen, nsplit=n, **kw) == workspace(varlen, nsplit=parts, **kw)


def test_refusals_of_sizes():
    d = lambda **kw: L.lib().srswa_cache8_attend(C.byref(desc(**kw)), *[1 << 20] * 6, 1 << 20, None, None, 1 << 20, None,  # noqa: E731
                                                 1 << 20, None, None, 0, None)
    assert d(K=513) == d(K=END) == d(W=1 << 31) == d(P=1 << 31) == L.ETOOLARGE


def lone(**kw):
    """Tensors whose dimensions of one element have odd strides."""
    import torch
    def odd(t, dim, stride):
        s = list(t.stride())
        s[dim] = stride
        return t.as_strided(t.shape, s)
    P, BS, D, R = 5, 64, 128, 1
    k, v = (torch.zeros(P, BS, 1, D, dtype=torch.uint8).view(torch.float8_e4m3fn) for _ in range(2))
    q = torch.zeros(1, 1, D, dtype=torch.bfloat16)
    a = dict(q=odd(odd(q, 0, 3), 1, 5), k=odd(k, 2, 7), v=odd(v, 2, 9), ks=odd(torch.ones(P, 1), 1, 3), vs=torch.ones(P, 1),
             bt=odd(torch.zeros(R, 4, dtype=torch.int32), 0, 1), lens=torch.ones(1, dtype=torch.int32))
    a.update(kw)
    return [a[x] for x in ("q", "k", "v", "ks", "vs", "bt", "lens")]


def test_strides_of_single_elements_do_not_count():
    """One row, one head, one request: their strides are never used.  (The call
    then stops at the CPU tensors.)"""
    from srswa import ops
    with pytest.raises(L.SrswaError, match="CUDA"):
        ops.cache8_attend(*lone())
    q, k, v, ks, vs, bt, lens = lone()
    with pytest.raises(L.SrswaError, match="CUDA"):
        ops.cache8_append(q, q, k, v, ks, vs, bt, lens)


def test_block_size_past_32_bits_is_refused():
    lib, X = L.lib(), 1 << 20
    for bs in (1 << 31, END):
        assert lib.srswa_pages_free(X, 1, X, 4, 4, 4, X, X, 8, bs, None) == L.ETOOLARGE
        assert lib.srswa_pages_extend(X, X, 1, X, 4, 4, 4, X, X, 8, bs, X, X, 1 << 30, None) == L.ETOOLARGE
        assert lib.srswa_pages_fork(X, X, 1, X, 4, 4, 4, X, X, 8, bs, None, 0, X, X, 1 << 30, None) == L.ETOOLARGE
