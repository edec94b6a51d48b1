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
