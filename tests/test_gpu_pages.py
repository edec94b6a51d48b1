"""Pages of a cache: free, extend, fork and compact against one-step-at-a-time
restatements (oracle/cache8.Pool).  Whole numbers and copies: equal."""

import numpy as np
import pytest
import torch

from oracle.cache8 import Pool

pytestmark = pytest.mark.gpu

from srswa import cache8, ops  # noqa: E402


def i32(x, dev):
    return torch.tensor(np.asarray(x, np.int32), device=dev)


def make(rng, dev, lens, P, W, BS, shared=0):
    """A table of random pages (some prefixes shared), its counts, and page
    data of several widths: 16-byte runs, 40-byte and 3-byte pages, a view in
    another order, a pool with gaps between pages."""
    R = len(lens)
    table = np.full((R, W), -1, np.int32)
    order = list(rng.permutation(P))
    for r, n in enumerate(lens):
        need = -(-n // BS)
        if shared and r and n >= BS * 2 and lens[r - 1] >= BS * 2:
            table[r, :2] = table[r - 1, :2]
            need0 = 2
        else:
            need0 = 0
        for b in range(need0, need):
            table[r, b] = order.pop()
    refs = np.zeros(P, np.int32)
    for p in table[table >= 0]:
        refs[p] += 1
    data = [rng.integers(0, 255, (P, 5, 2048)).astype(np.uint8), rng.integers(0, 9, (P, 10)).astype(np.int32),
            rng.integers(0, 255, (P, 3)).astype(np.uint8), rng.integers(0, 255, (P, 4, 6, 16)).astype(np.uint8),
            rng.integers(0, 255, (P, 70000)).astype(np.uint8)]
    t = [torch.from_numpy(d.copy()).to(dev) for d in data]
    t[3] = t[3].transpose(1, 2).contiguous().transpose(1, 2)
    wide = torch.zeros(P, 70016, dtype=torch.uint8, device=dev)
    wide[:, :70000] = t[4]
    t[4] = wide[:, :70000]
    pool = Pool(table, np.array(lens, np.int32), refs, BS, data)
    return pool, i32(table, dev), i32(lens, dev), i32(refs, dev), t


def same(pool, table, lens, refs, tensors, pages=None):
    np.testing.assert_array_equal(table.cpu().numpy(), pool.table)
    if lens is not None:
        np.testing.assert_array_equal(lens.cpu().numpy(), pool.lens)
    np.testing.assert_array_equal(refs.cpu().numpy(), pool.refs)
    for t, d in zip(tensors, pool.data):
        np.testing.assert_array_equal(t.cpu().numpy(), d)


LENS = [0, 1, 63, 64, 65, 200, 0, 640, 129, 0, 0, 0]


@pytest.mark.parametrize("rows", [[], [3], [7, 2, 7, 0, -1, 12, 5, 2], list(range(12))])
def test_free(cuda, rows):
    rng = np.random.default_rng(1)
    pool, table, lens, refs, t = make(rng, cuda, LENS, 80, 12, 64, shared=1)
    ops.pages_free(i32(rows, cuda), table, lens, refs, block_size=64)
    pool.free(rows)
    same(pool, table, lens, refs, t)


@pytest.mark.parametrize("P", [24, 27, 30, 60])
def test_extend(cuda, P):
    rng = np.random.default_rng(2)
    pool, table, lens, refs, t = make(rng, cuda, LENS, P, 12, 64)
    rows = [4, 9, 0, 4, 50, -3, 7, 1, 2, 10]
    new = [129, 64, 0, 700, 10, 10, 600, 13 * 64, 64, 200]
    short = ops.pages_extend(i32(rows, cuda), i32(new, cuda), table, lens, refs, block_size=64)
    assert int(short) == pool.extend(rows, new)
    same(pool, table, lens, refs, t)


@pytest.mark.parametrize("P", [22, 23, 25, 60])
@pytest.mark.parametrize("shared", [0, 1])
def test_fork(cuda, P, shared):
    rng = np.random.default_rng(3)
    pool, table, lens, refs, t = make(rng, cuda, LENS, P, 12, 64, shared)
    par = [5, 3, 0, 1, 5, 8, 4, 99, 2]
    kid = [6, 9, 10, 11, 9, 2, -1, 10, 10]
    short = ops.pages_fork(i32(par, cuda), i32(kid, cuda), table, lens, refs, t, block_size=64)
    assert int(short) == pool.fork(par, kid)
    same(pool, table, lens, refs, t)


@pytest.mark.parametrize("n", [1, 1500])
def test_fork_many(cuda, n):
    """More items than one CTA has threads, and more free pages than one pass of the scan."""
    rng = np.random.default_rng(4)
    lens = rng.integers(1, 200, n).tolist() + [0] * n
    P = 9000
    pool, table, lens_t, refs, t = make(rng, cuda, lens, P, 4, 64)
    pool.data, t = pool.data[1:3], t[1:3]
    par, kid = rng.permutation(n), n + rng.permutation(n)
    short = ops.pages_fork(i32(par, cuda), i32(kid, cuda), table, lens_t, refs, t, block_size=64)
    assert int(short) == pool.fork(par, kid)
    same(pool, table, lens_t, refs, t)


@pytest.mark.parametrize("inplace", [False, True])
@pytest.mark.parametrize("gone", [[], [7], [5, 8], [1, 2, 3, 4, 5, 7, 8]])
def test_compact(cuda, inplace, gone):
    rng = np.random.default_rng(5)
    pool, table, lens, refs, t = make(rng, cuda, LENS, 50, 12, 64, shared=1)
    ops.pages_free(i32(gone, cuda), table, lens, refs, block_size=64)
    pool.free(gone)
    kw = dict(out_table=table, out_refs=refs) if inplace else {}
    was = table.clone(), refs.clone()
    nt, nr, live = ops.pages_compact(table, refs, t, **kw)
    assert int(live) == pool.compact()
    same(pool, nt, None, nr, t)
    if not inplace:
        assert torch.equal(table, was[0]) and torch.equal(refs, was[1])


@pytest.mark.parametrize("P", [1, 1023, 1024, 5000, 70001])
def test_compact_sizes(cuda, P):
    rng = np.random.default_rng(6)
    refs = (rng.random(P) < 0.4).astype(np.int32) * rng.integers(1, 4, P).astype(np.int32)
    table = rng.permutation(P).astype(np.int32)[: max(1, P // 2)].reshape(1, -1)
    data = [rng.integers(0, 1 << 30, (P, 4)).astype(np.int32)]
    pool = Pool(table, np.zeros(1, np.int32), refs, 64, data)
    t = [torch.from_numpy(data[0].copy()).to(cuda)]
    nt, nr, live = ops.pages_compact(i32(table, cuda), i32(refs, cuda), t)
    assert int(live) == pool.compact()
    same(pool, nt, None, nr, t)


def test_random_life(cuda):
    """Extend, fork, free and compact at random over one pool: every step equal."""
    rng = np.random.default_rng(7)
    R, W, P, BS = 20, 10, 60, 16
    table = cache8.PageTable(R, W, P, BS, device=cuda)
    data = [rng.integers(0, 1 << 30, (P, 8)).astype(np.int32)]
    table.tensors = [torch.from_numpy(data[0].copy()).to(cuda)]
    pool = Pool(np.full((R, W), -1, np.int32), np.zeros(R, np.int32), np.zeros(P, np.int32), BS, data)
    for _ in range(120):
        what = rng.integers(0, 4)
        rows = rng.integers(0, R, rng.integers(1, 6))
        if what == 0:
            new = pool.lens[rows] + rng.integers(0, 70, len(rows))
            assert int(table.extend(i32(rows, cuda), i32(new, cuda))) == pool.extend(rows, new)
        elif what == 1:
            kids = rng.integers(0, R, len(rows))
            assert int(table.fork(i32(rows, cuda), i32(kids, cuda))) == pool.fork(rows, kids)
        elif what == 2:
            table.free(i32(rows[:2], cuda))
            pool.free(rows[:2])
        else:
            assert int(table.compact()) == pool.compact()
        same(pool, table.block_table, table.seq_lens, table.refs, table.tensors)
        used, count = np.unique(pool.table[pool.table >= 0], return_counts=True)
        assert (pool.refs[used] == count).all() and pool.refs.sum() == count.sum()
