"""CPU: what the block-pool entry points refuse, and the oracle's known answers."""
import numpy as np
import pytest
import torch

from nebulasd_b200 import _lib
from nebulasd_b200.block_pool import BlockPool, copy_blocks
from oracle import block_pool as oracle
from tests.block_pool_support import make_pool

L = _lib.lib
A = 4096  # a non-null, aligned address that no refused call follows


def _caches(k=A, v=A, nb=8, tiles=4, size=16, token=256):
    return [k, v, nb, tiles, size, token]


def _tables(table=A, rows=4, width=8, held=A, refs=A):
    return [table, rows, width, held, refs]


BAD_CACHES = [dict(k=None), dict(v=None), dict(k=A + 8), dict(nb=0), dict(nb=-1), dict(nb=2 ** 31), dict(tiles=0),
              dict(size=0), dict(token=0), dict(token=24), dict(tiles=2 ** 20, token=4096)]
BAD_TABLES = [dict(table=None), dict(held=None), dict(refs=None), dict(rows=0), dict(width=0),
              dict(rows=2 ** 16, width=2 ** 16)]


def _refused(rc):
    assert rc in (_lib.NEB_ERR_INVALID, _lib.NEB_ERR_UNSUPPORTED, _lib.NEB_ERR_WORKSPACE)
    assert L.neb_last_error()


def test_empty_lists_are_no_work():
    assert L.neb_copy_blocks(*_caches(), None, None, None, 0, None, None) == 0
    assert L.neb_fork_sequences(*_caches(), *_tables(), None, None, None, None, 0, None, 0, None, None) == 0
    assert L.neb_free_sequences(*_tables(), 8, None, 0, None, None) == 0


@pytest.mark.parametrize("kw", BAD_CACHES)
def test_bad_caches(kw):
    _refused(L.neb_copy_blocks(*_caches(**kw), A, A, None, 1, None, None))
    _refused(L.neb_fork_sequences(*_caches(**kw), *_tables(), A, A, A, None, 1, A, 1 << 30, None, None))
    _refused(L.neb_compact_blocks(*_caches(**kw), *_tables(), A, A, 1 << 30, None, None))


@pytest.mark.parametrize("kw", BAD_TABLES)
def test_bad_tables(kw):
    _refused(L.neb_fork_sequences(*_caches(), *_tables(**kw), A, A, A, None, 1, A, 1 << 30, None, None))
    _refused(L.neb_free_sequences(*_tables(**kw), 8, A, 1, None, None))
    _refused(L.neb_compact_blocks(*_caches(), *_tables(**kw), A, A, 1 << 30, None, None))


def test_bad_lists_and_workspaces():
    _refused(L.neb_copy_blocks(*_caches(), None, A, None, 1, None, None))
    _refused(L.neb_copy_blocks(*_caches(), A, None, None, 1, None, None))
    _refused(L.neb_copy_blocks(*_caches(), A, A, None, -1, None, None))
    fork = [*_caches(), *_tables()]
    need = L.neb_fork_workspace_bytes(8, 1)
    for lists, n, ws, size in (([None, A, A, None], 1, A, need), ([A, None, A, None], 1, A, need),
                               ([A, A, None, None], 1, A, need), ([A, A, A, None], -1, A, need),
                               ([A, A, A, None], 1, None, need), ([A, A, A, None], 1, A + 4, need),
                               ([A, A, A, None], 1, A, need - 1)):
        _refused(L.neb_fork_sequences(*fork, *lists, n, ws, size, None, None))
    _refused(L.neb_free_sequences(*_tables(), 8, None, 1, None, None))
    _refused(L.neb_free_sequences(*_tables(), 8, A, -1, None, None))
    _refused(L.neb_free_sequences(*_tables(), 0, A, 1, None, None))
    need = L.neb_compact_workspace_bytes(8)
    for new, ws, size in ((None, A, need), (A, None, need), (A, A + 4, need), (A, A, need - 1)):
        _refused(L.neb_compact_blocks(*fork, new, ws, size, None, None))
    assert L.neb_fork_workspace_bytes(0, 1) == L.neb_fork_workspace_bytes(8, -1) == 0
    assert L.neb_compact_workspace_bytes(0) == L.neb_compact_workspace_bytes(2 ** 31) == 0


def test_pools_beyond_the_plan():
    """Fork and compact plan pools of up to 2^23 blocks."""
    big, ws = 2 ** 23 + 1, 1 << 40
    assert L.neb_fork_sequences(*_caches(nb=big, tiles=1, size=1, token=16), *_tables(), A, A, A, None, 1, A, ws, None,
                                None) == _lib.NEB_ERR_UNSUPPORTED
    assert L.neb_compact_blocks(*_caches(nb=big, tiles=1, size=1, token=16), *_tables(), A, A, ws, None,
                                None) == _lib.NEB_ERR_UNSUPPORTED


def test_host_tensors_are_refused():
    k = torch.zeros((4, 1, 1, 16, 128), dtype=torch.float16)
    i = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError):
        copy_blocks(k, k.clone(), i, i)
    with pytest.raises(ValueError):
        BlockPool(k, k.clone(), i.view(1, 1), i, torch.zeros(4, dtype=torch.int32))


def test_oracle_known_answers():
    pool, groups, empty = make_pool(1, num_blocks=12, rows=4, width=4, lens=[40, 16], layers=1, heads=1, dim=8)
    a, b = groups[0][0], groups[1][0]
    c, d = empty
    start = pool.copy()
    free = [x for x in range(12) if pool.refs[x] == 0]
    # 40 tokens: two shared blocks, the third copied; 16 tokens: one shared; room for 17 takes a fresh block
    assert oracle.fork(pool, [a, b], [c, d], [40, 16], [0, 17]) == 0
    assert pool.table[c].tolist() == start.table[a, :2].tolist() + [free[0], -1]
    assert pool.table[d].tolist() == [start.table[b, 0], free[1], -1, -1]
    assert pool.refs[start.table[a, 0]] == 2 and pool.refs[free[0]] == 1 and pool.held[[c, d]].tolist() == [3, 2]
    assert np.array_equal(pool.k[free[0], :, :, :8], start.k[start.table[a, 2], :, :, :8])
    assert np.array_equal(pool.k[free[0], :, :, 8:], start.k[free[0], :, :, 8:])
    assert oracle.free(pool, [c, d, c]) == 0
    assert np.array_equal(pool.table, start.table) and np.array_equal(pool.refs, start.refs)
    bits, new = oracle.compact(pool)
    assert bits == 0 and pool.refs.tolist() == [1] * 4 + [0] * 8
    assert sorted(pool.table[pool.table >= 0].tolist()) == [0, 1, 2, 3]
    for r in (a, b):
        for j in range(start.held[r]):
            assert np.array_equal(pool.k[pool.table[r, j]], start.k[start.table[r, j]])
            assert new[start.table[r, j]] == pool.table[r, j]
    assert oracle.fork(pool, [a], [c], [49], None) == oracle.INVALID
    assert oracle.fork(pool, [a], [c], [0], [65]) == oracle.WIDTH
    assert oracle.fork(pool, [a, a], [c, c], [16, 16], None) == oracle.INVALID and pool.held[c] == 1


def test_oracle_counts_every_row_of_a_broken_pool():
    """A block in use that is counted as free is shared, given out as a fresh one too, and reported."""
    pool, groups, empty = make_pool(2, num_blocks=6, rows=4, width=4, lens=[40], layers=1, heads=1, dim=8)
    a, lost = groups[0][0], int(pool.table[groups[0][0], 1])
    pool.refs[lost] = 0
    for order in ([0, 1], [1, 0]):
        now, (c, d) = pool.copy(), empty[:2]
        lens, caps = np.array([32, 0])[order], np.array([32, 64])[order]  # takes all four free blocks
        assert oracle.fork(now, [a, a], [c, d], lens, caps) == oracle.REFS
        assert now.refs[lost] == 2 == sum(int((now.table[r] == lost).sum()) for r in (c, d))
    pool.refs[lost], last = 1, pool.table[a, 2]
    pool.refs[last] = 0
    now = pool.copy()
    assert oracle.fork(now, [a], [empty[0]], [40]) == oracle.REFS
    assert np.array_equal(now.k, pool.k)  # nothing copied from a block that may be given out


def test_error_words_that_are_missing():
    _refused(L.neb_take_error_bits(None, A, None))
    _refused(L.neb_take_error_bits(A, None, None))
