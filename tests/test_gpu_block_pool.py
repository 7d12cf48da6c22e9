"""GPU: blocks copied, forked, freed and compacted, bit for bit against the oracle."""
import numpy as np
import pytest
import torch

from oracle import block_pool as oracle
from tests.block_pool_support import ints, make_pool, same, to_device

pytestmark = pytest.mark.gpu

# layers, heads, block size, head dim, dtype
SHAPES = [(2, 2, 16, 128, torch.float16), (1, 1, 1, 8, torch.float16), (5, 3, 16, 64, torch.bfloat16),
          (1, 7, 5, 24, torch.float32), (36, 8, 16, 128, torch.float16)]


# ------------------------------------------------------------------------ copy
@pytest.mark.parametrize("layers,heads,size,dim,dtype", SHAPES)
@pytest.mark.parametrize("pairs", [1, 3, 20])
@pytest.mark.parametrize("partial", [False, True])
def test_copy(layers, heads, size, dim, dtype, pairs, partial, cuda):
    from nebulasd_b200.block_pool import copy_blocks, workspace_errors
    pool, _, _ = make_pool(pairs, num_blocks=41, rows=1, width=1, lens=[], layers=layers, heads=heads, size=size,
                           dim=dim, dtype=dtype)
    rng = np.random.default_rng(pairs)
    perm = rng.permutation(41)
    src, dst = perm[:pairs].tolist(), perm[-pairs:].tolist()
    tokens = rng.integers(0, size + 1, size=pairs).tolist() if partial else None
    h = to_device(pool, cuda, dtype)
    workspace_errors()
    copy_blocks(h.k_cache, h.v_cache, ints(src, cuda), ints(dst, cuda), ints(tokens, cuda) if partial else None)
    assert oracle.copy_blocks(pool.k, pool.v, src, dst, tokens) == 0 == workspace_errors()
    same(h, pool)


def test_copy_one_source_to_many(cuda):
    from nebulasd_b200.block_pool import copy_blocks, workspace_errors
    pool, _, _ = make_pool(4, num_blocks=700, rows=1, width=1, lens=[], layers=1, heads=1)
    h = to_device(pool, cuda)
    dst = [b for b in range(700) if b != 333]
    copy_blocks(h.k_cache, h.v_cache, ints([333] * 699, cuda), ints(dst, cuda))
    assert oracle.copy_blocks(pool.k, pool.v, [333] * 699, dst) == 0 == workspace_errors()
    same(h, pool)


@pytest.mark.parametrize("filler", [0, 400])
def test_copy_leaves_out_conflicts_and_bad_pairs(filler, cuda):
    """The same index twice, chains, a block onto itself, indices and counts out of range; with `filler` good pairs."""
    from nebulasd_b200.block_pool import copy_blocks, workspace_errors
    pool, _, _ = make_pool(5, num_blocks=20 + 2 * filler, rows=1, width=1, lens=[], layers=1, heads=2)
    src = [0, 1, 2, 3, 4, 5, -1, 6, 20 + 2 * filler, 7, 8, 9, 2 ** 31 - 1] + [20 + i for i in range(filler)]
    dst = [10, 10, 11, 2, 4, 12, 13, -7, 14, 15, 16, 17, -2 ** 31] + [20 + filler + i for i in range(filler)]
    tok = [16] * 10 + [17, -1, 3] + [5] * filler
    h = to_device(pool, cuda)
    workspace_errors()
    copy_blocks(h.k_cache, h.v_cache, ints(src, cuda), ints(dst, cuda), ints(tok, cuda))
    want = oracle.copy_blocks(pool.k, pool.v, src, dst, tok)
    assert want == oracle.BLOCK | oracle.INVALID | oracle.CONFLICT == workspace_errors()
    same(h, pool)
    copy_blocks(h.k_cache, h.v_cache, ints([], cuda), ints([], cuda))
    assert workspace_errors() == 0
    same(h, pool)


def test_copy_far_blocks(cuda):
    """Blocks whose bytes lie beyond 2^32."""
    from nebulasd_b200.block_pool import copy_blocks
    k = torch.zeros((20000, 8, 8, 16, 128), dtype=torch.float16, device=cuda)  # 5.2 GB
    v = torch.zeros_like(k)
    k[0], v[0], k[19998], v[19998] = 1.0, 2.0, 3.0, 4.0
    copy_blocks(k, v, ints([0, 19998], cuda), ints([19999, 1], cuda))
    assert bool((k[19999] == 1).all()) and bool((v[19999] == 2).all())
    assert bool((k[1] == 3).all()) and bool((v[1] == 4).all())
    assert int((k[2:19998] != 0).sum()) == 0


def test_error_bits_of_another_stream_are_kept(cuda):
    """Bits are read while a call on another stream records its own: every read takes some, none is lost."""
    from nebulasd_b200.block_pool import copy_blocks, workspace_errors
    pool, _, _ = make_pool(24, num_blocks=8, rows=1, width=1, lens=[], layers=1, heads=1)
    h = to_device(pool, cuda)
    bad, clash = (ints([0, 1], cuda), ints([4, 9], cuda)), (ints([2, 3], cuda), ints([6, 6], cuda))
    want = pool.copy()
    assert oracle.copy_blocks(want.k, want.v, [0, 1], [4, 9]) | oracle.copy_blocks(want.k, want.v, [2, 3], [6, 6]) \
        == oracle.BLOCK | oracle.CONFLICT
    workspace_errors()
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for turn in range(300):
        with torch.cuda.stream(side):
            torch.cuda._sleep(1500 * (turn % 50))  # up to some 40 us
            copy_blocks(h.k_cache, h.v_cache, *clash)
        copy_blocks(h.k_cache, h.v_cache, *bad)
        bits = workspace_errors()
        assert bits & oracle.BLOCK
        side.synchronize()
        assert bits | workspace_errors() == oracle.BLOCK | oracle.CONFLICT
    same(h, want)


# ------------------------------------------------------------------------ fork
def _fork(h, pool, parents, children, lens, caps, dev):
    h.fork(ints(parents, dev), ints(children, dev), ints(lens, dev), None if caps is None else ints(caps, dev))
    assert oracle.fork(pool, parents, children, lens, caps) == h.errors()
    same(h, pool)


@pytest.mark.parametrize("layers,heads,size,dim,dtype", SHAPES)
@pytest.mark.parametrize("room", [None, 0, 33])
def test_fork(layers, heads, size, dim, dtype, room, cuda):
    lens = [1, size - 1 or 1, size, size + 1, 3 * size, 3 * size + 2, 5 * size]
    pool, groups, empty = make_pool(3, num_blocks=150, rows=40, width=60, lens=lens, fan=2, layers=layers, heads=heads,
                                    size=size, dim=dim, dtype=dtype)
    h = to_device(pool, cuda, dtype)
    parents = [groups[i % 7][i % 2] for i in range(16)]
    at = [max(1, lens[i % 7] - i // 7) for i in range(16)]           # at the end, and before it
    caps = None if room is None else [n + min(room, 2 * size) for n in at]
    _fork(h, pool, parents, empty[:16], at, caps, cuda)
    # forks of forks
    _fork(h, pool, empty[:4], empty[16:20], at[:4], caps and caps[:4], cuda)


def test_fork_allocates_and_refuses(cuda):
    pool, groups, empty = make_pool(8, num_blocks=64, rows=20, width=9, lens=[40, 70, 16], layers=1, heads=1)
    a, b, c = (g[0] for g in groups)
    h = to_device(pool, cuda)
    e = empty
    # length 0: a new sequence, whatever the parent; no room: an empty one
    _fork(h, pool, [-5, 2 ** 31 - 1, a], [e[0], e[1], e[2]], [0, 0, 0], [40, 0, 16], cuda)
    # rows out of range, in use, listed twice; parent out of range; too long; too wide; negative
    _fork(h, pool, [a, a, a, a, a, 20, -1, a, a, c, b, a, a, a],
          [-1, 20, b, e[3], e[3], e[4], e[4], e[4], e[5], e[6], e[7], e[8], e[9], e[3]],
          [16, 16, 16, 17, 40, 3, 3, 49, -1, 17, 70, 0, 5, 16],
          [0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 145, -3, 144, 0], cuda)
    # an empty row as a parent, and one that becomes a child in the same call
    _fork(h, pool, [e[10], a], [e[11], e[10]], [4, 33], None, cuda)


def test_fork_spends_the_free_blocks_in_order(cuda):
    pool, groups, empty = make_pool(9, num_blocks=30, rows=16, width=12, lens=[100, 100, 100], layers=1, heads=2)
    h = to_device(pool, cuda)
    a = groups[0][0]
    # 9 free: 4 + 4 granted, 3 refused, then 0 needed granted, 1 refused (its turn is past the end)
    _fork(h, pool, [a] * 5, empty[:5], [96, 100, 96, 96, 97], [160, 160, 144, 96, 97], cuda)
    assert h.seq_blocks[ints(empty[:5], cuda).long()].tolist() == [10, 10, 0, 6, 0]
    pool2, _, e2 = make_pool(9, num_blocks=5, rows=3, width=5, lens=[80], layers=1, heads=1)
    h2 = to_device(pool2, cuda)  # none free
    _fork(h2, pool2, [0], [e2[0]], [0], [1], cuda)


def test_fork_reports_broken_tables(cuda):
    pool, groups, empty = make_pool(11, num_blocks=40, rows=6, width=8, lens=[70, 70], layers=1, heads=1)
    a, b = groups[0][0], groups[1][0]
    pool.table[a, 1], pool.table[a, 2] = 40, -9
    pool.table[b, 4] = 2 ** 31 - 1
    h = to_device(pool, cuda)
    _fork(h, pool, [a, b], empty[:2], [64, 70], None, cuda)


def test_fork_from_blocks_without_a_count(cuda):
    """Blocks in use that are counted as free (or less), handed out as fresh ones by the same call: shared, counted
    and reported whatever comes first, and not copied from."""
    broken, groups, empty = make_pool(14, num_blocks=40, rows=24, width=9, lens=[100, 100, 100], layers=3, heads=2)
    a, b, c = (g[0] for g in groups)
    broken.refs[broken.table[a, [2, 6]]] = 0   # 100 tokens: six full blocks and four tokens
    broken.refs[broken.table[b, [0, 6]]] = -2, -1
    parents, lens = [a, b, c, a, a, b, c, a, 0, 0], [100, 100, 100, 50, 100, 97, 16, 99, 0, 0]
    caps = [128, 128, 101, 80, 128, 97, 80, 144, 32, 32]
    for turn in range(30):
        pool, h = broken.copy(), to_device(broken, cuda)
        _fork(h, pool, parents, empty[:10], lens, caps, cuda)
        # all free blocks are spent: one counted zero is left, the -2 that two rows have raised
        assert int((pool.refs == 0).sum()) == 1 and pool.refs[pool.table[a, 2]] == 4 + 1
    # each alone: a shared block, a partial one
    for row, n in ((a, 48), (a, 99), (b, 16), (b, 97)):
        pool, h = broken.copy(), to_device(broken, cuda)
        h.fork(ints([row], cuda), ints(empty[:1], cuda), ints([n], cuda))
        assert oracle.fork(pool, [row], empty[:1], [n]) == h.errors() == oracle.REFS
        same(h, pool)


@pytest.mark.parametrize("n,num_blocks", [(300, 20000), (1500, 135168), (64, 1000003)])
def test_fork_many(n, num_blocks, cuda):
    rng = np.random.default_rng(n)
    lens = rng.integers(1, 400, size=20).tolist()
    pool, groups, empty = make_pool(n, num_blocks=num_blocks, rows=20 + n, width=40, lens=lens, layers=1, heads=1,
                                    dim=8, size=16)
    h = to_device(pool, cuda)
    pick = rng.integers(0, 20, size=n)
    at = [int(rng.integers(0, lens[i] + 1)) for i in pick]
    caps = [int(x) for x in rng.integers(0, 640, size=n)]
    _fork(h, pool, [groups[i][0] for i in pick], empty, at, caps, cuda)


def test_fork_many_that_meet(cuda):
    """More children than the plan takes at a time: rows listed again, parents that are children and the reverse, on
    both sides of the first 1,024; the free blocks run out among the later ones."""
    n = 2300
    pool, groups, empty = make_pool(17, num_blocks=3621, rows=2320, width=12, lens=[70, 100, 33, 160], layers=1, heads=1,
                                    dim=8)
    rng = np.random.default_rng(17)
    parents = [groups[i][0] for i in rng.integers(0, 4, size=n)]
    children, lens = empty[:n], [int(x) for x in rng.integers(1, 34, size=n)]
    caps = [x + int(y) for x, y in zip(lens, rng.integers(0, 32, size=n))]
    for i, j in ((1030, 3), (1500, 1023), (1024, 1023), (2100, 1500), (700, 20), (2290, 5)):
        children[i] = children[j]                       # listed again
    for i, j in ((1100, 8), (1800, 1700), (900, 30)):
        parents[i] = children[j]                        # a child of this call
    for i, j in ((9, 1200), (1050, 2000), (40, 60)):
        parents[i] = children[j]                        # one of a later entry
    lens[2200], caps[2200], lens[2250], caps[2250] = 16, 16, 0, 0  # need nothing, and get it
    h = to_device(pool, cuda)
    _fork(h, pool, parents, children, lens, caps, cuda)
    held = pool.held[children]
    assert (held[:1800] > 0).mean() > 0.98 and not held[2150:2200].any() and held[2200] == 1
    assert int((pool.refs == 0).sum()) < 6


# ------------------------------------------------------------------------ free
def _free(h, pool, rows, dev):
    h.free(ints(rows, dev))
    assert oracle.free(pool, rows) == h.errors()
    same(h, pool)


def test_free(cuda):
    lens = [1, 16, 17, 100, 640, 0, 33]
    pool, groups, empty = make_pool(2, num_blocks=120, rows=30, width=41, lens=lens, fan=3, layers=1, heads=1)
    h = to_device(pool, cuda)
    _free(h, pool, [groups[4][0], groups[3][1], groups[0][2], groups[5][0]], cuda)
    _free(h, pool, [groups[4][0], groups[4][1], groups[4][1], groups[2][0], empty[0], -1, 30], cuda)  # twice, empty, bad
    _free(h, pool, [], cuda)
    _free(h, pool, [r for g in groups for r in g], cuda)
    assert int(h.ref_counts.abs().sum()) == 0


def test_free_reports_broken_pools(cuda):
    pool, groups, _ = make_pool(6, num_blocks=40, rows=8, width=6, lens=[90, 90, 90, 50], fan=1, layers=1, heads=1)
    a, b, c, d = (g[0] for g in groups)
    pool.table[a, 2], pool.table[a, 3] = -1, 40
    pool.refs[pool.table[b, 1]] = 0
    pool.refs[pool.table[b, 2]] = -4
    pool.held[c], pool.held[d] = 7, -2
    h = to_device(pool, cuda)
    _free(h, pool, [a, b, c, d], cuda)


@pytest.mark.parametrize("rows,width", [(500, 77), (40, 8200)])
def test_free_many(rows, width, cuda):
    rng = np.random.default_rng(rows)
    lens = rng.integers(0, width * 16 // 3, size=rows // 4).tolist()
    pool, groups, _ = make_pool(rows, num_blocks=sum(-(-n // 16) + 2 for n in lens) + 10, rows=rows, width=width,
                                lens=lens, fan=2, layers=1, heads=1, dim=8)
    h = to_device(pool, cuda)
    _free(h, pool, [int(r) for r in rng.permutation(rows)[:rows // 2]], cuda)


# --------------------------------------------------------------------- compact
def _compact(h, pool):
    new = h.compact()
    bits, want = oracle.compact(pool)
    assert np.array_equal(new.cpu().numpy(), want)
    assert bits == h.errors()
    same(h, pool)


@pytest.mark.parametrize("layers,heads,size,dim,dtype", SHAPES)
def test_compact(layers, heads, size, dim, dtype, cuda):
    pool, groups, _ = make_pool(7, num_blocks=90, rows=30, width=12, lens=[size * 7 + 1, 3, size * 4, 0, size * 9],
                                fan=2, layers=layers, heads=heads, size=size, dim=dim, dtype=dtype)
    h = to_device(pool, cuda, dtype)
    _compact(h, pool)
    _compact(h, pool)  # nothing left to move
    assert bool((h.ref_counts[:int((h.ref_counts > 0).sum())] > 0).all())


@pytest.mark.parametrize("num_blocks,lens", [(1, []), (1, [16]), (7, []), (40, [640]), (33, [16] * 32), (2, [5])])
def test_compact_full_and_empty(num_blocks, lens, cuda):
    pool, _, _ = make_pool(num_blocks, num_blocks=num_blocks, rows=max(1, len(lens)), width=40, lens=lens, layers=1,
                           heads=1)
    _compact(to_device(pool, cuda), pool)


@pytest.mark.parametrize("num_blocks,live", [(20000, 9000), (135168, 70000), (300007, 20000)])
def test_compact_many(num_blocks, live, cuda):
    rng = np.random.default_rng(live)
    lens = (rng.integers(1, 2 * 16 * live // 40, size=40) * 0.95).astype(int).tolist()
    pool, _, _ = make_pool(live, num_blocks=num_blocks, rows=41, width=max(lens) // 16 + 2, lens=lens, layers=1, heads=1,
                           dim=8)
    _compact(to_device(pool, cuda), pool)


def test_compact_reports_broken_tables(cuda):
    pool, groups, _ = make_pool(13, num_blocks=60, rows=6, width=8, lens=[90, 90, 90], layers=1, heads=1)
    a, b, c = (g[0] for g in groups)
    pool.table[a, 1], pool.table[a, 2] = 60, -3
    pool.refs[pool.table[b, 0]] = 0  # in use and counted as free
    pool.held[c] = 3                 # entries beyond it are nobody's
    _compact(to_device(pool, cuda), pool)


# -------------------------------------------------------------------- together
def test_refusals_on_the_device(cuda):
    from nebulasd_b200.block_pool import BlockPool, copy_blocks
    pool, _, _ = make_pool(1, num_blocks=8, rows=4, width=4, lens=[16], layers=1, heads=1)
    h = to_device(pool, cuda)
    i = ints([1, 2], cuda)
    with pytest.raises(ValueError):
        copy_blocks(h.k_cache, h.v_cache[:4], i, i)
    with pytest.raises(ValueError):
        copy_blocks(h.k_cache.transpose(3, 4), h.v_cache.transpose(3, 4), i, i)
    for src, dst, tok in ((i.long(), i, None), (i, i[:1], None), (i, i, i[:1]), (i.cpu(), i, None), (i, i.view(1, 2), None),
                          (ints([1, 2, 3, 4], cuda)[::2], i, None)):
        with pytest.raises(ValueError):
            copy_blocks(h.k_cache, h.v_cache, src, dst, tok)
    for args in ((i, i, i.float()), (i[:1], i, i), (i, i, i, i[:1]), (i.cpu(), i, i)):
        with pytest.raises(ValueError):
            h.fork(*args)
    with pytest.raises(ValueError):
        h.free(i.long())
    k, v, t, s, r = h.k_cache, h.v_cache, h.block_table, h.seq_blocks, h.ref_counts
    for args in ((k, v, t.long(), s, r), (k, v, t, s[:2], r), (k, v, t, s, r[:7]), (k, v, t.t(), s, r),
                 (k, v.bfloat16(), t, s, r), (k[..., :4].contiguous(), v[..., :4].contiguous(), t, s, r)):
        with pytest.raises(ValueError):
            BlockPool(*args)
    same(h, pool)


@pytest.mark.parametrize("name", ["k_cache", "v_cache", "block_table", "seq_blocks", "ref_counts"])
def test_replaced_tensors_are_refused(name, cuda):
    """A pool whose tensor has other memory, or another tensor, neither reads nor writes where it was."""
    pool, groups, empty = make_pool(23, num_blocks=12, rows=4, width=4, lens=[40], layers=1, heads=1)
    h = to_device(pool, cuda)
    child, n = ints(empty[:1], cuda), ints([40], cuda)
    t, old = getattr(h, name), getattr(h, name).data
    other = old.clone()
    calls = (lambda: h.fork(ints(groups[0], cuda), child, n), lambda: h.free(child), h.compact)
    for put, back in ((lambda: setattr(t, "data", other), lambda: setattr(t, "data", old)),
                      (lambda: setattr(h, name, other), lambda: setattr(h, name, t))):
        put()
        for call in calls:
            with pytest.raises(ValueError, match="replaced"):
                call()
        back()
        same(h, pool)
    _fork(h, pool, groups[0], empty[:1], [40], None, cuda)


def test_captured_round(cuda):
    """Fork, copy, free and compact captured twice (two graphs of one pool), replayed with new lists in place."""
    from nebulasd_b200.block_pool import copy_blocks, workspace_errors
    pool, groups, empty = make_pool(21, num_blocks=200, rows=24, width=12, lens=[100, 70, 33, 150], fan=2, layers=2,
                                    heads=1)
    h = to_device(pool, cuda)
    workspace_errors()
    lists = [ints([0] * 4, cuda) for _ in range(4)]
    src, dst = ints([0, 0], cuda), ints([0, 0], cuda)
    rows = ints([0, 0], cuda)
    graphs, news = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            h.fork(*lists)
            copy_blocks(h.k_cache, h.v_cache, src, dst)
            h.free(rows)
            news.append(h.compact())
        graphs.append(g)
    rng = np.random.default_rng(2)
    same(h, pool)
    for turn in range(6):
        live = [r for r in range(24) if pool.held[r] > 0]
        parents = rng.choice(live, size=4).tolist()
        children = [r for r in range(24) if pool.held[r] == 0][:4]
        lens = [int(rng.integers(1, 16 * pool.held[r] + 1)) for r in parents]
        caps = [n + int(rng.integers(0, 20)) for n in lens]
        drop = rng.choice(live, size=2, replace=False).tolist()
        spare = [b for b in range(200) if pool.refs[b] == 0][-2:]
        s2 = [int(pool.table[drop[0], 0]), int(pool.table[drop[1], 0])]
        for t, values in zip([*lists, src, dst, rows], [parents, children, lens, caps, s2, spare, drop]):
            t.copy_(ints(values, cuda))
        graphs[turn % 2].replay()
        bits = oracle.fork(pool, parents, children, lens, caps)
        assert oracle.copy_blocks(pool.k, pool.v, s2, spare) == workspace_errors()
        bits |= oracle.free(pool, drop)
        more, want = oracle.compact(pool)
        assert bits | more == h.errors()
        assert np.array_equal(news[turn % 2].cpu().numpy(), want)
        same(h, pool)


def test_two_pools_at_once(cuda):
    """Rounds on two pools, each on its own stream."""
    pools, handles, lists = [], [], []
    for seed in (31, 32):
        pool, groups, empty = make_pool(seed, num_blocks=3000, rows=40, width=80, lens=[900, 1200, 33, 640], fan=2, layers=3,
                                        heads=2)
        pools.append(pool)
        handles.append(to_device(pool, cuda))
        live = [r for g in groups for r in g]
        lists.append((live, empty[:8], [900, 900, 1195, 1200, 33, 31, 640, 500], live[::2]))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in pools]
    args = [[ints(x, cuda) for x in some] for some in lists]
    torch.cuda.synchronize()
    for h, (parents, children, lens, drop), s in zip(handles, args, streams):
        with torch.cuda.stream(s):
            h.fork(parents, children, lens)
            h.free(drop)
            h.compact()
            h.fork(children, parents, lens)  # the dropped rows take them, the others refuse
    torch.cuda.synchronize()
    for pool, h, (parents, children, lens, drop) in zip(pools, handles, lists):
        bits = oracle.fork(pool, parents, children, lens) | oracle.free(pool, drop)
        bits |= oracle.compact(pool)[0]
        bits |= oracle.fork(pool, children, parents, lens)
        assert bits == h.errors() == oracle.INVALID
        same(h, pool)


def test_another_stream(cuda):
    pool, groups, empty = make_pool(22, num_blocks=100, rows=12, width=12, lens=[100, 70], layers=2, heads=1)
    h = to_device(pool, cuda)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    args = [ints(x, cuda) for x in ([groups[0][0], groups[1][0]], empty[:2], [97, 33])]
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        h.fork(*args)
        h.free(args[0])
        h.compact()
        assert h.errors() == 0
    oracle.fork(pool, args[0].tolist(), args[1].tolist(), args[2].tolist())
    oracle.free(pool, args[0].tolist())
    oracle.compact(pool)
    same(h, pool)
