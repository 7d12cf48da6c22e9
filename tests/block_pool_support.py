"""Pools in use, for the block-pool tests: the same arrays for the oracle and the device."""
import numpy as np
import torch

from oracle.block_pool import Pool


def make_pool(seed, *, num_blocks, rows, width, lens, fan=1, layers=2, heads=2, size=16, dim=128,
              dtype=torch.float16):
    """Sequences of `lens` tokens, each held by `fan` rows that share all but the last block; the other rows are
    empty.  Returns the pool (caches as raw words), the rows of each sequence and the empty rows."""
    rng = np.random.default_rng(seed)
    word = {2: np.uint16, 4: np.uint32}[torch.empty(0, dtype=dtype).element_size()]
    shape = (num_blocks, layers, heads, size, dim)
    k, v = (rng.integers(0, 2 ** 16, size=shape).astype(word) for _ in range(2))
    table, held = np.full((rows, width), -1, np.int32), np.zeros(rows, np.int32)
    order, blocks, used, groups = rng.permutation(rows), rng.permutation(num_blocks), 0, []
    for i, n in enumerate(lens):
        count = -(-n // size)
        group = order[i * fan:(i + 1) * fan]
        for f, r in enumerate(group):
            if count:
                table[r, :count - 1] = blocks[used:used + count - 1]
                table[r, count - 1] = blocks[used + count - 1 + f]
            held[r] = count
        used += count - 1 + fan if count else 0
        groups.append([int(r) for r in group])
    assert used <= num_blocks
    refs = np.bincount(table[table >= 0], minlength=num_blocks).astype(np.int32)
    return Pool(k, v, table, held, refs), groups, [int(r) for r in order[len(lens) * fan:]]


def to_device(pool, dev, dtype=torch.float16):
    from nebulasd_b200.block_pool import BlockPool
    signed = {2: np.int16, 4: np.int32}[pool.k.dtype.itemsize]
    k, v = (torch.from_numpy(a.view(signed).copy()).to(dev).view(dtype) for a in (pool.k, pool.v))
    return BlockPool(k, v, *(torch.from_numpy(a.copy()).to(dev) for a in (pool.table, pool.held, pool.refs)))


def same(handle, pool):
    """Bit for bit, caches included."""
    signed = {2: torch.int16, 4: torch.int32}[pool.k.dtype.itemsize]
    for got, want in ((handle.k_cache, pool.k), (handle.v_cache, pool.v)):
        assert np.array_equal(got.view(signed).cpu().numpy().view(pool.k.dtype), want)
    assert np.array_equal(handle.block_table.cpu().numpy(), pool.table)
    assert np.array_equal(handle.seq_blocks.cpu().numpy(), pool.held)
    assert np.array_equal(handle.ref_counts.cpu().numpy(), pool.refs)


def ints(values, dev):
    return torch.tensor(list(values), dtype=torch.int32, device=dev)
