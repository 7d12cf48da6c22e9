"""Restatement of the block pool's operators, one step at a time (CPU, numpy, bit copies).

TEST INFRASTRUCTURE ONLY (see ``oracle/__init__.py``).  The reference has no counterpart; this follows the
operators' definitions.  A pool is a ``Pool`` of numpy arrays: caches ``[num_blocks, layers, heads,
block_size, dim]``, ``table [rows, width]``, ``held [rows]`` (entries in use), ``refs [num_blocks]``.
Every function changes it in place and returns the error bits.
"""
from __future__ import annotations

import dataclasses

import numpy as np

BLOCK, ROW, WIDTH, INVALID, REFS, NO_BLOCK, CONFLICT = 1, 2, 4, 16, 128, 256, 512


@dataclasses.dataclass
class Pool:
    k: np.ndarray
    v: np.ndarray
    table: np.ndarray
    held: np.ndarray
    refs: np.ndarray

    def copy(self) -> "Pool":
        return Pool(*(getattr(self, f.name).copy() for f in dataclasses.fields(self)))


def copy_blocks(k, v, src, dst, tokens=None) -> int:
    bits, nb, size = 0, k.shape[0], k.shape[3]
    before_k, before_v = k.copy(), v.copy()
    for i, (s, d) in enumerate(zip(src, dst)):
        t = size if tokens is None else int(tokens[i])
        bad = 0
        if not (0 <= s < nb and 0 <= d < nb):
            bad |= BLOCK
        if not 0 <= t <= size:
            bad |= INVALID
        if any(j != i and (o == d or o == s) for j, o in enumerate(dst)):
            bad |= CONFLICT
        bits |= bad
        if not bad:
            k[d, :, :, :t], v[d, :, :, :t] = before_k[s, :, :, :t], before_v[s, :, :, :t]
    return bits


def fork(p: Pool, parents, children, lens, capacities=None) -> int:
    bits, (rows, width), size, nb = 0, p.table.shape, p.k.shape[3], p.refs.shape[0]
    start = p.copy()
    free = [b for b in range(nb) if p.refs[b] == 0]
    used, taken = 0, set()
    for i, (par, ch, n) in enumerate(zip(parents, children, lens)):
        par, ch, n = int(par), int(ch), int(n)
        cap = 0 if capacities is None else int(capacities[i])
        bad = 0
        if not 0 <= ch < rows or (n > 0 and not 0 <= par < rows):
            bad |= ROW
        if n < 0 or cap < 0:
            bad |= INVALID
        shared, total = max(n, 0) // size, -(-max(n, cap, 0) // size)
        if total > width:
            bad |= WIDTH
        if not bad and (start.held[ch] != 0 or (n > 0 and -(-n // size) > start.held[par])):
            bad |= INVALID
        if not bad:
            if ch in taken:
                bad |= INVALID
            taken.add(ch)
        bits |= bad
        if bad:
            continue
        need, first = total - shared, used
        used += need
        if need and used > len(free):
            bits |= NO_BLOCK
            continue
        for j in range(shared):
            b = int(start.table[par, j])
            if not 0 <= b < nb:
                bits |= BLOCK
                b = -1
            else:
                if start.refs[b] <= 0:
                    bits |= REFS
                p.refs[b] += 1
            p.table[ch, j] = b
        for j in range(need):
            b = free[first + j]
            p.refs[b] += 1
            p.table[ch, shared + j] = b
        p.held[ch] = total
        if n % size:
            s, d = int(start.table[par, shared]), free[first]
            if 0 <= s < nb and start.refs[s] <= 0:
                bits |= REFS
            elif 0 <= s < nb:
                p.k[d, :, :, :n % size], p.v[d, :, :, :n % size] = (start.k[s, :, :, :n % size],
                                                                    start.v[s, :, :, :n % size])
            else:
                bits |= BLOCK
    return bits


def free(p: Pool, rows) -> int:
    bits = 0
    for r in (int(x) for x in rows):
        if not 0 <= r < p.table.shape[0]:
            bits |= ROW
            continue
        n = int(p.held[r])
        if not 0 <= n <= p.table.shape[1]:
            bits |= WIDTH
        p.held[r] = 0
        for j in range(min(max(n, 0), p.table.shape[1])):
            b = int(p.table[r, j])
            p.table[r, j] = -1
            if not 0 <= b < p.refs.shape[0]:
                bits |= BLOCK
            elif p.refs[b] <= 0:
                bits |= REFS
            else:
                p.refs[b] -= 1
    return bits


def compact(p: Pool):
    bits, nb = 0, p.refs.shape[0]
    live = [b for b in range(nb) if p.refs[b] > 0]
    n = len(live)
    holes, movers = [b for b in range(n) if p.refs[b] <= 0], [b for b in live if b >= n]
    new = np.full(nb, -1, np.int32)
    new[live] = live
    for d, s in zip(holes, movers):
        new[s] = d
        p.k[d], p.v[d] = p.k[s], p.v[s]
        p.refs[d], p.refs[s] = p.refs[s], 0
    for r in range(p.table.shape[0]):
        for j in range(min(max(int(p.held[r]), 0), p.table.shape[1])):
            b = int(p.table[r, j])
            if not 0 <= b < nb:
                bits |= BLOCK
            else:
                if new[b] < 0:
                    bits |= REFS
                p.table[r, j] = new[b]
    return bits, new
