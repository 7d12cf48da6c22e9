"""Blocks of the paged KV cache copied, forked, freed and compacted on the GPU.

For programs that branch (best-of-n, beams, several answers to one prompt): a
fork shares its parent's full blocks and copies only the partial one, dropped
branches give their blocks back, and the holes that they leave are closed.
All of it is planned on the device from int32 tensors, so that branches chosen
there (``logprobs.token_logprobs``) need no host sync, and every result is the
same whatever the order of the threads.

``BlockPool`` names the caller's tensors: the caches ``[num_blocks, num_layers,
num_kv_heads, block_size, head_dim]`` and block table that ``store_kvcache``
and ``paged_attention`` use, ``seq_blocks`` (entries of each row in use) and
``ref_counts`` (rows that use each block; 0: free).  The reference's banks
(``nebulasd/src/nebulasd/workers/banks.py:43-60``) give every request blocks of
its own and keep no counts; a program on banks uses ``copy_blocks`` alone.
"""
from __future__ import annotations

import torch

from . import _lib
from ._workspace import ErrorWords, new_error_word, read_error_word
from .kernels.paged_attn import _raw_stream

_errors = ErrorWords("copy_blocks")


def _check_caches(k_cache: torch.Tensor, v_cache: torch.Tensor) -> tuple[int, int, int, int]:
    """(num_blocks, tiles per block, block_size, bytes of a token in a tile)."""
    if (k_cache.dim() != 5 or k_cache.shape != v_cache.shape or k_cache.dtype != v_cache.dtype
            or k_cache.get_device() < 0 or k_cache.get_device() != v_cache.get_device()
            or not k_cache.is_contiguous() or not v_cache.is_contiguous()):
        raise ValueError("k_cache and v_cache must be matching contiguous CUDA tensors "
                         "[num_blocks, num_layers, num_kv_heads, block_size, head_dim]")
    nb, layers, heads, size, dim = k_cache.shape
    token_bytes = dim * k_cache.element_size()
    if k_cache.numel() == 0 or token_bytes % 16:
        raise ValueError("the caches must hold blocks whose head rows are a multiple of 16 bytes")
    if layers * heads * size * token_bytes >= 1 << 31 or nb >= 1 << 31:
        raise ValueError("the caches must hold fewer than 2^31 blocks of less than 2 GiB")
    return nb, layers * heads, size, token_bytes


def _check_list(name: str, t: torch.Tensor, index: int, length: int | None = None) -> None:
    if (t.dtype != torch.int32 or t.dim() != 1 or t.get_device() != index or not t.is_contiguous()
            or t.numel() >= 1 << 31 or (length is not None and t.numel() != length)):
        raise ValueError(f"{name} must be a contiguous int32 vector on the caches' device"
                         + (f" of {length} elements" if length is not None else ""))


def copy_blocks(k_cache: torch.Tensor, v_cache: torch.Tensor, src: torch.Tensor, dst: torch.Tensor,
                num_tokens: torch.Tensor | None = None) -> None:
    """Block ``dst[i]`` gets the first ``num_tokens[i]`` tokens (default: all) of block ``src[i]``,
    every layer and head of both caches; its other tokens keep their contents.

    Lists are int32 vectors on the caches' device.  The pairs are copied at
    once, so a pair whose ``dst`` is another pair's ``dst``, or whose ``src`` is
    another pair's ``dst``, is left out and reported by ``workspace_errors``
    (bit 9), as is one with a block (bit 0) or token count (bit 4) out of range.
    Lists of more than some thousand pairs are better split: finding conflicts
    takes time with the square of their number.
    Runs on the current stream of the caches' device; its first call on a device
    must come before any graph capture.
    """
    nb, tiles, size, token_bytes = _check_caches(k_cache, v_cache)
    index, n = k_cache.get_device(), src.numel()
    _check_list("src", src, index)
    _check_list("dst", dst, index, n)
    if num_tokens is not None:
        _check_list("num_tokens", num_tokens, index, n)
    word = _errors.word(index)
    with _Device(index):
        rc = _lib.lib.neb_copy_blocks(k_cache.data_ptr(), v_cache.data_ptr(), nb, tiles, size, token_bytes,
                                      src.data_ptr(), dst.data_ptr(), _lib.ptr(num_tokens), n, word.data_ptr(),
                                      _raw_stream(index))
    _lib.check(rc, "copy_blocks")


def workspace_errors(device: torch.device | None = None) -> int:
    """Synchronise the device's current stream and return (and clear) the error bits of ``copy_blocks``."""
    return _errors.read(device)


class _Device:
    """``torch.cuda.device`` that costs nothing on the current device."""

    __slots__ = ("index", "guard")

    def __init__(self, index: int) -> None:
        self.index, self.guard = index, None

    def __enter__(self) -> None:
        if torch.cuda.current_device() != self.index:
            self.guard = torch.cuda.device(self.index)
            self.guard.__enter__()

    def __exit__(self, *exc) -> None:
        if self.guard is not None:
            self.guard.__exit__(*exc)


class BlockPool:
    """A paged cache with shared blocks.  Holds the caller's tensors, changes them in place.

    ``block_table`` int32 ``[rows, max_blocks]``, ``seq_blocks`` int32 ``[rows]``: the
    first ``seq_blocks[r]`` entries of row ``r`` are in use (0: an empty row);
    ``ref_counts`` int32 ``[num_blocks]``: how many rows use each block.  All
    contiguous, on the caches' device.  Methods run on the current stream of
    that device, and calls on one pool must be ordered.  What they refuse they
    leave as it was; ``errors`` tells why.  Lists must not be parts of the pool's
    own tensors.  A row gets all its blocks from the fork that makes it
    (``capacities``); none of the methods gives a row in use one more.  The tensors
    stay where they were when the pool was made: with one replaced or moved, every
    method raises.
    """

    def __init__(self, k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor,
                 seq_blocks: torch.Tensor, ref_counts: torch.Tensor) -> None:
        shape = _check_caches(k_cache, v_cache)
        index = k_cache.get_device()
        if (block_table.dtype != torch.int32 or block_table.dim() != 2 or block_table.get_device() != index
                or not block_table.is_contiguous() or not 0 < block_table.numel() < 1 << 31):
            raise ValueError("block_table must be a contiguous int32 [rows, max_blocks] tensor on the caches' "
                             "device, of fewer than 2^31 entries")
        _check_list("seq_blocks", seq_blocks, index, block_table.shape[0])
        _check_list("ref_counts", ref_counts, index, shape[0])
        self.k_cache, self.v_cache = k_cache, v_cache
        self.block_table, self.seq_blocks, self.ref_counts = block_table, seq_blocks, ref_counts
        self.num_blocks, self.block_size = shape[0], shape[2]
        self._index, self._device = index, k_cache.device
        self._caches = (k_cache.data_ptr(), v_cache.data_ptr(), *shape)
        self._tables = (block_table.data_ptr(), *block_table.shape, seq_blocks.data_ptr(), ref_counts.data_ptr())
        self._places = (*self._caches[:2], self._tables[0], *self._tables[3:])
        self._fork_bytes: dict[int, int] = {}
        self._compact_bytes = _lib.lib.neb_compact_workspace_bytes(shape[0])
        self._word = new_error_word(index, "BlockPool")
        self._error_ptr = self._word.data_ptr()

    def _check_tensors(self) -> None:
        if (self.k_cache.data_ptr(), self.v_cache.data_ptr(), self.block_table.data_ptr(), self.seq_blocks.data_ptr(),
                self.ref_counts.data_ptr()) != self._places:
            raise ValueError("a tensor of the pool has been replaced or moved since the pool was made")

    def _temporary(self, need: int) -> torch.Tensor:
        # From the caching allocator, so that calls on several streams and captured
        # graphs each have their own.
        return torch.empty(need, dtype=torch.uint8, device=self._device)

    def fork(self, parents: torch.Tensor, children: torch.Tensor, seq_lens: torch.Tensor,
             capacities: torch.Tensor | None = None) -> None:
        """Row ``children[i]`` becomes a sequence that starts with the first ``seq_lens[i]`` tokens of row
        ``parents[i]``, with blocks for ``capacities[i]`` tokens (default and at least ``seq_lens[i]``).

        The child shares the parent's full blocks and gets fresh ones (lowest free first, in the order of
        the list) for the rest, the tokens of the partial block copied, so that both may append.  Length 0
        makes a new sequence; its parent is not read.  Refused, leaving the child's row as it was: a child
        that is not empty or is listed before, a length beyond the parent's blocks (bit 4), rows out of range
        (bit 1), more than ``max_blocks`` blocks (bit 2), too few free blocks (bit 8).  A parent's block that
        no count vouches for is shared but not copied from (bit 7).  Int32 vectors.
        """
        self._check_tensors()
        index, n = self._index, children.numel()
        _check_list("children", children, index)
        _check_list("parents", parents, index, n)
        _check_list("seq_lens", seq_lens, index, n)
        if capacities is not None:
            _check_list("capacities", capacities, index, n)
        need = self._fork_bytes.get(n)
        if need is None:
            need = self._fork_bytes[n] = _lib.lib.neb_fork_workspace_bytes(self.num_blocks, n)
        with _Device(index):
            ws = self._temporary(need)
            rc = _lib.lib.neb_fork_sequences(*self._caches, *self._tables, parents.data_ptr(), children.data_ptr(),
                                             seq_lens.data_ptr(), _lib.ptr(capacities), n, ws.data_ptr(), need,
                                             self._error_ptr, _raw_stream(index))
        _lib.check(rc, "fork")

    def free(self, rows: torch.Tensor) -> None:
        """Empty the listed rows (int32): their blocks lose one reference each and are free at 0.  A row
        listed twice is freed once."""
        self._check_tensors()
        _check_list("rows", rows, self._index)
        with _Device(self._index):
            rc = _lib.lib.neb_free_sequences(*self._tables, self.num_blocks, rows.data_ptr(), rows.numel(),
                                             self._error_ptr, _raw_stream(self._index))
        _lib.check(rc, "free")

    def compact(self) -> torch.Tensor:
        """Move the blocks in use to the front of the pool; the free ones are one range behind them.

        Contents, counts and every row's entries move along.  Returns int32 ``[num_blocks]``: each block's
        new index (-1: it was free), for ids that the caller keeps elsewhere."""
        self._check_tensors()
        need = self._compact_bytes
        with _Device(self._index):
            ws = self._temporary(need)
            moved = torch.empty_like(self.ref_counts)
            rc = _lib.lib.neb_compact_blocks(*self._caches, *self._tables, moved.data_ptr(), ws.data_ptr(), need,
                                             self._error_ptr, _raw_stream(self._index))
        _lib.check(rc, "compact")
        return moved

    def errors(self) -> int:
        """Synchronise the current stream; return and clear the error bits that the pool's calls recorded
        (the bits of ``neb_fork_sequences`` and its neighbours in the C header)."""
        return read_error_word(self._word)
