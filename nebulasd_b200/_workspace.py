"""Device scratch for the attention kernels, one buffer per (device, stream).

The split-K kernels keep per-unit arrival counters and per-slot fp32 partials
in this buffer, and the verify kernel the work plan of its previous call (its
plan cache: calls on one buffer must be ordered on one stream) (the reference allocates its fp32 ``mid_o`` partials with
``torch.empty`` on every call, ``swiftLLM/swiftllm/worker/kernels/paged_attn.py:170-180``).
The counters must be zero when a call starts, and every call leaves them at
zero, so a buffer is zero-filled once when it is created and then reused by
the calls queued on its stream; calls on different streams (the compute
stream and the decoding piggyback stream of ``transformer_layer.py:169-185``,
or the two bank streams) get separate buffers, so they never race.
"""
from __future__ import annotations

import threading

import torch

from . import _lib

_lock = threading.Lock()
_buffers: dict[tuple[int, int], torch.Tensor] = {}


def attention_workspace(kernel: int, device: torch.device, stream: torch.cuda.Stream, num_rows: int,
                        num_q_heads: int, num_kv_heads: int) -> torch.Tensor:
    index = device.index if device.index is not None else torch.cuda.current_device()
    need = _lib.lib.neb_attention_workspace_bytes(kernel, index, max(num_rows, 1), num_q_heads, num_kv_heads)
    if need == 0:
        raise _lib.NebError(f"attention kernel {kernel} does not support {num_q_heads} q heads over "
                            f"{num_kv_heads} kv heads on device {index}")
    key = (index, stream.cuda_stream)
    with _lock:
        buf = _buffers.get(key)
        if buf is None or buf.numel() < need:
            # Round up so that slowly growing batches do not reallocate every call.
            size = max(need, 2 * buf.numel() if buf is not None else 0, 1 << 20)
            # Long-lived buffers are never inference tensors, even when the first
            # call comes from inside ``torch.inference_mode()`` (the reference's
            # model forward): callers may update them in place outside it.
            with torch.cuda.stream(stream), torch.inference_mode(False):
                buf = torch.zeros(size, dtype=torch.uint8, device=torch.device("cuda", index))
            _buffers[key] = buf
        return buf


def workspace_errors(buf: torch.Tensor, stream: torch.cuda.Stream) -> int:
    """Synchronise ``stream`` and return (and clear) the kernels' recorded error bits."""
    import ctypes
    bits = ctypes.c_uint32(0)
    _lib.check(_lib.lib.neb_workspace_status(buf.data_ptr(), ctypes.byref(bits), stream.cuda_stream),
               "neb_workspace_status")
    return bits.value


# Bumped whenever buffers are dropped, so that callers keeping a reference to
# the last buffer they used look it up again.
generation = 0


def release_all() -> None:
    global generation
    with _lock:
        _buffers.clear()
        generation += 1


_error_words: dict[int, torch.Tensor] = {}


def error_word(device: torch.device) -> torch.Tensor:
    """Per-device int32 where the store/RoPE kernels record out-of-range block ids (never a trap)."""
    index = device.index if device.index is not None else torch.cuda.current_device()
    with _lock:
        t = _error_words.get(index)
        if t is None:
            with torch.inference_mode(False):  # see attention_workspace
                t = torch.zeros(1, dtype=torch.int32, device=torch.device("cuda", index))
            _error_words[index] = t
        return t


class ErrorWords:
    """One int32 word per device where an operator's kernels record error bits (never a trap), for
    operators that keep no workspace of their own."""

    def __init__(self, what: str) -> None:
        self._what, self._words = what, {}

    def word(self, index: int) -> torch.Tensor:
        t = self._words.get(index)
        if t is not None:
            return t
        with _lock:
            t = self._words.get(index)
            if t is None:
                t = self._words[index] = new_error_word(index, self._what)
        return t

    def read(self, device: torch.device | None = None) -> int:
        """Synchronise the device's current stream; return and clear the bits recorded so far."""
        index = device.index if device is not None and device.index is not None else torch.cuda.current_device()
        return read_error_word(self.word(index))


def new_error_word(index: int, what: str) -> torch.Tensor:
    with torch.cuda.device(index):
        # Inside a capture its zero fill would run at each replay and not now.
        if torch.cuda.is_current_stream_capturing():
            raise _lib.NebError(f"{what}: its first call on a device must come before any graph capture")
        with torch.inference_mode(False):  # see attention_workspace
            t = torch.zeros(1, dtype=torch.int32, device=torch.device("cuda", index))
        torch.cuda.current_stream(index).synchronize()  # every stream uses the word from here on
    return t


def read_error_word(t: torch.Tensor) -> int:
    """Synchronise the current stream of the word's device; return and clear the bits, in one step on the device."""
    with torch.cuda.device(t.device):
        taken = torch.empty_like(t)
        rc = _lib.lib.neb_take_error_bits(t.data_ptr(), taken.data_ptr(), torch.cuda.current_stream().cuda_stream)
        _lib.check(rc, "neb_take_error_bits")
        return int(taken.item()) & 0xFFFFFFFF
