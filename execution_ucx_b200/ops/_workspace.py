"""What the operators that are called like a layer share: checks of arguments, the launch on a tensor's own device, and
zeroed words for kernels that count their CTAs."""
from __future__ import annotations

import ctypes as C
import itertools
import threading
import weakref

import torch

from . import _native


def require(ok: bool, message: str) -> None:
    if not ok:
        raise ValueError(message)


def require_rows(t: torch.Tensor, name: str, dtype, cols=None, rows=None) -> None:
    """A matrix whose rows the kernels can read in 16-byte pieces: unit inner stride, rows and base on 16 bytes, rows that
    do not overlap."""
    require(isinstance(t, torch.Tensor) and t.dim() == 2, f"{name} must be a matrix")
    require(t.dtype == dtype, f"{name} must be {dtype}, not {t.dtype}")
    require(cols is None or t.shape[1] == cols, f"{name} must have {cols} columns, not {t.shape[1]}")
    require(rows is None or t.shape[0] == rows, f"{name} must have {rows} rows, not {t.shape[0]}")
    unit = 16 // t.element_size()
    if t.numel():
        require(t.shape[1] == 1 or t.stride(1) == 1, f"{name} must have its columns side by side")
        require(t.shape[0] == 1 or (t.stride(0) % unit == 0 and t.stride(0) >= t.shape[1]), f"{name} must have rows {unit} elements aligned and apart")
        require(t.data_ptr() % 16 == 0, f"{name} must begin on 16 bytes")


def row_stride(t: torch.Tensor) -> int:
    """The distance of rows; any will do where there is one row."""
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def require_apart(out: torch.Tensor, other: torch.Tensor, name: str) -> None:
    """That ``out`` is ``other``, row for row, or shares no memory with it. Both are matrices that ``require_rows`` has seen."""
    a, b = (t.data_ptr() for t in (out, other))
    (n, wa, sa), (m, wb, sb) = ((t.shape[0], t.shape[1] * t.element_size(), row_stride(t) * t.element_size()) for t in (out, other))
    if not out.numel() or not other.numel() or a + (n - 1) * sa + wa <= b or b + (m - 1) * sb + wb <= a:
        return
    if (a, n, wa) == (b, m, wb) and (sa == sb or n == 1):
        return
    if sa == sb:  # columns beside each other, or a row's end within its distance to the next
        apart = (b - a) % sa
        shared = apart < wa or apart + wb > sa
    else:
        i = j = shared = 0
        while i < n and j < m and not shared:
            if a + i * sa + wa <= b + j * sb:
                i += 1
            elif b + j * sb + wb <= a + i * sa:
                j += 1
            else:
                shared = 1
    require(not shared, f"out may be {name} itself, and else must not share memory with it")


def require_dense(t: torch.Tensor, name: str, dtype, shape) -> None:
    require(isinstance(t, torch.Tensor) and tuple(t.shape) == tuple(shape), f"{name} must have the shape {tuple(shape)}")
    require(t.dtype == dtype, f"{name} must be {dtype}, not {t.dtype}")
    require(t.is_contiguous(), f"{name} must be contiguous")


def require_device(device, **tensors) -> None:
    for name, t in tensors.items():
        if t is not None:
            require(t.device == device, f"{name} is on {t.device}, not on {device}")


def require_cuda(device) -> None:
    require(device.type == "cuda", f"the kernels run on a CUDA device, not on {device}")


class on_device:
    """The given device as the current one, and its current stream: ``with on_device(index) as stream``."""

    def __init__(self, index: int):
        self.index = index

    def __enter__(self) -> int:
        self.before = torch.cuda.current_device()
        torch.cuda.set_device(self.index)
        return torch._C._cuda_getCurrentRawStream(self.index)

    def __exit__(self, *exc):
        torch.cuda.set_device(self.before)


def launch(function, desc, index: int, what: str) -> None:
    """One call of a launch function on device ``index`` and its current stream."""
    if torch._C._cuda_getDevice() == index:
        rc = function(desc, torch._C._cuda_getCurrentRawStream(index))
    else:
        with on_device(index) as stream:
            rc = function(desc, stream)
    if rc:
        _native.check(rc, what)


# What captured calls use of an object's own memory, by the token that their graph gives back when it is gone.
_held = {}
_tokens = itertools.count(1)


def _collect() -> None:
    """Gives what graphs that are gone had used back to where it came from, if that is still there."""
    tokens = (C.c_uint64 * 64)()
    while n := _native.load().eux_graphs_gone(tokens, 64):
        for token in tokens[:n]:
            _, words, owner = _held.pop(token, (None, None, None))  # none: the hold failed
            owner = owner and owner()
            if owner is not None and words is not None:
                owner._spare.append(words)


class CallScratch:
    """Memory for calls of a kernel: a workspace, and zeroed words that the kernel leaves zeroed. Calls that may run at the
    same time get memory of their own: those of one stream share some, and every captured call has its own, since graphs may
    be replayed beside each other and beside plain calls. ``keep`` is memory of the object's own that its calls use too. A
    graph keeps it, and the words, for as long as it is there itself, whatever becomes of the object; then others may have them."""

    SLOTS = 16

    def __init__(self, words: int, device, keep=()):
        self.words, self.device, self._keep = words, device, tuple(keep)
        self._of_stream = {}
        self._kept = []
        self._lock = threading.Lock()  # two threads that find nothing for their stream must not both make it
        with on_device(device.index):
            self._all = torch.zeros(self.SLOTS, words, dtype=torch.int32, device=device) if words else None
            self._spare = list(self._all.unbind(0)) if words else []
            torch.cuda.current_stream().synchronize()  # captured calls run on any stream

    def get(self, need: int):
        """The addresses of ``need`` bytes and of the words, for a call on the device's current stream, whether or not the device
        is the current one."""
        if torch._C._cuda_getDevice() != self.device.index:
            with on_device(self.device.index):
                return self.get(need)
        with self._lock:
            return self._get(need)

    def _get(self, need: int):
        stream = torch._C._cuda_getCurrentRawStream(self.device.index)
        if torch._C._cuda_isCurrentStreamCapturing():
            # In a capture a tensor's memory is the graph's; the words are zeroed by the graph itself where all that were zeroed
            # beforehand are given out.
            workspace = torch.empty(need, dtype=torch.uint8, device=self.device)
            _collect()
            mine = self._spare.pop() if self._spare else None
            words = mine if mine is not None or not self.words else torch.zeros(self.words, dtype=torch.int32, device=self.device)
            if mine is not None or self._keep:
                token = next(_tokens)
                _held[token] = (self._keep, mine, weakref.ref(self))
                if rc := _native.load().eux_graph_hold(stream, token):
                    if _held.pop(token, None) and mine is not None:
                        self._spare.append(mine)
                    _native.check(rc, "eux_graph_hold")
            return workspace.data_ptr(), words.data_ptr() if words is not None else 0
        mine = self._of_stream.get(stream)
        if mine is None or mine[2] < need:
            # A smaller workspace may be another thread's, which has yet to launch with it: it is kept. Powers of two: all that are kept come
            # to less than the largest.
            need = 1 << (need - 1).bit_length()
            words = mine[1] if mine else torch.zeros(self.words, dtype=torch.int32, device=self.device)
            if mine:
                self._kept.append(mine[0])
            else:
                for t in self._keep:  # made on another stream, perhaps, where it is not free before this one is done with it
                    t.record_stream(torch.cuda.current_stream())
            workspace = torch.empty(need, dtype=torch.uint8, device=self.device)
            mine = self._of_stream[stream] = (workspace, words, need, (workspace.data_ptr(), words.data_ptr()))
        return mine[3]

    def reset(self) -> None:
        """Zeroes all words, after a kernel that gave up: with nothing in flight."""
        for t in [m[1] for m in self._of_stream.values()] + ([self._all] if self.words else []):
            t.zero_()
