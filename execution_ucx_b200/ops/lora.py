"""Low-rank adapters of many requests at once, beside a shared projection (see ``csrc/kernels/lora.cu``).

``RemoteGemm`` and its block-scaled forms multiply every token with the one weight that a worker serves. ``LoraAdapters``
adds what is each request's own: ``out[t] = y[t] + scale[i] * B[i] (A[i] x[t])``, ``i = ids[t]``, for tokens of any
requests in any order, ``y`` being what the shared projection gave.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import _native
from . import _workspace as ws

_launches = 0


def launch_count() -> int:
    return _launches


class LoraAdapters:
    """The adapters of one projection: ``a`` ``[adapters, rank, K]`` and ``b`` ``[adapters, N, rank]``, bfloat16, and ``scale``
    ``[adapters]``, float32 (1 if not given). They are used where they lie: the object keeps their memory and copies nothing, so
    an adapter that is written into its place holds for the next call (a parameter whose ``data`` is set to other memory leaves the
    object with what it was given). ``rank`` is a multiple of 8 up to 128, K and N are
    multiples of 8. For inference: the result has no gradient. An object is made outside of graph captures; its calls may be
    captured, and made by several threads. A graph may outlive the object, but not the tensors given here."""

    MAX_RANK = 128

    def __init__(self, a: torch.Tensor, b: torch.Tensor, scale: Optional[torch.Tensor] = None):
        ws.require(isinstance(a, torch.Tensor) and a.dim() == 3, "a must be [adapters, rank, K]")
        ws.require(isinstance(b, torch.Tensor) and b.dim() == 3, "b must be [adapters, N, rank]")
        self.n_adapters, self.rank, self.K = a.shape
        self.N = b.shape[1]
        ws.require(self.n_adapters >= 1, "there must be an adapter")
        ws.require(8 <= self.rank <= self.MAX_RANK and self.rank % 8 == 0, f"the rank must be a multiple of 8 up to {self.MAX_RANK}, not {self.rank}")
        ws.require(self.K > 0 and self.N > 0 and self.K % 8 == 0 and self.N % 8 == 0, f"K and N must be multiples of 8, not {self.K} and {self.N}")
        ws.require_dense(a, "a", torch.bfloat16, (self.n_adapters, self.rank, self.K))
        ws.require_dense(b, "b", torch.bfloat16, (self.n_adapters, self.N, self.rank))
        if scale is not None:
            ws.require_dense(scale, "scale", torch.float32, (self.n_adapters,))
        self.device = a.device
        ws.require_device(self.device, b=b, scale=scale)
        ws.require_cuda(self.device)
        ws.require((a.data_ptr() | b.data_ptr()) % 16 == 0, "a and b must begin on 16 bytes")
        own = () if scale is not None else (torch.ones(self.n_adapters, dtype=torch.float32, device=self.device),)
        scale = own[0] if own else scale
        self._weights = (a.detach(), b.detach(), scale.detach())  # the memory, whatever becomes of the tensors: a parameter's may be exchanged
        self._weight_ptrs = (a.data_ptr(), b.data_ptr(), scale.data_ptr())
        self._index = self.device.index
        self._need = {}
        self._scratch = ws.CallScratch(0, self.device, keep=own)
        _native.load()

    a = property(lambda self: self._weights[0])
    b = property(lambda self: self._weights[1])
    scale = property(lambda self: self._weights[2])

    def __call__(self, x: torch.Tensor, ids: torch.Tensor, y: torch.Tensor, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """``x`` is ``[tokens, K]`` and ``y`` ``[tokens, N]``, bfloat16; ``ids`` ``[tokens]``, int32, names each token's adapter. A
        token whose id is not in ``[0, adapters)`` has none: its row of ``out`` is that of ``y``. ``out`` may be ``y``, but not
        share a part of its memory; the rows of all three may lie apart. Sums are of float32 and the
        result is rounded once. With few tokens nothing is rounded between; with many, which go in tiles of an adapter, ``A x`` is taken as two
        bfloat16 numbers, which lose 2^-16 of it: a token's last bits may depend on how many tokens and adapters there are. The same
        arguments give the same bits."""
        global _launches
        K, N = self.K, self.N
        # what a call usually brings, with as few questions as tell it from everything else
        if (isinstance(x, torch.Tensor) and isinstance(ids, torch.Tensor) and isinstance(y, torch.Tensor)
                and x.dtype is torch.bfloat16 and y.dtype is torch.bfloat16 and ids.dtype is torch.int32
                and ids.dim() == 1 and x.shape == (t := ids.numel(), K) and y.shape == (t, N)
                and x.is_contiguous() and y.is_contiguous() and ids.is_contiguous()
                and (x.data_ptr() | y.data_ptr()) % 16 == 0 and x.get_device() == y.get_device() == ids.get_device() == self._index):
            xs, ys = K, N
        else:
            self._require(x, ids, y)
            t, xs, ys = ids.shape[0], ws.row_stride(x), ws.row_stride(y)
        if out is None:
            out, os_ = torch.empty_strided((t, N), (N, 1), dtype=torch.bfloat16, device=self.device), N
        elif out is y:
            os_ = ys
        else:
            ws.require_rows(out, "out", torch.bfloat16, cols=N, rows=t)
            ws.require_device(self.device, out=out)
            ws.require_apart(out, y, "y")
            os_ = ws.row_stride(out)
        if t == 0:
            return out
        lib = _native.load()
        need = self._need.get(t)
        if need is None:
            need = self._need[t] = int(lib.eux_lora_workspace_bytes(self._desc(t)))
        workspace, _ = self._scratch.get(need)
        desc = self._desc(t, x.data_ptr(), ids.data_ptr(), y.data_ptr(), out.data_ptr(), workspace, xs, ys, os_)
        ws.launch(lib.eux_lora_launch, desc, self._index, "eux_lora_launch")
        few = t <= 512 and t * self.rank * (K + N) * 2 <= (128 if self.n_adapters >= t // 4 else 48) << 20  # as the launch chooses
        _launches += 2 if few else 3
        return out

    def _desc(self, tokens, x=0, ids=0, y=0, out=0, workspace=0, x_stride=0, y_stride=0, out_stride=0):
        return _native.descriptor(_native.LORA_DESC, _native.LoraDesc, x, ids, y, out, *self._weight_ptrs, workspace, x_stride, y_stride, out_stride,
                                  tokens, self.K, self.N, self.rank, self.n_adapters, 0)

    def _require(self, x, ids, y) -> None:
        ws.require_rows(x, "x", torch.bfloat16, cols=self.K)
        t = x.shape[0]
        ws.require_rows(y, "y", torch.bfloat16, cols=self.N, rows=t)
        ws.require_dense(ids, "ids", torch.int32, (t,))
        ws.require_device(self.device, x=x, ids=ids, y=y)


def reference(x: torch.Tensor, ids: torch.Tensor, y: torch.Tensor, a: torch.Tensor, b: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    """Plain PyTorch statement in 64 bits."""
    out = y.double().clone()
    for i in range(a.shape[0]):
        rows = (ids == i).nonzero().squeeze(1)
        if rows.numel():
            out[rows] += scale[i].double() * ((x[rows].double() @ a[i].double().t()) @ b[i].double().t())
    return out
