"""MoE token dispatch / combine over peer memory (see ``csrc/kernels/moe_dispatch.cu``).

``MoeAllToAll`` owns, per rank, a receive arena (``world`` regions of
``capacity`` rows), the 16-byte row headers and the flag block, all
peer-mapped. ``dispatch`` routes and pushes rows to the expert ranks,
``expert_ready`` is where an expert GEMM would run (identity here) and
``combine`` pulls the rows back with the gate-weighted sum fused into the read.

``route`` chooses the experts (``csrc/kernels/moe_route.cu``) and ``MoeExperts`` is
what they compute (``csrc/kernels/moe_experts.cu``): the whole layer of a few tokens
whose experts are on this GPU, or the experts of rows that a dispatch has brought.
"""
from __future__ import annotations

import ctypes as C
from typing import List, Optional, Tuple

import torch

from . import _native
from . import _workspace as ws
from ..parallel.peer import PeerGroup, SymmetricBuffer

_launches = 0
_ROUTE_SELF = 4096  # routing entries up to which the dispatch is one launch (kRouteSelf of moe_dispatch.cu)


def launch_count() -> int:
    return _launches


def row_bytes(hidden: int, fp8: bool) -> int:
    """Bytes of one row in a receive arena (the kernels' layout: ``eux_moe_row_bytes``)."""
    return int(_native.load().eux_moe_row_bytes(hidden, 1 if fp8 else 0))


class MoeAllToAll:
    def __init__(self, group: PeerGroup, n_tokens: int, hidden: int, topk: int, n_experts: int,
                 fp8: bool = False, capacity: Optional[int] = None,
                 buffers: Optional[tuple] = None, rank: Optional[int] = None):
        if n_experts % group.world or hidden % 128:
            raise ValueError("n_experts must divide by world and hidden by 128")
        self.group = group
        self.rank = group.rank if rank is None else rank
        self.world = group.world
        self.n_tokens, self.hidden, self.topk, self.n_experts, self.fp8 = n_tokens, hidden, topk, n_experts, fp8
        self.capacity = capacity or n_tokens * topk
        self.row_bytes = row_bytes(hidden, fp8)
        epr = n_experts // self.world
        if buffers is None:
            arena = group.alloc(self.world * self.capacity * self.row_bytes)
            meta = group.alloc(self.world * self.capacity * 16)
            flags = group.alloc((3 * self.world + self.world * epr) * 8)
            buffers = (arena, meta, flags)
        self.arena, self.meta, self.flags = buffers
        dev = group.device
        self.slot_of = torch.empty(n_tokens * topk, dtype=torch.int32, device=dev)
        self.counters = torch.zeros(self.world + n_experts + 8, dtype=torch.int32, device=dev)
        self.status = torch.zeros(1, dtype=torch.int32, device=dev)
        self.out = torch.empty(n_tokens, hidden, dtype=torch.bfloat16, device=dev)
        self.seq = 0
        self._x = self._idx = self._w = None

    def close(self) -> None:
        """Collective release of the peer-mapped buffers: every rank calls it."""
        self.group.free(self.arena, self.meta, self.flags)

    @classmethod
    def emulated(cls, world: int, n_tokens: int, hidden: int, topk: int, n_experts: int, fp8: bool = False,
                 capacity: Optional[int] = None) -> List["MoeAllToAll"]:
        """``world`` logical ranks on one GPU (for single-device checks)."""
        g = PeerGroup.emulated(world)
        cap = capacity or n_tokens * topk
        rb = row_bytes(hidden, fp8)
        epr = n_experts // world
        arenas = g.alloc_emulated(world * cap * rb)
        metas = g.alloc_emulated(world * cap * 16)
        flags = g.alloc_emulated((3 * world + world * epr) * 8)
        return [cls(g, n_tokens, hidden, topk, n_experts, fp8, cap, (arenas[r], metas[r], flags[r]), rank=r)
                for r in range(world)]

    def _desc(self):
        """An ``eux_moe_desc`` of the exchange under way."""
        x, idx, w = self._x, self._idx, self._w
        return _native.descriptor(
            _native.MOE_DESC, _native.MoeDesc, self.rank, self.world, self.n_tokens, self.hidden, self.topk, self.n_experts, int(self.fp8), self.capacity,
            x.data_ptr() if x is not None else 0, idx.data_ptr() if idx is not None else 0, w.data_ptr() if w is not None else 0,
            self.arena.ptr_table.data_ptr(), self.meta.ptr_table.data_ptr(), self.flags.ptr_table.data_ptr(),
            self.slot_of.data_ptr(), self.counters.data_ptr(), self.out.data_ptr(), self.seq, 2_000_000_000, self.status.data_ptr())

    def dispatch(self, x: torch.Tensor, topk_idx: torch.Tensor, topk_w: torch.Tensor, ctas: int = 0) -> None:
        global _launches
        assert x.dtype == torch.bfloat16 and x.is_contiguous() and x.shape == (self.n_tokens, self.hidden)
        assert topk_idx.dtype == torch.int32 and topk_w.dtype == torch.float32
        self._x, self._idx, self._w = x, topk_idx.contiguous(), topk_w.contiguous()
        self.seq += 1
        rc = _native.load().eux_moe_dispatch_launch(self._desc(), ctas, _native.current_stream_ptr())
        if rc:
            _native.check(rc, "eux_moe_dispatch_launch")
        _launches += 1 if self.n_tokens * self.topk <= _ROUTE_SELF else 2

    def expert_ready(self) -> None:
        global _launches
        rc = _native.load().eux_moe_expert_ready_launch(self._desc(), _native.current_stream_ptr())
        if rc:
            _native.check(rc, "eux_moe_expert_ready_launch")
        _launches += 1

    def combine(self, ctas: int = 0) -> torch.Tensor:
        global _launches
        rc = _native.load().eux_moe_combine_launch(self._desc(), ctas, _native.current_stream_ptr())
        if rc:
            _native.check(rc, "eux_moe_combine_launch")
        _launches += 1
        return self.out

    # -- views for tests / expert code --------------------------------------
    def recv_counts(self) -> torch.Tensor:
        """rows received from each source rank (valid after expert_ready)."""
        epr = self.n_experts // self.world
        return self.flags.view(torch.int64, 3 * self.world + self.world * epr)[self.world:2 * self.world]

    def recv_rows(self, src: int, n: int) -> torch.Tensor:
        off = src * self.capacity * self.row_bytes
        return self.arena.local[off: off + n * self.row_bytes].view(n, self.row_bytes)

    def recv_meta(self, src: int, n: int) -> torch.Tensor:
        off = src * self.capacity * 16
        return self.meta.local[off: off + n * 16].view(torch.int32).view(n, 4)

    def check_status(self) -> None:
        s = int(self.status.item())
        if s:
            raise RuntimeError(f"moe kernel status code={s & 0xff} where={s >> 8}")


def reference_dispatch_combine(x: torch.Tensor, topk_idx: torch.Tensor, topk_w: torch.Tensor, fp8: bool) -> torch.Tensor:
    """Plain PyTorch fp32 statement of dispatch -> identity expert -> weighted combine."""
    xf = x.float()
    if fp8:
        t, h = xf.shape
        g = xf.view(t, h // 128, 128)
        scale = g.abs().amax(-1, keepdim=True).clamp_min(1e-10) * (1.0 / 448.0)
        q = (g * (1.0 / scale)).to(torch.float8_e4m3fn).float()
        xf = (q * scale).view(t, h)
    valid = (topk_idx >= 0).float()
    wsum = (topk_w * valid).sum(-1, keepdim=True)
    return xf * wsum


# ---- choice of experts ---------------------------------------------------

ROUTE_MAX_EXPERTS = 1024


def route(logits: torch.Tensor, topk: int, *, scoring: str = "softmax", bias: Optional[torch.Tensor] = None, groups: int = 1,
          topk_groups: int = 1, renormalize: bool = True, scale: float = 1.0) -> Tuple[torch.Tensor, torch.Tensor]:
    """The ``topk`` experts of each token and their weights, as ``MoeAllToAll.dispatch`` and ``MoeExperts`` take them:
    int32 and float32, both ``[tokens, topk]``, largest score first, ties to the lowest expert.

    ``logits`` is ``[tokens, experts]``, float32 or bfloat16; its rows may lie apart. Scores are the softmax over all
    experts or the sigmoid of each. ``bias`` (float32, ``[experts]``) is added for the choice and left out of the weights.
    With ``groups`` the experts are that many equal runs, and only those of the ``topk_groups`` runs with the largest sum
    of two scores are chosen from. ``renormalize`` divides a token's weights by their sum (one that is zero in 64 bits gives weights
    of zero), ``scale`` multiplies them. An expert whose logit or bias is -inf or NaN is never chosen; where fewer than
    ``topk`` are left, the last places are expert -1 with weight 0. A logit of +inf weighs as the largest number does. For
    inference: the weights have no gradient."""
    global _launches
    ws.require(isinstance(logits, torch.Tensor) and logits.dim() == 2, "logits must be a matrix")
    dtype = logits.dtype
    t, e = logits.shape
    stride, inner_stride = logits.stride()
    if not (dtype is torch.float32 or dtype is torch.bfloat16):
        raise ValueError(f"logits must be float32 or bfloat16, not {dtype}")
    if not 1 <= e <= ROUTE_MAX_EXPERTS:
        raise ValueError(f"there must be 1 to {ROUTE_MAX_EXPERTS} experts, not {e}")
    if inner_stride != 1 and e != 1:
        raise ValueError("a token's logits must lie side by side")
    if not 1 <= topk <= min(32, e):
        raise ValueError(f"topk must be 1 to {min(32, e)}, not {topk}")
    if scoring not in ("softmax", "sigmoid"):
        raise ValueError(f"scoring must be softmax or sigmoid, not {scoring!r}")
    if not 1 <= groups <= 32 or e % groups:
        raise ValueError(f"{e} experts are not {groups} groups (of up to 32)")
    if not 1 <= topk_groups <= groups:
        raise ValueError(f"topk_groups must be 1 to {groups}, not {topk_groups}")
    device = logits.device
    if bias is not None:
        ws.require_dense(bias, "bias", torch.float32, (e,))
        ws.require_device(device, bias=bias)
    ws.require_cuda(device)
    idx = torch.empty_strided((t, topk), (topk, 1), dtype=torch.int32, device=device)
    w = torch.empty_strided((t, topk), (topk, 1), dtype=torch.float32, device=device)
    if t:
        desc = _native.descriptor(_native.ROUTE_DESC, _native.RouteDesc, logits.data_ptr(), bias.data_ptr() if bias is not None else 0,
                                  idx.data_ptr(), w.data_ptr(), stride, t, e, topk, _native.DT_F32 if dtype is torch.float32 else _native.DT_BF16,
                                  int(scoring == "sigmoid"), groups, topk_groups, int(renormalize), float(scale), 0)
        ws.launch(_native.load().eux_route_launch, desc, device.index, "eux_route_launch")
        _launches += 1
    return idx, w


# ---- the experts ------------------------------------------------------------

class MoeExperts:
    """The experts of one GPU: ``out[t] = sum_k w[t,k] * W_down[e] (silu(W_gate[e] x[t]) * (W_up[e] x[t]))``, ``e = idx[t,k]``.

    ``w_gate_up`` is ``[experts, 2 * inner, hidden]`` (gate rows, then up rows) and ``w_down`` ``[experts, hidden, inner]``,
    both bfloat16, or both float8_e4m3fn with float32 scales of 128 x 128 blocks: ``gate_up_scale`` ``[experts,
    ceil(2 * inner / 128), ceil(hidden / 128)]`` and ``down_scale`` ``[experts, ceil(hidden / 128), ceil(inner / 128)]`` (what
    ``remote_gemm.quantize_blocks_128x128`` gives for each expert). They are used where they lie: the object keeps their memory
    and copies nothing, so what is written into it holds for the next call (a parameter whose ``data`` is set to other memory leaves
    the object with what it was given). ``hidden`` and ``inner`` are multiples of 8 (16 for e4m3). e4m3 weights are no NaN, which is checked
    when they are given and not again: one that is written later counts as 480.

    Made for few tokens, where the layer is as fast as the weights of the named experts can be read: rows beyond
    ``MAX_TOKENS`` go in passes of that many, each of which reads its experts again. For inference: the result has no
    gradient. An object is made outside of graph captures; its calls may be captured, and made by several threads. A graph may
    outlive the object, but not the weights."""

    MAX_TOKENS = 128
    MAX_EXPERTS = 1024

    def __init__(self, w_gate_up: torch.Tensor, w_down: torch.Tensor, gate_up_scale: Optional[torch.Tensor] = None,
                 down_scale: Optional[torch.Tensor] = None):
        for name, w in (("w_gate_up", w_gate_up), ("w_down", w_down)):
            ws.require(isinstance(w, torch.Tensor) and w.dim() == 3, f"{name} must be [experts, rows, columns]")
        self.n_experts, self.hidden, self.inner = e, h, i = w_down.shape
        dtype = w_down.dtype
        ws.require(dtype in (torch.bfloat16, torch.float8_e4m3fn), f"weights must be bfloat16 or float8_e4m3fn, not {dtype}")
        self.fp8 = dtype == torch.float8_e4m3fn
        unit = 16 if self.fp8 else 8
        ws.require(1 <= e <= self.MAX_EXPERTS, f"there must be 1 to {self.MAX_EXPERTS} experts, not {e}")
        ws.require(h > 0 and i > 0 and h % unit == 0 and i % unit == 0, f"hidden and inner must be multiples of {unit}, not {h} and {i}")
        ws.require_dense(w_gate_up, "w_gate_up", dtype, (e, 2 * i, h))
        ws.require_dense(w_down, "w_down", dtype, (e, h, i))
        blocks = lambda n: -(-n // 128)  # noqa: E731
        ws.require((gate_up_scale is not None) == self.fp8 and (down_scale is not None) == self.fp8, "float8_e4m3fn weights have scales, bfloat16 weights none")
        if self.fp8:
            ws.require_dense(gate_up_scale, "gate_up_scale", torch.float32, (e, blocks(2 * i), blocks(h)))
            ws.require_dense(down_scale, "down_scale", torch.float32, (e, blocks(h), blocks(i)))
        self.device = w_down.device
        ws.require_device(self.device, w_gate_up=w_gate_up, gate_up_scale=gate_up_scale, down_scale=down_scale)
        ws.require_cuda(self.device)
        ws.require((w_gate_up.data_ptr() | w_down.data_ptr()) % 16 == 0, "weights must begin on 16 bytes")
        # the memory, whatever becomes of the tensors: a parameter's may be exchanged
        self._weights = tuple(w.detach() if w is not None else None for w in (w_gate_up, w_down, gate_up_scale, down_scale))
        self._weight_ptrs = tuple(w.data_ptr() if w is not None else 0 for w in self._weights)
        self.status = torch.zeros(1, dtype=torch.int32, device=self.device)
        self._status_ptr, self._index = self.status.data_ptr(), self.device.index
        self._need = {}
        lib = _native.load()
        if self.fp8:
            # the kernels widen e4m3 by moving bits, which has no place for NaN
            found = torch.zeros(1, dtype=torch.int32, device=self.device)
            with ws.on_device(self._index) as stream:
                for w in (w_gate_up, w_down):
                    _native.check(lib.eux_experts_find_nan(w.data_ptr(), w.numel(), found.data_ptr(), stream), "eux_experts_find_nan")
                ws.require(int(found.item()) == 0, "e4m3 weights must not be NaN")
        self._room = C.create_string_buffer(256 + 64)
        self._maps = (C.addressof(self._room) + 63) & ~63
        with ws.on_device(self._index):
            _native.check(lib.eux_experts_maps(self._desc(1, 1), self._maps), "eux_experts_maps")
        self._scratch = ws.CallScratch(int(lib.eux_experts_counter_words(self._desc(1, 1))), self.device, keep=(self.status,))

    w_gate_up = property(lambda self: self._weights[0])
    w_down = property(lambda self: self._weights[1])
    gate_up_scale = property(lambda self: self._weights[2])
    down_scale = property(lambda self: self._weights[3])

    def _desc(self, tokens, topk, x=0, idx=0, w=0, out=0, workspace=0, counters=0, x_stride=0, out_stride=0):
        """An ``eux_experts_desc`` of one pass."""
        return _native.descriptor(
            _native.EXPERTS_DESC, _native.ExpertsDesc, x, idx, w, out, *self._weight_ptrs, workspace, counters, self._status_ptr, self._maps,
            x_stride, out_stride, 2_000_000_000, tokens, self.hidden, self.inner, self.n_experts, topk, int(self.fp8))

    def __call__(self, x: torch.Tensor, topk_idx: torch.Tensor, topk_w: torch.Tensor, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """``x`` is ``[tokens, hidden]`` bfloat16, ``topk_idx`` (int32) and ``topk_w`` (float32) are ``[tokens, topk]``, up to 32
        per token. An entry whose expert is not in ``[0, experts)`` adds nothing: with the experts of one of several GPUs, pass
        the indices less the number of its first expert, and add up the GPUs' results. A token without entries gets zeros.
        ``out`` may be ``x`` itself, but beyond ``MAX_TOKENS`` rows not share a part of its memory; the rows of both may lie apart.
        Sums are in float32; what lies between the two products is rounded to bfloat16, or with up to eight tokens, of which no expert
        has more than four, to two such numbers: a token's last bits may depend on what else is in the call. The same arguments give
        the same bits. A wait in the kernels that runs out (two seconds) is told by ``check_status``; the result is none then."""
        global _launches
        index, hidden = self._index, self.hidden
        # what a call usually brings, with as few questions as tell it from everything else
        if (isinstance(x, torch.Tensor) and isinstance(topk_idx, torch.Tensor) and isinstance(topk_w, torch.Tensor)
                and x.dtype is torch.bfloat16 and topk_idx.dtype is torch.int32 and topk_w.dtype is torch.float32
                and topk_idx.dim() == 2 and (shape := topk_idx.shape) == topk_w.shape and x.shape == (shape[0], hidden) and 1 <= shape[1] <= 32
                and x.is_contiguous() and topk_idx.is_contiguous() and topk_w.is_contiguous() and x.data_ptr() % 16 == 0
                and x.get_device() == topk_idx.get_device() == topk_w.get_device() == index):
            xs = hidden
        else:
            self._require(x, topk_idx, topk_w)
            shape, xs = topk_idx.shape, ws.row_stride(x)
        t, topk = shape
        if out is None:
            out, os_ = torch.empty_strided((t, hidden), (hidden, 1), dtype=torch.bfloat16, device=self.device), hidden
        elif out is x:
            os_ = xs
        else:
            ws.require_rows(out, "out", torch.bfloat16, cols=hidden, rows=t)
            ws.require_device(self.device, out=out)
            if t > self.MAX_TOKENS:
                ws.require_apart(out, x, "x")  # a pass reads what the passes before it have not written
            os_ = ws.row_stride(out)
        lib = _native.load()
        for first in range(0, t, self.MAX_TOKENS):
            n = min(self.MAX_TOKENS, t - first)
            need = self._need.get((n, topk))
            if need is None:
                need = int(lib.eux_experts_workspace_bytes(self._desc(n, topk)))
                ws.require(need > 0, f"{n} x {topk} entries of {self.n_experts} experts of {hidden} x {self.inner} are too many for one call")
                self._need[n, topk] = need
            workspace, counters = self._scratch.get(need)
            desc = self._desc(n, topk, x.data_ptr() + 2 * first * xs, topk_idx.data_ptr() + 4 * first * topk, topk_w.data_ptr() + 4 * first * topk,
                              out.data_ptr() + 2 * first * os_, workspace, counters, xs, os_)
            ws.launch(lib.eux_experts_launch, desc, index, "eux_experts_launch")
            _launches += 3 if n > 8 or hidden % 128 else 2  # as the launch chooses
        return out

    def _require(self, x, topk_idx, topk_w) -> None:
        ws.require_rows(x, "x", torch.bfloat16, cols=self.hidden)
        t = x.shape[0]
        ws.require(isinstance(topk_idx, torch.Tensor) and topk_idx.dim() == 2 and topk_idx.shape[0] == t, f"topk_idx must be [{t}, topk]")
        topk = topk_idx.shape[1]
        ws.require(1 <= topk <= 32, f"topk must be 1 to 32, not {topk}")
        ws.require_dense(topk_idx, "topk_idx", torch.int32, (t, topk))
        ws.require_dense(topk_w, "topk_w", torch.float32, (t, topk))
        ws.require_device(self.device, x=x, topk_idx=topk_idx, topk_w=topk_w)

    def check_status(self) -> None:
        s = int(self.status.item())
        if s:
            torch.cuda.synchronize(self.device)  # calls on other streams still count in the words
            self._scratch.reset()
            self.status.zero_()
            raise RuntimeError(f"moe experts status code={s & 0xff} where={s >> 8}")


def reference_experts(x: torch.Tensor, topk_idx: torch.Tensor, topk_w: torch.Tensor, w_gate_up: torch.Tensor, w_down: torch.Tensor,
                      gate_up_scale: Optional[torch.Tensor] = None, down_scale: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Plain PyTorch statement of the experts in 64 bits."""
    def full(w, scale):
        w = w.double()
        if scale is None:
            return w
        return w * scale.double().repeat_interleave(128, 0)[:w.shape[0]].repeat_interleave(128, 1)[:, :w.shape[1]]
    e, h, i = w_down.shape
    out = torch.zeros(x.shape[0], h, dtype=torch.float64, device=x.device)
    for j in range(e):
        tok, slot = (topk_idx == j).nonzero(as_tuple=True)
        if tok.numel():
            gu = x[tok].double() @ full(w_gate_up[j], None if gate_up_scale is None else gate_up_scale[j]).t()
            y = (torch.nn.functional.silu(gu[:, :i]) * gu[:, i:]) @ full(w_down[j], None if down_scale is None else down_scale[j]).t()
            out.index_add_(0, tok, y * topk_w[tok, slot].double().unsqueeze(1))
    return out
