"""Ragged per-expert products on bf16 weights and their gradients, on the gfx950 HIP kernels.

The ``ragged_dot`` of the reference's ``skyrl/tx/layers/util.py:8-59`` for the expert kernels that
``LoRAExpert.__call__`` (skyrl/tx/layers/lora.py:394-444) holds unquantized: rows sorted by group,
``group_sizes[g]`` of them for group ``g``, rows beyond ``sum(group_sizes)`` giving zeros.  The
W8A8 form is ``w8a8_lora.grouped_lora_linear``.

Tensors are torch CUDA (ROCm) tensors; kernels are enqueued on torch's current stream.  Nothing is read
back to the host: the group sizes may come straight from ``w8a8_lora.moe_dispatch``.  There is no CPU
or eager fallback.
"""

from __future__ import annotations

import ctypes
import threading
import weakref

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from ... import _native
from .w8a8_lora import _on, _require_cuda, _stream_ptr

MAX_GROUPS = 1024
MAX_ROWS = 1 << 20
MAX_FEATURES = 65536


def _bf16(t: torch.Tensor, name: str) -> torch.Tensor:
    if t.dtype != torch.bfloat16:
        raise TypeError(f"{name} must be BF16, got {t.dtype}")
    _require_cuda(t, name)
    t = t.detach().contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()  # (a view into the middle of a buffer: the kernels load 16 bytes)


def whole_numbers(t: torch.Tensor, name: str, low: int, high: int) -> torch.Tensor:
    """``t`` as int32, with what that cannot hold at ``low`` or ``high``.  (Clamped as int64: a narrower type may not hold the bounds, and
    those of an unsigned one turn over.)"""
    if t.dtype.is_floating_point or t.dtype.is_complex or t.dtype in (torch.bool, torch.uint64):
        raise TypeError(f"{name} must be integers that int64 holds, got {t.dtype}")
    if t.dtype in (torch.int64, torch.uint32):
        t = t.to(torch.int64).clamp(low, high)
    return t.to(torch.int32)


def _geometry(rows: torch.Tensor, name: str, width: int, weight_shape, group_sizes: torch.Tensor):
    """``(m, k, n, groups, sizes)`` of a call, or what is wrong with it."""
    if len(weight_shape) != 3:
        raise ValueError(f"weight must be [groups, K, N], got {tuple(weight_shape)}")
    g, k, n = weight_shape
    if rows.ndim != 2 or rows.shape[0] <= 0 or rows.shape[1] != weight_shape[width]:
        raise ValueError(f"{name} must be [rows, {weight_shape[width]}] with at least one row, got {tuple(rows.shape)}")
    if group_sizes.ndim != 1 or group_sizes.shape[0] != g:
        raise ValueError(f"group_sizes must have shape ({g},), got {tuple(group_sizes.shape)}")
    m = rows.shape[0]
    sizes = whole_numbers(group_sizes.detach(), "group_sizes", 0, m)  # (what an int32 could not hold is more than there are rows)
    if k % 8 or n % 8 or not 0 < k <= MAX_FEATURES or not 0 < n <= MAX_FEATURES:
        raise ValueError(f"K and N must be positive multiples of 8 not exceeding {MAX_FEATURES}, got {k} and {n}")
    if not 0 < g <= MAX_GROUPS or m > MAX_ROWS:
        raise ValueError(f"at most {MAX_GROUPS} groups and {MAX_ROWS} rows are supported, got {g} and {m}")
    return m, k, n, g, sizes.to(rows.device).contiguous()


_TILES = (0, _native.FLAG_BF16_GROUPED_TILE_256X256, _native.FLAG_BF16_GROUPED_TILE_128X256, _native.FLAG_BF16_GROUPED_TILE_64X128)


def _check_flags(flags: int) -> None:
    """The tiles are all that a caller may force: the C calls know a flag for the type of dw too, which has to be that of the tensor."""
    if flags not in _TILES:
        raise ValueError(f"flags must be 0 or one of FLAG_BF16_GROUPED_TILE_*, got {flags!r}")


def _same_device(first: torch.Tensor, *others) -> None:
    for t in others:
        if t.device != first.device:
            raise ValueError(f"all operands must be on {first.device}, got {t.device}")


def grouped_matmul(x: torch.Tensor, weight: torch.Tensor, group_sizes: torch.Tensor, *, flags: int = 0) -> torch.Tensor:
    """``out[rows of g] = bf16(x[rows of g] @ weight[g])`` with float32 sums: x bf16 [rows, K], weight bf16
    [groups, K, N], group_sizes integers [groups].  Rows behind the last group are zero.  ``flags`` may force the tiles
    (``_native.FLAG_BF16_GROUPED_TILE_*``); by default they follow the sizes."""
    _check_flags(flags)
    host = _native.host() if isinstance(x, torch.Tensor) and x.is_cuda else None
    if host is not None:
        # an ordinary call goes through the host module; for any other it returns None
        result = host.grouped(x, weight, group_sizes, flags, _native.entry_address["bf16_grouped"],
                              _native.entry_address["bf16_grouped_workspace_bytes"], _stream_ptr(x.device))
        if type(result) is int:
            _native.check("mi355_w8a8_bf16_grouped_v1", result)
        if result is not None:
            return result
    xc, w = _bf16(x, "x"), _bf16(weight, "weight")
    _same_device(x, weight)
    m, k, n, g, sizes = _geometry(x, "x", 1, weight.shape, group_sizes)
    out = torch.empty((m, n), dtype=torch.bfloat16, device=x.device)
    lib = _native.load()
    ws = torch.empty(lib.mi355_w8a8_bf16_grouped_workspace_bytes(m, k, n, g, flags), dtype=torch.uint8, device=x.device)
    p = _native.Bf16GroupedProblem(ctypes.sizeof(_native.Bf16GroupedProblem), flags, m, k, n, g, xc.data_ptr(), w.data_ptr(),
                                   sizes.data_ptr(), out.data_ptr(), ws.data_ptr(), ws.numel())
    with _on(x.device):
        status = lib.mi355_w8a8_bf16_grouped_v1(ctypes.byref(p), _stream_ptr(x.device))
    _native.check("mi355_w8a8_bf16_grouped_v1", status)
    return out


def grouped_matmul_backward(x: torch.Tensor | None, dy: torch.Tensor, weight: torch.Tensor | None, group_sizes: torch.Tensor, *,
                            need_dx: bool = True, need_dw: bool = True, dw_dtype: torch.dtype = torch.bfloat16, flags: int = 0):
    """Cotangents ``(dx, dw)`` of ``grouped_matmul``: ``dx[rows of g] = bf16(dy[rows of g] @ weight[g].T)`` and
    ``dw[g] = x[rows of g].T @ dy[rows of g]`` in ``dw_dtype`` (bf16 or float32), both from float32 sums; None for the one
    that is not wanted.  ``x`` may be None without ``need_dw``, ``weight`` without ``need_dx``."""
    need_dx, need_dw = bool(need_dx), bool(need_dw)  # (the host module takes True alone for yes)
    if not need_dx and not need_dw:
        return None, None
    if (need_dw and x is None) or (need_dx and weight is None):
        raise ValueError("dw needs x and dx needs weight")
    if dw_dtype not in (torch.bfloat16, torch.float32):
        raise TypeError(f"dw_dtype must be BF16 or FP32, got {dw_dtype}")
    _check_flags(flags)
    host = _native.host() if isinstance(dy, torch.Tensor) and dy.is_cuda else None
    if host is not None:
        result = host.grouped_bwd(x, dy, weight, group_sizes, need_dx, need_dw, dw_dtype == torch.float32, flags,
                                  _native.entry_address["bf16_grouped_bwd"], _native.entry_address["bf16_grouped_bwd_workspace_bytes"],
                                  _stream_ptr(dy.device))
        if type(result) is int:
            _native.check("mi355_w8a8_bf16_grouped_bwd_v1", result)
        if result is not None:
            return result
    d = _bf16(dy, "dy")
    xc = _bf16(x, "x") if need_dw else None
    w = _bf16(weight, "weight") if need_dx else None
    _same_device(dy, *(t for t in (xc, w) if t is not None))
    shape = weight.shape if weight is not None else (group_sizes.shape[0] if group_sizes.ndim else 0, x.shape[-1], dy.shape[-1])
    m, k, n, g, sizes = _geometry(dy, "dy", 2, shape, group_sizes)
    if need_dw and tuple(x.shape) != (m, k):
        raise ValueError(f"x must be [{m}, {k}], got {tuple(x.shape)}")
    dx = torch.empty((m, k), dtype=torch.bfloat16, device=dy.device) if need_dx else None
    dw = torch.empty((g, k, n), dtype=dw_dtype, device=dy.device) if need_dw else None
    lib = _native.load()
    ws = torch.empty(lib.mi355_w8a8_bf16_grouped_bwd_workspace_bytes(m, k, n, g, flags, need_dx, need_dw), dtype=torch.uint8, device=dy.device)
    p = _native.Bf16GroupedBwdProblem(ctypes.sizeof(_native.Bf16GroupedBwdProblem),
                                      flags | (_native.FLAG_BF16_GROUPED_DW_F32 if dw_dtype == torch.float32 else 0), m, k, n, g,
                                      xc.data_ptr() if need_dw else None, d.data_ptr(), w.data_ptr() if need_dx else None,
                                      sizes.data_ptr(), dx.data_ptr() if need_dx else None, dw.data_ptr() if need_dw else None,
                                      ws.data_ptr(), ws.numel())
    with _on(dy.device):
        status = lib.mi355_w8a8_bf16_grouped_bwd_v1(ctypes.byref(p), _stream_ptr(dy.device))
    _native.check("mi355_w8a8_bf16_grouped_bwd_v1", status)
    return dx, dw


class _LeafUse:
    """One use of a leaf in an autograd graph; lives as long as the graph."""

    __slots__ = ("leaf", "stream", "__weakref__")

    def __init__(self, leaf, stream):
        self.leaf, self.stream = weakref.ref(leaf), stream


_leaf_uses: weakref.WeakSet = weakref.WeakSet()
_leaf_uses_lock = threading.RLock()  # (a set that grows in another thread cannot be walked)


_LIVING = ("a backward pass is captured while a graph of the same parameters, made on another stream, lives: "
           "let go of its outputs (the last loss, say) first, or run it on a stream of its own, the capture's for one")


def note_leaves(*tensors: torch.Tensor) -> list:
    """Uses of those ``tensors`` that are leaves, for the graph to keep and ``check_capture`` to look at."""
    uses = [_LeafUse(t, _stream_ptr(t.device)) for t in tensors if t.requires_grad and t.is_leaf]
    with _leaf_uses_lock:
        _leaf_uses.update(uses)
    return uses


def _leaves_behind(node):
    """The leaves whose gradients the backward of ``node`` leads to, through whatever operations."""
    seen, todo = set(), [node]
    while todo:
        for behind, _ in todo.pop().next_functions:
            if behind is None or behind in seen:
                continue
            seen.add(behind)
            if behind.name() == "torch::autograd::AccumulateGrad":
                yield behind.variable
            else:
                todo.append(behind)


def check_capture(uses: list, node=None) -> None:
    """Refuse a backward pass under stream capture that would draw the default stream into the capture, which ends the process.  Autograd adds to
    a leaf's gradient on the stream on which the leaf was first used, by any operation, since a graph of it last lived throughout: the
    host module knows that stream, ``node`` (the backward's) the leaves.  (Any other stream joins the capture and leaves it again: a warm-up on a
    side stream may live on.)  Without the module: refuse it beside a graph of the same leaves made here on another stream."""
    if (not uses and node is None) or not torch.cuda.is_current_stream_capturing():
        return
    host = _native.host() if node is not None else None
    if host is not None:
        if any(host.accumulation_stream(leaf) == 0 for leaf in _leaves_behind(node) if leaf.is_cuda):
            raise RuntimeError(_LIVING)
        return
    with _leaf_uses_lock:
        others = list(_leaf_uses)
    for other in others:
        leaf = other.leaf()
        if leaf is not None and any(use.leaf() is leaf and use.stream != other.stream for use in uses):
            raise RuntimeError(_LIVING)


def refuse_tangents(name: str, *tensors) -> None:
    """Forward-mode derivatives do not exist here; a dual tensor's would be lost without a word."""
    for t in tensors:
        if isinstance(t, torch.Tensor) and forward_ad.unpack_dual(t).tangent is not None:
            raise NotImplementedError(f"{name} has no forward-mode derivative")


class _GroupedMatmulFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, group_sizes):
        ctx.uses = note_leaves(x, weight)
        ctx.save_for_backward(x if ctx.needs_input_grad[1] else None, weight if ctx.needs_input_grad[0] else None, group_sizes)
        ctx.shape = tuple(weight.shape)
        return grouped_matmul(x, weight, group_sizes)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        check_capture(ctx.uses, ctx)
        x, weight, group_sizes = ctx.saved_tensors
        dx, dw = grouped_matmul_backward(x, dy, weight, group_sizes, need_dx=ctx.needs_input_grad[0], need_dw=ctx.needs_input_grad[1])
        return dx, dw, None


def bf16_grouped_linear(x: torch.Tensor, weight: torch.Tensor, group_sizes: torch.Tensor) -> torch.Tensor:
    """``grouped_matmul`` that autograd can differentiate in ``x`` and ``weight``."""
    refuse_tangents("bf16_grouped_linear", x, weight)
    if not (torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad)):
        return grouped_matmul(x, weight, group_sizes)
    return _GroupedMatmulFunction.apply(x, weight, group_sizes)


__all__ = ("MAX_FEATURES", "MAX_GROUPS", "MAX_ROWS", "bf16_grouped_linear", "grouped_matmul", "grouped_matmul_backward")
