"""The global norm over many gradient tensors and clipping by it, on the gfx950 HIP kernels.

The gradients of stacked adapters belong to different models that train side by side: with ``per_adapter`` the leading
axis of every tensor is the adapter, each adapter has its own norm over all tensors and is clipped to its own
limit.  Norms are taken in float64 and nothing is read back to the host.  Tensors are torch CUDA (ROCm)
tensors; kernels are enqueued on torch's current stream.  There is no CPU or eager fallback.
"""

from __future__ import annotations

import bisect
import math

import torch

from ... import _native
from .w8a8_lora import _on, _require_cuda, _stream_ptr, _scaling_vector

MAX_TENSORS = 65536
_TYPES = {torch.bfloat16: _native.GRAD_BF16, torch.float32: _native.GRAD_F32}


def _checked_table(grads, outs, per_adapter):
    """The C table of ``grads`` and ``outs`` and the adapters, or what is wrong with them."""
    dev = grads[0].device
    for i, g in enumerate(grads):
        if g.dtype not in _TYPES:
            raise TypeError(f"gradients must be BF16 or FP32, got {g.dtype} at {i}")
        _require_cuda(g, f"gradient {i}")
        if g.device != dev:
            raise ValueError(f"all gradients must be on {dev}, got {g.device} at {i}")
        if not g.is_contiguous():
            raise ValueError(f"gradients must be contiguous, got strides {g.stride()} at {i}")
        if per_adapter and (g.ndim == 0 or g.shape[0] != grads[0].shape[0]):
            raise ValueError(f"with per_adapter the leading axis of every gradient is the adapter, got {tuple(g.shape)} at {i}")
    adapters = grads[0].shape[0] if per_adapter else 1
    if not 0 < adapters <= 65535:
        raise ValueError(f"1 to 65535 adapters are supported, got {adapters}")
    if outs is not None:
        if len(outs) != len(grads):
            raise ValueError(f"out names {len(outs)} tensors for {len(grads)} gradients")
        for i, (g, o) in enumerate(zip(grads, outs)):
            if o.dtype != g.dtype or o.shape != g.shape or o.device != dev or not o.is_contiguous():
                raise ValueError(f"out must be contiguous {g.dtype} {tuple(g.shape)} on {dev} at {i}, got {o.dtype} {tuple(o.shape)}")
        spans = sorted((o.data_ptr(), o.data_ptr() + o.numel() * o.element_size()) for o in outs if o.numel())
        if any(start < end for (_, end), (start, _) in zip(spans, spans[1:])):
            raise ValueError("two outputs overlap in memory (a gradient given twice cannot be scaled in place)")
        starts = [start for start, _ in spans]
        for i, (g, o) in enumerate(zip(grads, outs)):
            behind = bisect.bisect_left(starts, g.data_ptr() + g.numel() * g.element_size())  # outputs that begin in front of the gradient's end
            if g.numel() and g.data_ptr() != o.data_ptr() and behind and spans[behind - 1][1] > g.data_ptr():
                raise ValueError(f"gradient {i} overlaps an output in memory (only its own, at the same place, may)")
    table = (_native.GradTensor * len(grads))()
    for i, g in enumerate(grads):
        table[i].grad = g.data_ptr()
        table[i].out = outs[i].data_ptr() if outs is not None else None
        table[i].count = g.numel() // adapters
        table[i].type = _TYPES[g.dtype]
    return table, adapters


class GradClipPlan:
    """Validated gradients, outputs, workspace and the C table of one norm-and-clip call; ``run()`` is a single C call on torch's
    current stream that neither allocates nor synchronizes, so it can be captured in a HIP graph.

    ``grads`` are contiguous bf16 or float32 tensors, read at every run where they lie: a loop whose backward writes the same
    buffers each step (``BackwardPlan``) builds the plan once.  ``max_norm`` is a number or a tensor (one value, or [adapters]
    with ``per_adapter``); None: only norms.  A contiguous float32 [adapters] tensor on the gradients' device is read at every
    run where it lies, any other form is copied when the plan is made.  Runs of a plan share its workspace: on one stream, or one behind the
    other; a graph that captured one needs the plan as long as it is replayed.  ``out`` names the tensors that the scaled gradients go
    to, of the same shapes and types; the gradients themselves scale in place."""

    def __init__(self, grads, max_norm=None, *, per_adapter: bool = False, out=None):
        grads = list(grads)
        if not grads:
            raise ValueError("at least one gradient is needed")
        if len(grads) > MAX_TENSORS:
            raise ValueError(f"at most {MAX_TENSORS} gradients are supported, got {len(grads)}")
        if type(per_adapter) is not bool:
            raise TypeError("per_adapter must be an exact bool")
        if max_norm is None and out is not None:
            raise ValueError("out given without max_norm")
        if max_norm is not None and not isinstance(max_norm, torch.Tensor) and not (math.isfinite(max_norm) and max_norm >= 0):
            raise ValueError(f"max_norm must be a finite number that is not negative, got {max_norm!r}")
        outs = None
        if max_norm is not None:
            outs = list(out) if out is not None else [torch.empty_like(g) for g in grads]
        # (2.5 us a tensor in Python: an ordinary table is made by the host module)
        host = _native.host() if isinstance(grads[0], torch.Tensor) and grads[0].is_cuda else None
        made = host.grad_table(grads, outs, per_adapter) if host is not None else None
        if made is not None:
            table, adapters = (_native.GradTensor * len(grads)).from_buffer_copy(made[0]), made[1]
        else:
            table, adapters = _checked_table(grads, outs, per_adapter)
        dev = grads[0].device
        limits = None
        if max_norm is not None:
            limits = _scaling_vector(max_norm if isinstance(max_norm, torch.Tensor) else float(max_norm), adapters, dev).detach()
            if tuple(limits.shape) != (adapters,):
                raise ValueError(f"max_norm must be a number or have shape ({adapters},), got {tuple(limits.shape)}")
        self._lib = _native.load()
        ws_bytes = int(self._lib.mi355_w8a8_grad_workspace_bytes(table, len(grads), adapters))
        if ws_bytes == 0:
            raise ValueError("the gradients hold more values than the native path supports")
        self.grads, self.out, self.limits, self.device = grads, outs, limits, dev
        self.norms = torch.empty(adapters, dtype=torch.float32, device=dev)
        self._per_adapter = per_adapter
        self._workspace = torch.empty(ws_bytes, dtype=torch.uint8, device=dev)
        self._table, self._adapters = table, adapters
        self._table_kept = 0  # FLAG_GRAD_TABLE_KEPT once a run has written the tensors' table into the workspace

    def run(self):
        """Enqueue the call; returns ``(out, norms)``, the reused outputs (None without ``max_norm``) and float32 norms ([adapters], or
        one value without ``per_adapter``) of the gradients before clipping."""
        ws, table = self._workspace, self._table
        with _on(self.device):
            flags = self._table_kept
            stream = _stream_ptr(self.device)
            if self.limits is None:
                status = self._lib.mi355_w8a8_grad_norm_v1(table, len(table), self._adapters, self.norms.data_ptr(), ws.data_ptr(), ws.numel(),
                                                           flags, stream)
            else:
                status = self._lib.mi355_w8a8_grad_clip_v1(table, len(table), self._adapters, self.limits.data_ptr(), self.norms.data_ptr(),
                                                           ws.data_ptr(), ws.numel(), flags, stream)
            written = not flags and not torch.cuda.is_current_stream_capturing()  # (a captured run has written nothing yet)
        _native.check("mi355_w8a8_grad_norm_v1" if self.limits is None else "mi355_w8a8_grad_clip_v1", status)
        if written:
            self._table_kept = _native.FLAG_GRAD_TABLE_KEPT
        return self.out, (self.norms if self._per_adapter else self.norms.reshape(()))


def grad_norm(grads, *, per_adapter: bool = False) -> torch.Tensor:
    """The norm over all ``grads`` together, float32: one value, or with ``per_adapter`` one for each index of their leading axis."""
    return GradClipPlan(grads, per_adapter=per_adapter).run()[1]


def clip_grad_norm(grads, max_norm, *, per_adapter: bool = False):
    """``(scaled gradients, norms)``: new tensors, each adapter's (or all) gradients times ``max_norm / norm`` where the norm is larger."""
    return GradClipPlan(grads, max_norm, per_adapter=per_adapter).run()


def clip_grad_norm_(grads, max_norm, *, per_adapter: bool = False) -> torch.Tensor:
    """``clip_grad_norm`` in place; returns the norms before clipping."""
    grads = list(grads)
    return GradClipPlan(grads, max_norm, per_adapter=per_adapter, out=grads).run()[1]


__all__ = ("GradClipPlan", "MAX_TENSORS", "clip_grad_norm", "clip_grad_norm_", "grad_norm")
