"""Embedding rows with scaling and the table's gradient by sorted tokens, on the gfx950 HIP kernels.

A table is ``[vocab, width]``, or ``[adapters, vocab, width]`` with one adapter and one factor for each token: the A
factors of a LoRA embedding, whose gradient is what its training needs.  Tensors are torch CUDA (ROCm)
tensors; kernels are enqueued on torch's current stream.  There is no CPU or eager fallback.
"""

from __future__ import annotations

import ctypes
import math

import torch
from torch.autograd.function import once_differentiable

from ... import _native
from .bf16_grouped_linear import check_capture, note_leaves, refuse_tangents, whole_numbers
from .w8a8_lora import _on, _require_cuda, _stream_ptr

MAX_TOKENS = 1 << 20
MAX_WIDTH = 65536
MAX_TABLE_ROWS = 1 << 30
_TYPES = {torch.bfloat16: 0, torch.float32: _native.FLAG_EMBEDDING_F32}


def _problem(ids, shape, scale, adapter_indices, dtype, dev):
    """The C struct of a call without its data tensors, and what it points at."""
    if dtype not in _TYPES:
        raise TypeError(f"embedding rows must be BF16 or FP32, got {dtype}")
    if ids.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"ids must be INT32 or INT64, got {ids.dtype}")
    _require_cuda(ids, "ids")
    if ids.device != dev:
        raise ValueError(f"ids must be on {dev}, got {ids.device}")
    if len(shape) not in (2, 3) or min(shape) <= 0:
        raise ValueError(f"the table must be [vocab, width] or [adapters, vocab, width], got {tuple(shape)}")
    vocab, width = shape[-2:]
    adapters = shape[0] if len(shape) == 3 else 0
    n = ids.numel()
    if n == 0:
        raise ValueError("ids must not be empty")
    if n > MAX_TOKENS or width > MAX_WIDTH or max(1, adapters) * vocab > MAX_TABLE_ROWS:
        raise ValueError(f"at most {MAX_TOKENS} ids, a width of {MAX_WIDTH} and {MAX_TABLE_ROWS} table rows are supported, got {n}, "
                         f"{width} and {max(1, adapters) * vocab}")
    flat = ids.detach().reshape(-1).contiguous()
    index = None
    if adapter_indices is not None:
        if not adapters:
            raise ValueError("adapter_indices given without a table of adapters")
        index = whole_numbers(adapter_indices.detach().reshape(-1), "adapter_indices", -1, adapters)
        if index.shape[0] != n:
            if index.shape[0] == 0 or n % index.shape[0]:
                raise ValueError(f"adapter_indices of length {index.shape[0]} do not divide {n} ids")
            index = index.repeat_interleave(n // index.shape[0])  # one entry per example
        index = index.to(dev).contiguous()
    elif adapters > 1:
        raise ValueError("a table of several adapters needs adapter_indices")
    scales, factor = None, 1.0
    if isinstance(scale, torch.Tensor):
        if scale.numel() != max(1, adapters) or scale.ndim > 1:
            raise ValueError(f"scale must be a number or have shape ({max(1, adapters)},), got {tuple(scale.shape)}")
        if not adapters:
            raise TypeError("the scale of a plain table must be a number")
        scales = scale.detach().to(device=dev, dtype=torch.float32).reshape(-1).contiguous()
    elif scale is not None:
        factor = ctypes.c_float(scale).value
        if not math.isfinite(factor):
            raise ValueError(f"scale must be finite as float32, got {scale!r}")
    p = _native.EmbeddingProblem(ctypes.sizeof(_native.EmbeddingProblem),
                                 _TYPES[dtype] | (_native.FLAG_EMBEDDING_IDS64 if flat.dtype == torch.int64 else 0), n, vocab, width, adapters,
                                 factor, 0)
    p.ids = flat.data_ptr()
    p.adapter_indices = index.data_ptr() if index is not None else None
    p.scales = scales.data_ptr() if scales is not None else None
    return p, (flat, index, scales)


def lookup(table: torch.Tensor, ids: torch.Tensor, scale=None, *, adapter_indices: torch.Tensor | None = None) -> torch.Tensor:
    """``scale * table[ids]`` (``scale[a] * table[a, ids]`` with ``a = adapter_indices`` for a table of adapters), the product
    in float32 and one rounding to the table's type.  ``ids`` int32 or int64 of any shape; ``scale`` a number, or for adapters
    float32 [adapters]; ``adapter_indices`` one entry per id, or per example (a divisor of the ids).  Ids and
    adapters out of range read zeros."""
    host = _native.host() if isinstance(table, torch.Tensor) and table.is_cuda else None
    if host is not None:
        # an ordinary call goes through the host module; for any other it returns None
        result = host.embedding(table, ids, scale, adapter_indices, _native.entry_address["embedding"], _stream_ptr(table.device))
        if type(result) is int:
            _native.check("mi355_w8a8_embedding_v1", result)
        if result is not None:
            return result
    _require_cuda(table, "table")
    p, keep = _problem(ids, tuple(table.shape), scale, adapter_indices, table.dtype, table.device)
    t = table.detach().contiguous()
    out = torch.empty((*ids.shape, p.width), dtype=table.dtype, device=table.device)
    p.table, p.out = t.data_ptr(), out.data_ptr()
    with _on(table.device):
        status = _native.load().mi355_w8a8_embedding_v1(ctypes.byref(p), _stream_ptr(table.device))
    _native.check("mi355_w8a8_embedding_v1", status)
    del keep
    return out


def lookup_backward(d_out: torch.Tensor, ids: torch.Tensor, table_shape, scale=None, *,
                    adapter_indices: torch.Tensor | None = None) -> torch.Tensor:
    """The table's gradient: ``scale * sum(d_out[t] for ids[t] == v)`` for every row v, in ``d_out``'s type (bf16 or
    float32) from float32 sums in the order of the ids, so that equal inputs give equal bits; zeros for rows that no id names."""
    shape = tuple(int(s) for s in table_shape)
    host = _native.host() if isinstance(d_out, torch.Tensor) and d_out.is_cuda else None
    if host is not None:
        result = host.embedding_bwd(d_out, ids, shape, scale, adapter_indices, _native.entry_address["embedding_bwd"],
                                    _native.entry_address["embedding_bwd_workspace_bytes"], _stream_ptr(d_out.device))
        if type(result) is int:
            _native.check("mi355_w8a8_embedding_bwd_v1", result)
        if result is not None:
            return result
    _require_cuda(d_out, "d_out")
    p, keep = _problem(ids, shape, scale, adapter_indices, d_out.dtype, d_out.device)
    if tuple(d_out.shape) != (*ids.shape, p.width):
        raise ValueError(f"d_out must have shape {(*ids.shape, p.width)}, got {tuple(d_out.shape)}")
    d = d_out.detach().contiguous()
    grad = torch.empty(shape, dtype=d_out.dtype, device=d_out.device)
    lib = _native.load()
    p.workspace_bytes = lib.mi355_w8a8_embedding_bwd_workspace_bytes(p.n_tokens, p.vocab, p.width, p.n_adapters, p.flags)
    ws = torch.empty(p.workspace_bytes, dtype=torch.uint8, device=d_out.device)
    p.d_out, p.out, p.workspace = d.data_ptr(), grad.data_ptr(), ws.data_ptr()
    with _on(d_out.device):
        status = lib.mi355_w8a8_embedding_bwd_v1(ctypes.byref(p), _stream_ptr(d_out.device))
    _native.check("mi355_w8a8_embedding_bwd_v1", status)
    del keep
    return grad


class _LookupFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, ids, scale, adapter_indices):
        ctx.uses = note_leaves(table)
        ctx.save_for_backward(ids, adapter_indices, scale if isinstance(scale, torch.Tensor) else None)
        ctx.shape, ctx.scale = tuple(table.shape), None if isinstance(scale, torch.Tensor) else scale
        return lookup(table, ids, scale, adapter_indices=adapter_indices)

    @staticmethod
    @once_differentiable
    def backward(ctx, d_out):
        check_capture(ctx.uses, ctx)
        ids, adapter_indices, scales = ctx.saved_tensors
        grad = lookup_backward(d_out, ids, ctx.shape, ctx.scale if scales is None else scales, adapter_indices=adapter_indices)
        return grad, None, None, None


def embed(table: torch.Tensor, ids: torch.Tensor, scale=None, *, adapter_indices: torch.Tensor | None = None) -> torch.Tensor:
    """``lookup`` that autograd can differentiate in the table (the scale is a constant)."""
    refuse_tangents("embed", table, scale)
    if isinstance(scale, torch.Tensor) and scale.requires_grad:
        raise ValueError("the scale of an embedding is a constant: detach it")
    if not (torch.is_grad_enabled() and table.requires_grad):
        return lookup(table, ids, scale, adapter_indices=adapter_indices)
    return _LookupFunction.apply(table, ids, scale, adapter_indices)


__all__ = ("MAX_TABLE_ROWS", "MAX_TOKENS", "MAX_WIDTH", "embed", "lookup", "lookup_backward")
