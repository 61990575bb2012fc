"""Token ids to drive: the stimulus table, and its gradient.

``stimulus_drive`` looks up ``scale * table[token]`` for every token, e.g. the soma drive of a
network that reads one token per tick; ``stimulus_gradient`` is its backward pass.  Both run in
CUDA kernels (``nsb_stimulus_drive``, ``nsb_stimulus_gradient``) on the current stream.

A token outside ``[0, len(table))`` (-1, say) stands for "no stimulus": its drive is zero, and it
takes no gradient.
"""

from __future__ import annotations

import ctypes

import torch

from .native import (VALUE_TYPES, _Matrix, dense_matrix, load_library, refuse_gradients, refuse_tangents,
                     token_call, written)


def _tokens(tokens: torch.Tensor, like: torch.Tensor) -> torch.Tensor:
    if tokens.dtype is not torch.int64 and tokens.dtype is not torch.int32:
        raise ValueError("tokens must be int32 or int64")
    if tokens.get_device() != like.get_device():
        raise ValueError("tokens must be on the table's CUDA device")
    return tokens if tokens.is_contiguous() else tokens.contiguous()


def _drive(tokens: torch.Tensor, table: torch.Tensor, scale: float, dtype: torch.dtype,
           out: torch.Tensor | None) -> torch.Tensor:
    view = dense_matrix(table, "table")
    tokens = _tokens(tokens, table)
    shape = (*tokens.shape, view.cols)
    given = out
    if out is None:
        out = table.new_empty(shape, dtype=dtype)
    elif out.shape != shape or out.dtype != dtype or out.device != table.device:
        raise ValueError("out must be a tensor of the drive's shape, dtype and device")
    elif not out.is_contiguous():
        raise ValueError("out must be contiguous")
    rows = _Matrix(out.data_ptr(), tokens.numel(), view.cols, view.cols, VALUE_TYPES[dtype])
    token_call(table, load_library().nsb_stimulus_drive, tokens.data_ptr(),
               tokens.element_size(), ctypes.byref(view), scale, ctypes.byref(rows))
    if given is not None:
        written(out)
    return out


class _StimulusDrive(torch.autograd.Function):
    @staticmethod
    def forward(ctx, tokens, table, scale, dtype):
        ctx.save_for_backward(tokens)
        ctx.scale, ctx.rows, ctx.dtype = scale, table.shape[0], table.dtype
        return _drive(tokens, table, scale, dtype, None)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        (tokens,) = ctx.saved_tensors
        return None, stimulus_gradient(tokens, grad, ctx.rows, scale=ctx.scale,
                                       dtype=ctx.dtype), None, None


def stimulus_drive(tokens: torch.Tensor, table: torch.Tensor, *, scale: float = 1.0,
                   dtype: torch.dtype | None = None,
                   out: torch.Tensor | None = None) -> torch.Tensor:
    """``scale * table[tokens]`` as [*tokens.shape, N], zero where a token is outside the table.

    ``tokens``: int32 or int64, any shape.  ``table``: [V, N] float32, float16 or bfloat16 with
    contiguous rows.  ``dtype``: the table's (the default) or float32; the product is taken in
    float32 and rounded once.  ``out`` (contiguous) receives the result where given; it cannot be
    combined with a table that requires a gradient.  There is no forward-mode derivative.
    """
    dtype = table.dtype if dtype is None else dtype
    if dtype != table.dtype and dtype != torch.float32:
        raise ValueError("dtype must be the table's or float32")
    refuse_tangents("stimulus_drive has no forward-mode derivative", table, out)
    if out is not None:
        refuse_gradients("out cannot be given where it or the table requires a gradient", table, out)
    elif table.requires_grad and torch.is_grad_enabled():
        return _StimulusDrive.apply(tokens, table, scale, dtype)
    return _drive(tokens, table, scale, dtype, out)


def stimulus_gradient(tokens: torch.Tensor, grad: torch.Tensor, rows: int, *, scale: float = 1.0,
                      dtype: torch.dtype | None = None) -> torch.Tensor:
    """The [rows, N] gradient of a stimulus table from the [*tokens.shape, N] gradient of its drive.

    Row v is ``scale`` times the float32 sum of the gradients of its tokens, in an order that the
    tokens alone fix: the same call gives the same bits.  ``dtype``: ``grad``'s (the default), or
    another where one of the two is float32.  It is not differentiable itself: a ``grad`` that requires
    a gradient is refused.
    """
    refuse_gradients("stimulus_gradient takes no gradients: call it under torch.no_grad() or on a detached grad", grad)
    if grad.dtype not in VALUE_TYPES or not grad.is_cuda:
        raise ValueError("grad must be a CUDA tensor of float32, float16 or bfloat16")
    dtype = grad.dtype if dtype is None else dtype
    if dtype not in VALUE_TYPES or (dtype != grad.dtype and torch.float32 not in (dtype, grad.dtype)):
        raise ValueError("dtype must be grad's, or one of the two float32")
    if grad.dim() == 0 or grad.shape[:-1] != tokens.shape:
        raise ValueError("grad must be [*tokens.shape, N]")
    if rows < 0:
        raise ValueError("rows must not be negative")
    tokens = _tokens(tokens, grad)
    flat = grad.reshape(tokens.numel(), grad.shape[-1])
    if flat.shape[1] > 1 and flat.stride(1) != 1 or flat.shape[0] > 1 and flat.stride(0) < flat.shape[1]:
        flat = flat.contiguous()  # e.g. the expanded gradient of a sum
    view = dense_matrix(flat, "grad")
    out = grad.new_empty((rows, view.cols), dtype=dtype)
    result = _Matrix(out.data_ptr(), rows, view.cols, view.cols, VALUE_TYPES[dtype])
    lib = load_library()
    size = lib.nsb_stimulus_gradient_workspace_size(view.rows, view.cols)
    workspace = grad.new_empty(size, dtype=torch.uint8)
    token_call(grad, lib.nsb_stimulus_gradient, tokens.data_ptr(), tokens.element_size(),
               ctypes.byref(view), scale, ctypes.byref(result), workspace.data_ptr(), size)
    return out
