"""Logits before the choice of a token: penalties for repeated tokens, biases and grammar masks.

One kernel (``nsb_adjust_logits``) reads each logit once, counts the history on the way, and can
make the greedy choice.
"""

from __future__ import annotations

import ctypes

import torch

from .native import _Logits, _Matrix, _RowValues, dense_matrix, load_library, refuse_gradients, token_call, written


_NONE = (None, 0)


def _row_values(value: float | torch.Tensor, name: str, rows: int, device: torch.device) -> _RowValues:
    if value.__class__ is float or not isinstance(value, torch.Tensor):
        return _RowValues(None, 0, float(value))
    shape = value.shape
    if value.dtype is not torch.float32 or value.device != device or shape not in ((), (1,), (rows,)):
        raise ValueError(f"{name} must be a number or a float32 tensor with one value per row")
    return _RowValues(value.data_ptr(), value.stride(0) if shape and shape[0] > 1 else 0, 1.0)


def _lengths(value: torch.Tensor, name: str, rows: int, device: torch.device) -> int:
    if (value.dtype != torch.int32 or value.device != device or tuple(value.shape) != (rows,)
            or not value.is_contiguous()):
        raise ValueError(f"{name} must be a contiguous int32 vector with one value per row")
    return value.data_ptr()


def _broadcast(value: torch.Tensor, name: str, dtype: torch.dtype, rows: int, columns: int,
               device: torch.device) -> tuple[int, int]:
    """(pointer, elements between rows) of a [columns] or [rows, columns] operand."""
    if (value.dtype != dtype or value.device != device
            or tuple(value.shape) not in ((columns,), (1, columns), (rows, columns))):
        raise ValueError(f"{name} must be {dtype} [{columns}] or one row for each row of logits")
    if columns > 1 and value.stride(-1) != 1:
        raise ValueError(f"{name} must have contiguous rows")
    return value.data_ptr(), value.stride(0) if value.dim() == 2 and value.shape[0] > 1 else 0


def adjust_logits(logits: torch.Tensor, *, history: torch.Tensor | None = None,
                  lengths: torch.Tensor | None = None,
                  prompt_lengths: torch.Tensor | None = None,
                  repetition: float | torch.Tensor = 1.0, presence: float | torch.Tensor = 0.0,
                  frequency: float | torch.Tensor = 0.0, bias: torch.Tensor | None = None,
                  mask: torch.Tensor | None = None, out: torch.Tensor | None = None,
                  choose: bool = False) -> torch.Tensor | tuple[torch.Tensor, torch.Tensor]:
    """Adjusted logits [B, V], and with ``choose`` the greedy choice [B] (int64) as well.

    With c the occurrences of a token in the generated part of its row's history,
    ``history[b, prompt_lengths[b]:lengths[b]]``, and "seen" for any occurrence in
    ``history[b, :lengths[b]]``::

        x = logit;  if seen: x = x / repetition if x > 0 else x * repetition
        x = x - frequency * c;  if c > 0: x = x - presence
        x = x + bias;  -inf where the mask bit is 0

    in float32, rounded once to the logits' type.  ``history``: int32 [B, L] (ids outside the
    vocabulary are skipped); ``lengths`` / ``prompt_lengths``: int32 [B] (default: L / 0);
    ``repetition`` (above 0), ``presence``, ``frequency``: numbers or float32 [B]; ``bias``: float32
    [V] or [B, V]; ``mask``: int32 [ceil(V / 32)] or [B, ceil(V / 32)], bit v % 32 of word v // 32
    set where token v is allowed.  ``out`` may be ``logits``, or share no element with them.  The choice is the lowest index of a
    row's largest adjusted logit, -1 where nothing is above -inf; a NaN is never chosen.

    There is no backward pass: where gradients are recorded, an argument that requires one is refused.
    """
    refuse_gradients("adjust_logits takes no gradients: call it under torch.no_grad() or on detached tensors",
                     logits, out, bias, repetition, presence, frequency)
    view = dense_matrix(logits, "logits")
    rows, vocabulary = view.rows, view.cols
    device = logits.device
    given = out
    if out is None:
        out = logits.new_empty((rows, vocabulary))
        result = _Matrix(out.data_ptr(), rows, vocabulary, vocabulary, view.type)
    elif out is logits:
        result = view
    elif out.shape != logits.shape or out.dtype != logits.dtype or out.device != device:
        raise ValueError("out must have the logits' shape, dtype and device")
    else:
        result = dense_matrix(out, "out")
    past, length, stride = None, 0, 0
    if history is not None:
        if (history.dtype != torch.int32 or history.device != device or history.dim() != 2
                or history.shape[0] != rows or (history.shape[1] > 1 and history.stride(1) != 1)):
            raise ValueError("history must be int32 [B, L] with contiguous rows")
        past, length, stride = history.data_ptr(), history.shape[1], history.stride(0)
    elif lengths is not None or prompt_lengths is not None:
        raise ValueError("lengths need a history")
    choice = logits.new_empty(rows, dtype=torch.int64) if choose else None
    args = _Logits(
        view, result, past, length, stride,
        None if lengths is None else _lengths(lengths, "lengths", rows, device),
        None if prompt_lengths is None else _lengths(prompt_lengths, "prompt_lengths", rows, device),
        _row_values(repetition, "repetition", rows, device),
        _row_values(presence, "presence", rows, device),
        _row_values(frequency, "frequency", rows, device),
        *(_NONE if bias is None else _broadcast(bias, "bias", torch.float32, rows, vocabulary, device)),
        *(_NONE if mask is None else _broadcast(mask, "mask", torch.int32, rows, (vocabulary + 31) // 32, device)),
        choice.data_ptr() if choose else None)
    token_call(logits, load_library().nsb_adjust_logits, ctypes.byref(args))
    if given is not None:
        written(out)
    return (out, choice) if choose else out
