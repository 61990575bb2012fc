"""Dense matrices in NVFP4, their product, and the readout of states through packed weights.

The format is the sparse weights' (E2M1 codes, an E4M3 scale per 16 elements, a float32 scale),
laid out row by row for the tensor cores:

* ``quantize_nvfp4`` packs a matrix, or its transpose, with one float32 scale per row or for the
  whole matrix (``per="tensor"`` gives the values of ``quantize_dequantize(x, "nvfp4")``);
* ``Nvfp4Matrix.dequantize`` reads it back;
* ``nvfp4_product`` multiplies two packed matrices, with float32 sums;
* ``nvfp4_readout`` quantises states row by row and multiplies them with the readout weights:
  packed ones for inference, floating-point ones for training.

A wait inside a product that runs out is reported by ``check_product_status``, which a program calls
where it reads results back anyway (``generate_tokens`` does).

A row of states is quantised by itself, whatever else is in the batch, and equal rows of a batch give equal
results.  The size of the batch decides how a product is cut into tiles and in which order its sums and
scales are taken: the same row gives results a few float32 roundings apart in batches of different sizes.
"""

from __future__ import annotations

import ctypes

import torch

from .native import (VALUE_TYPES, _Matrix, _Nvfp4, _raise_on_status, dense_matrix, load_library,
                     refuse_gradients, refuse_tangents, token_call, written)


class Nvfp4Matrix:
    """A packed [rows, columns] matrix; R = rows, K = columns.

    ``codes``: uint8 [R, 16 * ceil(K / 32)], two E2M1 codes per byte, the even column in the low
    nibble.  ``block_scales``: uint8 E4M3 [ceil(R / 128), 4 * ceil(K / 256), 512]; tile (i, j) holds
    rows 128 i ... and blocks of 16 columns 4 j ..., the scale of row r and block b at byte
    16 (r % 32) + 4 (r % 128 // 32) + b % 4.  ``scale``: float32 [R] or [1].  Codes and block scales
    beyond K are zero.  The tensors are used as they are, not copied, and stay the matrix's for good:
    kernels read them by their addresses.  It can be copied and pickled.
    """

    __slots__ = ("_codes", "_block_scales", "_scale", "_columns", "_view")

    def __init__(self, codes: torch.Tensor, block_scales: torch.Tensor, scale: torch.Tensor,
                 columns: int) -> None:
        if columns < 1:
            raise ValueError("an NVFP4 matrix needs at least one column")
        shape = codes.shape
        rows = shape[0] if shape else 0
        if codes.dtype is not torch.uint8 or shape != (rows, (columns + 31) // 32 * 16):
            raise ValueError("codes must be uint8 [rows, 16 * ceil(columns / 32)]")
        if (block_scales.dtype is not torch.uint8
                or block_scales.shape != ((rows + 127) // 128, (columns + 255) // 256 * 4, 512)):
            raise ValueError("block_scales must be uint8 [ceil(rows / 128), 4 * ceil(columns / 256), 512]")
        count = scale.numel()
        if scale.dtype is not torch.float32 or scale.dim() != 1 or (count != 1 and count != rows):
            raise ValueError("scale must be float32 [rows] or [1]")
        device = codes.get_device()
        if device < 0 or block_scales.get_device() != device or scale.get_device() != device:
            raise ValueError("codes, block_scales and scale must be on one CUDA device")
        if not (codes.is_contiguous() and block_scales.is_contiguous() and scale.is_contiguous()):
            raise ValueError("codes, block_scales and scale must be contiguous")
        self._codes, self._block_scales, self._scale, self._columns = codes, block_scales, scale, columns
        self._view = _Nvfp4(rows, columns, codes.data_ptr(), shape[1], block_scales.data_ptr(),
                            scale.data_ptr(), count)

    @classmethod
    def _own(cls, codes: torch.Tensor, block_scales: torch.Tensor, scale: torch.Tensor, rows: int,
             columns: int, count: int) -> "Nvfp4Matrix":
        """Of tensors made for it: nothing to check."""
        self = cls.__new__(cls)
        self._codes, self._block_scales, self._scale, self._columns = codes, block_scales, scale, columns
        self._view = _Nvfp4(rows, columns, codes.data_ptr(), (columns + 31) // 32 * 16,
                            block_scales.data_ptr(), scale.data_ptr(), count)
        return self

    def __reduce__(self):
        return Nvfp4Matrix, (self._codes, self._block_scales, self._scale, self._columns)

    @property
    def codes(self) -> torch.Tensor:
        return self._codes

    @property
    def block_scales(self) -> torch.Tensor:
        return self._block_scales

    @property
    def scale(self) -> torch.Tensor:
        return self._scale

    @property
    def columns(self) -> int:
        return self._columns

    @property
    def rows(self) -> int:
        return self._codes.shape[0]

    @property
    def shape(self) -> tuple[int, int]:
        return self._codes.shape[0], self._columns

    @property
    def device(self) -> torch.device:
        return self._codes.device

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """The values the codes stand for: level * (block scale * scale), rounded to ``dtype``."""
        if dtype not in VALUE_TYPES:
            raise ValueError("dtype must be float32, float16 or bfloat16")
        refuse_gradients("dequantize takes no gradients: its scale requires one", self._scale)
        rows, columns = self._view.rows, self._view.cols
        out = self._scale.new_empty((rows, columns), dtype=dtype)
        result = _Matrix(out.data_ptr(), rows, columns, columns, VALUE_TYPES[dtype])
        token_call(out, load_library().nsb_nvfp4_dequantize, ctypes.byref(self._view),
                   ctypes.byref(result))
        return out


def quantize_nvfp4(value: torch.Tensor, *, per: str = "row", transpose: bool = False) -> Nvfp4Matrix:
    """Pack a [M, K] float32, float16 or bfloat16 matrix, or (``transpose``) its transpose.

    ``per="row"``: a float32 scale for each row of the result, so that rows do not depend on one
    another; ``per="tensor"``: one for all.  Packing has no derivative: the result takes no part in
    autograd, whatever ``value`` requires.  A row (or tensor) with an infinity or a NaN is packed
    with the scale NaN, and reads back as NaN everywhere.
    """
    if per not in ("row", "tensor"):
        raise ValueError("per must be 'row' or 'tensor'")
    return _quantize(value.detach() if value.requires_grad else value, per == "row", transpose)


def _quantize(value: torch.Tensor, per_row: bool, transpose: bool) -> Nvfp4Matrix:
    view = dense_matrix(value, "value")
    rows, columns = (view.cols, view.rows) if transpose else (view.rows, view.cols)
    if view.cols < 1 or columns < 1:
        raise ValueError("an NVFP4 matrix needs at least one column")
    codes = value.new_empty((rows, (columns + 31) // 32 * 16), dtype=torch.uint8)
    scales = value.new_empty(((rows + 127) // 128, (columns + 255) // 256 * 4, 512), dtype=torch.uint8)
    count = rows if per_row else 1
    # A tensor without rows has the scale of zeros.
    scale = value.new_empty(count, dtype=torch.float32) if rows else value.new_ones(count, dtype=torch.float32)
    packed = Nvfp4Matrix._own(codes, scales, scale, rows, columns, count)
    lib = load_library()
    # A row's own scale needs no workspace; see nsb_nvfp4_quantize_workspace_size.
    size = 0 if per_row and not transpose else lib.nsb_nvfp4_quantize_workspace_size(
        view.rows, view.cols, int(transpose), count)
    workspace = value.new_empty(size, dtype=torch.uint8) if size else None
    token_call(value, lib.nsb_nvfp4_quantize, ctypes.byref(view), transpose,
               ctypes.byref(packed._view), None, 0,
               workspace.data_ptr() if size else None, size)
    return packed


def check_product_status(device: torch.device | str = "cuda") -> None:
    """Raise if a product on ``device`` gave up on a bounded wait since the last call, and left part of
    its result unwritten.  Waits for the current stream; what a graph replays counts like any other call.
    """
    index = torch.device(device).index
    code = ctypes.c_int32(0)
    with torch.cuda.device(torch.cuda.current_device() if index is None else index):
        lib = load_library()
        _raise_on_status(lib, lib.nsb_nvfp4_product_status(ctypes.byref(code), torch.cuda.current_stream().cuda_stream))
    if code.value:
        raise RuntimeError(f"NVFP4 product pipeline timeout (code {code.value})")


def nvfp4_product(a: Nvfp4Matrix, b: Nvfp4Matrix, *, bias: torch.Tensor | None = None,
                  dtype: torch.dtype = torch.float32,
                  out: torch.Tensor | None = None) -> torch.Tensor:
    """``a @ b.T (+ bias)`` of two packed matrices [M, K] and [N, K] as [M, N], with float32 sums.

    ``bias``: float32 [N].  The result is rounded once to ``dtype`` and depends on the operands
    alone (the same call gives the same bits).  ``out`` receives it where given (contiguous rows).
    Nothing here takes a gradient (:func:`nvfp4_readout` does).
    """
    refuse_gradients("nvfp4_product takes no gradients: use nvfp4_readout, or detached tensors", bias, out, a._scale, b._scale)
    m, n, device = a._view.rows, b._view.rows, a._scale.get_device()
    if a._columns != b._columns or device != b._scale.get_device():
        raise ValueError("the operands must have the same number of columns and the same device")
    if n < 1:
        raise ValueError("the second operand needs at least one row")
    _check_bias(bias, n, device)
    given = out
    if out is None:
        if dtype not in VALUE_TYPES:
            raise ValueError("dtype must be float32, float16 or bfloat16")
        out = a._scale.new_empty((m, n), dtype=dtype)
    elif out.shape != (m, n) or out.dtype != dtype or out.get_device() != device:
        raise ValueError("out must be [M, N] of the given dtype on the operands' device")
    result = dense_matrix(out, "out")
    token_call(out, load_library().nsb_nvfp4_product, ctypes.byref(a._view), ctypes.byref(b._view),
               None if bias is None else bias.data_ptr(), ctypes.byref(result), None)
    if given is not None:
        written(out)
    return out


def _check_bias(bias: torch.Tensor | None, n: int, device: int) -> None:
    if bias is not None and (bias.dtype is not torch.float32 or bias.shape != (n,)
                             or bias.get_device() != device or not bias.is_contiguous()):
        raise ValueError("bias must be a contiguous float32 [N] on the operands' device")


def _readout(state: torch.Tensor, weight: Nvfp4Matrix, bias: torch.Tensor | None,
             dtype: torch.dtype) -> torch.Tensor:
    """[M, K] states through packed weights in one call of the library."""
    view = dense_matrix(state, "state")
    rows, columns, n, device = view.rows, view.cols, weight._view.rows, state.get_device()
    if weight._scale.get_device() != device or n < 1:
        raise ValueError("weights must have at least one row and be on the states' device")
    _check_bias(bias, n, device)
    out = state.new_empty((rows, n), dtype=dtype)
    result = _Matrix(out.data_ptr(), rows, n, n, VALUE_TYPES[dtype])
    lib = load_library()
    size = lib.nsb_nvfp4_readout_workspace_size(rows, columns)
    workspace = state.new_empty(size, dtype=torch.uint8)
    token_call(state, lib.nsb_nvfp4_readout, ctypes.byref(view), ctypes.byref(weight._view),
               None if bias is None else bias.data_ptr(), ctypes.byref(result), workspace.data_ptr(), size,
               None)
    return out


class _Readout(torch.autograd.Function):
    """``y = Q(x) Q(w)^T + b`` with straight-through gradients, each product on operands quantised
    along its own sum: ``dx = Q(dy) Q(w^T)^T``, ``dw = Q(dy^T) Q(x^T)^T``, ``db = sum of dy``."""

    @staticmethod
    def forward(ctx, state, weight, bias, dtype):
        x, w = dense_matrix(state, "state"), dense_matrix(weight, "weight")
        device = state.get_device()
        if weight.get_device() != device or w.rows < 1:
            raise ValueError("weights must have at least one row and be on the states' device")
        _check_bias(bias, w.rows, device)
        out = state.new_empty((x.rows, w.rows), dtype=dtype)
        largest = state.new_empty(2, dtype=torch.float32)  # of state and weight, for the backward pass
        ctx.save_for_backward(state, weight, largest)
        lib = load_library()
        size = lib.nsb_nvfp4_train_workspace_size(x.rows, x.cols, w.rows)
        workspace = state.new_empty(size, dtype=torch.uint8)
        result = _Matrix(out.data_ptr(), x.rows, w.rows, w.rows, VALUE_TYPES[dtype])
        token_call(out, lib.nsb_nvfp4_train_forward, ctypes.byref(x), ctypes.byref(w),
                   None if bias is None else bias.data_ptr(), ctypes.byref(result), largest.data_ptr(),
                   workspace.data_ptr(), size, None)
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        refuse_tangents("nvfp4_readout has no forward-mode derivative", grad)
        state, weight, largest = ctx.saved_tensors
        wants_state, wants_weight, wants_bias, _ = ctx.needs_input_grad
        if state.shape[0] == 0:
            return (torch.zeros_like(state) if wants_state else None,
                    torch.zeros_like(weight) if wants_weight else None,
                    weight.new_zeros(weight.shape[0], dtype=torch.float32) if wants_bias else None, None)
        row_stride, stride = grad.stride()
        if stride != 1 and grad.shape[1] > 1 or row_stride < grad.shape[1] and grad.shape[0] > 1:
            grad = grad.contiguous()  # e.g. the expanded gradient of a sum
        x, w, d = dense_matrix(state, "state"), dense_matrix(weight, "weight"), dense_matrix(grad, "grad")
        dx = state.new_empty((x.rows, x.cols)) if wants_state else None
        dw = weight.new_empty((w.rows, w.cols)) if wants_weight else None
        db = weight.new_empty(w.rows, dtype=torch.float32) if wants_bias else None
        lib = load_library()
        size = lib.nsb_nvfp4_train_workspace_size(x.rows, x.cols, w.rows)
        workspace = state.new_empty(size, dtype=torch.uint8)
        token_call(grad, lib.nsb_nvfp4_train_backward, ctypes.byref(x), ctypes.byref(w), ctypes.byref(d),
                   largest.data_ptr(),
                   ctypes.byref(_Matrix(dx.data_ptr(), x.rows, x.cols, x.cols, x.type)) if wants_state else None,
                   ctypes.byref(_Matrix(dw.data_ptr(), w.rows, w.cols, w.cols, w.type)) if wants_weight else None,
                   db.data_ptr() if wants_bias else None, workspace.data_ptr(), size,
                   None)
        return dx, dw, db, None


def nvfp4_readout(state: torch.Tensor, weight: Nvfp4Matrix | torch.Tensor,
                  bias: torch.Tensor | None = None, *,
                  dtype: torch.dtype | None = None) -> torch.Tensor:
    """``Q(state) @ Q(weight).T + bias``: states [..., K] (e.g. soma states [B, N] or a recorded
    window [T, B, N]) to [..., N_out], multiplied in NVFP4 with float32 sums.

    The states are quantised per row.  ``weight``: an :class:`Nvfp4Matrix` [N_out, K] (inference
    only), or a floating-point [N_out, K], packed with one scale in the call; then state, weight and
    bias may require gradients (straight-through, see ``_Readout``).  ``bias``: float32 [N_out].
    ``dtype`` of the result: the states' by default.
    """
    dtype = state.dtype if dtype is None else dtype
    if dtype not in VALUE_TYPES:
        raise ValueError("dtype must be float32, float16 or bfloat16")
    packed = isinstance(weight, Nvfp4Matrix)
    scale = weight._scale if packed else None
    refuse_tangents("nvfp4_readout has no forward-mode derivative", state, scale if packed else weight, bias)
    shape = state.shape
    if not shape or shape[-1] != (weight._columns if packed else weight.shape[-1]):
        raise ValueError("states must be [..., K] for weights [N_out, K]")
    flat = state if len(shape) == 2 else state.reshape(-1, shape[-1])
    row_stride, stride = flat.stride()
    if (stride != 1 and shape[-1] > 1) or (row_stride < shape[-1] and flat.shape[0] > 1):
        flat = flat.contiguous()  # e.g. the neuron-major states of a batch
    wants = torch.is_grad_enabled() and (state.requires_grad
                                         or (bias is not None and bias.requires_grad)
                                         or (packed and scale.requires_grad))
    if packed:
        if wants:
            raise ValueError("packed weights take no gradients: pass floating-point weights")
        result = _readout(flat, weight, bias, dtype)
    elif wants or (torch.is_grad_enabled() and weight.requires_grad):
        result = _Readout.apply(flat, weight, bias, dtype)
    else:
        result = _readout(flat, _quantize(weight, False, False), bias, dtype)
    return result if len(shape) == 2 else result.view(*shape[:-1], result.shape[1])
