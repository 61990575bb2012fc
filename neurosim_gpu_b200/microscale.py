"""Dense matrices in NVFP4, their product, and the readout of states through packed weights.

The format is the sparse weights' (E2M1 codes, an E4M3 scale per 16 elements, a float32 scale),
laid out row by row for the tensor cores:

* ``quantize_nvfp4`` packs a matrix, or its transpose, with one float32 scale per row or for the
  whole matrix (``per="tensor"`` gives the values of ``quantize_dequantize(x, "nvfp4")``);
* ``Nvfp4Matrix.dequantize`` reads it back;
* ``nvfp4_product`` multiplies two packed matrices, with float32 sums;
* ``nvfp4_readout`` quantises states row by row and multiplies them with the readout weights:
  packed ones for inference, floating-point ones for training.

A row of the result depends on its own state alone, not on the rest of the batch.
"""

from __future__ import annotations

import ctypes
import functools
from dataclasses import dataclass

import torch

from .native import VALUE_TYPES, _Nvfp4, dense_matrix, load_library, token_call


@dataclass(frozen=True)
class Nvfp4Matrix:
    """A packed [rows, columns] matrix; R = rows, K = columns.

    ``codes``: uint8 [R, 16 * ceil(K / 32)], two E2M1 codes per byte, the even column in the low
    nibble.  ``block_scales``: uint8 E4M3 [ceil(R / 128), 4 * ceil(K / 256), 512]; tile (i, j) holds
    rows 128 i ... and blocks of 16 columns 4 j ..., the scale of row r and block b at byte
    16 (r % 32) + 4 (r % 128 // 32) + b % 4.  ``scale``: float32 [R] or [1].  Codes and block scales
    beyond K are zero.
    """

    codes: torch.Tensor
    block_scales: torch.Tensor
    scale: torch.Tensor
    columns: int

    def __post_init__(self) -> None:
        codes, scales, scale, columns = self.codes, self.block_scales, self.scale, self.columns
        if columns < 1:
            raise ValueError("an NVFP4 matrix needs at least one column")
        rows = codes.shape[0]
        if codes.dtype != torch.uint8 or tuple(codes.shape) != (rows, (columns + 31) // 32 * 16):
            raise ValueError("codes must be uint8 [rows, 16 * ceil(columns / 32)]")
        if (scales.dtype != torch.uint8
                or tuple(scales.shape) != ((rows + 127) // 128, (columns + 255) // 256 * 4, 512)):
            raise ValueError("block_scales must be uint8 [ceil(rows / 128), 4 * ceil(columns / 256), 512]")
        if scale.dtype != torch.float32 or scale.dim() != 1 or scale.shape[0] not in (1, rows):
            raise ValueError("scale must be float32 [rows] or [1]")
        if not (codes.is_cuda and codes.device == scales.device == scale.device):
            raise ValueError("codes, block_scales and scale must be on one CUDA device")
        if not (codes.is_contiguous() and scales.is_contiguous() and scale.is_contiguous()):
            raise ValueError("codes, block_scales and scale must be contiguous")

    @property
    def rows(self) -> int:
        return self.codes.shape[0]

    @property
    def shape(self) -> tuple[int, int]:
        return self.codes.shape[0], self.columns

    @property
    def device(self) -> torch.device:
        return self.codes.device

    def _view(self) -> _Nvfp4:
        return _Nvfp4(self.codes.shape[0], self.columns, self.codes.data_ptr(), self.codes.shape[1],
                      self.block_scales.data_ptr(), self.scale.data_ptr(), self.scale.shape[0])

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """The values the codes stand for: level * (block scale * scale), rounded to ``dtype``."""
        if dtype not in VALUE_TYPES:
            raise ValueError("dtype must be float32, float16 or bfloat16")
        out = torch.empty(self.shape, device=self.device, dtype=dtype)
        view, result = self._view(), dense_matrix(out, "out")
        token_call(self.device, load_library().nsb_nvfp4_dequantize, ctypes.byref(view),
                   ctypes.byref(result))
        return out


def quantize_nvfp4(value: torch.Tensor, *, per: str = "row", transpose: bool = False) -> Nvfp4Matrix:
    """Pack a [M, K] float32, float16 or bfloat16 matrix, or (``transpose``) its transpose.

    ``per="row"``: a float32 scale for each row of the result, so that rows do not depend on one
    another; ``per="tensor"``: one for all.  A row (or tensor) with an infinity or a NaN is packed
    with the scale NaN, and reads back as NaN everywhere.
    """
    if per not in ("row", "tensor"):
        raise ValueError("per must be 'row' or 'tensor'")
    return _quantize(value.detach(), per == "row", transpose)


def _quantize(value: torch.Tensor, per_row: bool, transpose: bool, amax: torch.Tensor | None = None,
              given: bool = False) -> Nvfp4Matrix:
    """``amax``: a float32 word that receives the largest |value|, or (``given``) holds it already."""
    view = dense_matrix(value, "value")
    rows, columns = (view.cols, view.rows) if transpose else (view.rows, view.cols)
    if view.cols < 1 or columns < 1:
        raise ValueError("an NVFP4 matrix needs at least one column")
    device = value.device
    codes = torch.empty((rows, (columns + 31) // 32 * 16), device=device, dtype=torch.uint8)
    scales = torch.empty(((rows + 127) // 128, (columns + 255) // 256 * 4, 512), device=device,
                         dtype=torch.uint8)
    # A tensor without rows has the scale of zeros.
    scale = (torch.empty if rows else torch.ones)(rows if per_row else 1, device=device,
                                                  dtype=torch.float32)
    packed = Nvfp4Matrix(codes, scales, scale, columns)
    lib = load_library()
    result = packed._view()
    size = lib.nsb_nvfp4_quantize_workspace_size(view.rows, view.cols, int(transpose), scale.shape[0])
    workspace = torch.empty(size, device=device, dtype=torch.uint8) if size else None
    token_call(device, lib.nsb_nvfp4_quantize, ctypes.byref(view), int(transpose),
               ctypes.byref(result), None if amax is None else amax.data_ptr(), int(given),
               workspace.data_ptr() if size else None, size)
    return packed


@functools.lru_cache(maxsize=None)
def _status(device: torch.device) -> torch.Tensor:
    """The word that products on ``device`` write an error code to (never inside a capture)."""
    with torch.inference_mode(False):
        return torch.zeros(1, device=device, dtype=torch.int32)


def check_product_status(device: torch.device | str = "cuda") -> None:
    """Raise if a product on ``device`` gave up on a bounded wait (reads the device)."""
    device = torch.device(device)
    if device.index is None:
        device = torch.device("cuda", torch.cuda.current_device())
    code = int(_status(device).item())
    if code:
        raise RuntimeError(f"NVFP4 product pipeline timeout (code {code})")


def nvfp4_product(a: Nvfp4Matrix, b: Nvfp4Matrix, *, bias: torch.Tensor | None = None,
                  dtype: torch.dtype = torch.float32,
                  out: torch.Tensor | None = None) -> torch.Tensor:
    """``a @ b.T (+ bias)`` of two packed matrices [M, K] and [N, K] as [M, N], with float32 sums.

    ``bias``: float32 [N].  The result is rounded once to ``dtype`` and depends on the operands
    alone (the same call gives the same bits).  ``out`` receives it where given (contiguous rows).
    """
    if a.columns != b.columns or a.device != b.device:
        raise ValueError("the operands must have the same number of columns and the same device")
    if b.rows < 1:
        raise ValueError("the second operand needs at least one row")
    if bias is not None and (bias.dtype != torch.float32 or tuple(bias.shape) != (b.rows,)
                             or bias.device != a.device or not bias.is_contiguous()):
        raise ValueError("bias must be a contiguous float32 [N] on the operands' device")
    if out is None:
        if dtype not in VALUE_TYPES:
            raise ValueError("dtype must be float32, float16 or bfloat16")
        out = torch.empty((a.rows, b.rows), device=a.device, dtype=dtype)
    elif tuple(out.shape) != (a.rows, b.rows) or out.dtype != dtype or out.device != a.device:
        raise ValueError("out must be [M, N] of the given dtype on the operands' device")
    x, y, result = a._view(), b._view(), dense_matrix(out, "out")
    token_call(a.device, load_library().nsb_nvfp4_product, ctypes.byref(x), ctypes.byref(y),
               None if bias is None else bias.data_ptr(), ctypes.byref(result),
               _status(a.device).data_ptr())
    return out


def _column_sums(value: torch.Tensor) -> torch.Tensor:
    view = dense_matrix(value, "value")
    out = torch.empty(value.shape[1], device=value.device, dtype=torch.float32)
    lib = load_library()
    size = lib.nsb_column_sums_workspace_size(*value.shape)
    workspace = torch.empty(size, device=value.device, dtype=torch.uint8)
    token_call(value.device, lib.nsb_column_sums, ctypes.byref(view), out.data_ptr(),
               workspace.data_ptr(), size)
    return out


class _Readout(torch.autograd.Function):
    """``y = Q(x) Q(w)^T + b`` with straight-through gradients, each product on operands quantised
    along its own sum: ``dx = Q(dy) Q(w^T)^T``, ``dw = Q(dy^T) Q(x^T)^T``, ``db = sum of dy``."""

    @staticmethod
    def forward(ctx, state, weight, bias, dtype):
        # The largest sizes of state and weight come with the forward's packing: the backward's needs no pass for them.
        most = torch.empty(2, device=state.device, dtype=torch.float32)
        ctx.save_for_backward(state, weight, most)
        return nvfp4_product(_quantize(state, True, False, most[:1]), _quantize(weight, False, False, most[1:]),
                             bias=None if bias is None else bias.detach(), dtype=dtype)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        state, weight, most = ctx.saved_tensors
        dx = dw = db = None
        if grad.stride(1) != 1 and grad.shape[1] > 1 or grad.shape[0] > 1 and grad.stride(0) < grad.shape[1]:
            grad = grad.contiguous()  # e.g. the expanded gradient of a sum
        grad_most = None
        if ctx.needs_input_grad[0]:
            if ctx.needs_input_grad[1]:
                grad_most = torch.empty(1, device=grad.device, dtype=torch.float32)
            dx = nvfp4_product(_quantize(grad, True, False, grad_most), _quantize(weight, False, True, most[1:], True),
                               dtype=state.dtype)
        if ctx.needs_input_grad[1]:
            if state.shape[0]:
                dw = nvfp4_product(_quantize(grad, False, True, grad_most, grad_most is not None),
                                   _quantize(state, False, True, most[:1], True), dtype=weight.dtype)
            else:
                dw = torch.zeros_like(weight)
        if ctx.needs_input_grad[2]:
            db = _column_sums(grad)
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
    if state.dim() < 1 or state.shape[-1] != (weight.columns if isinstance(weight, Nvfp4Matrix)
                                              else weight.shape[-1]):
        raise ValueError("states must be [..., K] for weights [N_out, K]")
    flat = state if state.dim() == 2 else state.reshape(-1, state.shape[-1])
    if flat.shape[0] > 1 and flat.stride(0) < flat.shape[1] or flat.shape[1] > 1 and flat.stride(1) != 1:
        flat = flat.contiguous()  # e.g. the neuron-major states of a batch
    wants = torch.is_grad_enabled() and (state.requires_grad
                                         or (bias is not None and bias.requires_grad))
    if isinstance(weight, Nvfp4Matrix):
        if wants:
            raise ValueError("packed weights take no gradients: pass floating-point weights")
        result = nvfp4_product(quantize_nvfp4(flat), weight, bias=bias, dtype=dtype)
    elif wants or (torch.is_grad_enabled() and weight.requires_grad):
        result = _Readout.apply(flat, weight, bias, dtype)
    else:
        result = nvfp4_product(quantize_nvfp4(flat), quantize_nvfp4(weight, per="tensor"), bias=bias,
                               dtype=dtype)
    return result if state.dim() == 2 else result.view(*state.shape[:-1], result.shape[1])
