"""NVFP4 matrices, their product and the readout against plain implementations in float64."""

from __future__ import annotations

import copy
import ctypes
import pickle
import subprocess
import sys
from pathlib import Path

import numpy as np
import pytest
import torch

from neurosim_gpu_b200 import (Nvfp4Matrix, check_product_status, native, nvfp4_product, nvfp4_readout,
                               quantize_dequantize, quantize_nvfp4)

DTYPES = [torch.float32, torch.float16, torch.bfloat16]
UNIT = {torch.float32: 2.0**-24, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}
LEVELS = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6, 0, -0.5, -1, -1.5, -2, -3, -4, -6])


def generator(seed):
    return torch.Generator().manual_seed(seed)


def blocks_of(x):
    rows, columns = x.shape
    out = np.zeros((rows, (columns + 15) // 16 * 16), np.float64)
    out[:, :columns] = x
    return out.reshape(rows, -1, 16)


def e4m3(x):
    """The E4M3 number nearest to x >= 0 (ties to even, at most 448), in float64."""
    x = np.asarray(x, np.float64)
    exponent = np.maximum(np.floor(np.log2(np.maximum(x, 2.0**-60))), -6)
    unit = 2.0 ** (exponent - 3)
    return np.minimum(np.round(x / unit) * unit, 448.0)


def quantized(x, per):
    """(values [R, K], block scales [R, blocks], scale) of the format's definition; the quotients
    that decide are float32 ones."""
    b = blocks_of(x.double().numpy())
    amax = np.abs(b).max((1, 2)) if per == "row" else np.full(len(b), np.abs(b).max())
    scale = np.maximum((amax.astype(np.float32) / np.float32(2688)), np.float32(2.0**-126))
    s = scale[:, None].astype(np.float32)
    block = e4m3(np.minimum(np.abs(b).max(2).astype(np.float32) / (np.float32(6) * s), np.float32(448)))
    step = s * block.astype(np.float32)
    ratio = np.abs(b).astype(np.float32) / np.where(step > 0, step, np.float32(1))[..., None]
    ratio = ratio.astype(np.float64)
    # Levels are 0.5 apart below 2, 1 apart below 4, then 2 apart: numpy rounds ties to even multiples.
    level = np.where(ratio < 2, np.round(ratio * 2) / 2, np.where(ratio < 4, np.round(ratio), np.round(ratio / 2) * 2))
    value = np.copysign(np.minimum(level, 6), b) * (block * s)[..., None].astype(np.float64)
    return value.reshape(len(b), -1)[:, : x.shape[1]], block, scale


def untiled(packed):
    tiles = packed.block_scales.cpu()
    flat = tiles.view(*tiles.shape[:2], 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(tiles.shape[0] * 128, -1)
    return flat.contiguous()


def check_packed(packed, x, per):
    """Codes, block scales, scale, padding and what is read back."""
    value, block, scale = quantized(x, per)
    rows, columns = x.shape
    assert packed.shape == (rows, columns)
    assert np.array_equal(packed.scale.cpu().numpy(), scale if per == "row" else scale[:1])
    got = untiled(packed)
    want = torch.zeros_like(got)
    want[:rows, : block.shape[1]] = torch.from_numpy(block).float().to(torch.float8_e4m3fn).view(torch.uint8)
    assert torch.equal(got, want)  # zeros beyond the matrix, too
    codes = packed.codes.cpu().numpy()
    codes = np.stack([codes & 15, codes >> 4], -1).reshape(rows, -1)
    assert not codes[:, columns:].any()
    step = np.repeat(block * packed.scale.cpu().numpy().astype(np.float32).reshape(-1, 1).astype(np.float64), 16, 1)[:, :columns]
    decoded = LEVELS[codes[:, :columns]] * step
    assert np.array_equal(decoded, value)
    assert np.array_equal(np.signbit(LEVELS[codes[:, :columns]]) | (codes[:, :columns] == 8), np.signbit(x.float().numpy()))
    # Read back: level * (block scale * scale), both products rounded to float32, then to the type.
    for dtype in DTYPES:
        back = packed.dequantize(dtype)
        want = torch.from_numpy(LEVELS[codes[:, :columns]].astype(np.float32) * step.astype(np.float32)).to(dtype)
        assert torch.equal(back.cpu(), want)


# -- refusals -------------------------------------------------------------------------------------


def test_entry_points_refuse_bad_arguments():
    lib = native.load_library()
    p = 0x1000  # never read: the checks fail first
    value = native._Matrix(p, 4, 40, 40, 0)

    def packed(rows=4, cols=40, codes=p, stride=32, scales=p, scale=p, count=1):
        return native._Nvfp4(rows, cols, codes, stride, scales, scale, count)

    def quantize(value=value, transpose=0, out=None, workspace=p, size=4, given=0):
        return lib.nsb_nvfp4_quantize(ctypes.byref(value), transpose, ctypes.byref(out or packed()), None, given, workspace, size, None)

    for bad in (packed(rows=5), packed(cols=41), packed(stride=16), packed(codes=p + 8), packed(scales=None),
                packed(scale=p + 2), packed(count=3), packed(codes=None), packed(rows=-1), packed(cols=0, stride=0)):
        assert quantize(out=bad) == -1
        assert lib.nsb_last_error()
    assert quantize(given=1) == -1 and quantize(transpose=1) == -1 and quantize(value=native._Matrix(p, 4, 40, 40, 7)) == -1
    assert quantize(workspace=None) == -3 and quantize(size=3) == -3 and quantize(workspace=p + 2) == -3
    out = native._Matrix(p, 4, 6, 6, 0)

    def product(a=None, b=None, out=out, bias=None):
        return lib.nsb_nvfp4_product(ctypes.byref(a or packed()), ctypes.byref(b or packed(rows=6)), bias,
                                     ctypes.byref(out), None, None)

    for bad in ({"b": packed(rows=6, cols=41)}, {"b": packed(rows=7)}, {"a": packed(rows=5)}, {"bias": p + 2},
                {"out": native._Matrix(p, 4, 6, 5, 0)}, {"out": native._Matrix(p + 2, 4, 6, 6, 0)}):
        assert product(**bad) == -1, bad
    assert product(a=packed(rows=0, codes=None, scales=None, scale=None),
                   out=native._Matrix(None, 0, 6, 6, 0)) == 0
    state, size = native._Matrix(p, 4, 40, 40, 0), lib.nsb_nvfp4_readout_workspace_size(4, 40)
    assert size >= 4 * 32 + 2048 + 16 and lib.nsb_nvfp4_readout_workspace_size(0, 40) == 0

    def readout(state=state, weight=packed(rows=6), out=out, workspace=p, size=size, bias=None):
        return lib.nsb_nvfp4_readout(ctypes.byref(state), ctypes.byref(weight), bias, ctypes.byref(out), workspace, size,
                                     None, None)

    for bad in ({"weight": packed(rows=7)}, {"weight": packed(rows=6, cols=41)}, {"bias": p + 2}, {"state": native._Matrix(p, 5, 40, 40, 0)}):
        assert readout(**bad) == -1, bad
    assert readout(size=size - 1) == -3 and readout(workspace=None) == -3 and readout(workspace=p + 8) == -3
    weight, grad, train = native._Matrix(p, 6, 40, 40, 0), native._Matrix(p, 4, 6, 6, 0), lib.nsb_nvfp4_train_workspace_size(4, 40, 6)
    assert train > size and lib.nsb_nvfp4_train_workspace_size(4, 0, 6) == 0

    def forward(weight=weight, out=out, largest=p, size=train):
        return lib.nsb_nvfp4_train_forward(ctypes.byref(state), ctypes.byref(weight), None, ctypes.byref(out), largest, p, size, None, None)

    def backward(grad=grad, dx=state, dw=weight, largest=p, size=train):
        return lib.nsb_nvfp4_train_backward(ctypes.byref(state), ctypes.byref(weight), ctypes.byref(grad), largest, ctypes.byref(dx),
                                            ctypes.byref(dw), None, p, size, None, None)

    assert forward(size=train - 1) == -3 and backward(size=train - 1) == -3
    assert forward(largest=None) == -1 and backward(largest=None) == -1 and backward(grad=out, dx=out) == -1
    assert forward(weight=native._Matrix(p, 6, 41, 41, 0)) == -1 and backward(dw=native._Matrix(p, 5, 40, 40, 0)) == -1
    assert lib.nsb_nvfp4_dequantize(ctypes.byref(packed()), ctypes.byref(native._Matrix(p, 4, 41, 41, 0)), None) == -1
    assert lib.nsb_column_sums(ctypes.byref(value), None, p, 10**6, None) == -1
    assert lib.nsb_column_sums(ctypes.byref(value), p, p, 1, None) == -3


def test_products_refuse_rows_that_32_bit_tiles_cannot_count():
    lib = native.load_library()
    p, rows = 0x1000, 2**31 - 256  # never read: the checks fail first

    def packed(rows):
        return ctypes.byref(native._Nvfp4(rows, 16, p, 16, p, p, 1))

    def dense(rows, cols):
        return ctypes.byref(native._Matrix(p, rows, cols, cols, 0))

    for m, n in ((rows, 6), (6, rows)):
        assert lib.nsb_nvfp4_product(packed(m), packed(n), None, dense(m, n), None, None) == -1
        assert b"2^31 - 256" in lib.nsb_last_error()
        assert lib.nsb_nvfp4_readout(dense(m, 16), packed(n), None, dense(m, n), p, 2**60, None, None) == -1
        assert lib.nsb_nvfp4_train_forward(dense(m, 16), dense(n, 16), None, dense(m, n), p, p, 2**60, None, None) == -1
        assert lib.nsb_nvfp4_train_backward(dense(m, 16), dense(n, 16), dense(m, n), p, dense(m, 16), dense(n, 16), None, p, 2**60,
                                            None, None) == -1
    assert lib.nsb_nvfp4_train_backward(dense(2, rows), dense(3, rows), dense(2, 3), p, dense(2, rows), dense(3, rows), None, p, 2**60,
                                        None, None) == -1


def test_functions_refuse_cpu_tensors():
    with pytest.raises(ValueError, match="CUDA"):
        quantize_nvfp4(torch.zeros(2, 32))


@pytest.mark.gpu
def test_functions_refuse_bad_arguments():
    x = torch.zeros(4, 40, device="cuda")
    q = quantize_nvfp4(x)
    for call in (lambda: quantize_nvfp4(x, per="block"), lambda: quantize_nvfp4(x.double()), lambda: quantize_nvfp4(x[0]),
                 lambda: quantize_nvfp4(x.t()), lambda: quantize_nvfp4(x[:, :0]), lambda: q.dequantize(torch.float64),
                 lambda: quantize_nvfp4(x[:0], transpose=True),
                 lambda: Nvfp4Matrix(q.codes, q.block_scales, q.scale, 70), lambda: Nvfp4Matrix(q.codes, q.block_scales, q.scale[:2], 40),
                 lambda: Nvfp4Matrix(q.codes, q.block_scales[:, :2], q.scale, 40), lambda: Nvfp4Matrix(q.codes.cpu(), q.block_scales, q.scale, 40),
                 lambda: nvfp4_product(q, quantize_nvfp4(x[:, :39])), lambda: nvfp4_product(q, q, bias=x[0, :4].half()),
                 lambda: nvfp4_product(q, q, bias=x[0, :3]), lambda: nvfp4_product(q, q, dtype=torch.float64),
                 lambda: nvfp4_product(q, q, out=x), lambda: nvfp4_readout(x[:, :39], q),
                 lambda: nvfp4_readout(x.clone().requires_grad_(), q), lambda: nvfp4_readout(x, q, dtype=torch.int32)):
        with pytest.raises(ValueError):
            call()


# -- the format -----------------------------------------------------------------------------------

SHAPES = [(1, 1), (1, 16), (2, 15), (3, 17), (1, 257), (130, 255), (257, 48), (128, 256), (5, 1000), (64, 4104), (33, 9000)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,columns", SHAPES)
def test_quantize(dtype, rows, columns):
    x = torch.randn(rows, columns, generator=generator(rows)) * torch.exp(2 * torch.randn(rows, 1, generator=generator(1)))
    x = x.to(dtype)
    for per in ("row", "tensor"):
        check_packed(quantize_nvfp4(x.cuda(), per=per), x, per)
        check_packed(quantize_nvfp4(x.cuda(), per=per, transpose=True), x.t().contiguous(), per)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("offset,odd", [(0, 0), (3, 1)])
@pytest.mark.parametrize("rows,columns", [(300, 4104), (2, 132_000), (3, 166_003), (129, 9001), (5, 70_017)])
def test_quantize_rows_longer_than_the_registers_hold(dtype, offset, odd, rows, columns):
    """Their last blocks are read twice, for the row's largest size and for the codes; the largest lies there."""
    stride = (columns + 15) // 16 * 16 + odd
    base = torch.randn(offset + rows * stride, generator=generator(rows)).to(dtype)
    x = base.as_strided((rows, columns), (stride, 1), offset)
    x[::2, -1] = 37.0
    x[1::2, -40] = -41.0
    check_packed(quantize_nvfp4(base.cuda().as_strided((rows, columns), (stride, 1), offset)), x, "row")


@pytest.mark.gpu
def test_quantize_strides_ties_and_small_values():
    g = generator(3)
    base = torch.randn(60 * 70, generator=g)
    for offset, stride in ((0, 64), (1, 64), (0, 65), (4, 60)):
        x = base.as_strided((50, 50), (stride, 1), offset)
        cuda = base.cuda().as_strided((50, 50), (stride, 1), offset)
        check_packed(quantize_nvfp4(cuda), x, "row")
        check_packed(quantize_nvfp4(cuda, per="tensor", transpose=True), x.t(), "tensor")
    # Scale 1 and block scale 448 or 1: every midpoint of the levels, and values one float32 beside it.
    middle = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0])
    line = torch.cat([middle, middle.nextafter(torch.tensor(9.0)), middle.nextafter(torch.tensor(0.0)), torch.tensor([6.0, 0.0, -0.0])])
    x = torch.zeros(3, 64)
    x[0, 0] = 2688.0
    x[0, 16:40], x[0, 40:64] = line, -line
    x[1] = x[0] * 2.0**-100
    x[2] = x[0] * 2.0**-140  # float32 subnormals: the scale stops at FLT_MIN
    check_packed(quantize_nvfp4(x.cuda()), x, "row")
    zeros = torch.zeros(2, 40)
    zeros[0, 3] = -0.0
    check_packed(quantize_nvfp4(zeros.cuda()), zeros, "row")


@pytest.mark.gpu
def test_packed_matrices_keep_their_tensors_and_can_be_copied():
    """The kernels go by the tensors' addresses, which an assignment would leave behind."""
    x = torch.randn(5, 70, generator=generator(18)).cuda()
    packed = quantize_nvfp4(x)
    for name in ("codes", "block_scales", "scale", "columns"):
        with pytest.raises(AttributeError):
            setattr(packed, name, getattr(packed, name))
    want = packed.dequantize()
    copies = [copy.deepcopy(packed), pickle.loads(pickle.dumps(packed)), copy.copy(packed)]
    assert copies[2].codes.data_ptr() == packed.codes.data_ptr()
    for other in copies[:2]:
        assert other.shape == packed.shape and other.codes.data_ptr() != packed.codes.data_ptr()
    packed.codes.zero_()
    assert not packed.dequantize().any()
    for other in copies[:2]:
        assert torch.equal(other.dequantize(), want)


@pytest.mark.gpu
def test_one_scale_gives_the_sparse_weights_values():
    x = torch.randn(37, 333, generator=generator(4)).cuda()
    assert torch.equal(quantize_nvfp4(x, per="tensor").dequantize(), quantize_dequantize(x, "nvfp4"))


@pytest.mark.gpu
@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan")])
def test_values_that_are_not_finite_stay_visible(value):
    x = torch.randn(40, 300, generator=generator(5)).cuda()
    want = quantize_nvfp4(x).dequantize()
    x[7, 299] = value
    back = quantize_nvfp4(x).dequantize()
    assert bool(back[7].isnan().all())
    keep = torch.arange(40, device="cuda") != 7
    assert torch.equal(back[keep], want[keep])
    back = quantize_nvfp4(x, transpose=True).dequantize()
    assert bool(back[299].isnan().all()) and not bool(back[:299].isnan().any())
    assert bool(quantize_nvfp4(x, per="tensor").dequantize().isnan().all())
    y = nvfp4_readout(x, quantize_nvfp4(want, per="tensor"))
    assert bool(y[7].isnan().all()) and not bool(y[keep].isnan().any())


# -- the product ----------------------------------------------------------------------------------

PRODUCTS = [(1, 1, 1), (1, 1000, 16), (1, 129, 4096), (2, 8, 17), (3, 257, 1000), (8, 1001, 5000), (16, 128, 64), (17, 300, 255),
            (33, 100, 256), (64, 131, 257), (127, 129, 512), (128, 128, 768), (129, 257, 63), (130, 2, 320), (255, 640, 1024),
            (256, 256, 2048), (257, 513, 300), (300, 77, 4104), (520, 1030, 272), (1025, 96, 1600), (2048, 2560, 520), (2300, 2420, 300), (2304, 20_000, 64)]


def exact_operand(rows, columns, seed):
    """A packed matrix of small integers at scale 1 (block scales 1 or 2), and its values."""
    g = generator(seed)
    codes = torch.tensor([0, 2, 4, 10, 12], dtype=torch.uint8)[torch.randint(0, 5, (rows, columns), generator=g)]  # 0 1 2 -1 -2
    blocks = (columns + 15) // 16
    twice = torch.randint(0, 2, (rows, blocks), generator=g)
    value = torch.from_numpy(LEVELS[codes.numpy()]) * torch.repeat_interleave(1 + twice, 16, 1)[:, :columns]
    wide = torch.zeros(rows, (columns + 31) // 32 * 32, dtype=torch.uint8)
    wide[:, :columns] = codes
    scales = torch.zeros((rows + 127) // 128 * 128, (columns + 255) // 256 * 16, dtype=torch.uint8)
    scales[:rows, :blocks] = 0x38 + 8 * twice.to(torch.uint8)  # E4M3 1.0 and 2.0
    tiles = scales.view(-1, 4, 32, scales.shape[1] // 4, 4).permute(0, 3, 2, 1, 4).reshape(scales.shape[0] // 128, -1, 512)
    packed = Nvfp4Matrix((wide[:, 0::2] | (wide[:, 1::2] << 4)).cuda(), tiles.contiguous().cuda(), torch.ones(1, device="cuda"), columns)
    return packed, value


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", PRODUCTS)
def test_product_of_integers_is_exact(m, n, k):
    a, x = exact_operand(m, k, 1)
    b, y = exact_operand(n, k, 2)
    assert torch.equal(a.dequantize().cpu().double(), x)
    bias = torch.randint(-9, 10, (n,), generator=generator(3)).float()
    want = x @ y.t()  # sums below 2^24: exact in float32 in any order
    got = nvfp4_product(a, b)
    assert torch.equal(got.cpu().double(), want)
    assert torch.equal(nvfp4_product(a, b, bias=bias.cuda()).cpu().double(), want + bias)
    wide = torch.full((m, n + 5), 7.0, device="cuda")
    nvfp4_product(a, b, out=wide[:, 1 : n + 1])
    assert torch.equal(wide[:, 1 : n + 1], got) and bool((wide[:, n + 1 :] == 7).all()) and bool((wide[:, 0] == 7).all())
    check_product_status()


def product_bound(x, y, dtype):
    """The float64 product and how far it may be off: blocks of 16 are exact in float32, each of the
    K / 16 additions, at most, loses 2^-23 of the sum of sizes (truncation), the scales three roundings."""
    want, size = x @ y.t(), x.abs() @ y.abs().t()
    return want, ((x.shape[1] + 15) // 16 + 4) * 2.0**-23 * size + 2 * UNIT[dtype] * want.abs() + 2.0**-25 * (dtype == torch.float16)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,n,k", [p for p in PRODUCTS if p[2] > 200])
def test_product(dtype, m, n, k):
    a = quantize_nvfp4(torch.randn(m, k, generator=generator(4)).cuda())
    b = quantize_nvfp4(torch.randn(n, k, generator=generator(5)).cuda() / k**0.5, per="tensor")
    bias = torch.randn(n, generator=generator(6))
    x, y = (torch.from_numpy(decode(p)) for p in (a, b))
    want, bound = product_bound(x, y, dtype)
    got = nvfp4_product(a, b, bias=bias.cuda(), dtype=dtype)
    assert got.dtype == dtype
    error = (got.cpu().double() - (want + bias.double())).abs()
    assert bool((error <= bound + (2.0**-23 + 2 * UNIT[dtype]) * bias.abs().unsqueeze(0)).all())
    assert torch.equal(nvfp4_product(a, b, bias=bias.cuda(), dtype=dtype), got)
    check_product_status()


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", [(8, 1001, 5000), (7, 300, 2100), (60, 200, 1100), (512, 130, 4096), (130, 2, 3200), (300, 700, 1300),
                                   (2304, 600, 1000)])
def test_equal_rows_give_equal_results(m, n, k):
    """Wherever in the batch they lie: tiles split along K over 2, 4 and 8 CTAs, whole ones, and pairs."""
    def wide(rows, seed):  # blocks of many sizes: sums that float32 rounds
        size = torch.exp(2 * torch.randn(rows, (k + 15) // 16, generator=generator(seed + 1)))
        return torch.randn(rows, k, generator=generator(seed)) * torch.repeat_interleave(size, 16, 1)[:, :k]

    x = wide(1, 15).cuda().expand(m, -1).contiguous()
    w = wide(n, 17)
    w[1::2] = w[0]
    y = nvfp4_readout(x, quantize_nvfp4(w.cuda(), per="tensor"))
    assert torch.equal(y, y[:1].expand(m, -1))
    assert torch.equal(y[:, 1::2], y[:, :1].expand(-1, n // 2))


def decode(packed):
    """The float64 values of a packed matrix, from its bytes."""
    codes = packed.codes.cpu().numpy()
    codes = np.stack([codes & 15, codes >> 4], -1).reshape(packed.rows, -1)[:, : packed.columns]
    scales = untiled(packed)[: packed.rows].view(torch.float8_e4m3fn).double().numpy()
    step = np.repeat(scales, 16, 1)[:, : packed.columns] * packed.scale.cpu().double().numpy().reshape(-1, 1)
    return LEVELS[codes] * step


@pytest.mark.gpu
def test_product_of_extreme_scales():
    """Scales at both ends of float32 and E4M3: the sum is scaled one operand at a time."""
    g = generator(7)
    for big, small in ((1e30, 1e-30), (1e-30, 1e20), (1e-38, 1.0)):
        x, y = big * torch.randn(5, 320, generator=g), small * torch.randn(9, 320, generator=g)
        x[:, 64:128] *= 1e-3
        a, b = quantize_nvfp4(x.cuda()), quantize_nvfp4(y.cuda())
        want, bound = product_bound(torch.from_numpy(decode(a)), torch.from_numpy(decode(b)), torch.float32)
        assert bool(((nvfp4_product(a, b).cpu().double() - want).abs() <= bound + 2.0**-149).all())


@pytest.mark.gpu
def test_product_past_32_bit_scale_offsets():
    """2^20 K tiles of 256 columns and more: their block scales lie beyond 2^31 bytes."""
    columns = 2**28 + 1287
    at = torch.tensor([0, 100, 2**27 + 3, 2**28 - 1, 2**28, 2**28 + 300, 2**28 + 1286])
    operands = []
    for rows, level in ((1, [1, 2, -1, 2, 1, 4, 6]), (3, [2, 1, 3, 1, -2, 6, 1])):
        codes = torch.zeros(rows, (columns + 31) // 32 * 16, dtype=torch.uint8, device="cuda")
        scales = torch.zeros(1, (columns + 255) // 256 * 4, 512, dtype=torch.uint8, device="cuda")
        for i, (c, v) in enumerate(zip(at.tolist(), level)):
            codes[:, c // 2] = int(np.flatnonzero(LEVELS == v)[0]) << (4 * (c % 2))
            block = c // 16
            for r in range(rows):
                scales[0, block // 4, 16 * r + block % 4] = 0x38 + 8 * (i % 2)  # E4M3 1.0 or 2.0
        operands.append(Nvfp4Matrix(codes, scales, torch.ones(1, device="cuda"), columns))
    want = sum(x * y * 4 ** (i % 2) for i, (x, y) in enumerate(zip([1, 2, -1, 2, 1, 4, 6], [2, 1, 3, 1, -2, 6, 1])))
    got = nvfp4_product(*operands)
    check_product_status()
    assert got.tolist() == [[want] * 3]
    del operands, codes, scales
    torch.cuda.empty_cache()


# One of each tile, split along K or not, and pairs of CTAs with few and with many K tiles.
@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 129, 4096), (17, 300, 255), (64, 131, 2570), (130, 2, 320), (256, 256, 2048),
                                   (2048, 2560, 520), (2300, 2420, 6000), (2304, 20_000, 64)])
def test_waits_that_run_out_report_and_leave_the_context_usable(m, n, k):
    lib = native.load_library()
    a, x = exact_operand(m, k, 1)
    b, y = exact_operand(n, k, 2)
    out, status = torch.full((m, n), 7.0, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    view = native.dense_matrix(out, "out")

    def product():
        native.token_call(out, lib.nsb_nvfp4_product, ctypes.byref(a._view), ctypes.byref(b._view), None, ctypes.byref(view),
                          status.data_ptr())

    lib.nsb_nvfp4_product_wait_limit(0)  # every wait gives up at once
    try:
        for _ in range(3):
            product()
        torch.cuda.synchronize()
    finally:
        lib.nsb_nvfp4_product_wait_limit(-1)
    assert int(status) != 0 and bool((out == 7.0).all())
    status.zero_()
    product()
    assert int(status) == 0
    assert torch.equal(out.cpu().double(), x @ y.t())


def test_products_refuse_a_status_word_that_is_not_aligned():
    lib = native.load_library()
    p, status = 0x1000, 0x1002  # never read: the checks fail first
    state, weight, out = (ctypes.byref(native._Matrix(p, *s, s[1], 0)) for s in ((4, 16), (6, 16), (4, 6)))
    a, b = (ctypes.byref(native._Nvfp4(rows, 16, p, 16, p, p, 1)) for rows in (4, 6))
    for result in (lib.nsb_nvfp4_product(a, b, None, out, status, None),
                   lib.nsb_nvfp4_readout(state, b, None, out, p, 2**40, status, None),
                   lib.nsb_nvfp4_train_forward(state, weight, None, out, p, p, 2**40, status, None),
                   lib.nsb_nvfp4_train_backward(state, weight, out, p, state, weight, None, p, 2**40, status, None)):
        assert result == -1 and b"status" in lib.nsb_last_error()


def test_status_needs_a_place_for_the_code():
    assert native.load_library().nsb_nvfp4_product_status(None, None) == -1


FIRST_PRODUCT_IN_A_CAPTURE = """
import torch
from neurosim_gpu_b200 import check_product_status, native, nvfp4_readout, quantize_nvfp4
lib = native.load_library()
x = torch.randn(3, 64, device="cuda")
w = quantize_nvfp4(torch.randn(5, 64, device="cuda"))
good, bad = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
with torch.cuda.graph(good):  # the process's first product
    y = nvfp4_readout(x, w)
check_product_status()        # nothing has run: nothing has failed
good.replay()
check_product_status()
want = nvfp4_readout(x, w)
assert torch.equal(y, want)
lib.nsb_nvfp4_product_wait_limit(0)
with torch.cuda.graph(bad):
    z = nvfp4_readout(x, w)
lib.nsb_nvfp4_product_wait_limit(-1)
bad.replay()
good.replay()                 # does not wipe the other's code
try:
    check_product_status()
except RuntimeError as e:
    assert "timeout" in str(e), e
else:
    raise AssertionError("the code was lost")
check_product_status()        # told once
bad.replay()
good.replay()
assert torch.equal(y, want)
try:
    check_product_status("cuda:0")
except RuntimeError:
    print("kept")
"""


@pytest.mark.gpu
def test_status_of_products_in_graphs():
    result = subprocess.run([sys.executable, "-c", FIRST_PRODUCT_IN_A_CAPTURE], capture_output=True, text=True, timeout=300,
                            cwd=Path(__file__).resolve().parent.parent)
    assert result.returncode == 0, result.stderr[-2000:]
    assert result.stdout.strip().endswith("kept")


@pytest.mark.gpu
def test_product_on_a_side_stream_and_in_a_graph():
    x, w = torch.randn(70, 700, generator=generator(8)).cuda(), torch.randn(200, 700, generator=generator(9)).cuda()
    packed = quantize_nvfp4(w, per="tensor")
    want = nvfp4_readout(x, packed)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        torch.cuda._sleep(20_000_000)
        later = torch.zeros_like(x)
        later.copy_(x)
        got = nvfp4_readout(later, packed)
    stream.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = nvfp4_readout(x, packed)
    y.zero_()
    graph.replay()
    assert torch.equal(y, want)


# -- the readout and its gradients ----------------------------------------------------------------


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape,n", [((1, 300), 40), ((5, 2, 300), 40), ((300,), 7), ((2, 0, 300), 7), ((140, 1000), 333)])
def test_readout(dtype, shape, n):
    state = torch.rand(*shape, generator=generator(10)).to(dtype)
    weight = torch.randn(n, shape[-1], generator=generator(11))
    bias = torch.randn(n, generator=generator(12))
    packed = quantize_nvfp4(weight.cuda(), per="tensor")
    got = nvfp4_readout(state.cuda(), packed, bias.cuda())
    assert got.shape == (*shape[:-1], n) and got.dtype == dtype
    flat = state.reshape(-1, shape[-1])
    if len(flat):
        want, bound = product_bound(torch.from_numpy(quantized(flat, "row")[0]), torch.from_numpy(quantized(weight, "tensor")[0]), dtype)
        error = (got.cpu().double().reshape(-1, n) - (want + bias.double())).abs()
        assert bool((error <= bound + (2.0**-23 + 2 * UNIT[dtype]) * bias.abs()).all())
    assert torch.equal(nvfp4_readout(state.cuda(), weight.cuda(), bias.cuda()), got)
    if len(shape) == 2:  # neuron-major states, as the batch tick leaves them
        assert torch.equal(nvfp4_readout(state.cuda().t().contiguous().t(), packed, bias.cuda()), got)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,k,n", [(1, 64, 1), (40, 130, 70), (129, 257, 300), (300, 1024, 128)])
def test_gradients_match_the_formula(dtype, m, k, n):
    g = generator(13)
    x = torch.rand(m, k, generator=g).to(dtype)
    w = torch.randn(n, k, generator=g).to(dtype)
    b = torch.randn(n, generator=g)
    d = torch.randn(m, n, generator=g).to(dtype)
    leaves = [t.cuda().requires_grad_() for t in (x, w, b)]
    y = nvfp4_readout(*leaves)
    grads = torch.autograd.grad(y, leaves, d.cuda())

    def q(t, per):
        return torch.from_numpy(quantized(t, per)[0])

    for got, left, right in ((grads[0], q(d, "row"), q(w.t(), "tensor")), (grads[1], q(d.t(), "tensor"), q(x.t(), "tensor"))):
        want, bound = product_bound(left, right, dtype)
        assert got.dtype == dtype
        assert bool(((got.cpu().double() - want).abs() <= bound).all())
    db = d.double().sum(0)
    assert bool(((grads[2].cpu().double() - db).abs() <= m * 2.0**-24 * d.double().abs().sum(0)).all())
    with torch.no_grad():
        assert torch.equal(y.detach(), nvfp4_readout(*leaves))


@pytest.mark.gpu
def test_gradients_match_differences():
    """On values that NVFP4 holds exactly the readout is the linear map itself, and so are its differences."""
    g = generator(14)
    x, w, d = (torch.randint(-1, 2, s, generator=g).double() for s in ((6, 48), (9, 48), (6, 9)))
    for t in (x, w, d):
        t[:, ::8] = 6.0  # every block holds its largest level, in both directions of the quantiser
        t[::6] = 6.0
        t *= 448.0  # ... so that every scale is 1 and every block scale 448: nothing is rounded anywhere
    leaves = [t.float().cuda().requires_grad_() for t in (x, w)]
    bias = torch.zeros(9, device="cuda", requires_grad=True)

    def loss(x, w, b):
        return (nvfp4_readout(x, w, b) * d.float().cuda()).sum(dtype=torch.float64)

    dx, dw, db = torch.autograd.grad(nvfp4_readout(*leaves, bias), (*leaves, bias), d.float().cuda())
    with torch.no_grad():
        for grad, i in ((dx, 0), (dw, 1)):
            for r, c in ((1, 1), (2, 13), (5, 47)):
                moved = [leaves[0].clone(), leaves[1].clone()]
                moved[i][r, c] = 448.0
                up = loss(*moved, bias)
                moved[i][r, c] = -448.0
                assert float(up - loss(*moved, bias)) / 896 == pytest.approx(float(grad[r, c]), rel=1e-6)
        step = torch.zeros_like(bias)
        step[4] = 448.0
        difference = float(loss(*leaves, bias + step) - loss(*leaves, bias)) / 448
        assert difference == pytest.approx(float(db[4]), rel=1e-6)


@pytest.mark.gpu
def test_gradients_of_some_and_of_empty_batches():
    x, w = torch.rand(5, 40, device="cuda"), torch.randn(6, 40, device="cuda", requires_grad=True)
    (dw,) = torch.autograd.grad(nvfp4_readout(x, w).sum(), w)  # an expanded gradient, no bias
    assert dw.shape == w.shape and bool(dw.any())
    (dw,) = torch.autograd.grad(nvfp4_readout(x[:0], w).sum(), w)
    assert not bool(dw.any())
    b = torch.zeros(6, device="cuda", requires_grad=True)
    (db,) = torch.autograd.grad(nvfp4_readout(x[:0], w.detach(), b).sum(), b)
    assert not bool(db.any())
