"""Logit penalties, biases, masks and the greedy choice against a plain implementation."""

from __future__ import annotations

import ctypes
import math

import numpy as np
import pytest
import torch

from neurosim_gpu_b200 import adjust_logits, native

DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def generator(seed):
    return torch.Generator().manual_seed(seed)


def plain(logits, history=None, lengths=None, prompts=None, repetition=1.0, presence=0.0, frequency=0.0,
          bias=None, mask=None, kind=np.float64):
    """The formula on the CPU, each step in `kind`; -> (adjusted [B, V] before the last rounding, counts)."""
    x = logits.float().numpy().astype(kind)
    rows, vocabulary = x.shape
    count = np.zeros((rows, vocabulary), np.int64)
    seen = np.zeros((rows, vocabulary), bool)
    if history is not None:
        h = history.numpy()
        for b in range(rows):
            end = h.shape[1] if lengths is None else min(max(int(lengths[b]), 0), h.shape[1])
            start = 0 if prompts is None else int(prompts[b])
            for i, v in enumerate(h[b, :end]):
                if 0 <= v < vocabulary:
                    seen[b, v] = True
                    count[b, v] += i >= start

    def column(value):
        value = value.numpy() if isinstance(value, torch.Tensor) else np.float32(value)
        return np.broadcast_to(np.asarray(value, np.float32).astype(kind).reshape(-1, 1), (rows, 1))

    r, p, f = column(repetition), column(presence), column(frequency)
    with np.errstate(invalid="ignore"):
        x = np.where(seen, np.where(x > 0, x / r, x * r), x)
        x = np.where(count > 0, x - f * count.astype(kind) - p, x)
        if bias is not None:
            x = x + bias.numpy().astype(kind)
    if mask is not None:
        bits = (mask.numpy().astype(np.uint32)[..., None] >> np.arange(32, dtype=np.uint32)) & 1
        bits = bits.reshape(*mask.shape[:-1], 32 * mask.shape[-1])[..., :vocabulary]
        x = np.where(bits == 0, -math.inf, x)
    return x, count


def choice_of(adjusted):
    x = np.where(np.isnan(adjusted), -math.inf, adjusted)
    best = x.argmax(1)  # the lowest index of equal ones
    return np.where(x.max(1) > -math.inf, best, -1)


def check(logits, dtype, **kw):
    names = {"prompts": "prompt_lengths"}
    device = {names.get(k, k): v.cuda() if isinstance(v, torch.Tensor) else v for k, v in kw.items()}
    got, choice = adjust_logits(logits.cuda(), choose=True, **device)
    steps, _ = plain(logits, kind=np.float32, **kw)
    want = torch.from_numpy(steps).to(dtype)
    assert got.dtype == dtype
    torch.testing.assert_close(got.cpu(), want, rtol=0, atol=0, equal_nan=True)  # the same float32 steps
    assert choice.cpu().tolist() == choice_of(want.float().numpy()).tolist()
    # ... and near the formula in float64: five float32 roundings of numbers no larger than the
    # parts' sizes, and the rounding to dtype.
    exact, count = plain(logits, **kw)
    size = np.abs(np.nan_to_num(logits.double().numpy())) * 2 + 2 + 2 * count
    if kw.get("bias") is not None:
        size = size + np.abs(np.nan_to_num(kw["bias"].numpy(), neginf=0.0))
    unit = {torch.float32: 0.0, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}[dtype]
    finite = np.isfinite(exact) & np.isfinite(got.float().cpu().numpy())
    with np.errstate(invalid="ignore"):
        error = np.abs(got.float().cpu().numpy().astype(np.float64) - exact)
    bound = 5 * 2.0**-24 * size + unit * np.abs(np.where(finite, exact, 0.0)) + 2.0**-24
    assert bool((error <= bound)[finite].all())
    assert np.array_equal(finite, np.isfinite(exact))
    return got, choice


def case(rows, vocabulary, length, seed=0):
    g = generator(seed)
    history = torch.randint(-2, vocabulary + 2, (rows, length), generator=g, dtype=torch.int32)
    if length:
        history[:, ::3] = history[:, ::3] % max(1, vocabulary // 50 + 1)  # some tokens repeat often
    return {
        "history": history,
        "lengths": torch.randint(-1, length + 3, (rows,), generator=g, dtype=torch.int32),
        "prompts": torch.randint(0, length + 1, (rows,), generator=g, dtype=torch.int32),
        "repetition": 1 + torch.rand(rows, generator=g), "presence": torch.rand(rows, generator=g),
        "frequency": torch.rand(rows, generator=g) - 0.3,
        "bias": torch.randn(vocabulary, generator=g),
        "mask": torch.randint(-(2**31), 2**31, (rows, (vocabulary + 31) // 32), generator=g).int(),
    }


def test_entry_point_refuses_bad_arguments():
    lib = native.load_library()
    p = 0x1000  # never read: the checks fail first

    def call(**kw):
        args = native._Logits()
        args.logits = args.out = native._Matrix(p, 2, 100, 100, 0)
        args.repetition.scalar = 1.0
        for name, value in kw.items():
            setattr(args, name, value)
        return lib.nsb_adjust_logits(ctypes.byref(args), None)

    for bad in ({"out": native._Matrix(p, 2, 99, 100, 0)}, {"out": native._Matrix(p, 2, 100, 100, 1)},
                {"logits": native._Matrix(None, 2, 100, 100, 0)}, {"history_length": 5}, {"history_length": -1},
                {"bias": p, "bias_stride": -1}, {"mask": p, "mask_stride": -1},
                {"repetition": native._RowValues(None, 0, 0.0)}, {"presence": native._RowValues(p, -1, 0.0)}):
        assert call(**bad) == -1, bad
        assert lib.nsb_last_error()
    assert lib.nsb_adjust_logits(None, None) == -1
    empty = native._Matrix(None, 0, 100, 100, 0)
    assert call(logits=empty, out=empty) == 0


def test_entry_points_refuse_results_that_overlap_with_what_they_read():
    lib = native.load_library()
    p = 0x10000  # never read: the checks fail first

    def adjust(out, logits=(0, 3, 100, 200)):
        args = native._Logits()
        args.logits, args.out = (native._Matrix(p + 4 * at, rows, cols, stride, 0) for at, rows, cols, stride in (logits, out))
        args.repetition.scalar = 0.0  # what the last check refuses
        assert lib.nsb_adjust_logits(ctypes.byref(args), None) == -1
        return b"overlap" not in lib.nsb_last_error()

    # The same matrix, before it, behind it, and the other columns of its rows.
    for at, stride in ((0, 200), (-500, 200), (500, 200), (500, 100), (100, 200), (-100, 200), (300, 200), (-300, 200)):
        assert adjust((at, 3, 100, stride)), (at, stride)
    for at, stride in ((1, 200), (-1, 200), (99, 200), (-99, 200), (0, 201), (0, 100), (499, 100), (200, 200), (101, 200)):
        assert not adjust((at, 3, 100, stride)), (at, stride)
    assert adjust((0, 1, 100, 150), (0, 1, 100, 100)) and adjust((100, 1, 100, 150), (0, 1, 100, 100))
    assert not adjust((99, 1, 100, 150), (0, 1, 100, 100))

    def drive(at, kind=0):
        table, out = native._Matrix(p, 10, 8, 8, 1 if kind == 1 else 0), native._Matrix(p + at, 4, 8, 8, kind)
        assert lib.nsb_stimulus_drive(None, 8, ctypes.byref(table), 1.0, ctypes.byref(out), None) == -1
        return b"overlap" not in lib.nsb_last_error()

    assert drive(320) and drive(-128) and drive(160, 1)
    assert not drive(316) and not drive(-124) and not drive(0) and not drive(158, 1)


def test_entry_point_refuses_addresses_that_are_not_aligned():
    lib = native.load_library()
    p = 0x10000  # never read: the checks fail first
    for name, step in (("history", 2), ("lengths", 1), ("prompt_lengths", 2), ("bias", 2), ("mask", 3), ("choice", 4), ("repetition", 2),
                       ("presence", 1), ("frequency", 2)):
        args = native._Logits()
        args.logits = args.out = native._Matrix(p, 2, 100, 100, 0)
        args.repetition.scalar = 1.0
        args.history, args.history_length = p, 5
        setattr(args, name, native._RowValues(p + step, 1, 1.0) if isinstance(getattr(args, name), native._RowValues) else p + step)
        assert lib.nsb_adjust_logits(ctypes.byref(args), None) == -1, name
        assert b"aligned" in lib.nsb_last_error(), name


def test_function_refuses_cpu_tensors():
    with pytest.raises(ValueError, match="CUDA"):
        adjust_logits(torch.zeros(2, 8))


def test_function_refuses_to_drop_a_gradient():
    x, leaf, row = torch.zeros(2, 8), torch.zeros(2, 8, requires_grad=True), torch.zeros(2, requires_grad=True)
    for call in (lambda: adjust_logits(leaf), lambda: adjust_logits(x, out=leaf), lambda: adjust_logits(x, bias=leaf),
                 lambda: adjust_logits(2 * leaf), lambda: adjust_logits(x, repetition=row), lambda: adjust_logits(x, presence=row),
                 lambda: adjust_logits(x, frequency=row)):
        with pytest.raises(ValueError, match="gradient"):
            call()
        with torch.no_grad(), pytest.raises(ValueError, match="CUDA"):
            call()


@pytest.mark.gpu
def test_logits_that_require_a_gradient():
    """Of a training readout's result: refused, in place and not, and taken under no_grad."""
    leaf = torch.randn(3, 50, device="cuda", requires_grad=True)
    y = 2 * leaf
    before = y.detach().clone()
    for kw in ({}, {"out": y}, {"choose": True}):
        with pytest.raises(ValueError, match="gradient"):
            adjust_logits(y, bias=torch.ones(50, device="cuda"), **kw)
    assert torch.equal(y, before)
    with torch.no_grad():
        got = adjust_logits(y, bias=torch.ones(50, device="cuda"))
    assert not got.requires_grad and torch.equal(got, before + 1)
    assert torch.equal(adjust_logits(y.detach(), bias=torch.ones(50, device="cuda")), got)


@pytest.mark.gpu
def test_function_refuses_bad_arguments():
    x = torch.zeros(2, 40, device="cuda")
    words = torch.zeros(2, 2, dtype=torch.int32, device="cuda")
    for bad in ({"history": words.long()}, {"history": words[:1]}, {"lengths": words[:, 0].contiguous()},
                {"history": words, "lengths": words[0, :1]}, {"bias": x[0, :39]}, {"bias": x[0].half()},
                {"mask": words[:, :1]}, {"mask": words.float()}, {"repetition": 0.0}, {"presence": x[:, 0].double()},
                {"frequency": torch.zeros(3, device="cuda")}, {"out": x[:1]}, {"out": x.half()}):
        with pytest.raises((ValueError, RuntimeError)):
            adjust_logits(x, **bad)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocabulary,length", [(0, 5, 3), (1, 1, 0), (1, 1, 4), (2, 31, 1), (1, 33, 17), (3, 1000, 0),
                                                    (5, 4097, 300), (2, 70_001, 5000), (1, 131_072, 64), (2, 200_003, 40_000),
                                                    (1, 600_000, 5000), (700, 130, 9)])
def test_adjust(dtype, rows, vocabulary, length):
    logits = (3 * torch.randn(rows, vocabulary, generator=generator(1))).to(dtype)
    check(logits, dtype, **case(rows, vocabulary, length))


@pytest.mark.gpu
def test_every_part_alone():
    rows, vocabulary = 3, 515
    logits = torch.randn(rows, vocabulary, generator=generator(2))
    full = case(rows, vocabulary, 200)
    check(logits, torch.float32)
    check(logits, torch.float32, bias=full["bias"])
    check(logits, torch.float32, mask=full["mask"])
    check(logits, torch.float32, mask=full["mask"][0], bias=torch.randn(rows, vocabulary))
    check(logits, torch.float32, history=full["history"], repetition=1.3)
    check(logits, torch.float32, history=full["history"], presence=0.5)
    check(logits, torch.float32, history=full["history"], lengths=full["lengths"], frequency=0.25, presence=-0.5)
    check(logits, torch.float32, history=full["history"], prompts=full["prompts"], repetition=0.5, frequency=1.0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_masked_rows_ties_and_values_that_are_not_finite(dtype):
    vocabulary = 9001
    logits = torch.zeros(6, vocabulary, dtype=dtype)
    mask = torch.full((6, (vocabulary + 31) // 32), -1, dtype=torch.int32)
    mask[0] = 0                                    # nothing left
    mask[1] = 0
    mask[1, 200] = 1 << 5                          # one token left
    logits[2, [70, 8999, 9000]] = 2.0              # equal largest: the lowest index
    logits[3] = torch.finfo(dtype).min             # the type's lowest value is still a choice
    logits[4, 10] = math.nan                       # never chosen
    logits[4, 20] = math.inf
    logits[5] = -math.inf
    for value in (math.nan, math.inf):             # in masked places they vanish
        logits[1, 7] = value
        got, choice = check(logits, dtype, mask=mask)
        assert choice.tolist() == [-1, 200 * 32 + 5, 70, 0, 20, -1]
        assert bool(torch.isneginf(got[0]).all()) and int(torch.isfinite(got[1]).sum()) == 1
    bias = torch.zeros(vocabulary)
    bias[70] = -math.inf                           # a bias can ban a token
    assert check(logits, dtype, mask=mask, bias=bias)[1].tolist()[2] == 8999


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_strided_rows_in_place_and_graph(dtype):
    rows, vocabulary = 4, 3001
    kw = case(rows, vocabulary, 90)
    base = torch.randn(rows * 3100 + 8, generator=generator(3)).to(dtype)
    for offset, stride in ((0, 3001), (1, 3008), (3, 3013), (8, 3024)):
        view = base.as_strided((rows, vocabulary), (stride, 1), offset)
        got, _ = check(view.clone(), dtype, **kw)
        device = {("prompt_lengths" if k == "prompts" else k): v.cuda() for k, v in kw.items()}
        strided = base.cuda().as_strided((rows, vocabulary), (stride, 1), offset)
        assert torch.equal(adjust_logits(strided, **device), got)
        out = torch.zeros(rows, 3030, dtype=dtype, device="cuda")[:, 2:3003]  # another place within 16 bytes
        assert torch.equal(adjust_logits(strided, out=out, **device), got)
        assert adjust_logits(strided, out=strided, **device) is strided
        assert torch.equal(strided, got)
    source = base[: rows * vocabulary].view(rows, vocabulary).cuda()
    want, choice = adjust_logits(source, choose=True, **device)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a, b = adjust_logits(source, choose=True, **device)
    a.zero_(), b.zero_()
    graph.replay()
    assert torch.equal(a, want) and torch.equal(b, choice)


@pytest.mark.gpu
def test_results_beside_the_logits_and_over_them():
    base = torch.randn(5, 90, generator=generator(6)).cuda()
    logits, bias = base[:, :45], torch.ones(45, device="cuda")
    want = logits + 1
    for bad in (base[:, 1:46], base[:, 44:89], base.view(-1)[: 5 * 45].view(5, 45)):
        with pytest.raises(RuntimeError, match="overlap"):
            adjust_logits(logits, bias=bias, out=bad)
    assert torch.equal(adjust_logits(logits, bias=bias, out=base[:, 45:]), want)  # the other half of each row
    assert torch.equal(adjust_logits(logits, bias=bias, out=base[:, :45]), want)  # another tensor, the same elements
    assert torch.equal(logits, want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocabulary,length", [(2, 131_071, 4096), (2, 200_003, 40_000), (1, 600_000, 5000), (3, 1001, 70_000)])
def test_long_histories_in_place(dtype, rows, vocabulary, length):
    logits = (3 * torch.randn(rows, vocabulary, generator=generator(4))).to(dtype)
    kw = case(rows, vocabulary, length)
    got, choice = check(logits, dtype, **kw)
    device = {("prompt_lengths" if k == "prompts" else k): v.cuda() for k, v in kw.items()}
    x = logits.cuda()
    again, same = adjust_logits(x, out=x, choose=True, **device)
    assert again is x and torch.equal(x, got) and torch.equal(same, choice)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocabulary", [(1, 131_072), (3, 40_001), (18, 33_000), (20, 33_000)])
def test_few_long_rows_without_a_history(dtype, rows, vocabulary):
    logits = (3 * torch.randn(rows, vocabulary, generator=generator(5))).to(dtype)
    kw = case(rows, vocabulary, 0)
    check(logits, dtype)
    check(logits, dtype, mask=kw["mask"], bias=kw["bias"])


@pytest.mark.gpu
def test_history_just_below_32_bits():
    """A walk over the history steps past its end: the place there is beyond 2^31."""
    length, vocabulary = 2**31 - 1, 40_000
    history = torch.full((1, length), -1, dtype=torch.int32, device="cuda")
    history[0, -3:] = torch.tensor([7, 39_999, 7])
    history[0, 5] = 11
    logits = torch.ones(1, vocabulary, device="cuda")
    prompts = torch.tensor([2**31 - 3], dtype=torch.int32, device="cuda")  # the last two are generated
    got = adjust_logits(logits, history=history, prompt_lengths=prompts, repetition=2.0, frequency=0.25, presence=1.0)
    want = torch.ones(vocabulary)
    want[[7, 39_999]] = 0.5 - 0.25 - 1.0
    want[11] = 0.5
    assert torch.equal(got[0].cpu(), want)
    negative = adjust_logits(logits, history=history[:, -3:], prompt_lengths=-prompts, frequency=0.25)  # no prompt
    assert negative[0, 7] == 0.5 and negative[0, 39_999] == 0.75
    del history
    torch.cuda.empty_cache()
