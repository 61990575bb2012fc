"""The stimulus lookup and its gradient against float64."""

from __future__ import annotations

import ctypes

import pytest
import torch

from neurosim_gpu_b200 import native, stimulus_drive, stimulus_gradient

DTYPES = [torch.float32, torch.float16, torch.bfloat16]
UNIT = {torch.float32: 2.0**-24, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}
TINY = {torch.float32: 2.0**-149, torch.float16: 2.0**-24, torch.bfloat16: 2.0**-133}


def generator(seed):
    return torch.Generator().manual_seed(seed)


def tokens_of(kind, count, rows, seed=0):
    g = generator(seed)
    if kind == "same":
        return torch.full((count,), rows - 1, dtype=torch.int64)
    if kind == "outside":
        return torch.tensor([-1, rows, 2**40, -(2**40)])[torch.arange(count) % 4]
    tokens = torch.randint(0, rows, (count,), generator=g)
    if kind == "few":  # a few tokens make up most of the batch, some are outside
        tokens = torch.where(torch.rand(count, generator=g) < 0.7, tokens % min(3, rows), tokens)
        tokens[torch.rand(count, generator=g) < 0.1] = -1
    return tokens


# -- refusals (no GPU needed for the C entry points) ---------------------------------------------


def test_entry_points_refuse_bad_arguments():
    lib = native.load_library()
    p = 0x1000  # never read: the checks fail first
    table = native._Matrix(p, 10, 8, 8, 0)
    out = native._Matrix(p, 4, 8, 8, 0)

    def drive(tokens=p, size=8, table=table, out=out):
        return lib.nsb_stimulus_drive(tokens, size, ctypes.byref(table), 1.0, ctypes.byref(out), None)

    for bad in ({"tokens": None}, {"size": 2}, {"tokens": p + 2}, {"out": native._Matrix(p, 4, 7, 7, 0)},
                {"out": native._Matrix(p, 4, 8, 7, 0)}, {"out": native._Matrix(None, 4, 8, 8, 0)},
                {"out": native._Matrix(p, 4, 8, 8, 1)}, {"table": native._Matrix(p, -1, 8, 8, 0)},
                {"table": native._Matrix(p, 10, 8, 8, 3)}, {"table": native._Matrix(p + 2, 10, 8, 8, 0)},
                {"table": native._Matrix(p, 10, 2**31, 2**31, 0)}):
        assert drive(**bad) == -1, bad
        assert lib.nsb_last_error()
    assert drive(out=native._Matrix(None, 0, 8, 8, 0), tokens=None) == 0  # nothing to do
    size = lib.nsb_stimulus_gradient_workspace_size(4, 8)
    assert size > 0 and lib.nsb_stimulus_gradient_workspace_size(0, 8) == 0
    for workspace, have in ((None, size), (p, size - 1), (p + 8, size)):
        assert lib.nsb_stimulus_gradient(p, 8, ctypes.byref(out), 1.0, ctypes.byref(table), workspace,
                                         have, None) == -3


def test_functions_refuse_cpu_tensors():
    with pytest.raises(ValueError, match="CUDA"):
        stimulus_drive(torch.zeros(3, dtype=torch.int64), torch.zeros(4, 8))
    with pytest.raises(ValueError, match="CUDA"):
        stimulus_gradient(torch.zeros(3, dtype=torch.int64), torch.zeros(3, 8), 4)


@pytest.mark.gpu
def test_functions_refuse_bad_arguments():
    table = torch.zeros(4, 8, device="cuda")
    tokens = torch.zeros(3, dtype=torch.int64, device="cuda")
    grad = torch.zeros(3, 8, device="cuda")
    for call in (lambda: stimulus_drive(tokens.float(), table), lambda: stimulus_drive(tokens.cpu(), table),
                 lambda: stimulus_drive(tokens, table.double()), lambda: stimulus_drive(tokens, table[0]),
                 lambda: stimulus_drive(tokens, table.t()), lambda: stimulus_drive(tokens, table, dtype=torch.float16),
                 lambda: stimulus_drive(tokens, table, out=torch.empty(2, 8, device="cuda")),
                 lambda: stimulus_drive(tokens, table.requires_grad_(), out=torch.empty(3, 8, device="cuda")),
                 lambda: stimulus_gradient(tokens, grad[:2], 4), lambda: stimulus_gradient(tokens, grad, -1),
                 lambda: stimulus_gradient(tokens, grad.half(), 4, dtype=torch.bfloat16)):
        with pytest.raises(ValueError):
            call()


# -- values ---------------------------------------------------------------------------------------


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("count,neurons,rows", [(0, 8, 4), (1, 1, 1), (1, 4096, 100), (5, 3, 2), (33, 1001, 7),
                                                (64, 64, 1), (300, 130, 1000), (20, 16600, 50)])
def test_drive(dtype, count, neurons, rows):
    table = torch.randn(rows, neurons, generator=generator(1)).to(dtype)
    tokens = tokens_of("few", count, rows)
    scale = 1.7
    inside = (tokens >= 0) & (tokens < rows)
    # Exact in float64, rounded to float32, then to the result's type: the kernel's own roundings.
    want = table.double()[tokens.clamp(0, rows - 1)] * float(torch.tensor(scale))
    want = torch.where(inside.unsqueeze(1), want, 0.0).float()
    for wide in (False, True):
        for size in (torch.int32, torch.int64):
            got = stimulus_drive(tokens.to(size).cuda(), table.cuda(), scale=scale,
                                 dtype=torch.float32 if wide else None)
            assert got.dtype == (torch.float32 if wide else dtype)
            assert torch.equal(got.cpu(), want.to(got.dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("offset,stride", [(0, 24), (1, 24), (0, 25), (4, 28), (2, 22)])
def test_drive_of_strided_tables_and_token_shapes(offset, stride):
    base = torch.randn(40 * stride, generator=generator(2)).cuda()
    table = base.as_strided((30, 20), (stride, 1), offset)
    tokens = tokens_of("any", 42, 30).view(6, 7).cuda().t()  # [7, 6], not contiguous
    out = torch.full((7, 6, 20), 9.0, device="cuda")
    assert stimulus_drive(tokens, table, out=out) is out
    assert torch.equal(out, table[tokens])
    empty = stimulus_drive(tokens, table[:0])  # no rows: every token is outside
    assert torch.equal(empty, torch.zeros_like(out))


@pytest.mark.gpu
def test_drive_reads_past_32_bit_offsets():
    rows, neurons = 70_000, 33_000  # 2.3e9 elements: the last rows lie beyond 2^31
    table = torch.zeros(rows, neurons, dtype=torch.float16, device="cuda")
    table[-1] = torch.arange(neurons, device="cuda") % 512
    tokens = torch.tensor([rows - 1, 0, rows - 1], device="cuda")
    got = stimulus_drive(tokens, table, scale=2.0)
    assert torch.equal(got[0], table[-1] * 2) and torch.equal(got[2], got[0]) and not got[1].any()
    del table, got
    torch.cuda.empty_cache()


def gradient_bound(tokens, grad, rows, scale, dtype):
    """(the float64 gradient, the largest error of float32 sums in any order, rounded to dtype)."""
    inside = (tokens >= 0) & (tokens < rows)
    index, g = tokens[inside], grad.double()[inside]
    want = torch.zeros(rows, grad.shape[1], dtype=torch.float64).index_add_(0, index, g) * scale
    size = torch.zeros_like(want).index_add_(0, index, g.abs()) * abs(scale)
    count = torch.zeros(rows, dtype=torch.float64).index_add_(0, index, torch.ones(len(index), dtype=torch.float64))
    # n - 1 additions and a multiplication, each off by 2^-24 relative, then the rounding to dtype.
    return want, (count + 1).unsqueeze(1) * 2.0**-24 * size + 2 * UNIT[dtype] * want.abs() + TINY[dtype]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,result", [(d, d) for d in DTYPES] + [(torch.bfloat16, torch.float32),
                                                                      (torch.float32, torch.float16)])
@pytest.mark.parametrize("kind,count,neurons,rows", [
    ("any", 0, 8, 5), ("any", 1, 1, 1), ("any", 2, 3, 300), ("same", 7, 1000, 2), ("same", 70_000, 24, 3),
    ("few", 33, 130, 70_000), ("few", 5000, 257, 40), ("few", 20_001, 64, 513), ("any", 9000, 8, 100_000),
    ("outside", 50, 16, 4), ("same", 300, 1026, 1)])
def test_gradient(dtype, result, kind, count, neurons, rows):
    tokens = tokens_of(kind, count, rows)
    grad = torch.randn(count, neurons, generator=generator(3)).to(dtype)
    scale = 1.5
    want, bound = gradient_bound(tokens, grad, rows, scale, result)
    got = stimulus_gradient(tokens.cuda(), grad.cuda(), rows, scale=scale, dtype=result)
    assert got.dtype == result and got.shape == (rows, neurons)
    assert bool(((got.cpu().double() - want).abs() <= bound).all())
    again = stimulus_gradient(tokens.int().cuda() if kind != "outside" else tokens.cuda(), grad.cuda(), rows,
                              scale=scale, dtype=result)
    assert torch.equal(again, got)


@pytest.mark.gpu
def test_autograd_matches_the_formula_and_differences():
    rows, neurons = 11, 36
    tokens = tokens_of("few", 60, rows).view(12, 5).cuda()
    g = generator(4)
    table = torch.randint(-8, 9, (rows, neurons), generator=g).float().cuda().requires_grad_()
    weight = torch.randint(-8, 9, (12, 5, neurons), generator=g).float().cuda()

    def loss(table):
        return (stimulus_drive(tokens, table, scale=0.5) * weight).sum(dtype=torch.float64)

    (grad,) = torch.autograd.grad(loss(table), table)
    want = torch.zeros(rows, neurons, dtype=torch.float64)
    for t, w in zip(tokens.flatten().tolist(), weight.view(-1, neurons).cpu().double()):
        if 0 <= t < rows:
            want[t] += 0.5 * w
    assert torch.equal(grad.cpu().double(), want)  # small integers: every sum is exact
    for v, n in ((0, 0), (1, 35), (rows - 1, 7)):
        step = torch.zeros_like(table)
        step[v, n] = 2.0
        with torch.no_grad():
            assert float(loss(table + step) - loss(table - step)) / 4.0 == float(grad[v, n])
    # The expanded gradient of a plain sum, and a drive wider than its table.
    narrow = table.detach().bfloat16().requires_grad_()
    (grad,) = torch.autograd.grad(stimulus_drive(tokens, narrow, dtype=torch.float32).sum(), narrow)
    count = torch.bincount(tokens[(tokens >= 0) & (tokens < rows)], minlength=rows).cpu()
    assert grad.dtype == torch.bfloat16
    assert torch.equal(grad.cpu().float(), count.unsqueeze(1).expand(-1, neurons).bfloat16().float())


@pytest.mark.gpu
def test_runs_on_the_current_stream():
    tokens = tokens_of("few", 4000, 50).cuda()
    grad = torch.randn(4000, 512, generator=generator(5)).cuda()
    want = stimulus_gradient(tokens, grad, 50)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        torch.cuda._sleep(20_000_000)  # the copy below lands late: a launch elsewhere would miss it
        later = torch.zeros_like(grad)
        later.copy_(grad)
        got = stimulus_gradient(tokens, later, 50)
        drive = stimulus_drive(tokens, got)
    stream.synchronize()
    assert torch.equal(got, want)
    assert torch.equal(drive, torch.where((tokens >= 0).unsqueeze(1), want[tokens.clamp(min=0)], 0.0))


@pytest.mark.gpu
def test_captured_in_a_graph():
    tokens = tokens_of("few", 257, 20).cuda()
    table = torch.randn(20, 96, generator=generator(6)).cuda()
    drive, grad = stimulus_drive(tokens, table), stimulus_gradient(tokens, table[tokens.clamp(0, 19)], 20)
    source = table[tokens.clamp(0, 19)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a, b = stimulus_drive(tokens, table), stimulus_gradient(tokens, source, 20)
    a.zero_(), b.zero_()
    graph.replay()
    assert torch.equal(a, drive) and torch.equal(b, grad)
