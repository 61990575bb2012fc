"""The token operators together, around a network."""

from __future__ import annotations

import pytest
import torch

from _util import make
from neurosim_gpu_b200 import (NativeDendriticMatrixRuntime, NativeDendriticPELSRuntime, adjust_logits,
                               generate_tokens, native, nvfp4_product, nvfp4_readout, quantize_nvfp4, stimulus_drive)

pytestmark = pytest.mark.gpu


def parts(n=97, batch=3, vocabulary=61):
    graph, model, state = make(n=n, batch=batch)
    g = torch.Generator().manual_seed(5)
    table = torch.randn(vocabulary, n, generator=g).cuda()
    weight = torch.randn(vocabulary, n, generator=g).cuda()
    bias = torch.randn(vocabulary, generator=g).cuda()
    prompt = torch.randint(0, vocabulary, (batch, 4), generator=g).cuda()
    mask = torch.full((batch, 2), -1, dtype=torch.int32, device="cuda")
    mask[0, 0] = 0x0000FFFF
    return graph, model, state, table, weight, bias, prompt, mask


def plainly(runtime, table, weight, bias, prompt, steps, mask, repetition, frequency):
    """The same chain from plain operations in float64, on the host; -> (tokens, smallest margin)."""
    values = quantize_nvfp4(weight, per="tensor").dequantize().cpu().double()
    history = [row.tolist() for row in prompt.cpu()]
    length, margin = prompt.shape[1], float("inf")
    bits = (mask.cpu().unsqueeze(-1) >> torch.arange(32, dtype=torch.int32)).bitwise_and(1).flatten(1)[:, : len(values)]
    for at in range(length + steps - 1):
        drive = torch.stack([0.7 * table[h[at]] if h[at] >= 0 else torch.zeros_like(table[0]) for h in history])
        with torch.inference_mode():
            runtime.step(drive, dendritic_drive=0.05)
        if at + 1 < length:
            continue
        state = quantize_nvfp4(runtime.state.contiguous()).dequantize().cpu().double()
        logits = state @ values.t() + bias.cpu().double()
        for b, h in enumerate(history):
            for v in set(h):
                if v >= 0:
                    logits[b, v] = logits[b, v] / repetition if logits[b, v] > 0 else logits[b, v] * repetition
                    logits[b, v] -= frequency * h[length:].count(v)
        logits[bits == 0] = -float("inf")
        best = logits.topk(2, dim=1).values
        margin = min(margin, float((best[:, 0] - best[:, 1]).min()))
        for h, v in zip(history, logits.argmax(1).tolist()):
            h.append(v)
    return torch.tensor(history)[:, length:], margin


@pytest.mark.parametrize("kind", [NativeDendriticMatrixRuntime, NativeDendriticPELSRuntime])
@pytest.mark.parametrize("batch", [1, 3])
def test_generate_matches_the_plain_chain(kind, batch):
    graph, model, state, table, weight, bias, prompt, mask = parts(batch=batch)
    kw = {} if kind is NativeDendriticMatrixRuntime else {"theta": 0.01}
    want, margin = plainly(kind(graph, model, state.clone(), **kw), table, weight, bias, prompt, 7, mask, 1.3, 0.2)
    # Logits of a few units, off by less than 1e-5; the choices can be told apart.  (PELS sums its current
    # with atomics, in no fixed order: 1e-6 in the state.)
    assert margin > 1e-4
    for readout in (weight, quantize_nvfp4(weight, per="tensor")):
        runtime = kind(graph, model, state.clone(), **kw)
        got = generate_tokens(runtime, table, readout, prompt, 7, bias=bias, scale=0.7, dendritic_drive=0.05,
                              repetition=1.3, frequency=0.2, mask=mask)
        assert got.cpu().tolist() == want.tolist()
        assert runtime.last_backend == "native"


def test_generate_with_nothing_allowed_and_refusals():
    graph, model, state, table, weight, bias, prompt, mask = parts()
    runtime = NativeDendriticMatrixRuntime(graph, model, state)
    mask[1] = 0
    got = generate_tokens(runtime, table, weight, prompt, 3, mask=mask, ticks=2)
    assert got[1].tolist() == [-1, -1, -1] and bool((got[[0, 2]] >= 0).all()) and bool(((got[0] < 16) | (got[0] >= 32)).all())
    assert generate_tokens(runtime, table, weight, prompt, 0).shape == (3, 0)
    for bad in (lambda: generate_tokens(runtime, table, weight, prompt[:2], 3), lambda: generate_tokens(runtime, table, weight, prompt[:, :0], 3),
                lambda: generate_tokens(runtime, table[:, :5], weight, prompt, 3), lambda: generate_tokens(runtime, table, weight, prompt.float(), 3),
                lambda: generate_tokens(runtime, table, weight, prompt, -1), lambda: generate_tokens(runtime, table, weight, prompt, 3, ticks=0)):
        with pytest.raises(ValueError):
            bad()


def test_training_through_the_network():
    """A loss on the logits reaches the stimulus table, the readout weights and the bias, and descent lowers it.
    (Not every single step does: between the codes' midpoints the quantised loss is flat.)"""
    graph, model, state, table, weight, bias, prompt, _ = parts()
    leaves = [t.clone().requires_grad_() for t in (table, weight, bias)]
    target = torch.tensor([3, 17, 60], device="cuda")

    def loss(table, weight, bias):
        runtime = NativeDendriticMatrixRuntime(graph, model, state.clone())
        for at in range(3):
            runtime.step(stimulus_drive(prompt[:, at], table, scale=0.7))
        return torch.nn.functional.cross_entropy(nvfp4_readout(runtime.state, weight, bias), target)

    first = loss(*leaves)
    first.backward()
    used = torch.zeros(table.shape[0], dtype=torch.bool, device="cuda")
    used[prompt[:, :3].flatten()] = True
    assert bool((leaves[0].grad.abs().sum(1) > 0)[used].all()) and not bool(leaves[0].grad[~used].any())
    for _ in range(30):
        now = loss(*leaves)
        for leaf, grad in zip(leaves, torch.autograd.grad(now, leaves)):
            with torch.no_grad():
                leaf -= 0.2 * grad
    assert float(now) < 0.5 * float(first)


@pytest.mark.parametrize("kind", [NativeDendriticMatrixRuntime, NativeDendriticPELSRuntime])
@pytest.mark.parametrize("batch", [1, 3])
def test_training_through_a_runtime_that_has_generated(kind, batch):
    graph, model, state, table, weight, bias, prompt, _ = parts(batch=batch)
    runtime = kind(graph, model, state, **({} if kind is NativeDendriticMatrixRuntime else {"theta": 0.01}))
    answer = generate_tokens(runtime, table, weight, prompt, 2)
    for value in (answer, runtime.state, runtime.dendritic_state, runtime.adaptation_state):
        assert not value.is_inference() and not value.requires_grad
    leaves = [t.clone().requires_grad_() for t in (table, weight, bias)]
    nvfp4_readout(runtime.state, *leaves[1:]).sum().backward()  # keeps the state for its backward pass
    assert bool(leaves[1].grad.any()) and bool(leaves[2].grad.any())
    runtime.step(stimulus_drive(answer[:, -1], leaves[0], scale=0.7))
    (grad,) = torch.autograd.grad(nvfp4_readout(runtime.state, weight, bias).sum(), leaves[0])
    assert bool(grad[answer[:, -1]].any())


def test_generate_reports_a_product_that_gave_up():
    graph, model, state, table, weight, bias, prompt, _ = parts()
    lib = native.load_library()
    want = generate_tokens(NativeDendriticMatrixRuntime(graph, model, state.clone()), table, weight, prompt, 3, bias=bias)
    lib.nsb_nvfp4_product_wait_limit(0)
    try:
        with pytest.raises(RuntimeError, match="timeout"):
            generate_tokens(NativeDendriticMatrixRuntime(graph, model, state.clone()), table, weight, prompt, 3, bias=bias)
    finally:
        lib.nsb_nvfp4_product_wait_limit(-1)
    again = generate_tokens(NativeDendriticMatrixRuntime(graph, model, state.clone()), table, weight, prompt, 3, bias=bias)
    assert torch.equal(again, want)


def test_autograd_learns_of_results_written_over_its_tensors():
    """exp() keeps its result for its backward pass, which refuses once that has been written over."""
    leaf = torch.randn(4, 40, device="cuda", requires_grad=True)
    packed = quantize_nvfp4(torch.randn(4, 64, device="cuda")), quantize_nvfp4(torch.randn(40, 64, device="cuda"))
    tokens = torch.zeros(4, dtype=torch.int64, device="cuda")
    for write in (lambda y: adjust_logits(y, out=y), lambda y: stimulus_drive(tokens, leaf, out=y),
                  lambda y: nvfp4_product(*packed, out=y)):
        y = leaf.exp()
        with torch.no_grad():
            assert write(y) is y
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.sum().backward()
    with torch.inference_mode():  # its tensors have no version
        y = torch.zeros(4, 40, device="cuda")
        assert adjust_logits(y, out=y) is y
