"""Derivatives that a token operator would drop are refused."""

from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

from neurosim_gpu_b200 import (Nvfp4Matrix, adjust_logits, nvfp4_product, nvfp4_readout, quantize_nvfp4, stimulus_drive,
                               stimulus_gradient)


def test_derivatives_that_would_be_dropped_are_refused():
    """Before anything else is looked at, so that tensors on the CPU show it."""
    plain, leaf, row = torch.zeros(3, 8), torch.zeros(3, 8, requires_grad=True), torch.zeros(3, requires_grad=True)
    tokens = torch.zeros(3, dtype=torch.int64)
    with pytest.raises(ValueError, match="gradient"):
        stimulus_gradient(tokens, leaf, 4)
    with pytest.raises(ValueError, match="gradient"):
        stimulus_drive(tokens, plain, out=leaf)
    with torch.no_grad():
        for call in (lambda: stimulus_gradient(tokens, leaf, 4), lambda: stimulus_drive(tokens, plain, out=leaf)):
            with pytest.raises(ValueError, match="CUDA"):
                call()
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(plain, torch.ones_like(plain))
        for call in (lambda: stimulus_drive(tokens, dual), lambda: stimulus_gradient(tokens, dual, 4), lambda: nvfp4_readout(dual, plain),
                     lambda: nvfp4_readout(plain, dual), lambda: nvfp4_readout(plain, plain, dual[0]), lambda: adjust_logits(dual),
                     lambda: adjust_logits(plain, bias=dual[0])):
            with pytest.raises(ValueError, match="forward-mode|gradients"):
                call()
        with pytest.raises(ValueError, match="CUDA"):  # no tangent: the check of the device is next
            stimulus_drive(tokens, plain)


@pytest.mark.gpu
def test_products_refuse_gradients_that_they_would_drop():
    x = torch.randn(4, 64, device="cuda")
    a, b = quantize_nvfp4(x.requires_grad_()), quantize_nvfp4(torch.randn(6, 64, device="cuda"))
    bias = torch.zeros(6, device="cuda", requires_grad=True)
    scaled = Nvfp4Matrix(a.codes, a.block_scales, a.scale.clone().requires_grad_(), 64)
    out = torch.zeros(4, 6, device="cuda", requires_grad=True)
    for call in (lambda: nvfp4_product(a, b, bias=bias), lambda: nvfp4_product(a, b, out=out), lambda: nvfp4_product(scaled, b),
                 lambda: nvfp4_product(b, scaled), scaled.dequantize, lambda: nvfp4_readout(x.detach(), scaled),
                 lambda: nvfp4_readout(x.detach(), b, bias)):
        with pytest.raises(ValueError, match="gradient"):
            call()
        with torch.no_grad():
            assert bool(call().isfinite().all())
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x.detach(), torch.ones_like(x))
        with pytest.raises(ValueError, match="forward-mode"):
            nvfp4_readout(dual, torch.randn(6, 64, device="cuda", requires_grad=True))


@pytest.mark.gpu
def test_backward_passes_refuse_tangents():
    """Forward over reverse: the gradient that comes in is a dual tensor."""
    leaf = torch.randn(6, 64, device="cuda", requires_grad=True)
    tokens = torch.tensor([1, 5, 1], device="cuda")
    for y in (nvfp4_readout(torch.randn(3, 64, device="cuda"), leaf), stimulus_drive(tokens, leaf)):
        with forward_ad.dual_level():
            dual = forward_ad.make_dual(torch.ones_like(y), torch.ones_like(y))
            with pytest.raises(ValueError, match="forward-mode|gradients"):
                torch.autograd.grad(y, leaf, dual, retain_graph=True)
        (grad,) = torch.autograd.grad(y, leaf, torch.ones_like(y))
        assert bool(grad.any())
