"""Tokens through a network: stimulus, ticks, readout and the choice of the next token.

``generate_tokens`` runs the chain ``token -> stimulus_drive -> ticks -> nvfp4_readout ->
adjust_logits -> token`` on the device, without reading anything back in between.
"""

from __future__ import annotations

import torch

from .logits import adjust_logits
from .microscale import Nvfp4Matrix, check_product_status, nvfp4_readout
from .stimulus import stimulus_drive


def generate_tokens(runtime, table: torch.Tensor, readout: Nvfp4Matrix | torch.Tensor,
                    prompt: torch.Tensor, steps: int, *, bias: torch.Tensor | None = None,
                    scale: float = 1.0, ticks: int = 1,
                    dendritic_drive: torch.Tensor | float = 0.0,
                    repetition: float | torch.Tensor = 1.0, presence: float | torch.Tensor = 0.0,
                    frequency: float | torch.Tensor = 0.0,
                    logit_bias: torch.Tensor | None = None,
                    mask: torch.Tensor | None = None) -> torch.Tensor:
    """The ``steps`` tokens [B, steps] (int64) that a network answers a prompt [B, P] with, P >= 1.

    Each token drives the network's B states for ``ticks`` ticks with ``scale * table[token]``
    (``table`` [V, N]; -1: no stimulus); the states are read out with ``readout`` ([V_out, N], packed
    or floating-point) and ``bias``, and the largest logit after penalties, ``logit_bias`` and
    ``mask`` (see :func:`adjust_logits`) is the next token, -1 where the mask leaves none.  The
    ``runtime`` (matrix or PELS) is advanced in place.  The call ends with the tokens on the device,
    and with a check that no product gave up (``RuntimeError``, see :func:`check_product_status`).
    """
    batch, neurons = runtime.state.shape
    if prompt.dim() != 2 or prompt.shape[0] != batch or prompt.shape[1] < 1:
        raise ValueError("prompt must be [B, P] with the runtime's B and P >= 1")
    if prompt.dtype not in (torch.int32, torch.int64) or prompt.device != table.device:
        raise ValueError("prompt must be int32 or int64 on the table's device")
    if table.dim() != 2 or table.shape[1] != neurons:
        raise ValueError("table must be [V, N] with the runtime's N")
    if steps < 0 or ticks < 1:
        raise ValueError("steps must not be negative, and ticks be at least 1")
    length = prompt.shape[1]
    with torch.no_grad():  # not inference mode: the runtime keeps the states, and may be trained through later
        history = torch.full((batch, length + steps), -1, device=prompt.device, dtype=torch.int32)
        history[:, :length] = prompt.clamp(-1, 2**31 - 1)  # what no table has stays outside it
        prompts = torch.full((batch,), length, device=prompt.device, dtype=torch.int32)
        answer = torch.empty((batch, steps), device=prompt.device, dtype=torch.int64)
        for at in range(length + steps - 1 if steps else 0):
            drive = stimulus_drive(history[:, at], table, scale=scale, dtype=torch.float32)
            for _ in range(ticks):
                runtime.step(drive, dendritic_drive=dendritic_drive)
            new = at + 1 - length
            if new < 0:
                continue  # the prompt's next token is known
            logits = nvfp4_readout(runtime.state, readout, bias, dtype=torch.float32)
            _, choice = adjust_logits(logits, history=history[:, : at + 1], prompt_lengths=prompts,
                                      repetition=repetition, presence=presence, frequency=frequency,
                                      bias=logit_bias, mask=mask, out=logits, choose=True)
            answer[:, new] = choice
            history[:, at + 1] = choice
        if steps:
            check_product_status(runtime.state.device)
    return answer
