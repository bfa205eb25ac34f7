"""AdamW over many tensors at once, for the parameters that Muon does not suit (embeddings, heads,
gains, biases) or for a whole model, with moments in 32 or in 8 bits, and the global gradient norm that
goes before a step of any optimizer class.

The reference's Adam (muon.py:104-109) keeps its moments in the parameter's type; that arithmetic stays
in ``adam_update`` and in the classes' auxiliary Adam. Here moments are float32, or 8-bit codes with
one float32 scale per 256 elements whatever the parameter's type, the arithmetic is float32, and
one launch takes hundreds of tensors. The formats are described in ``include/muon_b200.h``."""
from __future__ import annotations

import math
from typing import Sequence

import torch
from torch import Tensor

from ._lib import STATE_BLOCK
from ._tables import gradients
from .engine import _STATE_KINDS, get_backend


def adamw_step(params: Sequence[Tensor], grads: Sequence[Tensor], exp_avgs: Sequence[Tensor],
               exp_avg_sqs: Sequence[Tensor], steps, *, lr: float = 1e-3, betas: tuple[float, float] = (0.9, 0.999),
               eps: float = 1e-8, weight_decay: float = 1e-2, masters: Sequence[Tensor] | None = None,
               grad_scale: Tensor | None = None) -> None:
    """One AdamW step (decoupled weight decay) on lists of tensors, in place on ``params``, ``masters``,
    ``exp_avgs`` and ``exp_avg_sqs``.

    Arguments:
        params: all float32, all bfloat16 or all float16; any sizes, contiguous (or dense, with
            gradients and moments of the same strides).
        grads: of the parameters' type, or float32.
        exp_avgs, exp_avg_sqs: float32 moments.
        steps: the step number of every tensor, counted from 1, or one number for all.
        masters: float32 master weights of 16-bit parameters; the step is then taken on them and the
            parameters receive rounded copies.
        grad_scale: one float32 value on the device that every gradient is multiplied by (``grad_norm``
            returns one). When it is not finite nothing is changed.
    """
    get_backend().adamw_step(params, grads, exp_avgs, exp_avg_sqs, steps, lr, weight_decay, betas, eps, masters,
                             grad_scale)


def adamw8_step(params: Sequence[Tensor], grads: Sequence[Tensor], exp_avg_codes: Sequence[Tensor],
                exp_avg_scales: Sequence[Tensor], exp_avg_sq_codes: Sequence[Tensor],
                exp_avg_sq_scales: Sequence[Tensor], steps, *, lr: float = 1e-3,
                betas: tuple[float, float] = (0.9, 0.999), eps: float = 1e-8, weight_decay: float = 1e-2,
                masters: Sequence[Tensor] | None = None, grad_scale: Tensor | None = None, seed: int = 0) -> None:
    """``adamw_step`` with moments in 8 bits: for a tensor of n elements n uint8 codes per moment and
    ceil(n / 256) float32 scales. New state is all zeros. The parameters move by the unrounded moments
    of the step; the second moment is then rounded stochastically by a hash of ``seed``, step and element
    index (the same call gives the same result). ``eps`` must be at least 1e-16."""
    get_backend().adamw8_step(params, grads, exp_avg_codes, exp_avg_scales, exp_avg_sq_codes, exp_avg_sq_scales, steps,
                              lr, weight_decay, betas, eps, masters, grad_scale, seed)


def _gradients(tensors) -> list[Tensor]:
    """The gradients of parameters (those that have one), or the tensors themselves."""
    return gradients([tensors] if isinstance(tensors, Tensor) else tensors)


def grad_norm(tensors, max_norm: float = math.inf) -> tuple[Tensor, Tensor]:
    """2-norm of all elements of ``tensors`` (gradients, or parameters, meaning their ``.grad``)
    together, and the factor min(1, max_norm / (norm + 1e-6)) that brings it down to ``max_norm``: two
    float32 values on the device, without a synchronisation. Given to ``adamw_step`` or ``adamw8_step`` as
    ``grad_scale`` the factor clips the gradients without a pass of its own. It is NaN when the norm is
    not finite, which makes those calls change nothing. Tensors of different types may be mixed; all
    are on one device."""
    tensors = _gradients(tensors)
    if not tensors:
        return torch.zeros(()), torch.ones(())
    return get_backend().grad_norm(tensors, max_norm, clip=False).unbind()


def clip_grad_norm_(tensors, max_norm: float) -> Tensor:
    """Scale gradients in place so that their 2-norm together is at most ``max_norm`` (as
    ``torch.nn.utils.clip_grad_norm_`` does): gradients, or parameters, meaning their ``.grad``. Returns the norm
    before, on the device. Gradients whose norm is small enough are not written."""
    tensors = _gradients(tensors)
    if not tensors:
        return torch.zeros(())
    return get_backend().grad_norm(tensors, max_norm, clip=True)[0]


def _check_kind(kind: str) -> None:
    if kind not in _STATE_KINDS:
        raise ValueError(f"unknown kind of state {kind!r}; expected one of {sorted(_STATE_KINDS)}")


def quantize_state(tensors: Sequence[Tensor], kind: str, *, codes: Sequence[Tensor] | None = None,
                   scales: Sequence[Tensor] | None = None) -> tuple[Sequence[Tensor], Sequence[Tensor]]:
    """Moments (``kind``: "exp_avg" or "exp_avg_sq") as 8-bit codes and scales, rounded to nearest, into
    ``codes`` and ``scales`` or into new tensors. Values of "exp_avg_sq" must not be negative."""
    _check_kind(kind)
    if codes is None:
        codes = [torch.empty_like(t, dtype=torch.uint8) for t in tensors]
    if scales is None:
        scales = [torch.empty(-(-t.numel() // STATE_BLOCK), dtype=torch.float32, device=t.device) for t in tensors]
    get_backend().convert_state("quantize_state", tensors, codes, scales, kind, True)
    return codes, scales


def dequantize_state(codes: Sequence[Tensor], scales: Sequence[Tensor], kind: str, *,
                     dtype: torch.dtype = torch.float32, out: Sequence[Tensor] | None = None) -> Sequence[Tensor]:
    """What the codes and scales of 8-bit moments stand for, as tensors of ``dtype``, or in ``out``."""
    _check_kind(kind)
    if out is None:
        out = [torch.empty_like(c, dtype=dtype) for c in codes]
    get_backend().convert_state("dequantize_state", out, codes, scales, kind, False)
    return out
