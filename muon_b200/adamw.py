"""AdamW over many tensors at once, for the parameters that Muon does not suit (embeddings, heads,
gains, biases) or for a whole model, with moments in 32 or in 8 bits, and the global gradient norm that
goes before a step of any optimizer class.

The reference's Adam (muon.py:104-109) keeps its moments in the parameter's type; that arithmetic stays
in ``adam_update`` and in the classes' auxiliary Adam. Here moments are float32, or 8-bit codes with
one float32 scale per 256 elements whatever the parameter's type, the arithmetic is float32, and
one launch takes hundreds of tensors. The formats are described in ``include/muon_b200.h``."""
from __future__ import annotations

import math
from collections import OrderedDict
from typing import Sequence

import torch
from torch import Tensor

from ._lib import STATE_BLOCK
from ._tables import gradients
from .engine import _STATE_KINDS, get_backend, local_part, wait_for_mark


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

    No tensor that is written may share memory with another one of the call (a ValueError); gradients may with
    each other.
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
    """The gradients of parameters (those that have one; a plain leaf that requires gradients is a parameter too),
    or the tensors themselves."""
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
    return get_backend().grad_norm(tensors, max_norm, clip=False)


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


# ---- moments of a parameter as optimizer state -----------------------------------------------
# {"step", "moment_bits": 32, "exp_avg", "exp_avg_sq"} or {"step", "moment_bits": 8, "exp_avg_codes",
# "exp_avg_scales", "exp_avg_sq_codes", "exp_avg_sq_scales"}, with "master" where master weights are kept.
_MOMENT_KEYS = {32: ("exp_avg", "exp_avg_sq"),
                8: ("exp_avg_codes", "exp_avg_scales", "exp_avg_sq_codes", "exp_avg_sq_scales")}
_MIN_8BIT_NUMEL = 4096

_adam_moments = "param"


def set_adam_moments(kind: str = "param") -> None:
    """What the auxiliary Adam of ``MuonWithAuxAdam`` and ``SingleDeviceMuonWithAuxAdam`` keeps its
    moments in, for parameters whose state is created from now on. ``"param"`` (default): the parameter's
    type, with the reference's arithmetic (muon.py:104-109); ``"fp32"``: float32; ``"8bit"``: 8 bits,
    float32 for parameters of fewer than 4096 elements. The last two run ``adamw_step`` and
    ``adamw8_step``. (Not a param-group key: the reference asserts the exact key set, muon.py:155.)"""
    if kind not in ("param", "fp32", "8bit"):
        raise ValueError(f"unknown kind of moments {kind!r}; expected 'param', 'fp32' or '8bit'")
    global _adam_moments
    _adam_moments = kind


def get_adam_moments() -> str:
    return _adam_moments


def new_moments(state: dict, p: Tensor, bits: int, master: bool = False) -> None:
    """Fill an empty ``state`` with zero moments for ``p``."""
    state["step"] = 0
    state["moment_bits"] = bits
    for key in _MOMENT_KEYS[bits]:
        if key.endswith("_scales"):
            state[key] = torch.zeros(-(-p.numel() // STATE_BLOCK), dtype=torch.float32, device=p.device)
        else:
            state[key] = torch.zeros_like(p, dtype=torch.uint8 if bits == 8 else torch.float32,
                                          memory_format=torch.preserve_format)
    if master:
        state["master"] = _master_of(p)


def _master_of(p: Tensor) -> Tensor:
    return p.detach().to(torch.float32, copy=True, memory_format=torch.preserve_format)


def _same_order(a: Tensor, b: Tensor) -> bool:
    """Whether two tensors of one shape have their elements in the same order (dimensions of size 1 have none)."""
    return all(n == 1 or s == t for n, s, t in zip(a.shape, a.stride(), b.stride()))


def in_order_of(g: Tensor, p: Tensor) -> Tensor:
    """The gradient, or a copy of it with its elements in the order of its parameter's."""
    if g.stride() == p.stride() or _same_order(g, p):
        return g
    wait_for_mark(g)
    return torch.empty_like(p, dtype=g.dtype, memory_format=torch.preserve_format).copy_(g)


def moments_step(entries, lr: float, weight_decay: float, betas: tuple[float, float], eps: float,
                 grad_scale: Tensor | None = None, seed: int = 0) -> None:
    """One step for a list of (parameter, gradient in its order, state), state as ``new_moments`` lays it out: one
    call per combination of types and device. A state's step is counted when its call has been made."""
    kinds: "OrderedDict[tuple, list]" = OrderedDict()
    for p, g, state in entries:
        kinds.setdefault((p.dtype, g.dtype, p.device, state["moment_bits"], "master" in state), []).append((p, g, state))
    for (_, _, _, bits, master), members in kinds.items():
        states = [state for _, _, state in members]
        steps = [state["step"] + 1 for state in states]
        lists = [[state[key] for state in states] for key in _MOMENT_KEYS[bits]]
        more = dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, grad_scale=grad_scale,
                    masters=[state["master"] for state in states] if master else None)
        if bits == 8:
            more["seed"] = seed
        (adamw8_step if bits == 8 else adamw_step)([p for p, _, _ in members], [g for _, g, _ in members], *lists,
                                                   steps, **more)
        for state, now in zip(states, steps):
            state["step"] = now


def convert_moments(states: Sequence[dict], bits: int) -> None:
    """Turn the moments of these states into float32 or 8-bit ones."""
    states = [state for state in states if state["moment_bits"] != bits]
    by_device: dict = {}
    for state in states:
        by_device.setdefault(state[_MOMENT_KEYS[state["moment_bits"]][0]].device, []).append(state)
    for members in by_device.values():
        for kind in ("exp_avg", "exp_avg_sq"):
            if bits == 8:
                codes, scales = quantize_state([state[kind] for state in members], kind)
                new = [{f"{kind}_codes": c, f"{kind}_scales": s} for c, s in zip(codes, scales)]
            else:
                values = dequantize_state([state[f"{kind}_codes"] for state in members],
                                          [state[f"{kind}_scales"] for state in members], kind)
                new = [{kind: x} for x in values]
            for state, tensors in zip(members, new):
                state.update(tensors)
    for state in states:
        for key in _MOMENT_KEYS[state["moment_bits"]]:
            del state[key]
        state["moment_bits"] = bits


def restore_moments(p: Tensor, saved: dict) -> dict:
    """The tensors of a saved state for parameter ``p``, on its device, in the types they were saved in.
    (``torch.optim.Optimizer.load_state_dict`` casts every tensor to the parameter's type.) Moments of
    a parameter whose dimensions lie in another order in memory than when they were saved are
    brought into its order."""
    keep = {k: v.detach().to(p.device, copy=True) for k, v in saved.items() if torch.is_tensor(v)}
    laid_out = keep["exp_avg_codes" if saved["moment_bits"] == 8 else "exp_avg"]
    if laid_out.shape != p.shape:
        raise ValueError(f"moments of shape {tuple(laid_out.shape)} for a parameter of shape {tuple(p.shape)}")
    if _same_order(laid_out, p):
        return keep
    state = {"moment_bits": saved["moment_bits"], **keep}
    convert_moments([state], 32)
    for key in ("exp_avg", "exp_avg_sq", "master"):
        if key in state:
            state[key] = torch.empty_like(p, dtype=torch.float32, memory_format=torch.preserve_format).copy_(state[key])
    convert_moments([state], saved["moment_bits"])
    return {k: v for k, v in state.items() if torch.is_tensor(v)}


class KeepsMomentTypes:
    """``load_state_dict`` for optimizers whose state may hold ``new_moments``."""

    def load_state_dict(self, state_dict):
        super().load_state_dict(state_dict)
        ids = [i for group in state_dict["param_groups"] for i in group["params"]]
        for i, p in zip(ids, (p for group in self.param_groups for p in group["params"])):
            saved = state_dict["state"].get(i, {})
            if "moment_bits" in saved:
                self.state[p].update(restore_moments(local_part(p), saved))


# what a group of another Adam holds and AdamW has no use for
_FOREIGN_KEYS = {"amsgrad", "maximize", "foreach", "capturable", "differentiable", "fused", "decoupled_weight_decay", "use_muon"}


def _adopted(state_dict: dict, param_groups: list[dict]) -> dict:
    """The state dictionary of another Adam with decoupled decay as one of ``AdamW`` with float32 moments."""
    groups, states = [], {}
    for saved, mine in zip(state_dict["param_groups"], param_groups):
        missing = {"lr", "betas", "eps", "weight_decay"} - set(saved)
        if missing:
            raise ValueError(f"not the state of an AdamW: a group without {sorted(missing)}")
        for key in ("amsgrad", "maximize"):
            if saved.get(key):
                raise ValueError(f"AdamW does not take over a run with {key}")
        if not saved.get("decoupled_weight_decay", True) and saved["weight_decay"] != 0:
            raise ValueError("AdamW does not take over a run whose weight decay is not decoupled (torch.optim.Adam)")
        groups.append({**{k: v for k, v in mine.items() if k != "params"},
                       **{k: v for k, v in saved.items() if k not in _FOREIGN_KEYS}})
        for i in saved["params"]:
            if i in state_dict["state"]:
                states[i] = _adopted_state(state_dict["state"][i])
    return {**state_dict, "param_groups": groups + list(state_dict["param_groups"][len(groups):]), "state": states}


def _adopted_state(saved: dict) -> dict:
    if not saved or "moment_bits" in saved:
        return saved
    if set(saved) != {"step", "exp_avg", "exp_avg_sq"}:
        raise ValueError(f"not the state of an AdamW: {sorted(saved)}")
    return {"step": int(saved["step"]), "moment_bits": 32,
            **{key: local_part(saved[key]).detach().to(torch.float32) for key in ("exp_avg", "exp_avg_sq")}}


class AdamW(KeepsMomentTypes, torch.optim.Optimizer):
    """AdamW (decoupled weight decay) with one launch for all parameters of a type.

    Arguments:
        params, lr, betas, eps, weight_decay: as for ``torch.optim.AdamW``; parameters are float32,
            bfloat16 or float16. Parameters without a gradient are left as they are. Of a DTensor (sharded
            or replicated) the local part is updated and has its own moments.
        state_bits: 32 (float32 moments whatever the parameter's type) or 8.
        master_weights: keep a float32 copy of 16-bit parameters, which the steps are taken on.
        min_8bit_numel: parameters with fewer elements keep float32 moments.
        seed: of the stochastic rounding of 8-bit second moments.
        max_grad_norm: clip the gradients of all groups together to this norm. The factor stays on the
            device and is applied while the step reads the gradients; ``grad_norm`` holds the norm
            of the last step. A step whose norm is not finite changes nothing (it is counted).

    ``state_bits``, ``master_weights``, ``min_8bit_numel`` and ``seed`` may differ between groups. Steps are
    counted on the host, so ``step()`` cannot be captured into a CUDA graph (``adamw_step`` can)."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, *, state_bits=32,
                 master_weights=False, min_8bit_numel=_MIN_8BIT_NUMEL, seed=0, max_grad_norm=None):
        if max_grad_norm is not None and not max_grad_norm >= 0:
            raise ValueError(f"max_grad_norm must not be negative, got {max_grad_norm}")
        self.max_grad_norm = max_grad_norm
        self.grad_norm = None
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, state_bits=state_bits,
                                      master_weights=master_weights, min_8bit_numel=min_8bit_numel, seed=seed))

    def __getstate__(self):  # (torch's holds defaults, state and groups only)
        return {**super().__getstate__(), "max_grad_norm": self.max_grad_norm, "grad_norm": self.grad_norm}

    def __setstate__(self, state):  # (torch's load_state_dict passes state and groups only)
        super().__setstate__(state)
        self.__dict__.setdefault("max_grad_norm", None)
        self.__dict__.setdefault("grad_norm", None)

    def load_state_dict(self, state_dict):
        """State of this class is loaded as it was saved. That of ``torch.optim.AdamW`` (or of an Adam group of
        ``MuonWithAuxAdam``) is turned into this optimizer's: hyper-parameters from the dictionary,
        ``state_bits``, ``master_weights`` and ``seed`` from here. What has another meaning (AMSGrad, maximizing, a
        decay that is not decoupled, another optimizer's state) is refused."""
        own = all("state_bits" in group for group in state_dict["param_groups"])
        super().load_state_dict(state_dict if own else _adopted(state_dict, self.param_groups))
        if own:
            return
        for group in self.param_groups:
            held = [(p, self.state[p]) for p in group["params"] if self.state.get(p)]
            for p, state in held:
                local = local_part(p)
                if group["master_weights"] and local.dtype != torch.float32 and "master" not in state:
                    state["master"] = _master_of(local)
            if group["state_bits"] == 8:
                convert_moments([state for p, state in held if local_part(p).numel() >= group["min_8bit_numel"]], 8)

    def add_param_group(self, param_group):
        super().add_param_group(param_group)
        group = self.param_groups[-1]
        if group["state_bits"] not in (8, 32):
            self.param_groups.pop()
            raise ValueError(f"state_bits must be 8 or 32, got {group['state_bits']}")

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        if torch.cuda.is_available() and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("AdamW counts its steps on the host: a captured step would repeat one step number; "
                               "capture adamw_step or adamw8_step instead")
        work = []  # (group, [(parameter, gradient, state)])
        sharded = False
        for group in self.param_groups:
            entries = []
            for p in group["params"]:
                g, local = p.grad, local_part(p)
                if g is None:
                    continue
                if local is not p:
                    sharded = True
                    if g.placements != p.placements:  # one that is not reduced yet, say
                        wait_for_mark(g)
                        g = g.redistribute(placements=p.placements)
                    g = g.to_local()
                entries.append((local, in_order_of(g, local), self.state[p]))
            if entries:
                work.append((group, entries))
        if not work:
            return loss
        factor = None
        if self.max_grad_norm is not None:
            if sharded:
                raise ValueError("max_grad_norm needs whole gradients: clip sharded ones before step() "
                                 "(torch.nn.utils.clip_grad_norm_ takes DTensors)")
            self.grad_norm, factor = grad_norm([g for _, entries in work for _, g, _ in entries], self.max_grad_norm)
        for group, entries in work:
            for local, _, state in entries:
                if len(state) == 0:
                    bits = 8 if group["state_bits"] == 8 and local.numel() >= group["min_8bit_numel"] else 32
                    new_moments(state, local, bits, group["master_weights"] and local.dtype != torch.float32)
            moments_step(entries, float(group["lr"]), float(group["weight_decay"]), tuple(map(float, group["betas"])),
                         float(group["eps"]), factor, int(group["seed"]))
        return loss

    @torch.no_grad()
    def set_state_bits(self, bits: int) -> None:
        """Convert the moments of all parameters, and those still to come, to 8 or 32 bits (a run that
        goes on with another size of state, a checkpoint that was saved with one). To 8 bits: those of
        parameters with at least ``min_8bit_numel`` elements."""
        if bits not in (8, 32):
            raise ValueError(f"state_bits must be 8 or 32, got {bits}")
        for group in self.param_groups:
            group["state_bits"] = bits
            convert_moments([self.state[p] for p in group["params"] if len(self.state.get(p, {})) > 0
                             and (bits == 32 or local_part(p).numel() >= group["min_8bit_numel"])], bits)
