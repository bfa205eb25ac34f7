"""AdamW with 32-bit and 8-bit moments on the CPU: the formulas in 64 bits, and the 8-bit format by
its definition (value tables and searches, no bit arithmetic of the kernels' kind) and, for the codes
of a step, by the float32 operations that the format prescribes."""
from __future__ import annotations

import torch

BLOCK = 256
TOP = {"exp_avg": 448.0, "exp_avg_sq": 1.875}
TINY = {"exp_avg": 2.0 ** -110, "exp_avg_sq": 2.0 ** -120}


def code_values(kind: str) -> torch.Tensor:
    """What each of the 256 codes stands for, in units of the scale, float64."""
    c = torch.arange(256, dtype=torch.float64)
    if kind == "exp_avg_sq":
        return 2.0 ** ((c // 8) - 31) * (1 + (c % 8) / 8)
    sign = torch.where(c >= 128, -1.0, 1.0).double()
    c = c % 128
    exponent, mantissa = c // 8, c % 8
    value = torch.where(exponent == 0, mantissa / 8 * 2.0 ** -6, (1 + mantissa / 8) * 2.0 ** (exponent - 7))
    value[c == 127] = float("nan")
    return sign * value


def rows(x: torch.Tensor) -> torch.Tensor:
    """A flattened tensor as rows of BLOCK, the last one filled up with zeros."""
    x = x.reshape(-1)
    return torch.nn.functional.pad(x, (0, -x.numel() % BLOCK)).view(-1, BLOCK)


def dequantize(codes: torch.Tensor, scales: torch.Tensor, kind: str) -> torch.Tensor:
    """float32 values, flat: one rounding of code value times scale."""
    value = code_values(kind)[codes.reshape(-1).long()].float()
    return value * scales.repeat_interleave(BLOCK)[:codes.numel()]


def quantize(x: torch.Tensor, kind: str, bits=None):
    """Float32 values -> (uint8 codes, float32 scales). bits: the 20 random bits of every element
    ("exp_avg_sq" of a step); None: to nearest. The scale and the scaled value are float32 operations
    with one rounding each, as the format says; the code is then found in 64 bits."""
    n = x.numel()
    r = rows(x.float())
    top = torch.tensor(TOP[kind])
    amax = r.abs().amax(dim=1)
    tiny = amax < TINY[kind]
    scales = torch.where(tiny, torch.zeros(()), amax * (1.0 / top))
    factor = torch.where(tiny, torch.zeros(()), top / amax)
    y = (r * factor[:, None]).reshape(-1)[:n].double()
    values = code_values(kind)
    if kind == "exp_avg":
        positive = values[:127].contiguous()
        a = y.abs().clamp(max=448.0)
        hi = torch.searchsorted(positive, a).clamp(max=126)
        lo = (hi - 1).clamp(min=0)
        below, above = a - positive[lo], positive[hi] - a
        pick_hi = (above < below) | ((above == below) & (hi % 2 == 0))
        codes = torch.where(pick_hi, hi, lo)
        codes = torch.where(codes == 0, codes, codes + 128 * (y < 0))  # (a zero's sign is not compared)
        codes = torch.where(torch.isnan(y), torch.full_like(codes, 127), codes)
    else:
        u = torch.full((n,), 0.5, dtype=torch.float64) if bits is None else bits.double() / 2 ** 20
        lo = (torch.searchsorted(values, y, right=True) - 1).clamp(0, 255)
        width = 2.0 ** ((lo // 8).double() - 31) / 8  # between this code and the next
        codes = torch.floor(lo + (y - values[lo]) / width + u).clamp(0, 255)
        codes = torch.where(y < values[0], torch.zeros_like(codes), codes).long()  # 0 is the smallest, for 0 too
        codes = torch.where(torch.isnan(y), torch.full_like(codes, 255), codes)
    tiny_elem = tiny.repeat_interleave(BLOCK)[:n]
    codes = torch.where(tiny_elem, torch.zeros_like(codes), codes)
    return codes.to(torch.uint8), scales


def random_bits(n: int, seed: int, step: int) -> torch.Tensor:
    """The 20 random bits of elements 0 .. n-1 of a tensor."""
    return random_bits_at(torch.arange(n, dtype=torch.int64), seed, step)


def random_bits_at(i: torch.Tensor, seed: int, step: int) -> torch.Tensor:
    """The same for the elements of these indexes (32-bit arithmetic in Python integers for the key, in
    int64 tensors for the rest)."""
    mod = 1 << 32
    key = (seed * 0x3C6EF373 + step * 0xBB67AE85) % mod
    h = ((i // 4) * 0x9E3779B1 + key) % mod
    h = ((h ^ (h >> 16)) * 0x6A09E667) % mod
    h = ((h ^ (h >> 15)) * 0xBB67AE85) % mod
    h = h ^ (h >> 16)
    turn = 8 * (i % 4)
    return ((h >> turn) | (h << (32 - turn))) % (1 << 20)


def adamw64(p, g, m, v, step, lr, betas, eps, weight_decay, factor=1.0):
    """(p, m, v) after a step, all float64."""
    p, g, m, v = p.double(), g.double() * factor, m.double(), v.double()
    m = betas[0] * m + (1 - betas[0]) * g
    v = betas[1] * v + (1 - betas[1]) * g * g
    hat = (m / (1 - betas[0] ** step)) / ((v / (1 - betas[1] ** step)).sqrt() + eps)
    return p - lr * weight_decay * p - lr * hat, m, v


def moments32(g, m, v, betas, factor=1.0):
    """New moments by single float32 operations, in the order the 8-bit format prescribes."""
    f32 = lambda x: torch.tensor(x, dtype=torch.float32)  # noqa: E731
    g = g.float() * f32(factor)
    m = m.float() * f32(betas[0]) + g * f32(1 - betas[0])
    v = v.float() * f32(betas[1]) + (g * g) * f32(1 - betas[1])
    return m, v


def adamw_tolerance(p, g, m, v, step, lr, betas, eps, weight_decay, factor=1.0):
    """Bounds on |p|, |m|, |v| errors of one float32 step (before p is rounded to its type), from the
    roundings that are made: u = 2^-24 is half a step of float32.
    m: factor, g f, two constants, product, fused sum: 5 u (|b1 m| + |w1 g|).
    v: the same and a square, twice the relative error of g: 7 u v (no cancellation).
    p: decay constant and product and the last sum: 3 u (|p| + |update|); the update: m's error, v's
    halved by the root, root 2 u, its factor and eps and sum 4 u, quotient 4 u, step constant u."""
    u = 2.0 ** -24
    new_p, new_m, new_v = adamw64(p, g, m, v, step, lr, betas, eps, weight_decay, factor)
    g = g.double() * factor
    tol_m = 5 * u * (betas[0] * m.double().abs() + (1 - betas[0]) * g.abs())
    tol_v = 7 * u * new_v
    size = lr / (1 - betas[0] ** step) / ((new_v / (1 - betas[1] ** step)).sqrt() + eps)
    update = size * new_m.abs()
    tol_p = 3 * u * (p.double().abs() + update) + size * tol_m + update * 16 * u
    # products that fall under the smallest normal number lose up to 2^-149 each
    return tol_p + 1e-44, tol_m + 1e-44, tol_v + 4e-45
