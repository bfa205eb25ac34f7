"""CPU tests of the AdamW operators: the oracle's 8-bit format against its definition, the
refusals of the C entry points (which come before anything is launched) and of the Python ones."""
import ctypes
import math
from array import array

import pytest
import torch

from oracle import adamw_oracle as orc


def test_code_tables():
    sq = orc.code_values("exp_avg_sq")
    assert (sq[1:] > sq[:-1]).all() and float(sq[0]) == 2.0 ** -31 and float(sq[255]) == 1.875
    avg = orc.code_values("exp_avg")
    want = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    assert torch.equal(avg.nan_to_num(nan=-1e9), want.nan_to_num(nan=-1e9))


@pytest.mark.parametrize("kind", ["exp_avg", "exp_avg_sq"])
def test_oracle_codes_are_the_nearest(kind):
    """By search over all codes, in 64 bits: no other code is nearer than the one chosen."""
    gen = torch.Generator().manual_seed(0)
    x = torch.randn(5000, generator=gen) * torch.exp(4 * torch.randn(5000, generator=gen))
    x = x.abs() if kind == "exp_avg_sq" else x
    codes, scales = orc.quantize(x, kind)
    s = scales.repeat_interleave(256)[:5000].double()
    values = orc.code_values(kind)[:255 if kind == "exp_avg" else 256]
    values = values[~values.isnan()]
    best = (x.double()[:, None] - values[None, :] * s[:, None]).abs().amin(dim=1)
    got = (x.double() - orc.code_values(kind)[codes.long()] * s).abs()
    assert (got <= best + 1e-6 * x.double().abs()).all()
    again, _ = orc.quantize(orc.dequantize(codes, scales, kind), kind)
    assert (again.int() - codes.int()).abs().max() <= (1 if kind == "exp_avg_sq" else 128)


def test_oracle_steps_are_cut_at_the_random_bits():
    x = torch.full((256,), 1.0101)
    x[0] = 1.875
    values = orc.code_values("exp_avg_sq")
    below, above = 1.0, 1.125
    part = (float(x[1]) - below) / (above - below)
    for r, up in ((0, False), (int((1 - part) * 2 ** 20) - 2, False), (int((1 - part) * 2 ** 20) + 2, True), (2 ** 20 - 1, True)):
        codes, _ = orc.quantize(x, "exp_avg_sq", torch.full((256,), r))
        assert float(values[codes[1].long()]) == (above if up else below)


def test_random_bits_are_uniform_and_uncorrelated():
    n = 1 << 20
    r = orc.random_bits(n, 123, 7).double() / 2 ** 20
    se = 6 / math.sqrt(12 * n)  # six standard errors of a uniform mean
    assert abs(float(r.mean()) - 0.5) <= se
    for other in (orc.random_bits(n, 123, 8), orc.random_bits(n, 124, 7)):
        o = other.double() / 2 ** 20
        assert abs(float(((o - 0.5) * (r - 0.5)).mean()) * 12) <= 6 / math.sqrt(n)
    for lag in (2, 3, 4, 8, 256):
        assert abs(float(((r[lag:] - 0.5) * (r[:-lag] - 0.5)).mean()) * 12) <= 6 / math.sqrt(n - lag)


def _call(name, *tables_then_scalars):
    import muon_b200._lib as L
    keep = [L.address(x) if isinstance(x, array) else x for x in tables_then_scalars]
    rc = getattr(L.lib, name)(*keep)
    return rc, L.lib.muon_b200_last_error().decode()


def test_c_refusals_come_before_a_launch():
    """Addresses here are made up: an accepted call would end at the device check without a GPU, and none
    of these is accepted."""
    a, n, one = array("Q", [4096]), array("q", [8]), array("q", [1])
    zero, odd = array("Q", [0]), array("Q", [4097])
    hyper = (1e-3, 0.0, 0.9, 0.999, 1e-8)
    adamw = lambda p=a, w=None, g=a, m=a, v=a, n=n, s=one, c=1, pd=0, gd=0, h=hyper, f=None: _call(  # noqa: E731
        "muon_b200_adamw", p, w, g, m, v, n, s, c, pd, gd, *h, f, None)
    cases = [
        (adamw(p=None), -1, "parameter is NULL"), (adamw(p=zero), -1, "null parameter"),
        (adamw(g=zero), -1, "null gradient"), (adamw(m=zero), -1, "null exp_avg"), (adamw(v=zero), -1, "null exp_avg_sq"),
        (adamw(m=odd), -2, "exp_avg of tensor 0"), (adamw(p=odd), -2, "parameter of tensor 0"),
        (adamw(n=array("q", [-1])), -1, "elements"), (adamw(n=array("q", [1 << 41])), -1, "elements"),
        (adamw(n=None), -1, "numel"), (adamw(s=None), -1, "steps"), (adamw(s=array("q", [0])), -1, "count from 1"),
        (adamw(c=-1), -1, "count"), (adamw(pd=3), -1, "dtype"), (adamw(gd=1), -1, "gradients"),
        (adamw(w=a), -1, "master"), (adamw(pd=1, gd=1, w=zero), -1, "null master"),
        (adamw(h=(1e-3, 0.0, 1.0, 0.999, 1e-8)), -1, "betas"), (adamw(h=(1e-3, 0.0, 0.9, float("nan"), 1e-8)), -1, "betas"),
        (adamw(h=(1e-3, 0.0, 0.9, 0.999, -1.0)), -1, "eps"), (adamw(f=2), -2, "grad_scale"),
    ]
    a8 = lambda c=a, s=a, h=hyper: _call("muon_b200_adamw8", a, None, a, c, s, c, s, n, one, 1, 0, 0, *h, 0, None, None)  # noqa: E731
    cases += [(a8(c=zero), -1, "code"), (a8(s=zero), -1, "scale"), (a8(s=odd), -2, "scale"),
              (a8(h=(1e-3, 0.0, 0.9, 0.999, 1e-17)), -1, "eps")]
    norm = lambda t=a, n=n, d=array("i", [0]), m=1.0, o=4096, s=4096, b=1 << 30: _call(  # noqa: E731
        "muon_b200_grad_norm", t, n, d, 1, m, o, s, b, None)
    cases += [(norm(t=None), -1, "NULL"), (norm(t=zero), -1, "null"), (norm(d=None), -1, "dtypes"),
              (norm(d=array("i", [3])), -1, "dtype"), (norm(m=-1.0), -1, "max_norm"), (norm(m=float("nan")), -1, "max_norm"),
              (norm(o=0), -1, "output"), (norm(s=0), -1, "scratch"), (norm(s=4100), -2, "scratch"), (norm(t=array("Q", [4098])), -2, "aligned")]
    conv = lambda x=a, c=a, s=a, dt=0, k=0: _call("muon_b200_quantize_state", x, c, s, n, 1, dt, k, None)  # noqa: E731
    cases += [(conv(k=2), -1, "kind"), (conv(dt=3), -1, "dtype"), (conv(c=zero), -1, "code"), (conv(s=zero), -1, "scale"),
              (conv(x=zero), -1, "tensor")]
    for k, ((rc, text), code, match) in enumerate(cases):
        assert rc == code and match in text, f"case {k}: {rc} {text!r}"
    assert adamw(c=0, p=None, g=None, m=None, v=None, n=None, s=None)[0] == 0  # nothing to do


def test_no_cpu_fallback():
    import muon_b200 as mb
    x = lambda: [torch.zeros(4)]  # noqa: E731
    u = lambda: [torch.zeros(4, dtype=torch.uint8)]  # noqa: E731
    for call in (lambda: mb.adamw_step(x(), x(), x(), x(), 1), lambda: mb.grad_norm(x()), lambda: mb.clip_grad_norm_(x(), 1.0),
                 lambda: mb.adamw8_step(x(), x(), u(), [torch.zeros(1)], u(), [torch.zeros(1)], 1),
                 lambda: mb.quantize_state(x(), "exp_avg"), lambda: mb.dequantize_state(u(), [torch.zeros(1)], "exp_avg")):
        with pytest.raises(RuntimeError, match="no CPU implementation"):
            call()


def test_pointer_tables_refuse_what_is_no_cuda_tensor():
    from muon_b200._tables import collect
    with pytest.raises(RuntimeError, match="every gradient tensor of grad_norm .* no CPU implementation"):
        collect("grad_norm", (("gradient", [torch.zeros(3)], 7, 0, False),))
    for bad in ([1], [None], [[torch.zeros(1)]]):
        with pytest.raises(TypeError, match="is no tensor"):
            collect("grad_norm", (("gradient", bad, 7, 0, False),))
    with pytest.raises(TypeError):
        collect("grad_norm", (("gradient", 5, 7, 0, False),))
    device, numel, tables, found, codes = collect("grad_norm", (("gradient", [], 7, 0, False),))
    assert (device, numel, tables, found, codes) == (-1, b"", (b"",), (0,), b"")
