"""AdamW with 32-bit and 8-bit moments, the gradient norm and the conversion of moments, on the GPU,
against the 64-bit formulas and the format's definition (oracle/adamw_oracle.py). Tolerances: see
adamw_tolerance; storing a value in T adds half a step, finfo(T).eps / 2 relative to it."""
import math

import pytest
import torch

from oracle import adamw_oracle as orc

pytestmark = pytest.mark.gpu

# empty, single, around a vector of 8, around a block of 256, around a chunk, several chunks and a rest
SIZES = [0, 1, 7, 8, 255, 256, 257, 513, 8192, 8197, 3 * 8192 + 77]
BETAS, EPS, LR, WD = (0.9, 0.999), 1e-8, 3e-4, 0.1
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


@pytest.fixture(scope="module")
def mb():
    import muon_b200
    return muon_b200


def _place(ts, dtype, offset, device="cuda"):
    """Copies on the device, each `offset` elements behind a 256-byte boundary."""
    out = []
    for t in ts:
        buf = torch.empty(t.numel() + offset, dtype=dtype, device=device)
        out.append(buf[offset:].view(t.shape) if t.numel() else buf[offset:])
        out[-1].copy_(t)
    return out


def _inputs(sizes, seed, dtype=torch.float32):
    gen = torch.Generator().manual_seed(seed)
    p = [(torch.randn(n, generator=gen) * 0.02).to(dtype) for n in sizes]
    g = [(torch.randn(n, generator=gen) * 1e-3 * torch.exp(torch.randn(n, generator=gen))).to(dtype) for n in sizes]
    m = [torch.randn(n, generator=gen) * 3e-4 for n in sizes]
    v = [torch.rand(n, generator=gen) * 1e-6 for n in sizes]
    return p, g, m, v


def _assert_close(got, want, tol, what):
    got, want = got.detach().cpu().double().reshape(-1), want.reshape(-1)
    bad = ~((got - want).abs() <= tol.reshape(-1))
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} outside, first at {int(bad.nonzero()[0])}: "
                           f"{got[bad][0]:.9g} for {want[bad][0]:.9g}, allowed {tol.reshape(-1)[bad][0]:.3g}")


def _half_step(x, dtype):
    if dtype == torch.float32:
        return torch.zeros_like(x)  # the last float32 rounding is in the tolerance already
    info = torch.finfo(dtype)
    return x.abs() * (info.eps / 2) + info.tiny * info.eps / 2


# parameter type, master weights, gradient type
_FORMS = [("fp32", False, "same")] + [(d, w, g) for d in ("bf16", "fp16") for w in (False, True) for g in ("same", "fp32")]


@pytest.mark.parametrize("times", [1, 7, 18], ids=["few", "some", "many"])  # each size of table
@pytest.mark.parametrize("offset", [0, 1], ids=["aligned", "odd"])
@pytest.mark.parametrize("dtype,master,grad", _FORMS, ids=["-".join((d, "master" if w else "plain", g)) for d, w, g in _FORMS])
def test_adamw_step(mb, dtype, master, grad, offset, times):
    t = DTYPES[dtype]
    sizes = SIZES * times
    p, g, m, v = _inputs(sizes, 1, t)
    if grad == "fp32":
        g = [x.float() * 1.001 for x in g]
    gen = torch.Generator().manual_seed(2)
    w = [x.float() + torch.randn(x.shape, generator=gen) * 1e-5 for x in p] if master else None
    steps = [1 + (7 * i) % 5 for i in range(len(p))]
    P, M, V = _place(p, t, offset), _place(m, torch.float32, offset), _place(v, torch.float32, offset)
    G = _place(g, g[0].dtype, offset)
    W = _place(w, torch.float32, offset) if master else None
    factor = torch.tensor(0.37, device="cuda")
    mb.adamw_step(P, G, M, V, steps, lr=LR, betas=BETAS, eps=EPS, weight_decay=WD, masters=W, grad_scale=factor)
    f = float(torch.tensor(0.37))  # the factor as float32
    for i, n in enumerate(sizes):
        args = ((w or p)[i], g[i], m[i], v[i], steps[i], LR, BETAS, EPS, WD, f)
        want = orc.adamw64(*args)
        tol = orc.adamw_tolerance(*args)
        _assert_close(M[i], want[1], tol[1], f"exp_avg {n}")
        _assert_close(V[i], want[2], tol[2], f"exp_avg_sq {n}")
        if master:
            _assert_close(W[i], want[0], tol[0], f"master {n}")
            assert torch.equal(P[i], W[i].to(t)), "the parameter is the rounded master"
        else:
            _assert_close(P[i], want[0], tol[0] + _half_step(want[0], t), f"parameter {n}")
        assert torch.equal(G[i].cpu(), g[i]), "gradients are only read"


def _state8(m, v, offset):
    """8-bit state of the moments m, v: on the device and as the oracle sees it."""
    host, dev = {}, {}
    for name, kind, x in (("m", "exp_avg", m), ("v", "exp_avg_sq", v)):
        pairs = [orc.quantize(t, kind) for t in x]
        host[name] = pairs
        dev[name] = _place([c for c, _ in pairs], torch.uint8, offset)
        dev[name + "s"] = _place([s for _, s in pairs], torch.float32, offset)
    return host, dev


def _check_codes(got_codes, got_scales, want, kind, what):
    codes, scales = want
    assert torch.equal(got_scales.cpu(), scales), f"{what}: scales"
    a, b = got_codes.cpu().reshape(-1), codes.reshape(-1)
    if kind == "exp_avg":  # +0 and -0 are one value
        a, b = torch.where(a == 128, 0, a.int()), torch.where(b == 128, 0, b.int())
    bad = a != b
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} codes differ, first at {int(bad.nonzero()[0])}"


@pytest.mark.parametrize("times", [1, 7, 18], ids=["few", "some", "many"])  # each size of table
@pytest.mark.parametrize("offset", [0, 1], ids=["aligned", "odd"])
@pytest.mark.parametrize("dtype,master,grad", _FORMS, ids=["-".join((d, "master" if w else "plain", g)) for d, w, g in _FORMS])
def test_adamw8_step(mb, dtype, master, grad, offset, times):
    """Two steps: every code and scale equal to the format's definition, parameters within the
    bounds of the float32 arithmetic."""
    t = DTYPES[dtype]
    sizes = SIZES * times
    p, _, m, v = _inputs(sizes, 3, t)
    host, dev = _state8(m, v, offset)
    P = _place(p, t, offset)
    w = [x.float() for x in p] if master else None
    W = _place(w, torch.float32, offset) if master else None
    seed = 0x12345678F
    for step in (41, 42):
        g = _inputs(sizes, 100 + step, t if grad == "same" else torch.float32)[1]
        G = _place(g, g[0].dtype, offset)
        before = [x.cpu().clone() for x in (W or P)]
        mb.adamw8_step(P, G, dev["m"], dev["ms"], dev["v"], dev["vs"], step, lr=LR, betas=BETAS, eps=EPS,
                       weight_decay=WD, masters=W, seed=seed)
        for i, n in enumerate(sizes):
            m0 = orc.dequantize(*host["m"][i], "exp_avg")
            v0 = orc.dequantize(*host["v"][i], "exp_avg_sq")
            m1, v1 = orc.moments32(g[i], m0, v0, BETAS)
            host["m"][i] = orc.quantize(m1, "exp_avg")
            host["v"][i] = orc.quantize(v1, "exp_avg_sq", orc.random_bits(n, seed & 0xFFFFFFFF, step))
            _check_codes(dev["m"][i], dev["ms"][i], host["m"][i], "exp_avg", f"step {step}, exp_avg {n}")
            _check_codes(dev["v"][i], dev["vs"][i], host["v"][i], "exp_avg_sq", f"step {step}, exp_avg_sq {n}")
            args = (before[i], g[i], m0, v0, step, LR, BETAS, EPS, WD)
            want, tol = orc.adamw64(*args)[0], orc.adamw_tolerance(*args)[0]
            if master:
                _assert_close(W[i], want, tol, f"master {n}")
                assert torch.equal(P[i], W[i].to(t))
            else:
                _assert_close(P[i], want, tol + _half_step(want, t), f"parameter {n}")


class _Guarded:
    """Copies on the device with 64 other elements on either side, `offset` elements behind a boundary."""

    def __init__(self, ts, dtype, offset):
        self.bufs = [torch.full((t.numel() + 128 + offset,), 77, dtype=dtype, device="cuda") for t in ts]
        self.views = [b[64 + offset:64 + offset + t.numel()] for b, t in zip(self.bufs, ts)]
        self.offset = offset
        for v, t in zip(self.views, ts):
            v.copy_(t)

    def intact(self):
        return all((b[:64 + self.offset] == 77).all() and (b[len(b) - 64:] == 77).all() for b in self.bufs)


@pytest.mark.parametrize("offsets", [(1, 3, 2, 5, 7), (7, 7, 7, 7, 7), (0, 0, 1, 0, 0), (4, 2, 8, 13, 3), (0, 5, 0, 0, 2)])
@pytest.mark.parametrize("master", [False, True], ids=["plain", "master"])
@pytest.mark.parametrize("dtype", list(DTYPES))
def test_lists_that_start_anywhere(mb, dtype, master, offsets):
    """Every list at another distance from a 16-byte boundary, both steps: results as defined, and nothing
    beside the tensors is touched."""
    t = DTYPES[dtype]
    if t == torch.float32 and master:
        pytest.skip("float32 parameters have no masters")
    sizes = [15, 256, 271, 272, 273, 512, 528, 530, 256 * 40 + 100, 20001]
    p, g, m, v = _inputs(sizes, 40, t)
    w = [x.float() for x in p] if master else None
    po, go, mo, vo, wo = offsets
    P, G = _Guarded(p, t, po), _Guarded(g, t, go)
    W = _Guarded(w, torch.float32, wo) if master else None
    # float32 moments
    M, V = _Guarded(m, torch.float32, mo), _Guarded(v, torch.float32, vo)
    mb.adamw_step(P.views, G.views, M.views, V.views, 9, lr=LR, betas=BETAS, eps=EPS, weight_decay=WD,
                  masters=W.views if master else None)
    for i, n in enumerate(sizes):
        args = ((w or p)[i], g[i], m[i], v[i], 9, LR, BETAS, EPS, WD)
        want, tol = orc.adamw64(*args), orc.adamw_tolerance(*args)
        _assert_close(M.views[i], want[1], tol[1], f"exp_avg {n}")
        _assert_close(V.views[i], want[2], tol[2], f"exp_avg_sq {n}")
        if master:
            _assert_close(W.views[i], want[0], tol[0], f"master {n}")
        _assert_close(P.views[i], want[0], tol[0] + _half_step(want[0], t) * (1 + 2.0 ** -20), f"parameter {n}")
    assert all(x.intact() for x in (P, G, M, V)) and (W is None or W.intact())
    # 8-bit moments
    pairs = {k: [orc.quantize(x, kind) for x in y] for k, kind, y in (("m", "exp_avg", m), ("v", "exp_avg_sq", v))}
    C = {k: _Guarded([c for c, _ in pairs[k]], torch.uint8, o) for k, o in (("m", mo), ("v", vo))}
    S = {k: _Guarded([s for _, s in pairs[k]], torch.float32, o) for k, o in (("m", vo), ("v", mo))}
    before = [x.cpu().clone() for x in (W or P).views]
    mb.adamw8_step(P.views, G.views, C["m"].views, S["m"].views, C["v"].views, S["v"].views, 9, lr=LR, betas=BETAS, eps=EPS,
                   weight_decay=WD, masters=W.views if master else None, seed=4)
    for i, n in enumerate(sizes):
        m0, v0 = orc.dequantize(*pairs["m"][i], "exp_avg"), orc.dequantize(*pairs["v"][i], "exp_avg_sq")
        m1, v1 = orc.moments32(g[i], m0, v0, BETAS)
        _check_codes(C["m"].views[i], S["m"].views[i], orc.quantize(m1, "exp_avg"), "exp_avg", f"exp_avg {n}")
        _check_codes(C["v"].views[i], S["v"].views[i], orc.quantize(v1, "exp_avg_sq", orc.random_bits(n, 4, 9)), "exp_avg_sq",
                     f"exp_avg_sq {n}")
        args = (before[i], g[i], m0, v0, 9, LR, BETAS, EPS, WD)
        want, tol = orc.adamw64(*args)[0], orc.adamw_tolerance(*args)[0]
        if master:
            _assert_close(W.views[i], want, tol, f"master {n}")
            assert torch.equal(P.views[i], W.views[i].to(t))
        else:
            _assert_close(P.views[i], want, tol + _half_step(want, t), f"parameter {n}")
    assert all(x.intact() for x in (P, G, C["m"], C["v"], S["m"], S["v"])) and (W is None or W.intact())
    # conversions and clipping
    X = _Guarded([x.abs() for x in v], t, po)
    mb.quantize_state(X.views, "exp_avg_sq", codes=C["v"].views, scales=S["v"].views)
    mb.dequantize_state(C["v"].views, S["v"].views, "exp_avg_sq", out=X.views)
    for i, n in enumerate(sizes):
        want = orc.quantize(v[i].abs().to(t), "exp_avg_sq")
        _check_codes(C["v"].views[i], S["v"].views[i], want, "exp_avg_sq", f"quantized {n}")
        assert torch.equal(X.views[i].cpu(), orc.dequantize(*want, "exp_avg_sq").to(t))
    norm, factor = mb.grad_norm(G.views, 1e-3)
    mb.clip_grad_norm_(G.views, 1e-3)
    assert all(torch.equal(a.cpu(), (b.float() * factor.cpu()).to(t)) for a, b in zip(G.views, g))
    assert all(x.intact() for x in (X, G, C["v"], S["v"]))


def test_adamw8_from_zero_state_and_zero_gradients(mb):
    """New state is all zeros; a block without gradients stays zero and its parameters only decay."""
    p = [torch.randn(1000), torch.randn(512)]
    g = [torch.zeros(1000), torch.randn(512) * 1e-3]
    g[0][256:512] = torch.randn(256) * 1e-3
    P, G = _place(p, torch.float32, 0), _place(g, torch.float32, 0)
    z = [torch.zeros(n, dtype=torch.uint8, device="cuda") for n in (1000, 512, 1000, 512)]
    s = [torch.zeros(n, device="cuda") for n in (4, 2, 4, 2)]
    mb.adamw8_step(P, G, z[:2], s[:2], z[2:], s[2:], 1, lr=LR, betas=BETAS, eps=EPS, weight_decay=WD)
    assert s[0].cpu().nonzero().flatten().tolist() == [1] and s[2].cpu().nonzero().flatten().tolist() == [1]
    decayed = p[0] * torch.tensor(1 - LR * WD, dtype=torch.float32)
    assert torch.equal(P[0].cpu()[:256], decayed[:256]) and torch.equal(P[0].cpu()[512:], decayed[512:])
    for i in (0, 1):
        args = (p[i], g[i], torch.zeros_like(p[i]), torch.zeros_like(p[i]), 1, LR, BETAS, EPS, WD)
        _assert_close(P[i], orc.adamw64(*args)[0], orc.adamw_tolerance(*args)[0], "parameter")


def test_adamw8_range_of_a_block(mb):
    """One block whose gradients differ by 2^40, one of subnormal size, one of huge size, one NaN, one inf:
    codes as defined, trouble stays in its block of 256."""
    n = 256 * 6
    gen = torch.Generator().manual_seed(5)
    g = torch.randn(n, generator=gen)
    g[:256] *= 2.0 ** -(torch.arange(256) % 41).float()
    g[256:512] *= 1e-38
    g[512:768] *= 1e17
    g[768 + 5] = float("nan")
    g[1024 + 9] = float("inf")
    p = torch.randn(n, generator=gen)
    P, G = _place([p], torch.float32, 0), _place([g], torch.float32, 0)
    z = [torch.zeros(n, dtype=torch.uint8, device="cuda") for _ in range(2)]
    s = [torch.zeros(6, device="cuda") for _ in range(2)]
    mb.adamw8_step(P, G, [z[0]], [s[0]], [z[1]], [s[1]], 3, lr=LR, betas=BETAS, eps=EPS, weight_decay=0.0, seed=7)
    m1, v1 = orc.moments32(g, torch.zeros(n), torch.zeros(n), BETAS)
    fine = torch.tensor([0, 1, 2, 5])
    for codes, scales, x, kind, bits in ((z[0], s[0], m1, "exp_avg", None),
                                         (z[1], s[1], v1, "exp_avg_sq", orc.random_bits(n, 7, 3))):
        want = orc.quantize(x, kind, bits)
        got = codes.cpu().view(6, 256)[fine], scales.cpu()[fine]
        _check_codes(got[0], got[1], (want[0].view(6, 256)[fine], want[1][fine]), kind, kind)
        assert not torch.isfinite(scales.cpu()[3:5]).any()
    assert torch.isfinite(P[0].cpu().view(6, 256)[fine]).all()
    one = P[0].cpu().view(6, 256)
    assert torch.isnan(one[3, 5]) and torch.isfinite(one[3, 6:]).all()  # this step: that element only


def test_factor_that_is_not_finite_changes_nothing(mb):
    for bad in (float("nan"), float("inf"), -float("inf")):
        p, g, m, v = (_place(x, torch.float32, 0) for x in _inputs([300, 5000], 6))
        keep = [[t.clone() for t in x] for x in (p, m, v)]
        f = torch.tensor(bad, device="cuda")
        mb.adamw_step(p, g, m, v, 1, grad_scale=f)
        for x, k in zip((p, m, v), keep):
            assert all(torch.equal(a, b) for a, b in zip(x, k))
        z = [torch.full((n,), 3, dtype=torch.uint8, device="cuda") for n in (300, 5000)]
        s = [torch.full((-(-n // 256),), 1e-3, device="cuda") for n in (300, 5000)]
        mb.adamw8_step(p, g, z, s, [t.clone() for t in z], [t.clone() for t in s], 1, grad_scale=f)
        assert all((t == 3).all() for t in z) and all((t == torch.tensor(1e-3)).all() for t in s)
        assert all(torch.equal(a, b) for a, b in zip(p, keep[0]))


def test_more_tensors_than_a_launch_holds(mb):
    """1500 small tensors: several launches, every tensor updated once, in any order of sizes."""
    sizes = [1 + (37 * i) % 700 for i in range(1500)]
    p, g, m, v = _inputs(sizes, 8)
    P, G, M, V = (_place(x, torch.float32, 0) for x in (p, g, m, v))
    mb.adamw_step(P, G, M, V, 5, lr=LR, betas=BETAS, eps=EPS, weight_decay=WD)
    cat = lambda x: torch.cat([t.detach().cpu().reshape(-1) for t in x])  # noqa: E731
    args = (cat(p), cat(g), cat(m), cat(v), 5, LR, BETAS, EPS, WD)
    want, tol = orc.adamw64(*args), orc.adamw_tolerance(*args)
    for got, w, t in zip((P, M, V), want, tol):
        _assert_close(cat(got), w, t, "1500 tensors")
    norm, factor = mb.grad_norm(G, 0.25)
    exact = float(cat(g).double().norm())
    assert abs(float(norm) - exact) <= 2e-7 * exact and abs(float(factor) - 0.25 / (exact + 1e-6)) <= 4e-7 * float(factor)
    codes, scales = mb.quantize_state(V, "exp_avg_sq")
    for i in (0, 700, 1499):
        _check_codes(codes[i], scales[i], orc.quantize(V[i].cpu(), "exp_avg_sq"), "exp_avg_sq", f"tensor {i}")


@pytest.mark.parametrize("step8", [False, True], ids=["adamw", "adamw8"])
def test_same_result_alone_and_among_others(mb, step8):
    """What a tensor becomes does not depend on what else is in the call, nor on the run."""
    def run(order):
        p, g, m, v = _inputs([5000, 300, 70000], 9)
        P, G = _place(p, torch.float32, 0), _place(g, torch.float32, 0)
        if step8:
            _, d = _state8(m, v, 0)
            for idx in order:
                pick = lambda x: [x[i] for i in idx]  # noqa: E731
                mb.adamw8_step(pick(P), pick(G), pick(d["m"]), pick(d["ms"]), pick(d["v"]), pick(d["vs"]), 4, seed=11)
            return P + d["m"] + d["ms"] + d["v"] + d["vs"]
        M, V = _place(m, torch.float32, 0), _place(v, torch.float32, 0)
        for idx in order:
            pick = lambda x: [x[i] for i in idx]  # noqa: E731
            mb.adamw_step(pick(P), pick(G), pick(M), pick(V), 4)
        return P + M + V
    together, alone, again = run([[0, 1, 2]]), run([[2], [0], [1]]), run([[1, 2, 0]])
    assert all(torch.equal(a, b) and torch.equal(a, c) for a, b, c in zip(together, alone, again))


def test_strided_tensors(mb):
    """channels_last filters and a transposed matrix: dense in another order of dimensions."""
    gen = torch.Generator().manual_seed(10)
    shape = (8, 6, 3, 3)
    mk = lambda s: torch.randn(shape, generator=gen) * s  # noqa: E731
    p, g, m, v = mk(1), mk(1e-3), mk(1e-3), mk(1e-3).abs()
    cl = [x.cuda().to(memory_format=torch.channels_last) for x in (p, g, m, v)]
    q = [torch.randn(33, 17, generator=gen).cuda().t() for _ in range(3)] + [torch.rand(33, 17, generator=gen).cuda().t()]
    hosts = [[x.cpu() for x in y] for y in (cl, q)]
    mb.adamw_step([cl[0], q[0]], [cl[1], q[1]], [cl[2], q[2]], [cl[3], q[3]], 2, lr=LR, betas=BETAS, eps=EPS,
                  weight_decay=WD)
    for dev, host in zip((cl, q), hosts):
        args = (*host, 2, LR, BETAS, EPS, WD)
        for got, want, tol in zip((dev[0], dev[2], dev[3]), orc.adamw64(*args), orc.adamw_tolerance(*args)):
            _assert_close(got.cpu().contiguous(), want.contiguous(), tol.contiguous(), "strided")
    with pytest.raises(ValueError, match="strides"):  # another order than the parameter's
        mb.adamw_step([cl[0]], [g.cuda()], [cl[2]], [cl[3]], 2)
    with pytest.raises(ValueError, match="strides"):  # gaps
        w = torch.zeros(4, 8, device="cuda")[:, :4]
        mb.adamw_step([w], [w], [w], [w], 2)


# ------------------------------------------------------------------------------------ norm
def _norm_error(n):
    """float32 sums of 8 squares (each square and sum half a step: 8 u), float64 from there, a root
    that halves it and one rounding to float32."""
    return (4 + 1) * 2.0 ** -24


@pytest.mark.parametrize("times", [1, 3, 9, 18], ids=["one", "few", "some", "many"])  # one launch, each size of table
@pytest.mark.parametrize("offset", [0, 1], ids=["aligned", "odd"])
def test_grad_norm_and_clip(mb, offset, times):
    gen = torch.Generator().manual_seed(12)
    kinds = [torch.float32, torch.bfloat16, torch.float16]
    g = [(torch.randn(n, generator=gen) * 3).to(kinds[i % 3]) for i, n in enumerate(SIZES * times + [100003] * (times - 1))]
    G = [_place([x], x.dtype, offset)[0] for x in g]
    exact = math.sqrt(sum(float(x.double().square().sum()) for x in g))
    norm, factor = mb.grad_norm(G, 2.0)
    assert abs(float(norm) - exact) <= _norm_error(0) * exact
    assert abs(float(factor) - 2.0 / (exact + 1e-6)) <= 8 * 2.0 ** -24 * float(factor)
    assert all(torch.equal(a.cpu(), b) for a, b in zip(G, g))
    assert float(mb.grad_norm(G)[1]) == 1.0 and float(mb.grad_norm(G, 1e9)[1]) == 1.0
    assert torch.equal(mb.grad_norm(G, 2.0)[0], norm), "the same on every run"
    assert torch.equal(mb.clip_grad_norm_(G, 1e9), norm)
    assert all(torch.equal(a.cpu(), b) for a, b in zip(G, g)), "nothing to clip: not a bit changes"
    assert torch.equal(mb.clip_grad_norm_(G, 2.0), norm)
    for a, b in zip(G, g):
        assert torch.equal(a.cpu(), (b.float() * factor.cpu()).to(b.dtype))


@pytest.mark.parametrize("size", [1e30, 1e-30, 1e-42, 0.0])
def test_norm_over_the_whole_range(mb, size):
    x = torch.randn(5001, generator=torch.Generator().manual_seed(13)) * size
    exact = float(x.double().square().sum().sqrt())
    norm = float(mb.grad_norm([x.cuda()])[0])
    assert abs(norm - exact) <= _norm_error(0) * exact + 2.0 ** -150


def test_norm_that_is_not_finite(mb):
    for bad in (float("inf"), float("nan")):
        x = torch.randn(3000, device="cuda")
        x[1234] = bad
        norm, factor = mb.grad_norm([x], 1.0)
        assert math.isnan(float(factor)) and not math.isfinite(float(norm))
        y = x.clone()
        n = mb.clip_grad_norm_([x], 1.0)
        ref = torch.nn.Parameter(torch.zeros(3000, device="cuda"))
        ref.grad = y
        torch.nn.utils.clip_grad_norm_([ref], 1.0)
        assert torch.equal(torch.isnan(x), torch.isnan(y)) and torch.equal(x.nan_to_num(), y.nan_to_num())
        assert not math.isfinite(float(n))


def test_norm_of_parameters_and_of_nothing(mb):
    p = torch.nn.Parameter(torch.zeros(10, device="cuda"))
    q = torch.nn.Parameter(torch.zeros(10, device="cuda"))
    p.grad = torch.full((10,), 2.0, device="cuda")
    assert float(mb.clip_grad_norm_([p, q], 1.0)) == pytest.approx(math.sqrt(40), rel=1e-6)
    assert q.grad is None and float(p.grad.norm()) == pytest.approx(1.0, rel=1e-5)
    assert float(mb.clip_grad_norm_([q], 1.0)) == 0.0 and float(mb.grad_norm([q])[1]) == 1.0
    assert float(mb.clip_grad_norm_([torch.zeros(0, device="cuda")], 1.0)) == 0.0


def test_elements_past_32_bits(mb):
    """2^32 + 300 elements of bfloat16: the last ones are stepped, summed, scaled and expanded like others."""
    n, tail = (1 << 32) + 300, 700  # the last blocks, from a multiple of 256 on
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("needs 60 GB")
    first = (n - tail) // 256 * 256
    gen = torch.Generator().manual_seed(30)
    p, g = (torch.randn(n - first, generator=gen) * 0.02).bfloat16(), (torch.randn(n - first, generator=gen) * 0.01).bfloat16()
    P, G = torch.zeros(n, dtype=torch.bfloat16, device="cuda"), torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    P[first:], G[first:] = p.cuda(), g.cuda()
    codes = [torch.zeros(n, dtype=torch.uint8, device="cuda") for _ in range(2)]
    scales = [torch.zeros(-(-n // 256), device="cuda") for _ in range(2)]
    norm, factor = mb.grad_norm([G], 0.01)
    exact = float(g.double().norm())
    assert abs(float(norm) - exact) <= _norm_error(0) * exact
    mb.adamw8_step([P], [G], codes[:1], scales[:1], codes[1:], scales[1:], 1, lr=LR, betas=BETAS, eps=EPS, weight_decay=WD,
                   grad_scale=factor, seed=3)
    zeros = torch.zeros(n - first)
    f = float(factor)
    m, v = orc.moments32(g, zeros, zeros, BETAS, f)
    index = torch.arange(n - first) + first  # the hash is taken of the low 32 bits of index / 4: 2^32 / 4 is within
    bits = orc.random_bits_at(index, 3, 1)
    for k, (x, kind, r) in enumerate(((m, "exp_avg", None), (v, "exp_avg_sq", bits))):
        _check_codes(codes[k][first:], scales[k][first // 256:], orc.quantize(x, kind, r), kind, kind)
        out = mb.dequantize_state(codes[k:k + 1], scales[k:k + 1], kind, dtype=torch.bfloat16)[0]
        assert torch.equal(out[first:].cpu(), orc.dequantize(codes[k][first:].cpu(), scales[k][first // 256:].cpu(), kind).bfloat16())
        assert (out[:256] == 0).all() and (out[first - 512:first] == 0).all()
        del out
    args = (p, g, zeros, zeros, 1, LR, BETAS, EPS, WD, f)
    want = orc.adamw64(*args)[0]
    _assert_close(P[first:], want, orc.adamw_tolerance(*args)[0] + _half_step(want, torch.bfloat16), "parameter")
    assert torch.equal(mb.clip_grad_norm_([G], 0.01), norm)
    assert torch.equal(G[first:].cpu(), (g.float() * factor.cpu()).bfloat16()) and (G[:first] == 0).all()


# ------------------------------------------------------------------------------------ conversion
@pytest.mark.parametrize("times", [1, 7, 18], ids=["few", "some", "many"])
@pytest.mark.parametrize("offset", [0, 1], ids=["aligned", "odd"])
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("kind", ["exp_avg", "exp_avg_sq"])
def test_convert_state(mb, kind, dtype, offset, times):
    t = DTYPES[dtype]
    gen = torch.Generator().manual_seed(14)
    sizes = SIZES * times
    x = [(torch.randn(n, generator=gen) * torch.exp(2 * torch.randn(n, generator=gen))).to(t) for n in sizes]
    if kind == "exp_avg_sq":
        x = [y.abs() for y in x]
    for y in x:
        y[:300:7] = 0
    X = _place(x, t, offset)
    codes, scales = mb.quantize_state(X, kind)
    for i, n in enumerate(sizes):
        want = orc.quantize(x[i], kind)
        _check_codes(codes[i], scales[i], want, kind, f"{kind} {n}")
        assert codes[i].shape == x[i].shape and scales[i].numel() == -(-n // 256)
    C, S = _place([c.cpu() for c in codes], torch.uint8, offset), _place([s.cpu() for s in scales], torch.float32, offset)
    for got, c, s in zip(mb.dequantize_state(C, S, kind, dtype=t), codes, scales):
        want = orc.dequantize(c.cpu(), s.cpu(), kind)
        assert got.dtype == t and torch.equal(got.cpu(), want.to(t))
    out = _place([torch.zeros(n) for n in sizes], torch.float32, offset)
    assert mb.dequantize_state(C, S, kind, out=out) is out
    for got, y, s in zip(out, x, scales):  # half a code: 1/16 of the value, or half the smallest code
        y, s = y.double(), s.cpu().repeat_interleave(256)[:y.numel()].double()
        small = s * (2.0 ** -31 if kind == "exp_avg_sq" else 2.0 ** -10)
        assert ((got.cpu().double() - y).abs() <= y.abs() * (1 / 16) * (1 + 1e-6) + small).all()


def test_every_code(mb):
    """All 256 codes of either kind, through both directions."""
    codes = torch.arange(256, dtype=torch.uint8, device="cuda")
    scale = torch.ones(1, device="cuda")
    for kind in ("exp_avg", "exp_avg_sq"):
        x = mb.dequantize_state([codes], [scale], kind)[0]
        want = orc.code_values(kind)
        assert torch.equal(torch.isnan(x.cpu()), torch.isnan(want))
        assert torch.equal(x.cpu().nan_to_num(), want.float().nan_to_num())
        x = x.nan_to_num()
        back, s = mb.quantize_state([x], kind)
        assert float(s[0]) == 1.0  # the largest value of the table is in the block
        keep = ~torch.isnan(want)
        assert torch.equal(back[0].cpu()[keep], codes.cpu()[keep])


def test_stochastic_rounding_is_right_on_average(mb):
    """One value between two codes, 2^20 elements: the mean is the value (6 standard errors)."""
    n = 1 << 20
    for x, seed in ((1.0101, 1), (0.0371, 2), (3.3e-4, 3)):
        v = torch.full((n,), x)
        v[::256] = 1.875  # the scale of every block is 1
        g = torch.sqrt(v.double() / (1 - BETAS[1])).float()
        G, P = [g.cuda()], [torch.zeros(n, device="cuda")]
        z, s = [torch.zeros(n, dtype=torch.uint8, device="cuda") for _ in range(2)], [torch.zeros(n // 256, device="cuda") for _ in range(2)]
        mb.adamw8_step(P, G, [z[0]], [s[0]], [z[1]], [s[1]], 1, betas=BETAS, seed=seed)
        got = mb.dequantize_state([z[1]], [s[1]], "exp_avg_sq", dtype=torch.float32)[0].double()
        mask = torch.ones(n, dtype=torch.bool, device="cuda")
        mask[::256] = False
        got = got[mask]
        true = float(((g.double() ** 2) * (1 - BETAS[1]))[1])
        spread = float(got.std())
        assert spread > 0 and abs(float(got.mean()) - true) <= 6 * spread / math.sqrt(got.numel()) + 3e-7 * true


# ------------------------------------------------------------------------------------ streams, graphs, refusals
def test_on_another_stream(mb):
    p, g, m, v = _inputs([100000, 77], 15)
    P, G, M, V = (_place(x, torch.float32, 0) for x in (p, g, m, v))
    G = [torch.zeros_like(x) for x in G]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)  # the gradients arrive late, on the side stream
        for a, b in zip(G, g):
            a.copy_(b, non_blocking=True)
        norm, factor = mb.grad_norm(G, 0.5)
        mb.adamw_step(P, G, M, V, 3, lr=LR, betas=BETAS, eps=EPS, weight_decay=WD, grad_scale=factor)
        codes, scales = mb.quantize_state(M, "exp_avg")
        back = mb.dequantize_state(codes, scales, "exp_avg")
    torch.cuda.current_stream().wait_stream(side)
    f = float(factor)
    for i in range(2):
        args = (p[i], g[i], m[i], v[i], 3, LR, BETAS, EPS, WD, f)
        _assert_close(P[i], orc.adamw64(*args)[0], orc.adamw_tolerance(*args)[0], "parameter")
        assert (back[i] - M[i]).abs().max() <= M[i].abs().max() / 16


def test_two_streams_at_once(mb):
    """Norm, clipping and both steps on two streams side by side: each as alone."""
    def setup(seed):
        p, g, m, v = _inputs([700001, 333, 90000], seed)
        return dict(p=_place(p, torch.float32, 0), g=_place(g, torch.float32, 0), m=_place(m, torch.float32, 0),
                    v=_place(v, torch.float32, 0), d=_state8(m, v, 0)[1])

    def work(s):
        norms = []
        for step in range(3, 9):
            norm, f = mb.grad_norm(s["g"], 0.7)
            mb.adamw_step(s["p"], s["g"], s["m"], s["v"], step, grad_scale=f)
            d = s["d"]
            mb.adamw8_step(s["p"], s["g"], d["m"], d["ms"], d["v"], d["vs"], step, grad_scale=f, seed=step)
            norms += [norm, mb.clip_grad_norm_(s["g"], 0.6)]
        return norms

    alone = [setup(k) for k in (50, 51)]
    want = [work(s) for s in alone]
    both = [setup(k) for k in (50, 51)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], []
    for s, st in zip(both, streams):
        with torch.cuda.stream(st):
            got.append(work(s))
    torch.cuda.synchronize()
    for a, b, x, y in zip(alone, both, want, got):
        assert all(torch.equal(i, j) for i, j in zip(x, y))
        for key in ("p", "g", "m", "v"):
            assert all(torch.equal(i, j) for i, j in zip(a[key], b[key])), key
        for key in ("m", "ms", "v", "vs"):
            assert all(torch.equal(i, j) for i, j in zip(a["d"][key], b["d"][key])), key


def test_gradients_marked_ready_on_a_copy_stream(mb):
    p, g, m, v = _inputs([200000], 16)
    P, M, V = (_place(x, torch.float32, 0) for x in (p, m, v))
    G, host = [torch.zeros(200000, device="cuda")], g[0].pin_memory()
    copies = torch.cuda.Stream()
    with torch.cuda.stream(copies):
        torch.cuda._sleep(20_000_000)
        G[0].copy_(host, non_blocking=True)
        mb.mark_grad_ready(G[0])
    _, factor = mb.grad_norm(G, 1e9)
    mb.adamw_step(P, G, M, V, 1, lr=LR, betas=BETAS, eps=EPS, weight_decay=WD, grad_scale=factor)
    args = (p[0], g[0], m[0], v[0], 1, LR, BETAS, EPS, WD)
    _assert_close(P[0], orc.adamw64(*args)[0], orc.adamw_tolerance(*args)[0], "parameter")


def test_captured_and_replayed(mb):
    """Two graphs captured one after the other on one stream, replayed at the same time on two: each
    has norm scratch of its own. A replay repeats the call's step number and seed."""
    def setup(seed):
        p, g, m, v = _inputs([300000, 1234], seed)
        _, d = _state8(m, v, 0)
        return dict(p=_place(p, torch.float32, 0), g=_place(g, torch.float32, 0), m=_place(m, torch.float32, 0),
                    v=_place(v, torch.float32, 0), d=d)

    def call(s):
        norm, f = mb.grad_norm(s["g"], 0.5)
        mb.adamw_step(s["p"], s["g"], s["m"], s["v"], 3, grad_scale=f)
        d = s["d"]
        mb.adamw8_step(s["p"], s["g"], d["m"], d["ms"], d["v"], d["vs"], 3, grad_scale=f, seed=5)
        mb.clip_grad_norm_(s["g"], 0.5)
        return norm

    want = []
    for k in (20, 21):
        s = setup(k)
        norms = [call(s).clone() for _ in range(3)]
        want.append((s, norms[-1]))
    stream, graphs = torch.cuda.Stream(), []
    for k in (20, 21):
        s = setup(k)
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            norm = call(s)
        graphs.append((graph, s, norm))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(3):
        for (graph, _, _), st in zip(graphs, streams):
            with torch.cuda.stream(st):
                graph.replay()
    torch.cuda.synchronize()
    for (_, s, norm), (ref, ref_norm) in zip(graphs, want):
        assert torch.equal(norm, ref_norm)
        for key in ("p", "g", "m", "v"):
            assert all(torch.equal(a, b) for a, b in zip(s[key], ref[key])), key
        for key in ("m", "ms", "v", "vs"):
            assert all(torch.equal(a, b) for a, b in zip(s["d"][key], ref["d"][key])), key


def test_refusals(mb):
    f = lambda n=10, **k: torch.zeros(n, device="cuda", **k)  # noqa: E731
    good = lambda: ([f()], [f()], [f()], [f()])  # noqa: E731
    p, g, m, v = good()
    cases = [
        (lambda: mb.adamw_step([f()], [f(11)], [f()], [f()], 1), ValueError, "number of elements"),
        (lambda: mb.adamw_step([f()], [f()], [f(), f()], [f()], 1), ValueError, "2 exp_avg tensors for 1"),
        (lambda: mb.adamw_step([f()], [f(dtype=torch.bfloat16)], [f()], [f()], 1), ValueError, "gradient tensors must be"),
        (lambda: mb.adamw_step([f()], [f()], [f(dtype=torch.bfloat16)], [f()], 1), ValueError, "exp_avg tensors must be"),
        (lambda: mb.adamw_step([f(dtype=torch.float64)], [f()], [f()], [f()], 1), ValueError, "float64"),
        (lambda: mb.adamw_step([f(), f(dtype=torch.bfloat16)], [f(), f()], [f(), f()], [f(), f()], 1), ValueError, "one dtype"),
        (lambda: mb.adamw_step([f()], [f()], [f()], [f()], 1, masters=[f()]), ValueError, "no master"),
        (lambda: mb.adamw_step([f()], [f()], [f()], [f()], 0), mb.MuonB200Error, "steps count from 1"),
        (lambda: mb.adamw_step([f()], [f()], [f()], [f()], [1, 2]), ValueError, "2 steps for 1"),
        (lambda: mb.adamw_step([f()], [f()], [f()], [f()], 1, betas=(1.0, 0.9)), mb.MuonB200Error, "betas"),
        (lambda: mb.adamw_step([f()], [f()], [f()], [f()], 1, eps=-1.0), mb.MuonB200Error, "eps"),
        (lambda: mb.adamw_step([f()], [f()], [f()], [f()], 1, grad_scale=f(2)), ValueError, "grad_scale"),
        (lambda: mb.adamw_step([f()], [f()], [f()], [f()], 1, grad_scale=torch.ones(())), ValueError, "grad_scale"),
        (lambda: mb.adamw_step([f()], [torch.zeros(10)], [f()], [f()], 1), RuntimeError, "no CPU implementation"),
        (lambda: mb.adamw_step([p[0], p[0]], [f(), f()], [f(), f()], [f(), f()], 1), ValueError, "twice"),
        (lambda: mb.adamw_step([f(), f()], [f(), f()], [m[0], m[0]], [f(), f()], 1), ValueError, "twice"),
        (lambda: mb.adamw_step([p[0]], [f()], [p[0]], [f()], 1), ValueError, "twice"),
        (lambda: mb.adamw8_step([f()], [f()], [f()], [f(1)], [f()], [f(1)], 1), ValueError, "uint8"),
        (lambda: mb.adamw8_step([f()], [f()], [f(dtype=torch.uint8)], [f(2)], [f(dtype=torch.uint8)], [f(1)], 1), ValueError,
         "exp_avg scale tensor 0 has another number"),
        (lambda: mb.adamw8_step([f()], [f()], [f(dtype=torch.uint8)], [f(1)], [f(dtype=torch.uint8)], [f(1)], 1, eps=0.0),
         mb.MuonB200Error, "eps"),
        (lambda: mb.quantize_state([f()], "momentum"), ValueError, "kind"),
        (lambda: mb.dequantize_state([f(dtype=torch.uint8)], [f(1)], "exp_avg", dtype=torch.float64), ValueError, "float64"),
        (lambda: mb.clip_grad_norm_([p[0], p[0]], 1.0), ValueError, "twice"),
        (lambda: mb.clip_grad_norm_([p[0][:6], f(), p[0][5:]], 1.0), ValueError, "twice"),
        (lambda: mb.adamw_step([p[0][:6]], [f(6)], [p[0][4:]], [f(6)], 1), ValueError, "twice"),
        (lambda: mb.adamw_step([f()], [None], [f()], [f()], 1), TypeError, "is no tensor"),
        (lambda: mb.clip_grad_norm_([f()], -1.0), mb.MuonB200Error, "max_norm"),
        (lambda: mb.clip_grad_norm_([f()], float("nan")), mb.MuonB200Error, "max_norm"),
        (lambda: mb.grad_norm([f(dtype=torch.int32)]), ValueError, "int32"),
        (lambda: mb.grad_norm([torch.view_as_complex(f(20).view(10, 2)).conj().imag]), ValueError, "no memory of its own"),
        (lambda: mb.grad_norm([f().to_sparse()]), (ValueError, RuntimeError), "."),
    ]
    for k, (call, error, match) in enumerate(cases):
        with pytest.raises(error, match=match):
            call()
            pytest.fail(f"case {k} was accepted")
    mb.adamw_step([], [], [], [], 1)
    empty = f(0)
    mb.adamw_step([empty, f(0)], [f(0), f(0)], [f(0), f(0)], [f(0), f(0)], 1)
    assert mb.quantize_state([], "exp_avg") == ([], [])
