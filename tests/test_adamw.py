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
    keep = [x.buffer_info()[0] if isinstance(x, array) else x for x in tables_then_scalars]
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


def test_lists_refuse_what_is_no_cuda_tensor():
    import muon_b200 as mb
    with pytest.raises(RuntimeError, match="every gradient tensor of grad_norm .* no CPU implementation"):
        mb.grad_norm([torch.zeros(3)])
    for bad in ([1], [[torch.zeros(1)]], ["x"]):
        with pytest.raises(TypeError, match="is no tensor"):
            mb.grad_norm(bad)
    for bad in (5, None):
        with pytest.raises(TypeError):
            mb.clip_grad_norm_(bad, 1.0)
    assert [float(x) for x in mb.grad_norm([None])] == [0.0, 1.0] and float(mb.clip_grad_norm_([], 1.0)) == 0.0
    mb.adamw_step([], [], [], [], 1)
    mb.adamw8_step([], [], [], [], [], [], [])
    with pytest.raises(ValueError, match="1 gradient tensors for 0"):
        mb.adamw_step([], [torch.zeros(1)], [], [], 1)
    assert mb.dequantize_state([], [], "exp_avg") == []


# ------------------------------------------------------------------------------- the classes, without a GPU
class _OracleBackend:
    """Stand-in for the CUDA backend: the same calls on CPU tensors, from the oracle."""

    def __init__(self):
        self.calls = []

    def adamw_step(self, params, grads, ms, vs, steps, lr, weight_decay, betas, eps, masters, grad_scale):
        self.calls.append(("adamw", len(params), params[0].dtype, masters is not None))
        f = 1.0 if grad_scale is None else float(grad_scale)
        for i, p in enumerate(params):
            w = p if masters is None else masters[i]
            new = orc.adamw64(w, grads[i], ms[i], vs[i], steps[i], lr, betas, eps, weight_decay, f)
            w.copy_(new[0])
            p.copy_(w)
            ms[i].copy_(new[1])
            vs[i].copy_(new[2])

    def adamw8_step(self, params, grads, mc, msc, vc, vsc, steps, lr, weight_decay, betas, eps, masters, grad_scale, seed):
        self.calls.append(("adamw8", len(params), params[0].dtype, masters is not None))
        f = 1.0 if grad_scale is None else float(grad_scale)
        for i, p in enumerate(params):
            m = orc.dequantize(mc[i], msc[i], "exp_avg").view_as(p)
            v = orc.dequantize(vc[i], vsc[i], "exp_avg_sq").view_as(p)
            w = p if masters is None else masters[i]
            w.copy_(orc.adamw64(w, grads[i], m, v, steps[i], lr, betas, eps, weight_decay, f)[0])
            p.copy_(w)
            m, v = orc.moments32(grads[i], m, v, betas, f)
            for x, c, s, kind, bits in ((m, mc[i], msc[i], "exp_avg", None),
                                        (v, vc[i], vsc[i], "exp_avg_sq", orc.random_bits(p.numel(), seed, steps[i]))):
                codes, scales = orc.quantize(x.reshape(-1), kind, bits)
                c.view(-1).copy_(codes)
                s.copy_(scales)

    def grad_norm(self, tensors, max_norm, clip):
        norm = math.sqrt(sum(float(t.double().square().sum()) for t in tensors))
        return torch.tensor(norm), torch.tensor(min(1.0, max_norm / (norm + 1e-6)))

    def convert_state(self, what, values, codes, scales, kind, to_codes):
        for x, c, s in zip(values, codes, scales):
            if to_codes:
                new_c, new_s = orc.quantize(x.reshape(-1), kind)
                c.view(-1).copy_(new_c)
                s.copy_(new_s)
            else:
                x.view(-1).copy_(orc.dequantize(c, s, kind))

    def adam_step(self, params, grads, ms, vs, steps, lr, weight_decay, betas, eps):
        self.calls.append(("adam", len(params), params[0].dtype, False))


@pytest.fixture
def backend():
    from muon_b200 import engine
    stand_in = _OracleBackend()
    prev = engine._set_backend_for_testing(stand_in)
    yield stand_in
    engine._set_backend_for_testing(prev)


def _params(seed=0):
    gen = torch.Generator().manual_seed(seed)
    shapes = [(64, 80), (5,), (70, 3, 5, 5), (4096,)]
    kinds = [torch.float32, torch.float32, torch.bfloat16, torch.bfloat16]
    return [torch.nn.Parameter((torch.randn(s, generator=gen) * 0.1).to(k)) for s, k in zip(shapes, kinds)]


def _give_grads(params, seed):
    gen = torch.Generator().manual_seed(seed)
    for p in params:
        p.grad = (torch.randn(p.shape, generator=gen) * 0.01).to(p.dtype)


def test_adamw_class_groups_and_state(backend):
    import muon_b200 as mb
    params = _params()
    opt = mb.AdamW([dict(params=params[:2], lr=1e-2), dict(params=params[2:], state_bits=8, master_weights=True)],
                   weight_decay=0.0)
    opt.step()
    assert backend.calls == [] and len(opt.state) == 0  # nothing has a gradient
    _give_grads(params, 1)
    params[1].grad = None
    before = params[1].detach().clone()
    opt.step()
    assert backend.calls == [("adamw", 1, torch.float32, False), ("adamw8", 2, torch.bfloat16, True)]
    assert torch.equal(params[1], before) and len(opt.state.get(params[1], {})) == 0
    assert set(opt.state[params[0]]) == {"step", "moment_bits", "exp_avg", "exp_avg_sq"}
    s = opt.state[params[2]]
    assert s["exp_avg_codes"].dtype == torch.uint8 and s["exp_avg_codes"].shape == params[2].shape
    assert s["exp_avg_scales"].shape == (21,) and s["master"].dtype == torch.float32
    want = torch.optim.AdamW([params[0].detach().clone().requires_grad_()], lr=1e-2)  # the first step is lr * sign
    assert (opt.state[params[0]]["step"], s["step"]) == (1, 1) and want is not None
    backend.calls.clear()
    opt = mb.AdamW(params, state_bits=8, min_8bit_numel=4096 + 1)
    _give_grads(params, 2)
    opt.step()
    # by type and by size of state, in the order they come
    assert backend.calls == [("adamw8", 1, torch.float32, False), ("adamw", 1, torch.float32, False),
                             ("adamw8", 1, torch.bfloat16, False), ("adamw", 1, torch.bfloat16, False)]


def test_adamw_class_agrees_with_torch(backend):
    """Two steps on float32 parameters: the stand-in computes in 64 bits, torch in 32 (a few roundings)."""
    import muon_b200 as mb
    gen = torch.Generator().manual_seed(3)
    a = torch.nn.Parameter(torch.randn(50, 7, generator=gen))
    b = torch.nn.Parameter(a.detach().clone())
    ours, theirs = mb.AdamW([a], lr=1e-2, weight_decay=0.1), torch.optim.AdamW([b], lr=1e-2, weight_decay=0.1)
    for k in range(2):
        a.grad = torch.randn(50, 7, generator=gen)
        b.grad = a.grad.clone()
        ours.step()
        theirs.step()
        assert torch.allclose(a, b, rtol=1e-6, atol=1e-7)


def test_adamw_class_clips_all_groups_together(backend):
    import muon_b200 as mb
    gen = torch.Generator().manual_seed(4)
    ps = [torch.nn.Parameter(torch.randn(40, generator=gen)) for _ in range(3)]
    qs = [torch.nn.Parameter(p.detach().clone()) for p in ps]
    opt = mb.AdamW([dict(params=ps[:1]), dict(params=ps[1:])], max_grad_norm=0.5)
    ref = mb.AdamW([dict(params=qs[:1]), dict(params=qs[1:])])
    for p, q in zip(ps, qs):
        p.grad = torch.randn(40, generator=gen)
        q.grad = p.grad.clone()
    torch.nn.utils.clip_grad_norm_(qs, 0.5)
    opt.step()
    ref.step()
    assert float(opt.grad_norm) == pytest.approx(float(torch.cat([p.grad for p in ps]).norm()), rel=1e-6)
    for p, q in zip(ps, qs):
        assert torch.allclose(p, q, rtol=1e-6, atol=1e-7)
        assert torch.allclose(opt.state[p]["exp_avg"], ref.state[q]["exp_avg"], rtol=1e-5, atol=1e-9)


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_class_state_dict_keeps_types(backend, bits, tmp_path):
    import muon_b200 as mb
    params = _params(5)
    opt = mb.AdamW(params, state_bits=bits, master_weights=True)
    for k in range(2):
        _give_grads(params, 10 + k)
        opt.step()
    torch.save(opt.state_dict(), tmp_path / "state.pt")
    copies = [torch.nn.Parameter(p.detach().clone()) for p in params]
    again = mb.AdamW(copies, state_bits=40 - bits)
    again.load_state_dict(torch.load(tmp_path / "state.pt"))
    for p, q in zip(params, copies):
        a, b = opt.state[p], again.state[q]
        assert set(a) == set(b)
        for k in a:
            assert type(a[k]) is type(b[k])
            if torch.is_tensor(a[k]):
                assert a[k].dtype == b[k].dtype and torch.equal(a[k], b[k]) and a[k].data_ptr() != b[k].data_ptr(), k
            else:
                assert a[k] == b[k]
    _give_grads(params, 12)
    _give_grads(copies, 12)
    opt.step()
    again.step()
    assert all(torch.equal(p, q) for p, q in zip(params, copies))
    bad = opt.state_dict()
    bad["state"][0]["exp_avg" if bits == 32 else "exp_avg_codes"] = torch.zeros(3)
    with pytest.raises(ValueError, match="moments of shape"):
        again.load_state_dict(bad)


def test_adamw_class_changes_its_state_bits(backend):
    import muon_b200 as mb
    params = _params(6)
    opt = mb.AdamW(params)
    _give_grads(params, 1)
    opt.step()
    m = opt.state[params[0]]["exp_avg"].clone()
    opt.set_state_bits(8)
    assert [opt.state[p]["moment_bits"] for p in params] == [8, 32, 8, 8]
    assert opt.param_groups[0]["state_bits"] == 8 and "exp_avg" not in opt.state[params[0]]
    _give_grads(params, 2)
    opt.step()
    opt.set_state_bits(32)
    assert all(opt.state[p]["moment_bits"] == 32 and opt.state[p]["exp_avg"].shape == p.shape for p in params)
    assert [opt.state[p]["step"] for p in params] == [2] * 4 and m.shape == params[0].shape
    for bad in (16, "8"):
        with pytest.raises(ValueError, match="state_bits"):
            opt.set_state_bits(bad)
        with pytest.raises(ValueError, match="state_bits"):
            mb.AdamW(_params(), state_bits=bad)
    with pytest.raises(ValueError, match="max_grad_norm"):
        mb.AdamW(_params(), max_grad_norm=-1.0)


def test_auxiliary_adam_keeps_other_moments_when_asked(backend):
    """set_adam_moments: state made from then on; what exists keeps its kind; the default is the
    reference's arithmetic on the parameter's type."""
    import copy
    import muon_b200 as mb
    params = _params(7)
    assert mb.get_adam_moments() == "param"
    opt = mb.SingleDeviceMuonWithAuxAdam([dict(params=params[:1], use_muon=False)])
    _give_grads(params, 1)
    opt.step()
    assert backend.calls == [("adam", 1, torch.float32, False)] and "moment_bits" not in opt.state[params[0]]
    try:
        mb.set_adam_moments("8bit")
        opt.step()
        aux = mb.SingleDeviceMuonWithAuxAdam([dict(params=params, use_muon=False)])
        params[1].grad = None  # the reference's rule: zeros
        aux.step()
        mb.set_adam_moments("fp32")
        wide = mb.SingleDeviceMuonWithAuxAdam([dict(params=params, use_muon=False)])
        wide.step()
        with pytest.raises(ValueError, match="moments"):
            mb.set_adam_moments("int8")
    finally:
        mb.set_adam_moments()
    assert backend.calls[1][0] == "adam"
    assert [aux.state[p]["moment_bits"] for p in params] == [8, 32, 8, 8]
    assert [wide.state[p]["moment_bits"] for p in params] == [32] * 4
    assert wide.state[params[2]]["exp_avg"].dtype == torch.float32 and (params[1].grad == 0).all()
    for source in (aux, wide):
        target = mb.SingleDeviceMuonWithAuxAdam([dict(params=params, use_muon=False)])
        target.load_state_dict(copy.deepcopy(source.state_dict()))
        other = mb.SingleDeviceMuonWithAuxAdam([dict(params=params, use_muon=False)])
        mb.load_consolidated_state_dict(other, mb.consolidated_state_dict(source))
        for p in params:
            for key, value in source.state[p].items():
                for to in (target, other):
                    got = to.state[p][key]
                    assert (got.dtype == value.dtype and torch.equal(got, value)) if torch.is_tensor(value) else got == value


def test_adamw_class_on_dtensors(backend, tmp_path):
    """Row-sharded parameters on a mesh of one rank: the local part is stepped, with moments of its own; a
    gradient in another placement is brought into the parameter's; clipping is refused."""
    import torch.distributed as dist
    from torch.distributed.device_mesh import init_device_mesh
    from torch.distributed.tensor import DTensor, Partial, Shard
    import muon_b200 as mb
    dist.init_process_group("gloo", init_method=f"file://{tmp_path}/pg", rank=0, world_size=1)
    try:
        mesh = init_device_mesh("cpu", (1,))
        gen = torch.Generator().manual_seed(8)
        w, g = torch.randn(70, 80, generator=gen), torch.randn(70, 80, generator=gen)
        p = torch.nn.Parameter(DTensor.from_local(w.clone(), mesh, [Shard(0)]))
        q = torch.nn.Parameter(w.clone())
        ours, plain = mb.AdamW([p], state_bits=8), mb.AdamW([q], state_bits=8)
        for placement in (Shard(0), Partial()):
            p.grad = DTensor.from_local(g.clone(), mesh, [placement])
            q.grad = g.clone()
            ours.step()
            plain.step()
        assert torch.equal(p.to_local(), q) and ours.state[p]["exp_avg_codes"].shape == (70, 80)
        assert torch.equal(ours.state[p]["exp_avg_codes"], plain.state[q]["exp_avg_codes"])
        clipped = mb.AdamW([p], max_grad_norm=1.0)
        with pytest.raises(ValueError, match="whole gradients"):
            clipped.step()
    finally:
        dist.destroy_process_group()
