"""The AdamW class and the auxiliary Adam with float32 and 8-bit moments on the GPU: every step against
the 64-bit formulas from the state before it, checkpoints, and the operators together in a training loop."""
import copy
import math

import pytest
import torch

from oracle import adamw_oracle as orc

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def mb():
    import muon_b200
    return muon_b200


def _params(seed=0, device="cuda"):
    gen = torch.Generator().manual_seed(seed)
    shapes = [(300, 80), (5,), (70, 3, 5, 5), (8200,), (1000, 33), (0,)]
    kinds = [torch.float32, torch.float32, torch.bfloat16, torch.bfloat16, torch.float16, torch.float32]
    return [torch.nn.Parameter((torch.randn(s, generator=gen) * 0.1).to(k).to(device)) for s, k in zip(shapes, kinds)]


def _give_grads(params, seed, size=0.01):
    gen = torch.Generator().manual_seed(seed)
    for p in params:
        p.grad = (torch.randn(p.shape, generator=gen) * size).to(p.dtype).to(p.device)


def _values(state):
    """(first moment, second moment) of a state as flat float32 CPU tensors."""
    if state["moment_bits"] == 8:
        return tuple(orc.dequantize(state[f"{k}_codes"].cpu(), state[f"{k}_scales"].cpu(), k) for k in ("exp_avg", "exp_avg_sq"))
    return state["exp_avg"].cpu().reshape(-1), state["exp_avg_sq"].cpu().reshape(-1)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("master", [False, True], ids=["plain", "master"])
@pytest.mark.parametrize("max_norm", [None, 0.5])
def test_adamw_class_steps(mb, bits, master, max_norm):
    lr, betas, eps, wd = 1e-3, (0.9, 0.95), 1e-8, 0.1
    params = _params()
    opt = mb.AdamW(params, lr=lr, betas=betas, eps=eps, weight_decay=wd, state_bits=bits, master_weights=master,
                   min_8bit_numel=256, max_grad_norm=max_norm, seed=9)
    for step in range(1, 4):
        _give_grads(params, step)
        before = []
        for p in params:
            s = opt.state.get(p, {})
            zeros = torch.zeros(p.numel())
            m, v = _values(s) if s else (zeros, zeros)
            before.append((s["master"].cpu().clone() if "master" in s else p.detach().cpu().clone(), m.clone(), v.clone()))
        opt.step()
        f = 1.0
        if max_norm is not None:
            norm = math.sqrt(sum(float(p.grad.double().square().sum()) for p in params))
            assert abs(float(opt.grad_norm) - norm) <= 5 * 2.0 ** -24 * norm and norm > max_norm
            # the factor: the norm's error, and 4 roundings of its own
            f = min(1.0, max_norm / (norm + 1e-6))
        for p, (w, m, v) in zip(params, before):
            s = opt.state[p]
            assert s["step"] == step and s["moment_bits"] == (8 if bits == 8 and p.numel() >= 256 else 32)
            g = p.grad.cpu().reshape(-1)
            args = (w.reshape(-1), g, m, v, step, lr, betas, eps, wd, f)
            want, tol = orc.adamw64(*args), orc.adamw_tolerance(*args)
            extra = 0 if max_norm is None else 9 * 2.0 ** -24 * lr * 20  # 9 u of an update of at most 20 lr
            got = s["master"] if "master" in s else p.detach()
            assert ("master" in s) == (master and p.dtype != torch.float32)
            # half a step of the type: eps / 2 of the value, and under the smallest normal number (float16:
            # 2^-14, steps of 2^-24) half of the constant step, tiny * eps / 2 = 2^-25
            info = torch.finfo(got.dtype)
            half = 0 if got.dtype == torch.float32 else info.eps / 2 * (want[0].abs() + info.tiny)
            err = (got.cpu().double().reshape(-1) - want[0]).abs()
            assert (err <= tol[0] + extra + half).all(), (p.shape, float(err.max()))
            if "master" in s:
                assert torch.equal(p.detach(), s["master"].to(p.dtype))


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_class_checkpoint_goes_on_bit_for_bit(mb, bits, tmp_path):
    params = _params(1)
    opt = mb.AdamW(params, state_bits=bits, master_weights=True, max_grad_norm=1.0)
    for k in range(2):
        _give_grads(params, k)
        opt.step()
    torch.save(opt.state_dict(), tmp_path / "s.pt")
    copies = [torch.nn.Parameter(p.detach().clone()) for p in params]
    again = mb.AdamW(copies, max_grad_norm=1.0)
    again.load_state_dict(torch.load(tmp_path / "s.pt"))
    for k in range(2, 4):
        _give_grads(params, k)
        _give_grads(copies, k)
        opt.step()
        again.step()
    for p, q in zip(params, copies):
        assert torch.equal(p, q)
        for key, value in opt.state[p].items():
            got = again.state[q][key]
            assert torch.equal(got, value) and got.dtype == value.dtype if torch.is_tensor(value) else got == value


def test_moments_follow_a_parameter_into_another_memory_order(mb):
    """channels_last filters: moments in the filter's order; a checkpoint loaded into contiguous ones."""
    gen = torch.Generator().manual_seed(2)
    w = torch.randn(64, 16, 3, 3, generator=gen)
    p = torch.nn.Parameter(w.cuda().to(memory_format=torch.channels_last))
    q = torch.nn.Parameter(w.cuda())
    for bits in (32, 8):
        a, b = mb.AdamW([p], state_bits=bits), mb.AdamW([q])
        p.grad = torch.randn(w.shape, generator=gen).cuda()  # contiguous, unlike its parameter
        a.step()
        key = "exp_avg" if bits == 32 else "exp_avg_codes"
        assert a.state[p][key].stride() == p.stride()
        b.load_state_dict(copy.deepcopy(a.state_dict()))
        assert b.state[q][key].stride() == q.stride()
        a.set_state_bits(32)
        b.set_state_bits(32)
        one, two = a.state[p]["exp_avg"], b.state[q]["exp_avg"]
        # bits == 8: blocks of 256 are other elements in the other order, a second rounding of half a code
        assert torch.equal(one, two.to(memory_format=torch.channels_last)) if bits == 32 else \
            ((one - two).abs() <= one.abs() / 16 * (1 + 1e-6) + one.abs().max() * 2.0 ** -17).all()


def test_state_bits_of_a_run_are_changed(mb):
    params = _params(3)
    opt = mb.AdamW(params, min_8bit_numel=256)
    for k in range(2):
        _give_grads(params, k)
        opt.step()
    m = {p: opt.state[p]["exp_avg"].clone() for p in params}
    opt.set_state_bits(8)
    assert [opt.state[p]["moment_bits"] for p in params] == [8 if p.numel() >= 256 else 32 for p in params]
    opt.set_state_bits(32)
    for p in params:
        got = opt.state[p]["exp_avg"]
        top = m[p].abs().max() if p.numel() else 0.0
        assert ((got - m[p]).abs() <= m[p].abs() / 16 * (1 + 1e-6) + top * 2.0 ** -18).all()  # half a code
    _give_grads(params, 5)
    opt.step()
    assert all(torch.isfinite(p).all() for p in params)


def test_step_is_not_captured(mb):
    params = _params(4)
    opt = mb.AdamW(params)
    _give_grads(params, 1)
    opt.step()
    torch.cuda.synchronize()
    before = [p.detach().clone() for p in params]
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="captured"):
        with torch.cuda.graph(graph):
            opt.step()
    torch.cuda.synchronize()
    assert all(torch.equal(p, b) for p, b in zip(params, before)) and opt.state[params[0]]["step"] == 1


@pytest.mark.parametrize("moments", ["fp32", "8bit"])
def test_auxiliary_adam(mb, moments):
    """SingleDeviceMuonWithAuxAdam: matrices through Muon as before, the rest with other moments."""
    gen = torch.Generator().manual_seed(5)
    mat0, emb0, gain0 = torch.randn(128, 256, generator=gen) * 0.02, torch.randn(64, 100, generator=gen), torch.ones(256)
    grads = [[torch.randn(t.shape, generator=gen) * 0.1 for t in (mat0, emb0, gain0)] for _ in range(2)]

    def run(kind):
        ps = [torch.nn.Parameter(t.clone().cuda()) for t in (mat0, emb0, gain0)]
        mb.set_adam_moments(kind)
        try:
            opt = mb.SingleDeviceMuonWithAuxAdam([dict(params=ps[:1], use_muon=True), dict(params=ps[1:], use_muon=False, lr=1e-2)])
            for gs in grads:
                for p, g in zip(ps, gs):
                    p.grad = g.clone().cuda()
                opt.step()
        finally:
            mb.set_adam_moments()
        return ps, opt

    ps, opt = run(moments)
    ref, _ = run("param")
    assert torch.equal(ps[0], ref[0]), "Muon's part is untouched"
    assert [opt.state[p].get("moment_bits") for p in ps] == [None, 8 if moments == "8bit" else 32, 32]
    # float32 parameters: the float32 moments agree with the reference's arithmetic to its roundings; an
    # 8-bit first moment is off by 1/16, the root of a second by 1/16: two updates of about lr
    bound = 1e-6 if moments == "fp32" else 1e-2 * 2 * (1 / 16 + 1 / 16) * 1.2
    assert (ps[1] - ref[1]).abs().max() <= bound and (ps[2] - ref[2]).abs().max() <= 1e-6


def test_the_operators_in_a_training_loop(mb):
    """Clip, Muon for the matrices, AdamW with 8-bit moments for the rest: norms are the gradients', clipped
    gradients are within the bound, and a second loop from the same seeds gives the same norms."""
    def loop():
        torch.manual_seed(6)
        model = torch.nn.Sequential(torch.nn.Embedding(500, 64), torch.nn.Linear(64, 128), torch.nn.ReLU(),
                                    torch.nn.Linear(128, 500)).cuda()
        matrices = [model[1].weight]
        rest = [p for p in model.parameters() if p is not model[1].weight]
        muon, adamw = mb.SingleDeviceMuon(matrices, lr=0.02), mb.AdamW(rest, lr=1e-2, state_bits=8)
        tokens = torch.randint(0, 500, (4, 256), generator=torch.Generator().manual_seed(7)).cuda()
        norms = []
        for k in range(4):
            logits = model(tokens[k][:-1])
            logp = logits - logits.logsumexp(dim=-1, keepdim=True)
            (-logp.gather(1, tokens[k][1:, None]).mean()).backward()
            whole = torch.cat([p.grad.reshape(-1) for p in model.parameters()]).double().norm()
            norms.append(mb.clip_grad_norm_(model.parameters(), 0.1))
            assert abs(float(norms[-1]) - float(whole)) <= 1e-6 * float(whole)
            after = torch.cat([p.grad.reshape(-1) for p in model.parameters()]).double().norm()
            assert float(after) <= 0.1 * (1 + 1e-6)
            for opt in (muon, adamw):
                opt.step()
                opt.zero_grad()
        assert mb.device_status() == 0
        return [p.detach().clone() for p in model.parameters()], torch.stack(norms)

    a, norms = loop()
    _, again = loop()
    assert torch.isfinite(norms).all() and all(torch.isfinite(p).all() for p in a)
    # torch adds the embedding's gradient in no fixed order: a few roundings may differ
    assert torch.allclose(norms, again, rtol=1e-3)


def test_step_in_backward_with_other_moments(mb):
    """StepInBackward leaves the Adam groups to its step(): the same with 8-bit moments."""
    gen = torch.Generator().manual_seed(8)
    w0, e0 = torch.randn(64, 96, generator=gen) * 0.05, torch.randn(96, 96, generator=gen)
    x = torch.randn(32, 96, generator=gen).cuda()

    def run(in_backward):
        w, e = torch.nn.Parameter(w0.clone().cuda()), torch.nn.Parameter(e0.clone().cuda())
        opt = mb.SingleDeviceMuonWithAuxAdam([dict(params=[w], use_muon=True), dict(params=[e], use_muon=False)])
        stepper = mb.StepInBackward(opt) if in_backward else opt
        for _ in range(2):
            ((x @ e) @ w.t()).square().mean().backward()
            stepper.step()
            w.grad = e.grad = None
        return w, e, opt

    mb.set_adam_moments("8bit")
    try:
        a, b = run(False), run(True)
    finally:
        mb.set_adam_moments()
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    assert a[2].state[a[1]]["moment_bits"] == 8
