"""The AdamW operators and class, without a GPU: calls that lost state, counts or options."""
import pytest
import torch

from test_adamw import _OracleBackend, _give_grads, _params


@pytest.fixture
def backend():
    from muon_b200 import engine
    prev = engine._set_backend_for_testing(_OracleBackend())
    yield engine.get_backend()
    engine._set_backend_for_testing(prev)


def _assert_same_state(a, b):
    assert set(a) == set(b)
    for key, value in a.items():
        if torch.is_tensor(value):
            assert b[key].dtype == value.dtype and torch.equal(b[key], value) and b[key].data_ptr() != value.data_ptr(), key
        else:
            assert type(b[key]) is type(value) and b[key] == value, key


# ------------------------------------------------------------------------------- consolidated checkpoints
@pytest.mark.parametrize("bits", [32, 8])
def test_consolidated_checkpoint_of_the_adamw_class(backend, bits, tmp_path):
    import muon_b200 as mb
    params = _params(1)
    opt = mb.AdamW([dict(params=params[:2], lr=1e-2), dict(params=params[2:], master_weights=True)], state_bits=bits)
    for k in range(3):
        _give_grads(params, k)
        opt.step()
    torch.save(mb.consolidated_state_dict(opt), tmp_path / "state.pt")
    copies = [torch.nn.Parameter(p.detach().clone()) for p in params]
    again = mb.AdamW([dict(params=copies[:2]), dict(params=copies[2:])], state_bits=40 - bits)
    mb.load_consolidated_state_dict(again, torch.load(tmp_path / "state.pt"))
    assert [g["lr"] for g in again.param_groups] == [1e-2, 1e-3] and again.param_groups[0]["state_bits"] == bits
    for p, q in zip(params, copies):
        assert opt.state[p]["step"] == 3
        _assert_same_state(opt.state[p], again.state[q])
    _give_grads(params, 9)
    _give_grads(copies, 9)
    opt.step()
    again.step()
    assert all(torch.equal(p, q) for p, q in zip(params, copies))


def test_consolidated_checkpoints_of_other_kinds_are_refused(backend):
    """Muon state for an AdamW group or the reverse, an optimizer whose state is neither: refused, and what
    the optimizer holds stays."""
    import muon_b200 as mb
    params = _params(2)[:1]
    adamw, muon = mb.AdamW(params), mb.SingleDeviceMuon(params)
    _give_grads(params, 1)
    adamw.step()
    muon.state[params[0]]["momentum_buffer"] = torch.ones(64, 80)
    of_adamw, of_muon = mb.consolidated_state_dict(adamw), mb.consolidated_state_dict(muon)
    for target, source in ((adamw, of_muon), (muon, of_adamw)):
        with pytest.raises(ValueError, match="state of"):
            mb.load_consolidated_state_dict(target, source)
    assert adamw.state[params[0]]["step"] == 1 and (muon.state[params[0]]["momentum_buffer"] == 1).all()
    other = torch.optim.AdamW(params)
    other.step()
    with pytest.raises(ValueError, match="exp_avg"):
        mb.consolidated_state_dict(other)


def test_consolidated_checkpoint_of_sharded_parameters_is_refused(backend, tmp_path):
    """The state of a DTensor is that of this rank's rows: one rank's would be taken for all."""
    import torch.distributed as dist
    from torch.distributed.device_mesh import init_device_mesh
    from torch.distributed.tensor import DTensor, Shard
    import muon_b200 as mb
    dist.init_process_group("gloo", init_method=f"file://{tmp_path}/pg", rank=0, world_size=1)
    try:
        mesh = init_device_mesh("cpu", (1,))
        p = torch.nn.Parameter(DTensor.from_local(torch.randn(8, 4), mesh, [Shard(0)]))
        p.grad = DTensor.from_local(torch.randn(8, 4), mesh, [Shard(0)])
        opt = mb.AdamW([p])
        opt.step()
        with pytest.raises(ValueError, match="DTensor"):
            mb.consolidated_state_dict(opt)
    finally:
        dist.destroy_process_group()


# ------------------------------------------------------------------------------- marked gradients
class _Stream:
    """Stand-in for a CUDA stream: the events it was made to wait for, and what ran on it, in order."""

    def __init__(self):
        self.log = []

    def wait_event(self, event):
        self.log.append(event)


class _Event:
    def __init__(self):
        self.after = None

    def record(self, stream):
        self.after = list(stream.log)


@pytest.fixture
def streams(monkeypatch):
    """The current stream as a stand-in, and the marks; `streams.now` may be set to another stream."""
    from muon_b200 import engine

    class Streams:
        now = _Stream()

    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: Streams.now)
    monkeypatch.setattr(torch.cuda, "Event", _Event)
    monkeypatch.setattr(engine, "_grad_ready", {})
    return Streams


@pytest.mark.parametrize("clip", [False, True])
def test_a_norm_leaves_the_marks_to_the_step(streams, monkeypatch, clip):
    """A norm on one stream waits for marked gradients, and so does the step on another stream that follows it;
    after clipping the step waits for the clipped values."""
    from muon_b200 import engine
    calls = engine.CudaBackend()

    class Tables:
        @staticmethod
        def grad_norm(tensors, max_norm, clip, scratch):
            streams.now.log.append("norm")
            return 0, torch.ones(()), torch.ones(())

        @staticmethod
        def adamw(*args):
            streams.now.log.append("step")
            return 0

    monkeypatch.setattr(engine, "_tables", Tables)
    a, b = torch.zeros(4), torch.zeros(4)
    arrived = _Event()
    engine._grad_ready[a.data_ptr()] = arrived
    first = streams.now
    calls.grad_norm([a, b], 1.0, clip)
    assert first.log == [arrived, "norm"]
    streams.now = second = _Stream()
    calls.adamw_step([a, b], [a, b], [a, b], [a, b], 1, 1e-3, 0.0, (0.9, 0.999), 1e-8)
    assert len(second.log) == 2 and second.log[1] == "step"
    if clip:
        assert second.log[0].after == [arrived, "norm"]  # an event behind the clipping
    else:
        assert second.log[0] is arrived
    assert not engine._grad_ready


class _Arrival(_Event):
    """A gradient in flight: its values are there once a stream has waited for them."""

    def __init__(self, gradient, values):
        super().__init__()
        self.gradient, self.values = gradient, values


@pytest.fixture
def in_flight(streams, monkeypatch):
    """in_flight(gradient) makes it NaN until a wait for its mark brings its values."""
    from muon_b200 import engine

    def put(gradient):
        engine._grad_ready[gradient.data_ptr()] = _Arrival(gradient, gradient.clone())
        gradient.fill_(float("nan"))

    monkeypatch.setattr(_Stream, "wait_event", lambda self, event: event.gradient.copy_(event.values))
    yield put
    assert not engine._grad_ready


def test_copies_of_gradients_wait_for_their_marks(in_flight, backend):
    """A gradient in another order of dimensions is copied before the kernels read it."""
    import muon_b200 as mb
    gen = torch.Generator().manual_seed(5)
    grad = lambda: torch.randn(80, 64, generator=gen).t()  # noqa: E731
    p = torch.nn.Parameter(torch.zeros(64, 80))
    seen = []
    backend.adam_step = lambda ps, gs, *rest: seen.extend(g.clone() for g in gs)
    backend.muon_step = lambda ps, gs, *rest, **more: seen.extend(g.clone() for g in gs)
    backend.adamw_step = lambda ps, gs, *rest: seen.extend(g.clone() for g in gs)
    optimizers = [mb.SingleDeviceMuonWithAuxAdam([dict(params=[p], use_muon=False)]),
                  mb.SingleDeviceMuonWithAuxAdam([dict(params=[p], use_muon=True)]), mb.SingleDeviceMuon([p]), mb.AdamW([p])]
    for opt in optimizers:
        p.grad = grad()
        want = p.grad.clone()
        in_flight(p.grad)
        opt.step()
        assert torch.equal(seen.pop(), want), type(opt).__name__


def test_sharded_gradients_wait_for_their_marks(in_flight, backend, monkeypatch, tmp_path):
    """Gradients that are DTensors are marked by the memory of their local part, and redistributed or sent off
    after it is there."""
    import torch.distributed as dist
    from torch.distributed.device_mesh import init_device_mesh
    from torch.distributed.tensor import DTensor, Partial, Shard
    import muon_b200 as mb
    from muon_b200 import engine
    dist.init_process_group("gloo", init_method=f"file://{tmp_path}/pg", rank=0, world_size=1)
    try:
        mesh = init_device_mesh("cpu", (1,))
        gen = torch.Generator().manual_seed(6)
        g = torch.randn(8, 4, generator=gen)
        p = torch.nn.Parameter(DTensor.from_local(torch.zeros(8, 4), mesh, [Shard(0)]))
        seen = []
        backend.adamw_step = lambda ps, gs, *rest: seen.extend(g.clone() for g in gs)
        for placement in (Partial(), Shard(0)):
            p.grad = DTensor.from_local(g.clone(), mesh, [placement])
            if isinstance(placement, Partial):  # (a whole one is waited for by the call itself)
                in_flight(p.grad.to_local())
            mb.AdamW([p]).step()
            assert torch.equal(seen.pop(), g)
        backend.muon_orthogonalize = lambda grads, *rest: seen.extend(g.clone() for g in grads)
        backend.apply_update = lambda *args: None
        in_flight(p.grad.to_local())
        mb.ShardedMuon([p]).step()
        assert torch.equal(seen.pop(), g)
        monkeypatch.setattr(engine, "_require_cuda", lambda *args: None)
        for x in (p, p.grad):
            mb.mark_grad_ready(x)
            assert list(engine._grad_ready) == [p.grad.to_local().data_ptr()]
            engine._grad_ready.clear()
    finally:
        dist.destroy_process_group()


# ------------------------------------------------------------------------------- copies of an optimizer
@pytest.mark.parametrize("how", ["deepcopy", "pickle"])
@pytest.mark.parametrize("max_norm", [None, 0.05])
def test_a_copied_optimizer_steps_as_the_original(backend, how, max_norm):
    import copy
    import pickle
    import muon_b200 as mb
    params = _params(3)
    opt = mb.AdamW(params, lr=1e-2, state_bits=8, max_grad_norm=max_norm)
    _give_grads(params, 1)
    opt.step()
    again = copy.deepcopy(opt) if how == "deepcopy" else pickle.loads(pickle.dumps(opt))
    copies = again.param_groups[0]["params"]
    assert again.max_grad_norm == max_norm and (max_norm is None) == (again.grad_norm is None)
    _give_grads(params, 2)
    _give_grads(copies, 2)
    opt.step()
    again.step()
    for p, q in zip(params, copies):
        assert p is not q and torch.equal(p, q)
        _assert_same_state(opt.state[p], again.state[q])
    again.load_state_dict(opt.state_dict())
    assert again.max_grad_norm == max_norm


# ------------------------------------------------------------------------------- state of other optimizers
def _two_runs(seed, kinds=(torch.float32, torch.float32)):
    gen = torch.Generator().manual_seed(seed)
    ps = [torch.nn.Parameter((torch.randn(s, generator=gen) * 0.1).to(k)) for s, k in zip(((70, 80), (5,)), kinds)]
    return ps, [torch.nn.Parameter(p.detach().clone()) for p in ps]


@pytest.mark.parametrize("bits", [32, 8])
def test_a_run_of_torch_adamw_goes_on(backend, bits):
    """Moments, step numbers and the hyper-parameters of torch.optim.AdamW are taken over, into this optimizer's
    kind of state. The stand-in computes in 64 bits, torch in 32; moments in 8 bits are half a code off."""
    import muon_b200 as mb
    theirs, ours = _two_runs(1)
    run = torch.optim.AdamW([dict(params=theirs[:1], lr=1e-2), dict(params=theirs[1:])], lr=2e-3, betas=(0.8, 0.9),
                            eps=1e-7, weight_decay=0.1)
    for k in range(3):
        _give_grads(theirs, k)
        run.step()
    for p, q in zip(theirs, ours):
        q.data.copy_(p)
    opt = mb.AdamW([dict(params=ours[:1], seed=4), dict(params=ours[1:])], state_bits=bits)
    opt.load_state_dict(run.state_dict())
    assert [(g["lr"], g["betas"], g["eps"], g["weight_decay"], g["state_bits"], g["seed"]) for g in opt.param_groups] == [
        (1e-2, (0.8, 0.9), 1e-7, 0.1, bits, 4), (2e-3, (0.8, 0.9), 1e-7, 0.1, bits, 0)]
    assert set(opt.param_groups[0]) == set(mb.AdamW([ours[0]]).param_groups[0])
    assert [(opt.state[p]["step"], opt.state[p]["moment_bits"]) for p in ours] == [(3, bits), (3, 32)]
    if bits == 32:
        for p, q in zip(theirs, ours):
            for key in ("exp_avg", "exp_avg_sq"):
                assert torch.equal(run.state[p][key], opt.state[q][key])
    _give_grads(theirs, 9)
    _give_grads(ours, 9)
    run.step()
    opt.step()
    for p, q in zip(theirs, ours):
        # Half a code is 1/16 of either moment. With these betas |m| <= 1.18 sqrt(v) (Cauchy-Schwarz), at step 4 an
        # update is at most 1.17 lr and the codes are worth 0.062 (m) + 0.038 (v) of lr
        assert torch.allclose(p, q, rtol=1e-6, atol=1e-7 if bits == 32 or q.numel() == 5 else 1.2e-3)


def test_torch_state_of_16_bit_parameters_becomes_float32(backend):
    import muon_b200 as mb
    theirs, ours = _two_runs(2, (torch.bfloat16, torch.float16))
    run = torch.optim.AdamW(theirs)
    _give_grads(theirs, 1)
    run.step()
    opt = mb.AdamW(ours, master_weights=True)
    opt.load_state_dict(run.state_dict())
    for p, q in zip(theirs, ours):
        s = opt.state[q]
        assert s["exp_avg"].dtype == s["exp_avg_sq"].dtype == s["master"].dtype == torch.float32
        assert torch.equal(s["exp_avg"], run.state[p]["exp_avg"].float()) and torch.equal(s["master"], q.float())
    _give_grads(ours, 2)
    opt.step()


def test_adam_groups_of_other_classes_are_taken_over(backend):
    import muon_b200 as mb
    ours = _params(4)[:2]
    try:
        for moments in ("param", "fp32", "8bit"):
            mb.set_adam_moments(moments)
            run = mb.SingleDeviceMuonWithAuxAdam([dict(params=ours, use_muon=False)])
            _give_grads(ours, 1)
            run.step()
            opt = mb.AdamW(ours)
            opt.load_state_dict(run.state_dict())
            assert "use_muon" not in opt.param_groups[0] and [opt.state[p]["step"] for p in ours] == [1, 1]
            assert [opt.state[p]["moment_bits"] for p in ours] == ([8, 32] if moments == "8bit" else [32, 32])
            opt.step()
    finally:
        mb.set_adam_moments()


def test_state_that_means_something_else_is_refused(backend):
    """Before anything changes."""
    import muon_b200 as mb
    theirs, ours = _two_runs(3)
    opt = mb.AdamW(ours, lr=5e-4)
    _give_grads(ours, 1)
    opt.step()
    for run, match in ((torch.optim.AdamW(theirs, amsgrad=True), "amsgrad"), (torch.optim.AdamW(theirs, maximize=True), "maximize"),
                       (torch.optim.Adam(theirs, weight_decay=0.1), "decoupled"), (torch.optim.SGD(theirs, momentum=0.9), "betas"),
                       (torch.optim.Adamax(theirs), "exp_inf"), (mb.SingleDeviceMuon(theirs[:1]), "betas")):
        _give_grads(theirs, 1)
        if not isinstance(run, mb.SingleDeviceMuon):
            run.step()
        with pytest.raises(ValueError, match=match):
            opt.load_state_dict(run.state_dict())
        assert opt.param_groups[0]["lr"] == 5e-4 and [opt.state[p]["step"] for p in ours] == [1, 1]
    plain = torch.optim.Adam(theirs)  # without decay the two are the same
    _give_grads(theirs, 1)
    plain.step()
    opt.load_state_dict(plain.state_dict())
    opt.step()
    assert [opt.state[p]["step"] for p in ours] == [2, 2]


def test_torch_state_of_dtensors(backend, tmp_path):
    """torch keeps DTensors as moments, this class the local parts."""
    import torch.distributed as dist
    from torch.distributed.device_mesh import init_device_mesh
    from torch.distributed.tensor import DTensor, Shard
    import muon_b200 as mb
    dist.init_process_group("gloo", init_method=f"file://{tmp_path}/pg", rank=0, world_size=1)
    try:
        mesh = init_device_mesh("cpu", (1,))
        make = lambda: torch.nn.Parameter(DTensor.from_local(torch.ones(8, 4), mesh, [Shard(0)]))  # noqa: E731
        a, b = make(), make()
        for p in (a, b):
            p.grad = DTensor.from_local(torch.arange(32.0).view(8, 4), mesh, [Shard(0)])
        run, opt = torch.optim.AdamW([a]), mb.AdamW([b])
        run.step()
        opt.load_state_dict(run.state_dict())
        assert type(opt.state[b]["exp_avg"]) is torch.Tensor
        assert torch.equal(opt.state[b]["exp_avg"], run.state[a]["exp_avg"].to_local())
        opt.step()
    finally:
        dist.destroy_process_group()


# ------------------------------------------------------------------------------- steps that are refused
@pytest.mark.parametrize("aux", [False, True])
def test_a_refused_step_is_not_counted(backend, aux):
    """The step number counts the steps that were taken: a call that refuses its lists leaves it. What the calls
    before it in the same step() did stays done, and counted."""
    import muon_b200 as mb
    params = _params(5)[:2]
    _give_grads(params, 1)
    if aux:
        mb.set_adam_moments("8bit")
        opt = mb.SingleDeviceMuonWithAuxAdam([dict(params=params, use_muon=False)])
    else:
        opt = mb.AdamW(params, state_bits=8)

    def refuse(*args):
        raise ValueError("refused")

    try:
        opt.step()
        kept, backend.adamw_step = backend.adamw_step, refuse
        with pytest.raises(ValueError, match="refused"):
            opt.step()
        assert [opt.state[p]["step"] for p in params] == [2, 1]  # (the 8-bit call comes first)
        backend.adamw_step = kept
        opt.step()
        assert [opt.state[p]["step"] for p in params] == [3, 2]
    finally:
        mb.set_adam_moments()


# ------------------------------------------------------------------------------- order of memory
def _like(x, order):
    """A copy of x whose memory has these strides."""
    out = torch.empty_strided(x.shape, order)
    return out.copy_(x)


# shape, strides of the parameter, strides of the gradient: sizes of 1 have no order
_SAME_ORDER = [((96, 64, 1, 1), (64, 1, 1, 1), (64, 1, 64, 64)), ((96, 64, 1, 1), (64, 1, 64, 64), (64, 1, 1, 1)),
               ((1, 80, 64), (5120, 64, 1), (7, 64, 1)), ((64, 24, 3, 1), (72, 1, 24, 24), (72, 1, 24, 72))]


@pytest.mark.parametrize("shape,of_p,of_g", _SAME_ORDER)
@pytest.mark.parametrize("aux", [False, True])
def test_sizes_of_one_have_no_order(backend, shape, of_p, of_g, aux):
    """The gradient is handed over as it is, and moments saved for one such parameter are loaded for another code for
    code."""
    import muon_b200 as mb
    gen = torch.Generator().manual_seed(7)
    seen = []

    def step(ps, gs, mc, msc, vc, vsc, *rest):  # (the stand-in's own takes contiguous codes only)
        seen.extend(g.data_ptr() for g in gs)
        for codes in mc + vc:
            codes.copy_(torch.randint(0, 256, shape, generator=gen))

    backend.adamw8_step = step

    def make(order):
        p = torch.nn.Parameter(_like(torch.ones(shape), order))
        if aux:
            return p, mb.SingleDeviceMuonWithAuxAdam([dict(params=[p], use_muon=False)])
        return p, mb.AdamW([p], state_bits=8)

    try:
        if aux:
            mb.set_adam_moments("8bit")
        p, opt = make(of_p)
        q, again = make(of_g)
        p.grad = _like(torch.randn(shape, generator=gen), of_g)
        opt.step()
        assert seen == [p.grad.data_ptr()]
        again.load_state_dict(opt.state_dict())
        for key in ("exp_avg_codes", "exp_avg_sq_codes"):
            assert torch.equal(again.state[q][key], opt.state[p][key]), key
    finally:
        mb.set_adam_moments()


def test_channels_last_gradients_of_the_auxiliary_adam_are_not_copied(backend):
    import muon_b200 as mb
    p = torch.nn.Parameter(torch.ones(64, 24, 3, 3).to(memory_format=torch.channels_last))
    seen = []
    backend.adamw_step = lambda ps, gs, *rest: seen.extend(g.data_ptr() for g in gs)
    try:
        mb.set_adam_moments("fp32")
        opt = mb.SingleDeviceMuonWithAuxAdam([dict(params=[p], use_muon=False)])
        p.grad = torch.randn(64, 24, 3, 3).to(memory_format=torch.channels_last)
        grad = p.grad
        opt.step()
        opt.step()
    finally:
        mb.set_adam_moments()
    assert p.grad is grad and seen == [grad.data_ptr()] * 2
    backend.adam_step = lambda ps, gs, *rest: seen.extend(g.is_contiguous() for g in gs)
    mb.SingleDeviceMuonWithAuxAdam([dict(params=[p], use_muon=False)]).step()  # the parameter's type: as before
    assert seen[-1] is True


def test_clipping_takes_the_gradients_that_a_step_takes(backend):
    """A gradient that is a slice of a larger buffer, or one value for all elements, is copied into its
    parameter's order: with clipping before the norm, which needs dense memory."""
    import muon_b200 as mb
    gen = torch.Generator().manual_seed(8)
    plain = backend.grad_norm

    def norm(tensors, max_norm, clip):
        assert all(t.is_contiguous() for t in tensors)
        return plain(tensors, max_norm, clip)

    backend.grad_norm = norm
    results = []
    for max_norm in (None, 1e9):
        params = [torch.nn.Parameter(torch.ones(6, 10)), torch.nn.Parameter(torch.ones(7))]
        params[0].grad = torch.arange(120.0).view(6, 20)[:, ::2]
        params[1].grad = torch.full((1,), 0.5).expand(7)
        mb.AdamW(params, max_grad_norm=max_norm).step()
        results.append(params)
    assert all(torch.equal(p, q) for p, q in zip(*results))


def test_a_parameter_may_be_a_plain_leaf(streams, monkeypatch):
    """As for torch.optim and torch.nn.utils: a tensor that requires gradients of its own is a parameter, and its
    .grad is meant (clip_grad_norm_ must not scale the weights). A gradient that has a graph behind it is none."""
    from muon_b200 import engine
    from muon_b200._tables import gradients
    import muon_b200 as mb
    leaf = torch.ones(3, requires_grad=True)
    parameter, plain = torch.nn.Parameter(torch.ones(3)), torch.ones(3)
    frozen = torch.nn.Parameter(torch.ones(3), requires_grad=False)
    assert gradients([leaf, parameter, frozen]) == []
    leaf.grad, parameter.grad = torch.full((3,), 2.0), torch.full((3,), 3.0)
    with_graph = leaf * 2
    got = gradients([leaf, plain, with_graph, parameter, frozen])
    assert len(got) == 4 and all(a is b for a, b in zip(got, (leaf.grad, plain, with_graph, parameter.grad)))
    monkeypatch.setattr(engine, "_require_cuda", lambda *args: None)
    mb.mark_grad_ready(leaf)
    assert list(engine._grad_ready) == [leaf.grad.data_ptr()]
    leaf.grad = None
    with pytest.raises(ValueError, match="no gradient"):
        mb.mark_grad_ready(leaf)


# ------------------------------------------------------------------------------- the build
def _build_module():
    import importlib.util
    import os
    spec = importlib.util.spec_from_file_location("_build", os.path.join(_package(), "build.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def _package():
    import os
    import muon_b200
    return os.path.dirname(muon_b200.__file__)


def test_the_extension_is_built_again_for_another_torch(tmp_path):
    """_tables.so is bound to the torch and the Python it was built for, whose files are newer or older than it."""
    build = _build_module()
    built = []
    build._run = lambda cmd, verbose=False: built.append(cmd)
    build._older = lambda target, names: False
    stamp = build.TABLES_STAMP = str(tmp_path / "stamp")
    assert build.is_stale()  # nothing says what it was built for
    build.build_library()
    assert len(built) == 1 and any("tables.cpp" in x for x in built[0])
    assert not build.is_stale()
    build.build_library()
    assert len(built) == 1
    with open(stamp) as f:
        text = f.read()
    assert torch.__version__ in text
    with open(stamp, "w") as f:
        f.write(text.replace(torch.__version__, "1.0"))
    assert build.is_stale()
    build.build_library()
    assert len(built) == 2 and not build.is_stale()


def test_an_extension_that_does_not_load_says_what_to_do(tmp_path):
    import os
    import subprocess
    import sys
    package = tmp_path / "muon_b200"
    package.mkdir()
    for name in os.listdir(_package()):
        if name.endswith(".py") or name == "libmuon_b200.so":
            os.symlink(os.path.join(_package(), name), package / name)
    for content in (None, b"no library"):
        if content is not None:
            (package / "_tables.so").write_bytes(content)
        out = subprocess.run([sys.executable, "-c", "import muon_b200"], cwd=tmp_path, capture_output=True, text=True,
                             env={**os.environ, "PYTHONPATH": str(tmp_path)})
        assert out.returncode != 0 and "python muon_b200/build.py" in out.stderr and "_tables.so" in out.stderr


def test_consolidated_checkpoints_of_the_auxiliary_adam_and_of_adamw_are_not_mixed(backend):
    """Their groups hold different options, and their states different kinds of moments."""
    import muon_b200 as mb
    params = _params(6)[:2]
    _give_grads(params, 1)
    aux, adamw = mb.SingleDeviceMuonWithAuxAdam([dict(params=params, use_muon=False)]), mb.AdamW(params)
    aux.step()
    adamw.step()
    for target, source in ((aux, adamw), (adamw, aux)):
        before = [dict(g) for g in target.param_groups]
        with pytest.raises(ValueError, match="options of"):
            mb.load_consolidated_state_dict(target, mb.consolidated_state_dict(source))
        assert [dict(g) for g in target.param_groups] == before
        assert all(target.state[p]["step"] == 1 for p in params)
        target.load_state_dict(target.state_dict())
