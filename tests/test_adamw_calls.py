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
