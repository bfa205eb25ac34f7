"""Calls on the AdamW operators at the edges of what their documentation allows, on the GPU."""
import pytest
import torch

from oracle import adamw_oracle as orc
from test_gpu_adamw import _place

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def mb():
    import muon_b200
    return muon_b200


# ------------------------------------------------------------------------------------ conversion
@pytest.mark.parametrize("offset", [0, 1], ids=["aligned", "odd"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_signed_zeros_of_second_moments(mb, dtype, offset):
    """-0.0 is not negative: it gets the code of 0, the smallest. So do values under 0 that the rounding of an
    earlier run may have left; a block whose largest magnitude counts as zero has codes 0 and scale 0."""
    gen = torch.Generator().manual_seed(30)
    x = [torch.rand(n, generator=gen) for n in (256, 600, 1, 257)]
    x[0][::3] = -0.0
    x[1][1::2] = -0.0
    x[2][0] = -0.0
    x[3][256] = -0.0
    for k, y in enumerate((-1e-38, -1e-12, -2.0 ** -31, -1e-7, -1e-3, -0.5)):
        x[0][10 + k] = y
        x[1][300 + k] = y
    tiny = torch.full((300,), 2.0 ** -125) * torch.where(torch.arange(300) % 2 == 0, 1.0, -1.0)
    tiny[5], tiny[299] = -0.0, -0.0
    x = [y.to(dtype) for y in x + [tiny]]
    codes, scales = mb.quantize_state(_place(x, dtype, offset), "exp_avg_sq")
    for y, c, s in zip(x, codes, scales):
        want_c, want_s = orc.quantize(y, "exp_avg_sq")
        assert torch.equal(c.cpu(), want_c) and torch.equal(s.cpu(), want_s)
        assert (c.cpu()[torch.signbit(y)] == 0).all()
    assert (codes[4] == 0).all() and (scales[4] == 0).all()


# ------------------------------------------------------------------------------------ memory
def test_memory_that_is_read_and_written_is_refused(mb):
    """A block would read what another one has written already. Each call is refused before a launch and leaves
    the memory as it was; lists that lie close together in one buffer, or share what they only read, are not."""
    f = lambda n=600, **k: torch.ones(n, device="cuda", **k)  # noqa: E731
    u = lambda n=600: f(n, dtype=torch.uint8)  # noqa: E731
    buf = f(1200)
    codes = u(4800)
    lie = codes.view(torch.float32)  # 1200 floats in the same memory
    cases = [
        lambda: mb.adamw_step([buf[:600]], [buf[300:900]], [f()], [f()], 1),
        lambda: mb.adamw_step([buf[:600]], [buf[:600]], [f()], [f()], 1),
        lambda: mb.adamw_step([f()], [buf[:600]], [buf[599:1199]], [f()], 1),
        lambda: mb.adamw_step([f(), f()], [f(), buf[:600]], [f(), f()], [buf[500:1100], f()], 1),
        lambda: mb.adamw_step([buf[:600]], [f()], [f()], [f()], 1, grad_scale=buf[599]),
        lambda: mb.adamw_step([f(dtype=torch.bfloat16)], [buf[:600]], [f()], [f()], 1, masters=[buf[1:601]]),
        lambda: mb.adamw8_step([f()], [lie[:600]], [codes[:600]], [f(3)], [u()], [f(3)], 1),
        lambda: mb.adamw8_step([f()], [buf[:600]], [u()], [buf[598:601]], [u()], [f(3)], 1),
        lambda: mb.quantize_state([lie[:600]], "exp_avg", codes=[codes[2399:2999]]),
        lambda: mb.quantize_state([buf[:600]], "exp_avg", scales=[buf[597:600]]),
        lambda: mb.dequantize_state([codes[:600]], [f(3)], "exp_avg", out=[lie[:600]]),
        lambda: mb.dequantize_state([u()], [buf[600:603]], "exp_avg", out=[buf[1:601]]),
    ]
    for k, call in enumerate(cases):
        with pytest.raises(ValueError, match="overlaps memory that is read"):
            call()
            pytest.fail(f"case {k} was accepted")
    assert (buf == 1).all() and (codes == 1).all()
    buf = f(2404)
    mb.adamw_step([buf[:600]], [buf[600:1200]], [buf[1200:1800]], [buf[1800:2400]], 1, grad_scale=buf[2400])
    assert (buf[600:1200] == 1).all() and (buf[:600] != 1).all() and buf[2400] == 1
    g = f()
    mb.adamw_step([f(), f()], [g, g], [f(), f()], [f(), f()], 1)
    codes, scales = mb.quantize_state([g, g[:300]], "exp_avg")
    mb.dequantize_state([codes[0], codes[0][:256]], [scales[0], scales[0][:1]], "exp_avg")


# ------------------------------------------------------------------------------------ marked gradients
@pytest.mark.parametrize("clip", [False, True])
def test_norm_and_step_of_marked_gradients_on_two_streams(mb, clip):
    """Gradients that arrive on a copy stream, their norm on a second stream, the step on a third: the marks alone
    order them."""
    n = 1 << 20
    gen = torch.Generator().manual_seed(31)
    p, g = torch.randn(n, generator=gen) * 0.02, (torch.randn(n, generator=gen) * 1e-3).pin_memory()
    P, G = _place([p], torch.float32, 0), [torch.zeros(n, device="cuda")]
    M, V = ([torch.zeros(n, device="cuda")] for _ in range(2))
    copies, norms, steps = (torch.cuda.Stream() for _ in range(3))
    torch.cuda.synchronize()
    with torch.cuda.stream(copies):
        torch.cuda._sleep(20_000_000)
        G[0].copy_(g, non_blocking=True)
        mb.mark_grad_ready(G[0])
    with torch.cuda.stream(norms):
        norm = mb.clip_grad_norm_(G, 0.5) if clip else mb.grad_norm(G, 0.5)[0]
    with torch.cuda.stream(steps):
        mb.adamw_step(P, G, M, V, 1, weight_decay=0.0)
    torch.cuda.synchronize()
    want_norm = float(g.double().norm())
    assert abs(float(norm) - want_norm) <= 5 * 2.0 ** -24 * want_norm
    factor = min(1.0, 0.5 / (want_norm + 1e-6)) if clip else 1.0
    want = 0.1 * factor * g.double()  # roundings: norm 5, sum and quotient 2, the product, constant and product of the moment 2
    assert ((M[0].cpu().double() - want).abs() <= 10.5 * 2.0 ** -24 * want.abs() + 1e-44).all()
    from muon_b200 import engine
    assert not engine._grad_ready


# ------------------------------------------------------------------------------------ order of memory
@pytest.mark.parametrize("shape,of_p,of_g", [((96, 64, 1, 1), (64, 1, 1, 1), (64, 1, 64, 64)),
                                             ((64, 24, 3, 1), (72, 1, 24, 24), (72, 1, 24, 72)),
                                             ((1, 24, 3, 64), (7, 1, 24, 72), (4608, 1, 24, 72))])
def test_lists_whose_sizes_of_one_have_other_strides(mb, shape, of_p, of_g):
    """The elements are in one order, so the call takes them; every other difference of strides is refused."""
    gen = torch.Generator().manual_seed(32)
    p, g = torch.randn(shape, generator=gen), torch.randn(shape, generator=gen)
    place = lambda x, order: torch.empty_strided(shape, order, device="cuda").copy_(x)  # noqa: E731
    P, G, M, V = place(p, of_p), place(g, of_g), place(p * 0, of_g), place(p * 0, of_p)
    mb.adamw_step([P], [G], [M], [V], 1, lr=1e-2, weight_decay=0.1)
    args = (p, g, p * 0, p * 0, 1, 1e-2, (0.9, 0.999), 1e-8, 0.1)
    tol = orc.adamw_tolerance(*args)
    for got, want, t in zip((P, M, V), orc.adamw64(*args), tol):
        assert ((got.cpu().double() - want).abs() <= t).all()
    codes, scales = mb.quantize_state([M], "exp_avg")
    out = [place(p, of_g)]
    mb.dequantize_state(codes, scales, "exp_avg", out=out)
    want = orc.dequantize(*orc.quantize(torch.as_strided(M, (M.numel(),), (1,)).cpu(), "exp_avg"), "exp_avg")
    assert torch.equal(torch.as_strided(out[0], (M.numel(),), (1,)).cpu(), want)
    if not P.is_contiguous():
        with pytest.raises(ValueError, match="strides"):
            mb.adamw_step([P], [G.contiguous()], [M], [V], 2)


# ------------------------------------------------------------------------------------ autograd
def test_what_is_written_counts_a_version(mb):
    """A tensor that a later backward pass has saved is not changed in silence, as with torch's own in-place
    functions. State of an optimizer, what is only read and a refused call leave the counters."""
    f = lambda n=600: torch.ones(n, device="cuda")  # noqa: E731
    u = lambda: torch.zeros(600, dtype=torch.uint8, device="cuda")  # noqa: E731
    w = torch.nn.Parameter(f())
    loss = (w * w).sum()
    mb.adamw_step([w], [f()], [f()], [f()], 1)
    with pytest.raises(RuntimeError, match="inplace operation"):
        loss.backward()
    w.grad = None
    h = f()
    loss = (w * h).sum()
    mb.clip_grad_norm_([h], 1.0)
    with pytest.raises(RuntimeError, match="inplace operation"):
        loss.backward()

    def versions(written, read, call):
        before = [t._version for t in written + read]
        call()
        return [t._version - v for t, v in zip(written + read, before)] == [1] * len(written) + [0] * len(read)

    p, g, m, v, f1 = f(), f(), f(), f(), f(1)
    assert versions([p], [g, f1, m, v], lambda: mb.adamw_step([p], [g], [m], [v], 1, grad_scale=f1))
    q, master = f().bfloat16(), f()
    c = [u(), torch.zeros(3, device="cuda"), u(), torch.zeros(3, device="cuda")]
    assert versions([q], [g, master, *c], lambda: mb.adamw8_step([q], [g], *([x] for x in c), 1, masters=[master]))
    assert versions([], [p, g], lambda: mb.grad_norm([p, g]))
    assert versions([p, g], [], lambda: mb.clip_grad_norm_([p, g], 1e9))
    assert versions([], [m, *c[:2]], lambda: mb.quantize_state([m], "exp_avg", codes=[c[0]], scales=[c[1]]))
    assert versions([m], c[:2], lambda: mb.dequantize_state([c[0]], [c[1]], "exp_avg", out=[m]))

    def refused():
        with pytest.raises((ValueError, mb.MuonB200Error)):
            mb.adamw_step([p], [g], [m], [v], 0)
        with pytest.raises((ValueError, mb.MuonB200Error)):
            mb.adamw_step([p], [g], [m], [p], 1)

    assert versions([], [p, g, m, v], refused)
    opt = mb.AdamW([w], state_bits=8, min_8bit_numel=1, max_grad_norm=1.0)
    w.grad = f()
    opt.step()
    loss = (w * w).sum()
    opt.step()
    with pytest.raises(RuntimeError, match="inplace operation"):
        loss.backward()
    with torch.inference_mode():
        i = f()  # has no counter
    mb.adamw_step([i], [f()], [f()], [f()], 1)
    assert float(i[0]) != 1.0


def test_lists_from_iterators_of_views(mb):
    """Views that nothing but the iterator makes: they live until the call is made."""
    flat = {k: torch.ones(40 * 64, device="cuda") for k in "pgmv"}
    views = lambda k: (flat[k][64 * i:64 * (i + 1)] for i in range(40))  # noqa: E731
    before = {k: t._version for k, t in flat.items()}
    mb.adamw_step(*(views(k) for k in "pgmv"), 1)
    mb.clip_grad_norm_(views("g"), 1e9)
    assert {k: t._version - before[k] for k, t in flat.items()} == {"p": 40, "g": 40, "m": 0, "v": 0}
    assert all((t == t[0]).all() for t in flat.values()) and float(flat["p"][0]) < 1.0
