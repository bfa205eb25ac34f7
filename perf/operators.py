"""The optimizer operators as they are measured: the AdamW step over many tensors with 32-bit and
with 8-bit moments, the global gradient norm with clipping, and the conversion of moments between
32 and 8 bits.

``own = False``: elementary torch operations in 32 bits on the tensors laid end to end.
``own = True``: the calls a user makes of ``muon_b200``.

The 8-bit format. A flattened tensor is cut into blocks of 256 elements (the last may be shorter),
each with one float32 scale per moment.

* First moment: e4m3 codes, value = code * scale, scale = amax / 448, nearest even.
* Second moment: unsigned codes c of 5 exponent and 3 mantissa bits, value = scale * w(c) with
  w(c) = 2^((c >> 3) - 31) * (1 + (c & 7) / 8), scale = amax / 1.875. A step rounds it
  stochastically: with x = v * (1.875 / amax) as float32 bits, c = ((bits + r) >> 20) - 768, clamped
  to 0..255, r a 20-bit number from a hash of seed, step and element index. A plain conversion uses
  r = 2^19 (nearest).
* A block whose amax is under 2^-110 (first) or 2^-120 (second moment) gets scale 0 and codes 0.
"""
import math
import random

import torch

own = False

BLOCK = 256
E4M3_MAX, SQ_MAX = 448.0, 1.875
TINY = {"exp_avg": 2.0 ** -110, "exp_avg_sq": 2.0 ** -120}
FIRST_STEP = 100          # the states are those of a run at this step
LR, EPS, WD = 3e-4, 1e-8, 0.1
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}

# one decoder layer of the benchmark's Llama-3-8B-shaped configuration
LLAMA_LAYER = [4096 * 4096] * 2 + [1024 * 4096] * 2 + [14336 * 4096] * 3


# ------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # the gain vectors beside GPT-2-small-sized matrices, the smallest group an auxiliary Adam gets: latency
        dict(name="adamw gains", op="adamw", tensors="gains", dtype="fp32", master=False, max_norm=0.0, packed=False),
        # a convolutional network's 128 filters, all under AdamW, gradients clipped to norm 1
        dict(name="adamw conv clipped", op="adamw", tensors="conv", dtype="fp32", master=False, max_norm=1.0, packed=False),
        # bfloat16 parameters and gradients of four decoder layers, float32 moments: the largest
        dict(name="adamw llama 4 layers", op="adamw", tensors="llama4", dtype="bf16", master=False, max_norm=0.0, packed=False),
        # views into one flat float16 buffer, odd sizes, so hardly any starts on a 16-byte boundary; float32 master weights
        dict(name="adamw packed fp16", op="adamw", tensors="ragged", dtype="fp16", master=True, max_norm=1.0, packed=True,
             count=150, mean=100000, shapes=7),
        # the same three kinds of call with moments in 8 bits
        dict(name="adamw8 gains", op="adamw8", tensors="gains", dtype="fp32", master=False, max_norm=0.0, packed=False),
        dict(name="adamw8 conv", op="adamw8", tensors="conv", dtype="fp32", master=False, max_norm=0.0, packed=False),
        dict(name="adamw8 llama 2 layers", op="adamw8", tensors="llama2", dtype="bf16", master=False, max_norm=1.0, packed=False),
        # clipping in place before a step of another optimizer class: a few vectors, a layer, odd sizes
        dict(name="clip gains", op="clip", tensors="gains", dtype="fp32", master=False, max_norm=0.5, packed=False),
        dict(name="clip llama layer", op="clip", tensors="llama1", dtype="bf16", master=False, max_norm=1.0, packed=False),
        dict(name="clip packed", op="clip", tensors="ragged", dtype="fp32", master=False, max_norm=1.0, packed=True,
             count=90, mean=60000, shapes=3),
        # a run's float32 moments turned into 8-bit ones and read back (switching a run, checking a checkpoint)
        dict(name="convert llama layer", op="convert", tensors="llama1", dtype="bf16", master=False, max_norm=0.0, packed=False),
        # 8-bit moments of many filters expanded for a checkpoint
        dict(name="expand conv", op="expand", tensors="conv", dtype="fp32", master=False, max_norm=0.0, packed=False),
    ]


def draw(rng):
    """One more case: any operator, 1 to 300 tensors of sizes around 1 to 20 million elements."""
    op = rng.choice(["adamw", "adamw8", "clip", "convert", "expand"])
    count = int(round(math.exp(rng.uniform(0.0, math.log(300)))))
    mean = int(round(math.exp(rng.uniform(math.log(20), math.log(min(2e7, 3e8 / count))))))
    dtype = rng.choice(["fp32", "bf16", "fp16"])
    return dict(op=op, tensors="ragged", dtype=dtype, master=op in ("adamw", "adamw8") and dtype != "fp32" and rng.random() < 0.5,
                max_norm=rng.choice([0.5, 1.0, 4.0]) if op == "clip" or rng.random() < 0.5 else 0.0,
                packed=rng.random() < 0.3, count=count, mean=mean, shapes=rng.randrange(1 << 30))


def _sizes(case):
    kind = case["tensors"]
    if kind == "gains":
        return [768] * 25
    if kind == "conv":
        return [256 * 256 * 9] * 64 + [128 * 128 * 9] * 64
    if kind.startswith("llama"):
        return LLAMA_LAYER * int(kind[5:])
    rng = random.Random(case["shapes"])  # odd sizes around the mean, an empty tensor and a single element among many
    sizes = [max(1, int(case["mean"] * math.exp(rng.uniform(-1.5, 0.7)))) for _ in range(case["count"])]
    if len(sizes) > 8:
        sizes[3], sizes[5] = 0, 1
    return sizes


# ------------------------------------------------------------------------------------ inputs
def _device():
    return torch.device("cuda", 0)


def _carve(sizes, dtype, packed):
    """One buffer and a view of it per tensor: as an allocator places them (every 256 bytes), or packed
    one behind the other from an odd element on."""
    at, starts = 1 if packed else 0, []
    for n in sizes:
        starts.append(at)
        at += n if packed else -(-n // 128) * 128
    flat = torch.zeros(max(1, at), dtype=dtype, device=_device())
    return flat, [flat[s:s + n] for s, n in zip(starts, sizes)]


def prepare(case, seed):
    gen = torch.Generator(device=_device()).manual_seed(int(seed))
    sizes, packed, dtype = _sizes(case), case["packed"], DTYPES[case["dtype"]]
    state = dict(case=case, sizes=sizes, steps=[FIRST_STEP] * len(sizes), seed=int(seed) & 0xFFFFFFFF)

    def randn(like):
        return torch.empty(like.shape, dtype=torch.float32, device=_device()).normal_(generator=gen)

    # gradients whose size differs from weight to weight by a factor of e either way, moments to match
    state["grad_flat"], state["grads"] = _carve(sizes, dtype, packed)
    sigma = randn(state["grad_flat"]).exp_().mul_(1e-3)
    state["grad_flat"].copy_(randn(sigma).mul_(sigma))
    if case["op"] == "clip":
        return state
    state["m_flat"], state["m"] = _carve(sizes, torch.float32, packed)
    state["v_flat"], state["v"] = _carve(sizes, torch.float32, packed)
    state["m_flat"].copy_(randn(sigma).mul_(sigma).mul_(0.25))
    state["v_flat"].copy_(randn(sigma).square_().mul_(0.5).add_(0.2).mul_(sigma).mul_(sigma))
    del sigma
    if case["op"] in ("adamw", "adamw8"):
        state["p_flat"], state["p"] = _carve(sizes, dtype, packed)
        weights = randn(state["p_flat"]).mul_(0.02)
        state["p_flat"].copy_(weights)
        state["w_flat"] = state["w"] = None
        if case["master"]:
            state["w_flat"], state["w"] = _carve(sizes, torch.float32, packed)
            state["w_flat"].copy_(weights)
        del weights
    if case["op"] == "adamw":
        return state
    # moments in 8 bits: codes of the tensor's size, one scale for each 256 of them
    blocks = [-(-n // BLOCK) for n in sizes]
    for name, kind in (("m", "exp_avg"), ("v", "exp_avg_sq")):
        codes, state[name + "_codes"] = _carve(sizes, torch.uint8, packed)
        scales, state[name + "_scales"] = _carve(blocks, torch.float32, packed)
        if case["op"] != "convert":
            c, s = _quantize(_blocked(state[name]).float(), kind, 1 << 19)
            _put(state[name + "_codes"], _unblocked(c, sizes))
            _put(state[name + "_scales"], s.split(blocks))
            del state[name], state[name + "_flat"]
        state[name + "_value"], state[name + "_values"] = _carve(
            sizes, torch.float32 if case["op"] == "expand" else torch.bfloat16, packed)
    if case["op"] in ("convert", "expand"):
        del state["grads"], state["grad_flat"]
    return state


# ------------------------------------------------------------------------------------ one pass
def run(state):
    return {"adamw": _run_adamw, "adamw8": _run_adamw8, "clip": _run_clip, "convert": _run_convert,
            "expand": _run_expand}[state["case"]["op"]](state)


def _betas(state):
    return (0.9, 0.95) if state["case"]["dtype"] == "fp32" else (0.9, 0.999)


def _out(state, **more):
    out = dict(more)
    for key in ("p_flat", "w_flat"):
        if state.get(key) is not None:
            out[key] = state[key]
    return out


def _run_adamw(state):
    s, max_norm = state, state["case"]["max_norm"]
    s["steps"] = steps = [t + 1 for t in s["steps"]]
    out = {}
    if own:
        import muon_b200
        scale = None
        if max_norm:
            out["norm"], scale = muon_b200.grad_norm(s["grads"], max_norm)
        muon_b200.adamw_step(s["p"], s["grads"], s["m"], s["v"], steps, lr=LR, betas=_betas(s), eps=EPS, weight_decay=WD,
                             masters=s["w"], grad_scale=scale)
    else:
        g = _flat(s["grads"]).float()
        if max_norm:
            out["norm"], scale = _norm(g, max_norm)
            g = g * scale
        b1, b2 = _betas(s)
        m = _flat(s["m"]) * b1 + g * (1 - b1)
        v = _flat(s["v"]) * b2 + g * g * (1 - b2)
        p = _moved(_flat(s["w"] or s["p"]).float(), m, v, steps[0], _betas(s))
        _put(s["m"], m.split(s["sizes"]))
        _put(s["v"], v.split(s["sizes"]))
        _put(s["p"], p.split(s["sizes"]))
        if s["w"] is not None:
            _put(s["w"], p.split(s["sizes"]))
    return _out(s, m=s["m_flat"], v=s["v_flat"], **out)


def _run_adamw8(state):
    s, max_norm = state, state["case"]["max_norm"]
    s["steps"] = steps = [t + 1 for t in s["steps"]]
    out = {}
    if own:
        import muon_b200
        scale = None
        if max_norm:
            out["norm"], scale = muon_b200.grad_norm(s["grads"], max_norm)
        muon_b200.adamw8_step(s["p"], s["grads"], s["m_codes"], s["m_scales"], s["v_codes"], s["v_scales"], steps, lr=LR,
                              betas=_betas(s), eps=EPS, weight_decay=WD, masters=s["w"], grad_scale=scale, seed=s["seed"])
    else:
        g = _blocked(s["grads"]).float()
        if max_norm:
            out["norm"], scale = _norm(g, max_norm)
            g = g * scale
        b1, b2 = _betas(s)
        m = _values(s, "m", "exp_avg") * b1 + g * (1 - b1)
        v = _values(s, "v", "exp_avg_sq") * b2 + (g * g) * (1 - b2)
        p = _moved(_blocked(s["w"] or s["p"]).float(), m, v, steps[0], _betas(s))
        _put(s["p"], _unblocked(p, s["sizes"]))
        if s["w"] is not None:
            _put(s["w"], _unblocked(p, s["sizes"]))
        _store(s, "m", m, "exp_avg", None)
        _store(s, "v", v, "exp_avg_sq", _random_bits(s["sizes"], s["seed"], steps[0]))
    _expand(s)
    return _out(s, m=s["m_value"], v=s["v_value"], **out)


def _run_clip(state):
    s, max_norm = state, state["case"]["max_norm"]
    if own:
        import muon_b200
        norm = muon_b200.clip_grad_norm_(s["grads"], max_norm)
    else:
        g = _flat(s["grads"]).float()
        norm, scale = _norm(g, max_norm)
        _put(s["grads"], (g * scale).split(s["sizes"]))
    return dict(norm=norm, grads=s["grad_flat"])


def _run_convert(state):
    s = state
    if own:
        import muon_b200
        muon_b200.quantize_state(s["m"], "exp_avg", codes=s["m_codes"], scales=s["m_scales"])
        muon_b200.quantize_state(s["v"], "exp_avg_sq", codes=s["v_codes"], scales=s["v_scales"])
    else:
        _store(s, "m", _blocked(s["m"]), "exp_avg", None)
        _store(s, "v", _blocked(s["v"]), "exp_avg_sq", 1 << 19)
    _expand(s)
    return dict(m=s["m_value"], v=s["v_value"])


def _run_expand(state):
    _expand(state)
    return dict(m=state["m_value"], v=state["v_value"])


def _expand(s):
    """What the codes stand for: bfloat16 beside a step or a conversion, float32 for a checkpoint."""
    if own:
        import muon_b200
        muon_b200.dequantize_state(s["m_codes"], s["m_scales"], "exp_avg", out=s["m_values"])
        muon_b200.dequantize_state(s["v_codes"], s["v_scales"], "exp_avg_sq", out=s["v_values"])
    else:
        _put(s["m_values"], _unblocked(_values(s, "m", "exp_avg"), s["sizes"]))
        _put(s["v_values"], _unblocked(_values(s, "v", "exp_avg_sq"), s["sizes"]))


# ------------------------------------------------------------------------------------ the plain forms' parts
def _flat(tensors):
    return torch.cat([t.reshape(-1) for t in tensors])


def _blocked(tensors):
    """All tensors as rows of 256, each filled up with zeros."""
    return torch.cat([torch.nn.functional.pad(t.reshape(-1), (0, -t.numel() % BLOCK)) for t in tensors]).view(-1, BLOCK)


def _unblocked(x, sizes):
    return [c[:n] for c, n in zip(x.reshape(-1).split([-(-n // BLOCK) * BLOCK for n in sizes]), sizes)]


def _put(tensors, values):
    [t.copy_(x) for t, x in zip(tensors, values)]


def _norm(g, max_norm):
    """Norm (summed in 64 bits: many elements) and the factor that brings it down to max_norm."""
    norm = g.double().square().sum().sqrt().float()
    return norm, (max_norm / (norm + 1e-6)).clamp(max=1.0)


def _moved(p, m, v, step, betas):
    c1, c2 = 1 - betas[0] ** step, 1 - betas[1] ** step
    return p * (1 - LR * WD) - (LR / c1) * (m / (v.sqrt() * c2 ** -0.5 + EPS))


def _quantize(x, kind, r):
    """Rows of 256 float32 values -> codes and scales; `r`: the 20 random bits of the second moment."""
    amax = x.abs().amax(dim=1)
    top = E4M3_MAX if kind == "exp_avg" else SQ_MAX
    small = amax < TINY[kind]
    scale = torch.where(small, 0.0, amax * (1.0 / top))
    y = x * torch.where(small, 0.0, torch.full_like(amax, top) / amax)[:, None]
    if kind == "exp_avg":
        codes = y.clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn).view(torch.uint8)
    else:
        codes = (((y.contiguous().view(torch.int32).long() + r) >> 20) - 768).clamp(0, 255).to(torch.uint8)
    return torch.where(small[:, None], 0, codes).to(torch.uint8), scale


def _values(s, name, kind):
    codes, scales = _blocked(s[name + "_codes"]), _flat(s[name + "_scales"])
    if kind == "exp_avg":
        return codes.view(torch.float8_e4m3fn).float() * scales[:, None]
    return ((codes.int() + 768) << 20).view(torch.float32) * scales[:, None]


def _store(s, name, x, kind, r):
    codes, scales = _quantize(x, kind, r)
    _put(s[name + "_codes"], _unblocked(codes, s["sizes"]))
    _put(s[name + "_scales"], scales.split([-(-n // BLOCK) for n in s["sizes"]]))


def _random_bits(sizes, seed, step):
    """20 random bits for each element, from its index in its tensor: one 32-bit hash for four elements,
    each taking the low 20 bits of another rotation of it."""
    low = 0xFFFFFFFF
    key = (seed * 0x3C6EF373 + step * 0xBB67AE85) & low
    index = torch.cat([torch.arange(-(-n // BLOCK) * BLOCK, device=_device()) for n in sizes]).view(-1, BLOCK)
    h = ((index >> 2) * 0x9E3779B1 + key) & low
    h = ((h ^ (h >> 16)) * 0x6A09E667) & low
    h = ((h ^ (h >> 15)) * 0xBB67AE85) & low
    h = h ^ (h >> 16)
    turn = (index & 3) * 8
    return ((h >> turn) | (h << (32 - turn))) & 0xFFFFF


# ------------------------------------------------------------------------------------ work, exact values
def work(case):
    sizes, op = _sizes(case), case["op"]
    n, b = sum(sizes), 4 if case["dtype"] == "fp32" else 2
    scales = 4 * sum(-(-k // BLOCK) for k in sizes)
    moved = b + 8 if case["master"] else 2 * b
    return {"adamw": dict(bytes=n * (moved + b + 16), flops=16 * n),
            "adamw8": dict(bytes=n * (moved + b + 4 + 4) + 4 * scales, flops=40 * n),
            "clip": dict(bytes=n * 2 * b, flops=3 * n),
            "convert": dict(bytes=n * 2 * (4 + 1 + 2) + 2 * scales, flops=12 * n),
            "expand": dict(bytes=n * 2 * (1 + 4) + 2 * scales, flops=4 * n)}[op]


def exact(case, seed):
    """The operators from their definitions, tensor by tensor in 64 bits."""
    s = prepare(case, seed)
    op, betas, step = case["op"], _betas(s), FIRST_STEP + 1
    out = {}
    if op == "clip" or (op in ("adamw", "adamw8") and case["max_norm"]):
        norm = math.sqrt(sum(float(g.double().pow(2).sum()) for g in s["grads"]))
        out["norm"] = torch.tensor(norm, dtype=torch.float64)
        factor = min(1.0, case["max_norm"] / (norm + 1e-6))
    else:
        factor = 1.0
    if op == "clip":
        out["grads"] = _wide(s["grad_flat"], s["grads"], [g.double() * factor for g in s["grads"]])
        return out
    if op in ("convert", "expand"):
        for name, kind in (("m", "exp_avg"), ("v", "exp_avg_sq")):
            if op == "convert":
                values = [_exact_rounded(x.double(), kind, 0.5) for x in s[name]]
            else:
                values = [_exact_values(c, k, kind) for c, k in zip(s[name + "_codes"], s[name + "_scales"])]
            out[name] = _wide(s[name + "_value"], s[name + "_values"], values)
        return out
    new = {"p": [], "m": [], "v": []}
    for i, g in enumerate(s["grads"]):
        g = g.double() * factor
        if op == "adamw":
            m, v = s["m"][i].double(), s["v"][i].double()
        else:
            m = _exact_values(s["m_codes"][i], s["m_scales"][i], "exp_avg")
            v = _exact_values(s["v_codes"][i], s["v_scales"][i], "exp_avg_sq")
        m = betas[0] * m + (1 - betas[0]) * g
        v = betas[1] * v + (1 - betas[1]) * g * g
        hat = m / (1 - betas[0] ** step) / ((v / (1 - betas[1] ** step)).sqrt() + EPS)
        p = (s["w"] or s["p"])[i].double()
        new["p"].append(p - LR * WD * p - LR * hat)
        if op == "adamw8":
            m = _exact_rounded(m, "exp_avg", None)
            v = _exact_rounded(v, "exp_avg_sq", _exact_random(v.numel(), s["seed"], step))
        new["m"].append(m)
        new["v"].append(v)
    out["p_flat"] = _wide(s["p_flat"], s["p"], new["p"])
    if s["w"] is not None:
        out["w_flat"] = _wide(s["w_flat"], s["w"], new["p"])
    flat, views = ("_flat", "") if op == "adamw" else ("_value", "_values")
    out["m"] = _wide(s["m" + flat], s["m" + views], new["m"])
    out["v"] = _wide(s["v" + flat], s["v" + views], new["v"])
    return out


def _wide(flat, views, values):
    """A 64-bit copy of a buffer with `values` in the place of its views."""
    out = flat.double()
    for view, x in zip(views, values):
        at = view.storage_offset() - flat.storage_offset()
        out[at:at + view.numel()] = x
    return out


def _exact_values(codes, scales, kind):
    c = codes.double()
    if kind == "exp_avg":
        sign, c = torch.where(c >= 128, -1.0, 1.0), c % 128
        e, f = torch.floor(c / 8), c % 8
        w = sign * torch.where(e == 0, f / 8 * 2.0 ** -6, (1 + f / 8) * 2.0 ** (e - 7))
    else:
        w = (1 + c % 8 / 8) * 2.0 ** (torch.floor(c / 8) - 31)
    return w * scales.double().repeat_interleave(BLOCK)[:c.numel()]


def _exact_rounded(x, kind, u):
    """What the codes of x stand for; u in [0, 1): what is added before the second moment is cut."""
    n = x.numel()
    if n == 0:
        return x
    rows = torch.nn.functional.pad(x, (0, -n % BLOCK)).view(-1, BLOCK)
    amax = rows.abs().amax(dim=1, keepdim=True)
    scale = amax / (E4M3_MAX if kind == "exp_avg" else SQ_MAX)
    y = (rows / torch.where(amax > 0, scale, 1.0)).reshape(-1)[:n]
    scale = torch.where(amax < TINY[kind], 0.0, scale).expand(-1, BLOCK).reshape(-1)[:n]
    if kind == "exp_avg":
        unit = 2.0 ** (torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
        return torch.round(y / unit) * unit * scale
    e = torch.floor(torch.log2(y.clamp(min=2.0 ** -40)))
    e = torch.where(y < 2.0 ** e, e - 1, torch.where(y >= 2.0 ** (e + 1), e + 1, e))
    c = torch.floor(8 * (e + 31) + 8 * (y / 2.0 ** e - 1) + u).clamp(0, 255)
    return (1 + c % 8 / 8) * 2.0 ** (torch.floor(c / 8) - 31) * scale


def _exact_random(n, seed, step):
    """The same 20-bit numbers as a share of 2^20, by 32-bit words held in 64."""
    word, mod = torch.arange(n, device=_device()) // 4, 2 ** 32
    h = (word * 0x9E3779B1 + (seed * 0x3C6EF373 + step * 0xBB67AE85) % mod) % mod
    h = (torch.bitwise_xor(h, h // 2 ** 16) * 0x6A09E667) % mod
    h = (torch.bitwise_xor(h, h // 2 ** 15) * 0xBB67AE85) % mod
    h = torch.bitwise_xor(h, h // 2 ** 16)
    shift = 2 ** (8 * (torch.arange(n, device=_device()) % 4))
    return (h // shift + h * (mod // shift)) % 2 ** 20 / 2.0 ** 20
