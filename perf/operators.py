"""The operators of a training step around the layers' products, as a program uses them.

    listed()             the cases
    draw(rng)            one more case of the same ranges
    prepare(case, seed)  inputs on the GPU, and the optimizer that a program keeps
    run(state)           one pass: in plain torch operations, or (``own``) through the framework's entry points
    work(case)           bytes and flop that the pass cannot do without
    exact(case, seed)    what run() returns for these inputs, from the definition in 64 bits

Two kinds of case:

norm    ``cuda_funcs.residual_norm``: the residual stream x and a block's output f joined and normed,
            h = residual_scale x + block_scale gate N_f(f),    y = N(h),
        forward, or forward and backward.  N, N_f: layer norm or root-mean-square norm with weight and bias.
adamw   ``optim.AdamW.step``: one update of all tensors of a model, moments in 32 or 8 bits, gradients clipped by their
        common norm or not.  The moments are returned as the float32 values they stand for.

The 8-bit moments: 64 consecutive elements of a tensor share a scale 2^(s - 127), s one byte.
  exp_avg     e4m3; the largest finite magnitude of the block is scaled into [128, 256).
  exp_avg_sq  no sign, 5 exponent bits E, 3 mantissa bits M: (8 + M) 2^(E - 33), and M 2^-32 for E = 0; the largest value
              is scaled into [1, 2).  What is not zero does not become zero.
  Both are rounded down or up with the odds of their distance: floor(x / step + u), u = (2 k + 1) / 2^17, k 16 bits of
  a hash of the step's number and of the element's place (low half: exp_avg, high half: exp_avg_sq).
A tensor's elements begin at a multiple of 64 of the group's flat moments.
"""
import math

import torch

own = False

F32, F64 = torch.float32, torch.float64
DTYPE = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
EPS, ALIGN = 1e-5, 64


def _layers(count, dim, ff):
    """Shapes of the tensors of ``count`` transformer layers and a few vectors that no multiple of 64 divides."""
    one = [(dim, dim)] * 4 + [(ff, dim), (dim, ff), (dim,), (dim,), (ff,), (dim - 1,), (3,), (1,)]
    return one * count


# The default regressor: embedding, four layers of width 128 with their value encodings, head (65 tensors, 0.95 M elements)
_REGRESSOR = ([(128, 98)]
              + [(128, 128), (128, 128), (128, 128), (384,), (128,), (8, 16, 64), (8, 16, 64), (8, 16, 64), (8, 16, 64),
                 (128, 128), (128,), (512, 128), (512,), (128, 512), (128,)] * 4
              + [(128, 128), (128,), (1, 128), (1,)])


def listed():
    norm = dict(kind="norm", rows=13, dim=128, dtype="float32", weights="float32", norm="layer", block_norm="", gate="",
                residual_scale=1.0, block_scale=1.0, residual=False, train=False)
    adamw = dict(kind="adamw", model="layers", count=1, dim=128, ff=512, dtype="float32", bits=8, clip=False, steps=1000)
    return [
        # one crystal of 13 atoms through the norm behind a block: a relaxation loop, launches and host time alone
        dict(norm, name="norm_infer_13"),
        # the norm behind a block for the default training batch (256 crystals of 1 to 60 atoms), forward and backward
        dict(norm, name="norm_train_2372", rows=2372, train=True),
        # a prompt of a wide model in serving: residual stream and its root-mean-square norm
        dict(norm, name="norm_infer_wide", rows=4096, dim=5120, dtype="bfloat16", weights="bfloat16", norm="rms", residual=True),
        # pre-norm training with a learned scale per channel on the block, odd row count
        dict(norm, name="norm_train_channel", rows=8190, dim=2048, dtype="bfloat16", norm="rms", gate="channel", residual=True,
             residual_scale=1.0, block_scale=0.22, train=True),
        # norms before and after the block, gated per sequence (8 sequences of 2048): the largest training step of the range
        dict(norm, name="norm_train_sandwich", rows=16384, dim=4096, dtype="bfloat16", weights="bfloat16", norm="rms",
             block_norm="rms", gate="sequence", residual=True, train=True),
        # odd sizes, gated per element, layer norms on both sides
        dict(norm, name="norm_train_odd", rows=1021, dim=1001, dtype="float16", weights="float16", norm="layer", block_norm="layer",
             gate="element", residual=True, residual_scale=0.87, train=True),
        # the default regressor, moments in 8 bits
        dict(adamw, name="adamw_regressor_8", model="regressor", steps=40),
        # the same with the clip that its training step has before the update
        dict(adamw, name="adamw_regressor_8_clip", model="regressor", clip=True, steps=40),
        # first step of a model in bfloat16 with moments in 32 bits
        dict(adamw, name="adamw_bf16_32", count=2, dim=1024, ff=4096, dtype="bfloat16", bits=32, steps=0),
        # the same model, moments in 8 bits, far into training
        dict(adamw, name="adamw_bf16_8", count=2, dim=1024, ff=4096, dtype="bfloat16", bits=8, steps=100000),
        # a step over 151 M float32 parameters, clipped, moments in 8 bits and in 32
        dict(adamw, name="adamw_large_8_clip", count=3, dim=2048, ff=8192, clip=True),
        dict(adamw, name="adamw_large_32_clip", count=3, dim=2048, ff=8192, clip=True, bits=32),
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, spread over the logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    if rng.random() < 0.55:
        dim = _spread(rng, 16, 8192)
        if rng.random() < 0.5:
            dim = max(64, dim // 64 * 64)
        rows = _spread(rng, 1, min(65536, (1 << 26) // dim))
        gate = rng.choice(["", "channel", "sequence", "element"])
        if gate == "sequence":
            rows = max(4, rows // 4 * 4)
        dtype = rng.choice(["float32", "bfloat16", "float16"])
        return dict(kind="norm", rows=rows, dim=dim, dtype=dtype, weights=rng.choice(["float32", dtype]),
                    norm=rng.choice(["layer", "rms"]), block_norm=rng.choice(["", "", "layer", "rms"]), gate=gate,
                    residual_scale=rng.choice([1.0, 1.0, round(rng.uniform(0.5, 3.0), 3)]),
                    block_scale=rng.choice([1.0, 1.0, round(rng.uniform(0.1, 1.0), 3)]),
                    residual=rng.random() < 0.6, train=rng.random() < 0.65)
    model = rng.choice(["regressor", "layers", "layers", "layers"])
    dim = _spread(rng, 64, 2048)
    return dict(kind="adamw", model=model, count=rng.choice([1, 2, 3]) if dim < 1500 else 1, dim=dim,
                ff=rng.choice([dim * 4, dim * 3 + rng.randrange(64)]), dtype=rng.choice(["float32", "bfloat16", "float16"]),
                bits=rng.choice([8, 8, 32]), clip=rng.random() < 0.5, steps=_spread(rng, 1, 200000) - 1)


# ------------------------------------------------------------------------------------------------ inputs
def _gate_rows(case):
    return {"": 0, "channel": 1, "element": case["rows"],
            "sequence": 8 if case["rows"] % 8 == 0 else 4}[case["gate"]]


def _shapes(case):
    return _REGRESSOR if case["model"] == "regressor" else _layers(case["count"], case["dim"], case["ff"])


def _offsets(shapes):
    """Where each tensor begins in the flat moments, and how long these are."""
    at, offs = 0, []
    for shape in shapes:
        offs.append(at)
        at += -(-math.prod(shape) // ALIGN) * ALIGN
    return offs, at


def _prepare_norm(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    dt, wt, N, D = DTYPE[case["dtype"]], DTYPE[case["weights"]], case["rows"], case["dim"]
    new = lambda *shape, at=0.0, by=1.0, to=dt: (at + by * torch.randn(*shape, generator=gen, device=dev)).to(to)  # noqa: E731
    G = _gate_rows(case)
    # tokens of one sequence have something in common, channels differ in size, and a stream grows along the layers
    channel = torch.exp(0.5 * torch.randn(D, generator=gen, device=dev))
    x = ((torch.randn(N, D, generator=gen, device=dev) + 0.3 * torch.randn(D, generator=gen, device=dev)) * channel * 2.0).to(dt)
    f = new(N, D, at=0.1, by=1.3)
    s = dict(case=case, x=x, f=f, gate=None, weight=new(D, at=1.0, by=0.1, to=wt), bias=None, block_weight=None, block_bias=None)
    if case["norm"] == "layer":
        s["bias"] = new(D, by=0.1, to=wt)
    if case["block_norm"]:
        s["block_weight"] = new(D, at=1.0, by=0.1, to=wt)
        s["block_bias"] = new(D, by=0.1, to=wt) if case["block_norm"] == "layer" else None
    if G == 1:
        s["gate"] = new(D, at=0.5, by=0.2)
    elif G == N:
        s["gate"] = new(N, D, at=0.5, by=0.5)
    elif G:      # a program's layout: sequences, positions, channels
        s["gate"] = new(G, 1, D, at=0.5, by=0.5)
        s["x"], s["f"] = s["x"].view(G, N // G, D), s["f"].view(G, N // G, D)
    if case["train"]:
        s["gy"] = new(*s["x"].shape, by=0.5)
        s["gh"] = new(*s["x"].shape, by=0.5) if case["residual"] else None
        for k in _LEAVES:
            if s[k] is not None:
                s[k].requires_grad_(True)
    return s


_LEAVES = ("x", "f", "gate", "weight", "bias", "block_weight", "block_bias")


def _prepare_adamw(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    dt, shapes = DTYPE[case["dtype"]], _shapes(case)
    offs, total = _offsets(shapes)
    normal = lambda: torch.randn(total, generator=gen, device=dev)  # noqa: E731
    # gradients of a tensor's rows differ in size by some powers of ten, as those of rare features and dead units do
    size = 10.0 ** (torch.rand(total // ALIGN, generator=gen, device=dev) * 3.0 - 5.0)
    size = size.repeat_interleave(ALIGN)
    live = torch.zeros(total, dtype=torch.bool, device=dev)
    for o, shape in zip(offs, shapes):
        live[o:o + math.prod(shape)] = True
    p = (normal() * 0.05).mul_(live).to(dt)
    g = (normal() * size).mul_(live).to(dt)
    m = v = None
    if case["steps"]:
        m = (normal() * size * 0.3).mul_(live)
        v = (normal() * size).square_().add_(0.1 * size * size).mul_(live)
    else:
        m, v = torch.zeros(total, device=dev), torch.zeros(total, device=dev)
    # the norm of the gradients is about twice what they are clipped to
    s = dict(case=case, p=p, g=g, t=case["steps"], lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01,
             max_norm=0.5 * float(g.double().norm()) if case["clip"] else None)
    if case["bits"] == 8:
        half = torch.full((total // ALIGN, ALIGN), 0.5, dtype=F64, device=dev)
        s["m"], s["m_scale"] = _encode_m(m.double().view(-1, ALIGN), half)
        s["v"], s["v_scale"] = _encode_v(v.double().view(-1, ALIGN), half)
    else:
        s["m"], s["v"] = m, v
    if own:
        s["optimizer"] = _optimizer(s, shapes, offs)
    return s


def _optimizer(s, shapes, offs):
    """The optimizer of a program in the midst of training: made as always, its state loaded as from a checkpoint."""
    from crystalframer_amd import optim
    part = lambda t, o, shape: t[o:o + math.prod(shape)].view(shape)  # noqa: E731
    params = []
    for o, shape in zip(offs, shapes):
        params.append(torch.nn.Parameter(part(s["p"], o, shape)))
        params[-1].grad = part(s["g"], o, shape)
    case = s["case"]
    opt = optim.AdamW(params, lr=s["lr"], betas=s["betas"], eps=s["eps"], weight_decay=s["weight_decay"],
                      state_bits=case["bits"], max_grad_norm=s["max_norm"])
    state, step = {}, torch.tensor([s["t"]])
    for k, (o, shape) in enumerate(zip(offs, shapes)):
        state[k] = dict(step=step, exp_avg=part(s["m"], o, shape), exp_avg_sq=part(s["v"], o, shape))
        if case["bits"] == 8:
            blocks = slice(o // ALIGN, o // ALIGN + -(-math.prod(shape) // ALIGN))
            state[k].update(exp_avg_scale=s["m_scale"][blocks], exp_avg_sq_scale=s["v_scale"][blocks])
    whole = opt.state_dict()
    whole["state"] = state
    opt.load_state_dict(whole)
    return opt


def prepare(case, seed):
    return _prepare_norm(case, seed) if case["kind"] == "norm" else _prepare_adamw(case, seed)


# ------------------------------------------------------------------------------------------------ passes
def run(state):
    if state["case"]["kind"] == "norm":
        return _own_norm(state) if own else _plain_norm(state)
    return _own_adamw(state) if own else _plain_adamw(state)


def _own_norm(s):
    from crystalframer_amd import cuda_funcs
    case = s["case"]
    if not case["train"]:
        with torch.no_grad():
            out = _own_norm_forward(cuda_funcs, s)
        return dict(zip(("h", "y"), out)) if case["residual"] else dict(y=out)
    out = _own_norm_forward(cuda_funcs, s)
    leaves = [k for k in _LEAVES if s[k] is not None]
    outs, gs = (out, (s["gh"], s["gy"])) if case["residual"] else ((out,), (s["gy"],))
    grads = torch.autograd.grad(outs, [s[k] for k in leaves], gs)
    return dict(zip(("h", "y") if case["residual"] else ("y",), (o.detach() for o in outs)),
                **{"grad_" + k: g for k, g in zip(leaves, grads)})


def _own_norm_forward(cuda_funcs, s):
    case = s["case"]
    return cuda_funcs.residual_norm(
        s["x"], s["f"], s["weight"], s["bias"], norm=case["norm"], eps=EPS, gate=s["gate"], residual_scale=case["residual_scale"],
        block_scale=case["block_scale"], block_norm=case["block_norm"] or None, block_weight=s["block_weight"],
        block_bias=s["block_bias"], block_eps=EPS, keep_residual=case["residual"])


def _own_adamw(s):
    opt = s["optimizer"]
    opt.step()
    (m, v), = opt.moments()
    out = dict(params=s["p"], exp_avg=m, exp_avg_sq=v)
    if s["max_norm"] is not None:
        out["grad_norm"] = opt.grad_norm
    return out


def _plain_one_norm(h, kind, weight, bias):
    if kind == "layer":
        h = h - h.mean(-1, keepdim=True)
    y = h * torch.rsqrt((h * h).mean(-1, keepdim=True) + EPS) * weight
    return y if bias is None else y + bias


def _plain_norm(s):
    case, dt = s["case"], s["x"].dtype
    t = {k: None if s[k] is None else s[k].detach().to(F32, copy=True).requires_grad_(case["train"]) for k in _LEAVES}
    a = _plain_one_norm(t["f"], case["block_norm"], t["block_weight"], t["block_bias"]) if case["block_norm"] else t["f"]
    if t["gate"] is not None:
        a = a * t["gate"]
    h = case["residual_scale"] * t["x"] + case["block_scale"] * a
    y = _plain_one_norm(h, case["norm"], t["weight"], t["bias"])
    out = dict(h=h.detach().to(dt), y=y.detach().to(dt)) if case["residual"] else dict(y=y.detach().to(dt))
    if case["train"]:
        leaves = [k for k in _LEAVES if t[k] is not None]
        outs, gs = ((h, y), (s["gh"].float(), s["gy"].float())) if case["residual"] else ((y,), (s["gy"].float(),))
        grads = torch.autograd.grad(outs, [t[k] for k in leaves], gs)
        out.update({"grad_" + k: g.to(s[k].dtype) for k, g in zip(leaves, grads)})
    return out


def _times(x, e):
    """x 2^e; the power is put together from its bits, so that nothing is rounded."""
    return x * (torch.as_tensor(e).to(torch.int64) + 1023 << 52).view(F64)


# A code of 8 bits without its sign: E = code >> 3, M = code & 7; ``low``: the exponent of the smallest normal value (E = 1).
def _decode(code, low):
    code = code.to(torch.int64)
    E = code >> 3
    return _times(((code & 7) + torch.where(E > 0, 8, 0)).to(F64), torch.clamp_min(E, 1) - 1 + low - 3)


def _encode(x, scale, low, u):
    t = _times(x, -scale)
    e = torch.where(t > 0, torch.clamp_min(torch.frexp(t).exponent - 1, low), low)
    return ((e - low) * 8 + torch.floor(_times(t, 3 - e) + u)).to(torch.int64)


def _scale(x, top):
    """Exponents that bring the largest of each row of ``x`` into [2^top, 2^(top + 1))."""
    largest = x.amax(1, keepdim=True)
    e = torch.clamp(torch.frexp(largest).exponent - 1 - top, -127, 127)
    return torch.where(largest > 0, e, -127)


def _encode_m(m, u):
    scale = _scale(m.abs(), 7)
    code = _encode(m.abs(), scale, -6, u) | torch.where(torch.signbit(m), 128, 0)
    return code.to(torch.uint8).view(-1).view(torch.float8_e4m3fn), (scale + 127).to(torch.uint8).view(-1)


def _encode_v(v, u):
    scale = _scale(v, 0)
    code = _encode(v, scale, -29, u)
    code = torch.where((v > 0) & (code == 0), 1, code)
    return code.to(torch.uint8).view(-1), (scale + 127).to(torch.uint8).view(-1)


def _value_m(code, scale):
    code = code.view(torch.uint8).view(-1, ALIGN).to(torch.int64)
    return _times(_decode(code & 127, -6), scale.to(torch.int64)[:, None] - 127) * torch.where(code > 127, -1.0, 1.0)


def _value_v(code, scale):
    return _times(_decode(code.view(-1, ALIGN), -29), scale.to(torch.int64)[:, None] - 127)


def _fractions(t, n, dev):
    """u of exp_avg and of exp_avg_sq for the elements 0 ... n - 1 in step ``t``."""
    mask = 0xffffffff
    k = t * 0x6A09E667 & mask
    k = (k ^ k >> 15) * 0x9E3779B1 & mask
    k ^= k >> 16
    x = torch.arange(n, device=dev) * 0x9E3779B1 + k & mask
    x = (x ^ x >> 16) * 0xBB67AE85 & mask
    x ^= x >> 15
    return tuple((2 * y + 1).to(F64).mul_(2.0 ** -17).view(-1, ALIGN) for y in (x & 0xffff, x >> 16))


def _plain_adamw(s):
    (b1, b2), eight = s["betas"], s["case"]["bits"] == 8
    s["t"] += 1
    g = s["g"].to(F64 if eight else F32)
    if s["max_norm"] is not None:
        norm = s["g"].double().square().sum().sqrt()
        g = g * torch.clamp_max(s["max_norm"] / (norm + 1e-6), 1.0).to(F32)
    if eight:       # in 64 bits: a moment next to a border between two codes goes the same way wherever it is computed
        g = g.view(-1, ALIGN)
        m = b1 * _value_m(s["m"], s["m_scale"]) + (1 - b1) * g
        v = b2 * _value_v(s["v"], s["v_scale"]) + (1 - b2) * g * g
        um, uv = _fractions(s["t"], g.numel(), g.device)
        s["m"], s["m_scale"] = _encode_m(m, um)
        s["v"], s["v_scale"] = _encode_v(v, uv)
        new_m, new_v = (x.float().view(-1) for x in (_value_m(s["m"], s["m_scale"]), _value_v(s["v"], s["v_scale"])))
        m, v = m.float().view(-1), v.float().view(-1)
    else:
        new_m = m = s["m"].mul_(b1).add_((1 - b1) * g)
        new_v = v = s["v"].mul_(b2).add_((1 - b2) * g * g)
    c1, c2 = -math.expm1(s["t"] * math.log(b1)), -math.expm1(s["t"] * math.log(b2))
    p = s["p"].float() * (1 - s["lr"] * s["weight_decay"])
    p = p - s["lr"] / c1 * m / (torch.sqrt(v) / math.sqrt(c2) + s["eps"])
    s["p"].copy_(p)
    out = dict(params=s["p"], exp_avg=new_m, exp_avg_sq=new_v)
    if s["max_norm"] is not None:
        out["grad_norm"] = norm.to(F32)
    return out


# ------------------------------------------------------------------------------------------------ what a pass needs
def work(case):
    size = lambda t: DTYPE[t].itemsize  # noqa: E731
    if case["kind"] == "norm":
        N, D, G = case["rows"], case["dim"], _gate_rows(case)
        arrays = 3 + case["residual"]                                            # x, f; y and h
        flops = 10 + (8 if case["block_norm"] else 0) + (1 if G else 0)
        vectors = 1 + (case["norm"] == "layer") + (1 + (case["block_norm"] == "layer") if case["block_norm"] else 0)
        if case["train"]:
            arrays += 3 + case["residual"]                                       # gy and gh; gradients of x and f
            flops *= 3
        ways = 2 if case["train"] else 1
        return {"bytes": (arrays * N + ways * G) * D * size(case["dtype"]) + ways * vectors * D * size(case["weights"]),
                "flops": flops * N * D}
    n = sum(math.prod(shape) for shape in _shapes(case))
    moments = 4 + 4 / ALIGN + 8 if case["bits"] == 8 else 16       # read, written; those of 8 bits returned in 32 as well
    return {"bytes": int(n * (3 * size(case["dtype"]) + moments)), "flops": (16 + 2 * case["clip"]) * n}


# ------------------------------------------------------------------------------------------------ the definition in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return _exact_norm(s) if case["kind"] == "norm" else _exact_adamw(s)


def _exact_normed(h, kind, weight, bias):
    """y, and what its derivative needs: the normed rows and one over their deviation."""
    centre = h.mean(-1, keepdim=True) if kind == "layer" else 0.0
    spread = ((h - centre).square().mean(-1, keepdim=True) + EPS).sqrt()
    unit = (h - centre) / spread
    return unit * weight + (0.0 if bias is None else bias), unit, 1.0 / spread


def _exact_back(g, kind, weight, unit, inverse):
    """Gradients of the normed rows' input, of weight and of bias for the gradient ``g`` of y."""
    rows = tuple(range(g.dim() - 1))
    u = g * weight
    d = u - unit * (u * unit).mean(-1, keepdim=True)
    if kind == "layer":
        d = d - u.mean(-1, keepdim=True)
    return d * inverse, (g * unit).sum(rows), g.sum(rows)


def _exact_norm(s):
    case = s["case"]
    x, f, gate, w, b, wf, bf = (None if s[k] is None else s[k].detach().to(F64) for k in _LEAVES)
    a = f
    if case["block_norm"]:
        a, unit_f, inverse_f = _exact_normed(f, case["block_norm"], wf, bf)
    alpha, beta = case["residual_scale"], case["block_scale"]
    h = alpha * x + beta * (a if gate is None else gate * a)
    y, unit, inverse = _exact_normed(h, case["norm"], w, b)
    out = dict(h=h, y=y) if case["residual"] else dict(y=y)
    if not case["train"]:
        return out
    dh, dw, db = _exact_back(s["gy"].to(F64), case["norm"], w, unit, inverse)
    if case["residual"]:
        dh = dh + s["gh"].to(F64)
    da = beta * dh if gate is None else beta * gate * dh
    out.update(grad_x=alpha * dh, grad_weight=dw)
    if gate is not None:
        dg = beta * a * dh
        out["grad_gate"] = dg.sum(0) if gate.dim() == 1 else dg.sum(1, keepdim=True) if gate.dim() == 3 else dg
    if b is not None:
        out["grad_bias"] = db
    out["grad_f"] = da
    if case["block_norm"]:
        out["grad_f"], out["grad_block_weight"], dbf = _exact_back(da, case["block_norm"], wf, unit_f, inverse_f)
        if bf is not None:
            out["grad_block_bias"] = dbf
    return out


def _exact_table(codes, low):
    """The values of the first ``codes`` codes."""
    return torch.tensor([(c % 8 + 8 * (c >= 8)) * 2.0 ** (max(c // 8, 1) - 1 + low - 3) for c in range(codes)], dtype=F64, device="cuda")


def _exact_units(largest, top):
    """The powers of two, 2^-127 to 2^127, that bring ``largest`` into [2^top, 2^(top + 1)) or as near as they can."""
    powers = torch.tensor([2.0 ** e for e in range(-127, 128)], dtype=F64, device="cuda")
    return powers[torch.searchsorted(powers * 2.0 ** top, largest.contiguous(), right=True).sub(1).clamp_min(0)]


def _exact_rounded(x, table, top, u):
    """x (blocks, 64), not negative, as the 8 bits hold it: the block's scale, and of the two values of the table around it
    the upper one where its share of the way reaches 1 - u."""
    largest = x.amax(1, keepdim=True)
    unit = _exact_units(largest, top)
    t = x / unit
    at = torch.searchsorted(table, t.contiguous(), right=True) - 1
    under, over = table[at], table[at + 1]
    return torch.where((t - under) / (over - under) + u >= 1.0, over, under) * unit


def _exact_fractions(t, n):
    import numpy as np
    A, B, C = np.uint32(0x9E3779B1), np.uint32(0xBB67AE85), np.uint32(0x6A09E667)
    with np.errstate(over="ignore"):
        k = np.array([t & 0xffffffff], dtype=np.uint32) * C
        k = (k ^ (k >> np.uint32(15))) * A
        k = k ^ (k >> np.uint32(16))
        x = np.arange(n, dtype=np.uint32) * A + k
        x ^= x >> np.uint32(16)
        x *= B
        x ^= x >> np.uint32(15)
    both = [torch.from_numpy(y.astype(np.uint16).view(np.int16)).cuda().to(torch.int32) & 0xffff for y in (x, x >> np.uint32(16))]
    return [((y.to(F64) + 0.5) / 65536).view(-1, ALIGN) for y in both]


def _exact_adamw(s):
    (b1, b2), t = s["betas"], s["t"] + 1
    g = s["g"].to(F64)
    norm = torch.linalg.vector_norm(g)
    if s["max_norm"] is not None:      # the factor is held in 32 bits: the 8-bit moments go by it
        g = g * min(1.0, float(torch.tensor(s["max_norm"] / (float(norm) + 1e-6), dtype=F32)))
    if s["case"]["bits"] == 8:
        low, high = _exact_table(128, -6), _exact_table(256, -29)
        blocks = lambda c: c.view(torch.uint8).long().view(-1, ALIGN)  # noqa: E731
        powers = torch.tensor([2.0 ** (e - 127) for e in range(255)], dtype=F64, device="cuda")
        unit = lambda c: powers[c.long()][:, None]  # noqa: E731
        old = blocks(s["m"])
        m = (torch.where(old < 128, low[old % 128], -low[old % 128]) * unit(s["m_scale"])).view(-1)
        v = (high[blocks(s["v"])] * unit(s["v_scale"])).view(-1)
    else:
        m, v = s["m"].to(F64), s["v"].to(F64)
    m = m * b1 + g * (1 - b1)
    v = v * b2 + g.square() * (1 - b2)
    p = s["p"].to(F64) * (1 - s["lr"] * s["weight_decay"])
    p -= s["lr"] * (m / (1 - b1 ** t)) / ((v / (1 - b2 ** t)).sqrt() + s["eps"])
    if s["case"]["bits"] == 8:
        um, uv = _exact_fractions(t, m.numel())
        m = torch.copysign(_exact_rounded(m.abs().view(-1, ALIGN), low, 7, um).view(-1), m)
        w = _exact_rounded(v.view(-1, ALIGN), high, 0, uv)
        least = _exact_units(v.view(-1, ALIGN).amax(1, keepdim=True), 0) * high[1]
        v = torch.where((v.view(-1, ALIGN) > 0) & (w == 0), least, w).view(-1)
    out = dict(params=p, exp_avg=m, exp_avg_sq=v)
    if s["max_norm"] is not None:
        out["grad_norm"] = norm
    return out
