"""``cuda_funcs.residual_norm`` against float64: values and all gradients, over types, sizes, gates, strides.

Tolerances count roundings.  A result is rounded once to its type (half a unit) and computed in float32 from terms of some
magnitude: sums over D or N terms run over at most 16 consecutive additions per lane and then trees, and what is summed has
been through a dozen operations, so that 64 roundings (2^-24 each) of the largest magnitude cover a value.  Magnitudes: of y and of
the gradients of rows the largest |term| of the row's formula, of column sums the sum of the terms' magnitudes."""
import pytest
import torch

import training_reference as TR

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _make(shape, dtype, wtype, norm, block_norm, gate, block=True, seed=0, offset=0.3, biases=False):
    gen = torch.Generator().manual_seed(seed)
    D = shape[-1]
    rnd = lambda s, at, by, t: (at + by * torch.randn(s, generator=gen)).to(t)  # noqa: E731
    k = dict(x=rnd(shape, offset, 1.5, dtype))
    if block:
        k["block"] = rnd(shape, 0.1, 0.8, dtype)
    if gate is not None:
        k["gate"] = rnd(gate, 0.6, 0.5, dtype)
    if norm:
        k["weight"] = rnd((D,), 1.0, 0.2, wtype)
        if norm == "layer" or biases:
            k["bias"] = rnd((D,), 0.0, 0.2, wtype)
    if block_norm:
        k["block_weight"] = rnd((D,), 1.0, 0.2, wtype)
        if block_norm == "layer" or biases:
            k["block_bias"] = rnd((D,), 0.0, 0.2, wtype)
    return k, gen


def _check(got, ref, size, what):
    got = got.detach().cpu().double()
    tol = TR.tolerance(ref, what[1], size)
    bad = (got - ref).abs() > tol
    assert got.shape == ref.shape and not bad.any(), (what, float(((got - ref).abs() / tol).max()))


def _compare(shape, dtype, wtype=None, norm="layer", block_norm=None, gate=None, keep=True, block=True, scales=(1.0, 1.0), eps=1e-5,
             seed=0, place=lambda name, t: t.cuda(), train=True, biases=False):
    from crystalframer_amd import cuda_funcs
    wtype = wtype or dtype
    tensors, gen = _make(shape, dtype, wtype, norm, block_norm, gate, block, seed, biases=biases)
    opts = dict(norm=norm, eps=eps, residual_scale=scales[0], block_scale=scales[1], block_norm=block_norm, block_eps=eps)
    dev = {k: place(k, t).requires_grad_(train) for k, t in tensors.items()}
    ref = {k: t.double().requires_grad_(train) for k, t in tensors.items()}
    out = cuda_funcs.residual_norm(**dev, **opts, keep_residual=keep)
    h, y = TR.residual_norm(**ref, **opts)
    outs, refs = ((out,), (h if norm is None else y,)) if norm is None or not keep else (out, (h, y))
    D = shape[-1]
    rows = lambda t: t.detach().abs().amax(-1, keepdim=True)  # noqa: E731
    wmax = ref["weight"].detach().abs().max() if norm else 1.0
    terms = rows(scales[0] * ref["x"])
    ra = hat_a = None
    if block:
        a = ref["block"]
        if block_norm:
            a, hat_a, ra = TR.norm_forward(ref["block"], block_norm, ref["block_weight"], ref.get("block_bias"), eps)
            size_a = (rows(ref["block"]) * ra.detach() + 1) * ref["block_weight"].detach().abs().max() + 0.5
        else:
            size_a = rows(a)
        gmax = ref["gate"].detach().abs().max() if gate is not None else 1.0
        terms = terms + abs(scales[1]) * gmax * size_a
    sizes = [terms]
    hat = r = None
    if norm:
        _, hat, r = TR.norm_forward(h.detach(), norm, None, None, eps)
        # errors of h are carried by r; layer norm's mean is subtracted from values of size |h|
        sizes.append((terms * r * wmax + 1.0) * (1.0 + rows(hat) / max(D, 1) ** 0.5))
    sizes = [sizes[-1]] if not keep else sizes
    for o, e, s, n in zip(outs, refs, sizes, ("h", "y")):
        _check(o, e.detach(), s, (n, dtype))
        assert o.dtype == dtype
    if not train:
        return
    gs = [(0.1 + torch.randn(shape, generator=gen)).to(dtype) for _ in outs]
    leaves = list(dev)
    got = torch.autograd.grad(outs, [dev[k] for k in leaves], [g.cuda() for g in gs])
    want = torch.autograd.grad(refs, [ref[k] for k in leaves], [g.double() for g in gs])
    gh = gs[0].double() if keep or norm is None else torch.zeros(shape).double()
    gy = gs[-1].double() if norm else None
    size_h = rows(gh)
    if norm:
        u = rows(gy) * wmax
        err_hat = 1.0 + terms * r          # what a rounding of h makes of a normed value
        size_h = size_h + r * u * (1 + rows(hat)) * err_hat
    size_a_grad = size_h
    sums = dict(x=abs(scales[0]) * size_h)
    N = gh.numel() // D
    flat = lambda t, w=D: (t + torch.zeros(shape, dtype=torch.float64)).reshape(N, D)  # noqa: E731
    if block:
        size_da = abs(scales[1]) * gmax * size_h
        sums["block"] = size_da
        if gate is not None:
            per = abs(scales[1]) * size_h * size_a + torch.zeros(shape, dtype=torch.float64)
            G = ref["gate"].shape
            sums["gate"] = per if G == tuple(shape) else per.reshape(-1, D).sum(0) if len(G) == 1 else \
                per.reshape(*G[:sum(1 for a, b in zip(G[:-1], shape) if a == b)], -1, D).sum(-2).reshape(G)
        if block_norm:
            wa = ref["block_weight"].detach().abs().max()
            err_a = 1.0 + rows(ref["block"]) * ra.detach()
            sums["block"] = ra.detach() * size_da * wa * (1 + rows(hat_a)) * err_a
            sums["block_weight"] = flat(size_da * (rows(hat_a) + err_a)).sum(0)
            sums["block_bias"] = flat(size_da).sum(0)
    if norm:
        sums["weight"] = flat(rows(gy) * (rows(hat) + err_hat)).sum(0)
        sums["bias"] = flat(rows(gy)).sum(0)
    for k, g, w in zip(leaves, got, want):
        assert g.dtype == dev[k].dtype
        _check(g, w, sums[k], ("gradient of " + k, g.dtype))


SIZES = [(1, 1), (3, 2), (5, 3), (1, 17), (2, 63), (7, 64), (65, 65), (13, 127), (300, 128), (33, 129), (4, 255), (70, 256), (9, 511),
         (17, 513), (6, 1000), (5, 1001), (3, 1024), (3, 2047), (2, 2049), (5, 4096), (2, 4100), (1, 8192), (3, 8200), (2, 12288), (2, 12345), (2, 16384)]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("shape", SIZES, ids=str)
def test_sizes(shape, dtype):
    _compare(shape, dtype, norm="layer", seed=1)
    _compare(shape, dtype, wtype=F32, norm="rms", block_norm="layer", gate=(shape[-1],), seed=2)
    _compare(shape, dtype, norm="layer", block_norm="rms", gate=shape, scales=(0.7, 1.3), seed=3)


@pytest.mark.parametrize("dtype,wtype", [(F32, F32), (BF16, BF16), (BF16, F32), (F16, F32)])
@pytest.mark.parametrize("gate", [None, (96,), (6, 1, 96), (6, 10, 96), (1, 1, 96)])
@pytest.mark.parametrize("norm,block_norm", [("layer", None), ("rms", None), ("layer", "layer"), ("rms", "rms"), (None, "layer"), (None, None)])
def test_forms(norm, block_norm, gate, dtype, wtype):
    for keep in (True, False) if norm else (True,):
        _compare((6, 10, 96), dtype, wtype, norm, block_norm, gate, keep, scales=(1.0, 0.22))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_without_a_block(dtype):
    for norm in ("layer", "rms"):
        for keep in (True, False):
            _compare((19, 200), dtype, norm=norm, block=False, keep=keep)
    _compare((19, 200), dtype, norm="layer", block=False, keep=True, scales=(0.5, 1.0))


@pytest.mark.parametrize("rows,dim", [(5000, 128), (2049, 1024), (1500, 40)])
@pytest.mark.parametrize("gate", ["channel", "sequence"])
def test_many_rows(rows, dim, gate):
    """Sums over rows that take several workgroups, with gates that end inside and between them."""
    shape = (rows, dim) if gate == "channel" or rows % 3 else (rows // 500, 500, dim)
    if gate == "sequence" and len(shape) == 2:
        shape = (3, rows // 3, dim)
    g = (dim,) if gate == "channel" else (shape[0], 1, dim)
    _compare(shape, F32, norm="layer", block_norm="rms", gate=g)
    _compare(shape, BF16, norm="rms", gate=g, wtype=F32)


def test_many_short_sequences():
    _compare((700, 2, 72), F32, norm="layer", gate=(700, 1, 72))
    _compare((350, 3, 2, 72), F32, norm="layer", gate=(350, 3, 1, 72))
    _compare((350, 3, 2, 72), F32, norm="layer", gate=(350, 1, 1, 72))


@pytest.mark.parametrize("dim", [1032, 2048])
def test_short_sequences_of_long_rows(dim):
    """More rows of a gate than workgroups that add them, in rows whose column sums have a kernel of their own."""
    _compare((700, 2, dim), BF16, norm="layer", block_norm="layer", gate=(700, 1, dim))
    _compare((90, 3, dim), F16, F32, norm="layer", block_norm="layer", gate=(90, 1, dim))
    _compare((350, 3, dim), F16, F32, norm="layer", block_norm="layer", gate=(350, 1, dim))
    _compare((130, 3, 16384), BF16, norm="rms", gate=(130, 1, 16384))


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("dim", [1000, 1001, 1024, 5000])
def test_gates_over_many_rows_of_16_bits(dim, dtype):
    """Column sums in a kernel of their own (from 2^20 elements on), for each kind of gate and mixture of norms."""
    rows = (1 << 20) // dim // 2 + 1
    for gate in ((dim,), (2, rows, dim), (2, 1, dim)):
        _compare((2, rows, dim), dtype, norm="layer", block_norm="layer", gate=gate, keep=dim % 2 == 0)
        _compare((2, rows, dim), dtype, F32, norm="rms", block_norm="layer", gate=gate)
        _compare((2, rows, dim), dtype, norm=None, block_norm="layer", gate=gate)


def test_more_sequences_than_a_grid_is_high():
    from crystalframer_amd import cuda_funcs
    B, S, D = 66000, 2, 1032
    gen = torch.Generator(device="cuda").manual_seed(3)
    rnd = lambda s, at, by: (at + by * torch.randn(s, generator=gen, device="cuda", dtype=BF16))  # noqa: E731
    t = dict(x=rnd((B, S, D), 0.3, 1.5), block=rnd((B, S, D), 0.1, 0.8), gate=rnd((B, 1, D), 0.6, 0.5), weight=rnd((D,), 1.0, 0.2), bias=rnd((D,), 0.0, 0.2),
             block_weight=rnd((D,), 1.0, 0.2), block_bias=rnd((D,), 0.0, 0.2))
    t = {k: v.requires_grad_() for k, v in t.items()}
    gy = rnd((B, S, D), 0.1, 1.0)
    y = cuda_funcs.residual_norm(**t, block_norm="layer", keep_residual=False)
    dg, dx, db = torch.autograd.grad(y, (t["gate"], t["x"], t["bias"]), gy)
    _check(db, gy.cpu().double().sum((0, 1)), gy.abs().sum((0, 1), dtype=torch.float32).cpu().double(), ("gradient of bias", BF16))
    for part in (slice(0, 5), slice(65530, 65540), slice(B - 5, B)):
        ref = {k: (v.detach()[part] if v.dim() == 3 else v.detach()).cpu().double().requires_grad_() for k, v in t.items()}
        h, ry = TR.residual_norm(**ref, block_norm="layer")
        wg, wx = torch.autograd.grad(ry, (ref["gate"], ref["x"]), gy[part].cpu().double())
        # normed values to 5 deviations, weights to 2, deviations of h from a half on: terms of dh below 2 * 2 * 5 * (1 + 5), of the gate's 10 such
        _check(dx[part], wx, 120.0, ("gradient of x", BF16))
        _check(dg[part], wg, 2 * 10 * 120.0, ("gradient of gate", BF16))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("dim", [96, 1032, 16384])
def test_biases_beside_root_mean_squares(dim, dtype):
    """Also where their gradients are not wanted: the others' are the same, bit for bit."""
    from crystalframer_amd import cuda_funcs
    shape, opts = (9, 4, dim), dict(norm="rms", block_norm="rms")
    _compare(shape, dtype, gate=(9, 1, dim), biases=True, **opts)
    for given in (("bias",), ("block_bias",), ("bias", "block_bias")):
        t, gen = _make(shape, dtype, dtype, "rms", "rms", (9, 1, dim), biases=True)
        t = {k: v.cuda() for k, v in t.items() if k not in ("bias", "block_bias") or k in given}
        g = torch.randn(shape, generator=gen).to(dtype).cuda()
        grads = []
        for frozen in ((), given):
            dev = {k: v.detach().clone().requires_grad_(k not in frozen) for k, v in t.items()}
            wanted = [k for k in t if k not in given]
            grads.append(torch.autograd.grad(cuda_funcs.residual_norm(**dev, **opts, keep_residual=False), [dev[k] for k in wanted], g))
        assert all(torch.equal(a, b) for a, b in zip(*grads)), given


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_layouts(dtype):
    """Rows with gaps between them, addresses off every alignment, transposed and expanded tensors."""
    def gaps(name, t):
        if t.dim() == 1:
            return torch.cat([t.new_zeros(3), t]).cuda()[3:]
        big = t.new_zeros(t.shape[0], t.shape[1] + 7).cuda()
        big[:, 5:5 + t.shape[1]] = t.cuda()
        return big[:, 5:5 + t.shape[1]]

    def transposed(name, t):
        return t.cuda() if t.dim() == 1 else t.t().contiguous().cuda().t()
    for place in (gaps, transposed):
        for dim in (100, 128, 131):
            _compare((37, dim), dtype, norm="layer", block_norm="rms", gate=(37, dim), place=lambda n, t: place(n, t).detach())
    from crystalframer_amd import cuda_funcs
    x = torch.randn(12, 80).to(dtype).cuda().requires_grad_()
    cuda_funcs.residual_norm(x, x, keep_residual=False).sum().backward()         # a gradient of stride zero, one tensor twice
    y = torch.randn(80).to(dtype).cuda()
    h, _ = cuda_funcs.residual_norm(x.detach(), y.expand(12, 80))
    assert torch.equal(h, (x.detach().float() + y.float()).to(dtype))


def test_rows_that_are_constant_or_no_numbers_stay_by_themselves():
    from crystalframer_amd import cuda_funcs
    x, f = torch.randn(9, 300), torch.randn(9, 300)
    w, b = torch.rand(300) + 0.5, torch.randn(300)
    plain = cuda_funcs.residual_norm(x.cuda(), f.cuda(), w.cuda(), b.cuda())
    x2, f2 = x.clone(), f.clone()
    x2[2], f2[2] = 3.0, -3.0                # zero everywhere
    x2[4], f2[4] = 1.0, 0.5                 # constant
    x2[5, 7] = float("inf")
    f2[6, 299] = float("nan")
    X, Fb = x2.cuda().requires_grad_(), f2.cuda().requires_grad_()
    h, y = cuda_funcs.residual_norm(X, Fb, w.cuda(), b.cuda())
    keep = [0, 1, 3, 7, 8]
    assert torch.equal(h[keep], plain[0][keep]) and torch.equal(y[keep], plain[1][keep])
    assert torch.equal(y[2].cpu(), b) and torch.equal(y[4].cpu(), b)
    assert torch.isnan(y[5]).all() and torch.isnan(y[6]).all()
    gx, = torch.autograd.grad(y, X, torch.ones_like(y) * w.cuda())
    assert torch.isfinite(gx[[0, 1, 2, 3, 4, 7, 8]]).all() and torch.isnan(gx[[5, 6]]).all()


def test_gradients_against_differences():
    """Directional differences of the float64 loss of float32 outputs: step 2^-6, so that the second-order remainder (2^-12 of the
    third derivative) and the rounding of the outputs (2^-24 / 2^-6 of their norm) are below 2e-3 of the slope's scale."""
    from crystalframer_amd import cuda_funcs
    t, gen = _make((4, 5, 48), F32, F32, "layer", "rms", (4, 1, 48), seed=5)
    ch, cy = torch.randn(4, 5, 48, generator=gen).double(), torch.randn(4, 5, 48, generator=gen).double()

    def loss(tensors):
        h, y = cuda_funcs.residual_norm(**{k: v.cuda() for k, v in tensors.items()}, norm="layer", block_norm="rms", residual_scale=0.9)
        return float((h.cpu().double() * ch).sum() + (y.cpu().double() * cy).sum())
    leaves = {k: v.cuda().requires_grad_() for k, v in t.items()}
    h, y = cuda_funcs.residual_norm(**leaves, norm="layer", block_norm="rms", residual_scale=0.9)
    grads = torch.autograd.grad((h, y), list(leaves.values()), (ch.float().cuda(), cy.float().cuda()))
    for (k, v), g in zip(t.items(), grads):
        d = torch.randn(v.shape, generator=gen)
        e = 2.0 ** -6
        slope = (loss({**t, k: v + e * d}) - loss({**t, k: v - e * d})) / (2 * e)
        scale = float(g.double().norm().cpu() * d.double().norm())
        assert abs(slope - float((g.cpu().double() * d.double()).sum())) < 2e-3 * scale, k


def test_one_output_alone_has_a_gradient():
    from crystalframer_amd import cuda_funcs
    t, gen = _make((21, 160), F32, F32, "layer", None, (160,))
    for which in (0, 1):
        dev = {k: v.cuda().requires_grad_() for k, v in t.items()}
        ref = {k: v.double().requires_grad_() for k, v in t.items()}
        g = torch.randn(21, 160, generator=gen)
        got = torch.autograd.grad(cuda_funcs.residual_norm(**dev)[which], list(dev.values()), g.cuda(), allow_unused=True)
        want = torch.autograd.grad(TR.residual_norm(**ref)[which], list(ref.values()), g.double(), allow_unused=True)
        for k, a, b in zip(t, got, want):
            b = torch.zeros(t[k].shape).double() if b is None else b
            assert a is not None and (a.cpu().double() - b).abs().max() <= 64 * 2.0 ** -24 * max(float(b.abs().max()), 1.0), (which, k)
    # gradients of some leaves only
    dev = {k: v.cuda().requires_grad_(k in ("block", "bias")) for k, v in t.items()}
    h, y = cuda_funcs.residual_norm(**dev)
    a, b = torch.autograd.grad((h, y), (dev["block"], dev["bias"]), (h.detach(), y.detach()))
    full = {k: v.cuda().requires_grad_() for k, v in t.items()}
    h, y = cuda_funcs.residual_norm(**full)
    c, d = torch.autograd.grad((h, y), (full["block"], full["bias"]), (h.detach(), y.detach()))
    assert torch.equal(a, c) and torch.equal(b, d)


def test_the_same_tensor_as_stream_and_block():
    from crystalframer_amd import cuda_funcs
    x = torch.randn(11, 72, device="cuda", requires_grad=True)
    g = torch.randn(11, 72, device="cuda")
    for scales in ((1.0, 1.0), (0.5, 1.25)):
        opts = dict(residual_scale=scales[0], block_scale=scales[1])
        both, = torch.autograd.grad(cuda_funcs.residual_norm(x, x, **opts), x, (g, g))
        a, b = x.detach().clone().requires_grad_(), x.detach().clone().requires_grad_()
        cuda_funcs.residual_norm(a, b, **opts)[1].backward(g, retain_graph=True)
        one = a.grad.clone()
        b.grad.add_(1.0)                         # (the gradients are two tensors, also where they are equal)
        assert torch.equal(a.grad, one)
        ga, gb = torch.autograd.grad(cuda_funcs.residual_norm(a, b, **opts), (a, b), (g, g))
        assert (both - (ga + gb)).abs().max() <= 2.0 ** -23 * (ga.abs() + gb.abs()).max()


def test_no_rows():
    from crystalframer_amd import cuda_funcs
    x = torch.zeros(0, 64, device="cuda", requires_grad=True)
    w, b = (torch.ones(64, device="cuda", requires_grad=True) for _ in range(2))
    g = torch.ones(64, device="cuda", requires_grad=True)
    h, y = cuda_funcs.residual_norm(x, x * 2, w, b, gate=g)
    assert h.shape == y.shape == (0, 64)
    for t in torch.autograd.grad((h, y), (w, b, g), (h, y)):
        assert torch.equal(t, torch.zeros(64, device="cuda"))


def test_equal_runs_give_equal_bits_and_graphs_replay_them():
    from crystalframer_amd import cuda_funcs
    t, _ = _make((1201, 130), F32, F32, "layer", "rms", (130,))
    dev = {k: v.cuda().requires_grad_() for k, v in t.items()}
    gh, gy = torch.randn(1201, 130).cuda(), torch.randn(1201, 130).cuda()

    def once():
        h, y = cuda_funcs.residual_norm(**dev, block_norm="rms")
        return (h.detach(), y.detach()) + torch.autograd.grad((h, y), list(dev.values()), (gh, gy))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = once()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(first, once()))
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = once()
        graphs.append((graph, held))
    for k in range(3):
        with torch.no_grad():
            dev["x"].add_(0.25)
        for graph, _ in graphs:
            graph.replay()
        want = once()
        torch.cuda.synchronize()
        for _, held in graphs:
            assert all(torch.equal(a, b) for a, b in zip(held, want)), k


def test_capture_beside_an_eager_graph_of_the_same_leaves_is_refused():
    from crystalframer_amd import cuda_funcs
    w = torch.ones(64, device="cuda", requires_grad=True)
    x = torch.randn(7, 64, device="cuda")
    loss = cuda_funcs.residual_norm(x, None, w, keep_residual=False).sum()           # kept
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="let go"):
        with torch.cuda.graph(graph):
            cuda_funcs.residual_norm(x, None, w, keep_residual=False).sum().backward()
    y = []
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):               # (the forward pass alone is nothing to refuse)
        y.append(cuda_funcs.residual_norm(x, None, w, keep_residual=False).detach())
    graph.replay()
    assert torch.equal(y[0], cuda_funcs.residual_norm(x, None, w, keep_residual=False).detach())
    del loss
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cuda_funcs.residual_norm(x, None, w, keep_residual=False).sum().backward()
    for k in range(3):
        w.grad.zero_()
        graph.replay()
        torch.cuda.synchronize()
        want = cuda_funcs.residual_norm(x, None, torch.ones(64, device="cuda"), keep_residual=False).sum(0)
        assert (w.grad - want).abs().max() <= 64 * 2.0 ** -24 * 7 * 3, k


def test_offsets_beyond_32_bits():
    from crystalframer_amd import cuda_funcs
    rows, dim = (1 << 31) // 16384 + 5, 16384
    x = torch.zeros(rows, dim, dtype=BF16, device="cuda")
    g = torch.zeros(rows, dim, dtype=BF16, device="cuda")
    tail = torch.randn(9, dim).to(BF16)
    x[-9:], g[-9:] = tail.cuda(), tail.flip(0).cuda()
    w = torch.ones(dim, device="cuda", requires_grad=True)
    x.requires_grad_()
    y = cuda_funcs.residual_norm(x, None, w, norm="rms", keep_residual=False)
    small = x.detach()[-9:].clone().requires_grad_()
    w2 = w.detach().clone().requires_grad_()
    y2 = cuda_funcs.residual_norm(small, None, w2, norm="rms", keep_residual=False)
    assert torch.equal(y[-9:], y2)
    gx, gw = torch.autograd.grad(y, (x, w), g)
    gx2, gw2 = torch.autograd.grad(y2, (small, w2), g[-9:])
    assert torch.equal(gx[-9:], gx2) and not gx[:-9].any()
    assert (gw - gw2).abs().max() <= 64 * 2.0 ** -24 * 9 * gw2.abs().max()


def test_refusals():
    from crystalframer_amd import cuda_funcs
    N = cuda_funcs.residual_norm
    x = torch.zeros(4, 6, 32, device="cuda")
    v = torch.zeros(32, device="cuda")
    for error, call in [
            (ValueError, lambda: N(x, norm="batch")), (ValueError, lambda: N(x, block_norm="layer")), (ValueError, lambda: N(x, gate=v)),
            (ValueError, lambda: N(x, x, norm=None, keep_residual=False)), (ValueError, lambda: N(x, x, v, norm=None)),
            (ValueError, lambda: N(x, x, block_weight=v)), (ValueError, lambda: N(x, x[:2])), (ValueError, lambda: N(x, x, v[:31])),
            (ValueError, lambda: N(x, x, gate=x[:, :, :1])), (ValueError, lambda: N(x, x, gate=x[:1])), (ValueError, lambda: N(x, x, gate=x[0])),
            (ValueError, lambda: N(x, x, eps=-1.0)), (ValueError, lambda: N(torch.zeros(2, 16385, device="cuda"))),
            (ValueError, lambda: N(torch.zeros((), device="cuda"))), (ValueError, lambda: N(torch.zeros(3, 0, device="cuda"))),
            (TypeError, lambda: N(x.double())), (TypeError, lambda: N(x, x.half())), (TypeError, lambda: N(x, x, gate=v.half())),
            (TypeError, lambda: N(x, x, v.half())), (TypeError, lambda: N(x.half(), None, v.half(), v)), (RuntimeError, lambda: N(x, x.cpu()))]:
        with pytest.raises(error):
            call()
    a = torch.randn(3, 8, device="cuda", requires_grad=True)
    g, = torch.autograd.grad(N(a, keep_residual=False).square().sum(), a, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()
