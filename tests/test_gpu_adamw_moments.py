"""optim.AdamW with parameters of several types, moments in 32 and 8 bits and clipping, against float64 (training_reference).

Moments in 8 bits are compared code by code: the kernel decides in 64 bits, so that a code differs only where the moment
lies within 2^-50 of a border.  Parameters: half a unit of their type, and eight float32 roundings (a product, a quotient, a
square root, sums) of the step's size; exp_avg in 32 bits is rounded three times a step, each time relative to the terms of its
sum, which may cancel: the size is that of the step with the sum of the terms' magnitudes in the place of exp_avg."""
import copy
import io

import numpy as np
import pytest
import torch

import training_reference as TR

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
SHAPES = [(128, 128), (1,), (3,), (7, 5), (63,), (64,), (65,), (1023,), (4097,), (8, 16, 64), (5, 0), (20011,)]
HYPER = dict(lr=3e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2)


def _params(dtype, shapes=SHAPES, seed=0):
    gen = torch.Generator().manual_seed(seed)
    types = dtype if isinstance(dtype, list) else [dtype] * len(shapes)
    return [torch.nn.Parameter((0.1 * torch.randn(s, generator=gen)).to(t).cuda()) for s, t in zip(shapes, types)]


def _grads(params, step, scale=None):
    gen = torch.Generator().manual_seed(100 + step)
    for k, p in enumerate(params):
        spread = 10.0 ** (-3.0 * torch.rand(p.shape, generator=gen)) * (0.05 + 0.2 * (k % 4))
        p.grad = (torch.randn(p.shape, generator=gen) * spread * (1.0 if scale is None else scale)).to(p.dtype).cuda()


class Reference:
    def __init__(self, params, bits, start=0):
        first, self.states, self.t = 0, [], start
        for p in params:
            self.states.append(TR.State(p.numel(), bits, first))
            first += -(-p.numel() // 64) * 64

    def step(self, before, grads, factor=1.0, hyper=HYPER):
        self.t += 1
        return [s.step(p, g, self.t, hyper["lr"], hyper["betas"], hyper["eps"], hyper["weight_decay"], factor)
                for s, p, g in zip(self.states, before, grads)]


def _numbers(ts):
    return [t.detach().cpu().double().numpy().ravel() for t in ts]


def _check(opt, params, before, want, ref, bits):
    # The kernel of float32 parameters with 32-bit moments and no clipping takes 1 - beta2 from beta2 in float32, which is off by half
    # of its last place, 2^-25: 2^-25 / (1 - beta2) of what is added to exp_avg_sq, half of that in its root.
    whole = opt._flat[id(opt.param_groups[0])]["legacy"] and opt.max_grad_norm is None
    slack = 2.0 ** -25 / (1.0 - HYPER["betas"][1]) if whole else 0.0
    for k, (p, b, w, s) in enumerate(zip(params, _numbers(before), want, ref.states)):
        got = p.detach().cpu().double().numpy().ravel()
        tol = TR.HALF[p.dtype] * np.abs(w) + TR.TINY[p.dtype] + 8 * 2.0 ** -24 * (s.size + np.abs(b)) + slack * s.size
        assert (np.abs(got - w) <= tol).all(), (k, np.abs(got - w).max())
        st = opt.state[p]
        if bits == 8:
            for name, codes in (("exp_avg", s.cm), ("exp_avg_sq", s.cv), ("exp_avg_scale", s.sm), ("exp_avg_sq_scale", s.sv)):
                got = st[name].view(torch.uint8).cpu().numpy().ravel().astype(np.int64)
                assert np.array_equal(got, codes), (k, name, np.flatnonzero(got != codes)[:5])
        else:
            # three roundings a step, of terms no larger than the largest that was added
            for name, x in (("exp_avg", s.m), ("exp_avg_sq", s.v)):
                got = st[name].cpu().double().numpy().ravel()
                assert (np.abs(got - x) <= slack * np.abs(x) + 8 * ref.t * 2.0 ** -24 * (np.abs(x) + (np.abs(x).max() if len(x) else 0.0))).all(), (k, name)


@pytest.mark.parametrize("clip", [None, 0.5, 1e9])
@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("dtype", [F32, BF16, F16, "mixed"])
def test_steps(dtype, bits, clip):
    from crystalframer_amd import optim
    types = [[F32, BF16, F16][k % 3] for k in range(len(SHAPES))] if dtype == "mixed" else dtype
    params = _params(types)
    opt = optim.AdamW(params, **HYPER, state_bits=bits, max_grad_norm=clip)
    ref = Reference(params, bits)
    for step in range(4):
        _grads(params, step)
        before = [p.detach().clone() for p in params]
        grads = _numbers([p.grad for p in params])
        kept = [p.grad.clone() for p in params]
        norm = float(np.sqrt(sum((g * g).sum() for g in grads)))
        factor = 1.0 if clip is None else float(np.float32(min(1.0, clip / (norm + 1e-6))))
        opt.step()
        _check(opt, params, before, ref.step(_numbers(before), grads, factor), ref, bits)
        assert all(torch.equal(p.grad, g) for p, g in zip(params, kept))
        if clip is not None:
            assert opt.grad_norm.dtype == F32 and opt.grad_norm.shape == () and abs(float(opt.grad_norm) - norm) <= 2.0 ** -23 * norm
    (m, v), = opt.moments()
    assert m.dtype == v.dtype == F32
    for s in ref.states:
        if bits == 8:
            a, b = s.values()
            assert np.array_equal(m[s.first:s.first + s.n].cpu().numpy(), a.astype(np.float32))
            assert np.array_equal(v[s.first:s.first + s.n].cpu().numpy(), b.astype(np.float32))


def test_float32_with_clipping_is_the_plain_step_of_clipped_gradients():
    from crystalframer_amd import optim
    mine, other = _params(F32), _params(F32)
    a, b = optim.AdamW(mine, **HYPER, max_grad_norm=0.3), torch.optim.AdamW(other, **HYPER)
    for step in range(3):
        _grads(mine, step), _grads(other, step)
        a.step()
        norm = torch.nn.utils.clip_grad_norm_(other, 0.3)
        b.step()
        assert abs(float(a.grad_norm) - float(norm)) <= 1e-5 * float(norm)
        for x, y in zip(mine, other):
            assert x.numel() == 0 or (x - y).abs().max() <= 2e-6 * (step + 1) * y.abs().max()


def test_many_tensors_views_and_missing_gradients():
    """More tensors than one launch takes, at addresses off every alignment, some without a gradient, some frozen."""
    from crystalframer_amd import optim
    for bits, dtype in ((8, BF16), (32, F16), (8, F32)):
        base = torch.randn(200 * 131 + 1).mul_(0.1).to(dtype).cuda()
        gbase = torch.randn(200 * 131 + 1).to(dtype).cuda()
        params = [torch.nn.Parameter(base[1 + 131 * k:1 + 131 * k + 1 + (k * 37) % 131]) for k in range(200)]
        frozen = torch.nn.Parameter(torch.ones(9, device="cuda"), requires_grad=False)
        opt = optim.AdamW(params[:50] + [frozen] + params[50:], **HYPER, state_bits=bits)
        ref = Reference(params, bits)
        for step in range(2):
            for k, p in enumerate(params):
                p.grad = None if k % 11 == 3 else gbase[1 + 131 * k:1 + 131 * k + p.numel()]
            before = [p.detach().clone() for p in params]
            opt.step()
            ref.t += 1
            want = [s.step(b, g, ref.t, **dict(zip(("lr", "betas", "eps", "wd"), HYPER.values()))) if k % 11 != 3 else b for k, (s, b, g) in
                    enumerate(zip(ref.states, _numbers(before), _numbers([gbase[1 + 131 * k:1 + 131 * k + p.numel()] for k, p in enumerate(params)])))]
            _check(opt, params, before, want, ref, bits)
        assert torch.equal(frozen, torch.ones(9, device="cuda"))


def test_values_that_are_no_numbers_stay_with_their_element():
    from crystalframer_amd import optim
    g = torch.randn(200) * 1e-3
    g[5], g[70], g[71] = float("nan"), float("inf"), -float("inf")
    g[130] = 3e38
    p, q = (torch.nn.Parameter(torch.ones(200, device="cuda")) for _ in range(2))
    opt, clean = optim.AdamW([p], **HYPER, state_bits=8), optim.AdamW([q], **HYPER, state_bits=8)
    hit = torch.tensor([5, 70, 71])
    for step in range(3):
        p.grad = g.cuda() if step == 0 else torch.full((200,), 1e-3, device="cuda")
        q.grad = torch.where(torch.isfinite(g), g, 0.0).cuda() if step == 0 else torch.full((200,), 1e-3, device="cuda")
        opt.step(), clean.step()
    others = torch.ones(200, dtype=torch.bool)
    others[hit] = False
    assert torch.isnan(p.detach().cpu()[hit]).all() and torch.equal(p.detach().cpu()[others], q.detach().cpu()[others])
    (m, v), = opt.moments()
    assert torch.isnan(m[hit]).all() and torch.isinf(v[[5, 70, 71, 130]]).all() and torch.isfinite(m[:200].cpu()[others]).all()
    # a norm that is no number is one for all, as the framework's clipping has it
    opt = optim.AdamW([q], **HYPER, state_bits=8, max_grad_norm=1.0)
    q.grad = g.cuda()
    opt.step()
    assert torch.isnan(opt.grad_norm) and torch.isnan(q).all()


def test_extreme_gradients():
    """Zero, the smallest and the largest values, and blocks that hold both."""
    from crystalframer_amd import optim
    g = torch.zeros(64 * 7)
    g[64:128] = 1e-30
    g[128:192] = torch.logspace(-18, 18, 64)
    g[192:256] = 1e-45
    g[256] = 1.0
    g[320:384] = torch.logspace(-8, 0, 64)
    p = torch.nn.Parameter(torch.ones(64 * 7, device="cuda"))
    opt = optim.AdamW([p], **HYPER, state_bits=8)
    ref = Reference([p], 8)
    for step in range(4):
        p.grad = (g if step % 2 == 0 else g * 0).cuda()
        before = [p.detach().clone()]
        opt.step()
        want = ref.step(_numbers(before), _numbers([p.grad]))
        _check(opt, [p], before, want, ref, 8)
        assert (p - before[0]).abs().max() < 0.1


def test_moments_follow_their_gradients_on_average():
    """What moves by less than a code's step a time moves nevertheless.  Gradients of size 1 for 300 steps, then of size 0.1 for 2000:
    exp_avg_sq falls to 0.0437.  An element wanders: a step of 0.1 % is a step of one code, 1/8 at most, with odds of 0.008 at
    least, which adds 0.001 / 8 to the variance of its logarithm, over 2000 steps 0.25 if nothing pulled it back.  An average of 65536
    elements is then within 0.5 / 256 of the whole, a tenth of what is asked; the furthest of them, five deviations, by a factor of
    e^2.5."""
    from crystalframer_amd import optim
    p = torch.nn.Parameter(torch.zeros(65536, device="cuda"))
    opt = optim.AdamW([p], lr=0.0, state_bits=8)
    want_m = want_v = 0.0
    for step in range(2300):
        size = 1.0 if step < 300 else 0.1
        p.grad = torch.full_like(p, size) if step in (0, 300) else p.grad
        opt.step()
        want_m, want_v = 0.9 * want_m + 0.1 * size, 0.999 * want_v + 0.001 * size * size
    (m, v), = opt.moments()
    assert abs(float(m.double().mean()) - want_m) < 0.01 * want_m
    assert abs(float(v.double().mean()) - want_v) < 0.05 * want_v and want_v / 12.2 < float(v.min()) and float(v.max()) < 12.2 * want_v


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_state_dict_goes_round(dtype, bits):
    from crystalframer_amd import optim
    a = _params(dtype)
    one = optim.AdamW(a, **HYPER, state_bits=bits, max_grad_norm=1.0)
    for step in range(3):
        _grads(a, step)
        one.step()
    file = io.BytesIO()
    torch.save(one.state_dict(), file)
    file.seek(0)
    saved = torch.load(file, weights_only=True, map_location="cpu")
    b = [torch.nn.Parameter(p.detach().clone()) for p in a]
    two = optim.AdamW(b, state_bits=8 if bits == 32 else 32, max_grad_norm=1.0)      # a checkpoint brings its own
    two.load_state_dict(saved)
    assert two.param_groups[0]["state_bits"] == bits and two.param_groups[0]["lr"] == HYPER["lr"]
    c = copy.deepcopy(a)
    three = copy.deepcopy(one)
    for x, y in zip(three.param_groups[0]["params"], c):
        assert torch.equal(x, y)
    c = three.param_groups[0]["params"]
    three.max_grad_norm = 1.0
    for step in range(3, 5):
        for ps, o in ((a, one), (b, two), (c, three)):
            _grads(ps, step)
            o.step()
        assert all(torch.equal(x, y) and torch.equal(x, z) for x, y, z in zip(a, b, c))
    for x, y in zip(one.moments()[0], two.moments()[0]):
        assert torch.equal(x, y)


def test_checkpoints_of_the_frameworks_optimizer_load():
    from crystalframer_amd import optim
    a, b = _params(BF16), _params(BF16)
    theirs = torch.optim.AdamW(_params(F32), **HYPER)
    _grads(theirs.param_groups[0]["params"], 0)
    theirs.step()
    mine = optim.AdamW(a, state_bits=32)
    mine.load_state_dict(theirs.state_dict())
    for p, q in zip(a, theirs.param_groups[0]["params"]):
        assert mine.state[p]["exp_avg"].dtype == F32 and torch.equal(mine.state[p]["exp_avg"], theirs.state[q]["exp_avg"])
        assert int(mine.state[p]["step"]) == 1


def test_groups_share_the_norm():
    from crystalframer_amd import optim
    a, b = _params(F32, SHAPES[:5]), _params(BF16, SHAPES[5:], seed=1)
    opt = optim.AdamW([dict(params=a, lr=1e-3), dict(params=b, state_bits=8, weight_decay=0.0)], **HYPER, max_grad_norm=0.1)
    refs = Reference(a, 32), Reference(b, 8)
    for step in range(2):
        _grads(a, step), _grads(b, step + 10)
        before = [[p.detach().clone() for p in ps] for ps in (a, b)]
        grads = [_numbers([p.grad for p in ps]) for ps in (a, b)]
        norm = float(np.sqrt(sum((g * g).sum() for gs in grads for g in gs)))
        opt.step()
        assert abs(float(opt.grad_norm) - norm) <= 2.0 ** -23 * norm
        factor = float(np.float32(0.1 / (norm + 1e-6)))
        for ps, old, gs, ref, hyper, bits in zip((a, b), before, grads, refs, (dict(HYPER, lr=1e-3), dict(HYPER, weight_decay=0.0)), (32, 8)):
            _check(opt, ps, old, ref.step(_numbers(old), gs, factor, hyper), ref, bits)
    assert len(opt.moments()) == 2


@pytest.mark.parametrize("bits", [8, 32])
def test_captured_steps_keep_counting(bits):
    from crystalframer_amd import optim
    a, b = _params(BF16), _params(BF16)
    one, two = (optim.AdamW(ps, **HYPER, state_bits=bits, max_grad_norm=0.2) for ps in (a, b))
    _grads(a, 0), _grads(b, 0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        one.step()
    torch.cuda.current_stream().wait_stream(side)
    two.step()
    held = [p.grad for p in a]
    graphs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()]
    norms = []
    for graph in graphs:
        with torch.cuda.graph(graph):
            one.step()
        norms.append(one.grad_norm)
    for step in range(1, 7):
        _grads(b, step)
        for h, p in zip(held, b):
            h.copy_(p.grad)
        graphs[step % 2].replay()
        two.step()
        torch.cuda.synchronize()
        assert torch.equal(norms[step % 2], two.grad_norm)
        assert all(torch.equal(x, y) for x, y in zip(a, b)), step
    assert all(torch.equal(x, y) for x, y in zip(one.moments()[0], two.moments()[0]))


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("eps", [0.0, 1e-30])
def test_small_roots_beside_a_small_eps(bits, eps):
    """exp_avg_sq around 2^-130, where float32 holds 19 bits of it: 2^-19 of the update, and what the other steps round."""
    from crystalframer_amd import optim
    p = torch.nn.Parameter(torch.linspace(0.5, 1.0, 200, device="cuda"))
    g = 1e-18 * (1.0 + torch.arange(200, dtype=torch.float64) % 7 / 7) * (1 - 2 * (torch.arange(200) % 2))
    p.grad = g.float().cuda()
    q = p.detach().cpu().double()
    opt = optim.AdamW([p], lr=3e-3, eps=eps, weight_decay=0.0, state_bits=bits, max_grad_norm=1.0)
    opt.step()
    want = q - 3e-3 * g / (g.abs() + eps)
    assert ((p.detach().cpu().double() - want).abs() <= 8 * 2.0 ** -24 + 3e-3 * 2.0 ** -19).all()


def test_a_group_in_float32_is_stepped_alike_beside_others():
    from crystalframer_amd import optim
    a, b, c = _params(F32), _params(F32), _params(BF16, seed=1)
    one, two = optim.AdamW(a, **HYPER), optim.AdamW([dict(params=b), dict(params=c, state_bits=8)], **HYPER)
    for step in range(3):
        _grads(a, step), _grads(b, step), _grads(c, step)
        one.step(), two.step()
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_elements_beyond_what_one_table_entry_counts():
    from crystalframer_amd import optim
    n = (1 << 30) + 200
    p = torch.nn.Parameter(torch.zeros(n, dtype=BF16, device="cuda"))
    p.grad = torch.zeros(n, dtype=BF16, device="cuda")
    ends = [slice(0, 100), slice((1 << 30) - 64, n)]
    for s in ends:
        p.grad[s] = torch.randn(s.stop - s.start).to(BF16).cuda()
    opt = optim.AdamW([p], **HYPER, state_bits=8, max_grad_norm=1.0)
    opt.step()
    g = [p.grad[s].cpu().double().numpy() for s in ends]
    norm = np.sqrt(sum((x * x).sum() for x in g))
    assert abs(float(opt.grad_norm) - norm) <= 2.0 ** -23 * norm
    for s, x in zip(ends, g):
        ref = TR.State(s.stop - s.start, 8, s.start)
        want = ref.step(np.zeros(len(x)), x, 1, HYPER["lr"], HYPER["betas"], HYPER["eps"], HYPER["weight_decay"],
                        float(np.float32(min(1.0, 1.0 / (norm + 1e-6)))))
        got = p.detach()[s].cpu().double().numpy()
        assert (np.abs(got - want) <= 2.0 ** -8 * np.abs(want) + 8 * 2.0 ** -24 * ref.size).all()
        assert np.array_equal(opt.state[p]["exp_avg"].view(torch.uint8)[s].cpu().numpy(), ref.cm.astype(np.uint8))
    assert not p.detach()[1000:1 << 29].any()


def test_refusals():
    from crystalframer_amd import optim
    p = torch.nn.Parameter(torch.zeros(70, device="cuda", dtype=BF16))
    for bad in (dict(state_bits=16), dict(max_grad_norm=-1.0)):
        with pytest.raises(ValueError):
            optim.AdamW([p], **bad)
    opt = optim.AdamW([torch.nn.Parameter(torch.zeros(3, device="cuda", dtype=torch.float64))])
    opt.param_groups[0]["params"][0].grad = torch.zeros(3, device="cuda", dtype=torch.float64)
    with pytest.raises(RuntimeError, match="float32"):
        opt.step()
    opt = optim.AdamW([p], state_bits=8)
    p.grad = torch.ones(70, device="cuda", dtype=BF16)
    opt.step()
    saved = opt.state_dict()
    opt.param_groups[0]["state_bits"] = 32
    with pytest.raises(RuntimeError, match="state_bits"):
        opt.step()
    opt.param_groups[0]["state_bits"] = 8
    q = torch.nn.Parameter(torch.zeros(70, device="cuda"))
    q.grad = torch.ones_like(q)
    for form in (dict(state_bits=8), dict(max_grad_norm=1.0)):
        new = optim.AdamW([q], **form)
        with pytest.raises(RuntimeError, match="before the capture"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                new.step()
    with pytest.warns(UserWarning):
        new = optim.AdamW([q, q], state_bits=8)
    with pytest.raises(RuntimeError, match="twice"):
        new.step()
    old = p.data
    for other in (torch.zeros(71, device="cuda", dtype=BF16), old.float(), torch.zeros(140, device="cuda", dtype=BF16)[::2]):
        p.grad = None
        p.data = other
        p.grad = torch.ones(other.shape, device="cuda", dtype=other.dtype)
        if other.dtype == F32:
            opt.step()            # a parameter may change its type; its moments stay
            continue
        with pytest.raises(RuntimeError):
            opt.step()
    p.grad = None
    p.data = old
    for name, wrong in (("exp_avg", torch.zeros(69).to(torch.float8_e4m3fn)), ("exp_avg_scale", torch.zeros(1, dtype=torch.uint8)),
                        ("exp_avg_sq", torch.zeros(70))):
        broken = copy.deepcopy(saved)
        broken["state"][0][name] = wrong
        with pytest.raises(RuntimeError, match=name):
            optim.AdamW([torch.nn.Parameter(old.clone())], state_bits=8).load_state_dict(broken)
