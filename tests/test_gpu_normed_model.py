"""Encoders with layer norms: the joined residual norm inside the model against torch.nn.LayerNorm and the addition, and a whole
training run of it (norms forward and backward, the gradients' norm, AdamW with 8-bit moments) as its user makes it.

Both paths compute the same formula in float32 and differ by rounding; frames are switched off (distances alone), so that no choice
between two axes can turn on a last bit.  A rounding of 2^-24 is carried through two layers and their norms (each may multiply it by
one over a row's deviation, about 1 here): 1e-4 of the largest magnitude is what the model is held to everywhere else."""
import copy

import pytest
import torch

import helpers as Hh

pytestmark = pytest.mark.gpu


def _model(norm_first=False, seed=0, dropout=0.0):
    from crystalframer_amd import latticeformer, params
    import crystalframer_amd as cf
    cf.KernelManager.SYMM_BREAK_NOISE = 0.0
    torch.manual_seed(seed)
    model = latticeformer.Latticeformer(params.ModelParams(num_layers=2, value_pe_angle_real=0, t_fixup_init=False, symm_break_noise=0.0,
                                                           dropout=dropout)).cuda()
    for layer in model.encoder.layers:
        layer.norm_first = norm_first
    with torch.no_grad():
        for n, p in model.named_parameters():
            if ".norm" in n:
                p.add_(0.1 * torch.randn_like(p))
    return model


def _batch(seed=3):
    from crystalframer_amd import synthetic
    return synthetic.make_batch(9, atoms="uniform", atoms_lo=1, atoms_hi=7, len_lo=3.0, len_hi=9.0, ang_lo=65.0, ang_hi=115.0, seed=seed).to("cuda")


def _calls(monkeypatch):
    from crystalframer_amd import norms
    seen, real = [], norms.residual_norm

    def counted(*args, **kw):
        seen.append(kw.get("keep_residual"))
        return real(*args, **kw)
    monkeypatch.setattr(norms, "residual_norm", counted)
    return seen


@pytest.mark.parametrize("norm_first", [False, True])
def test_model_against_the_modules(norm_first, monkeypatch):
    from crystalframer_amd import encoder
    seen = _calls(monkeypatch)
    a = _model(norm_first)
    batch = _batch()
    a(batch).sum().backward()                 # the first training pass stores the normalisation of the Gaussian widths
    a.zero_grad()
    b = copy.deepcopy(a)
    del seen[:]
    out = a(batch)
    out.square().mean().backward()
    assert len(seen) == 5                     # two norms for each of two layers, and the last
    monkeypatch.setattr(encoder, "FUSED_RESIDUAL_NORM", False)
    ref = b(batch)
    ref.square().mean().backward()
    assert len(seen) == 5
    assert Hh.rel_err(out, ref) < 1e-4
    for (n, p), q in zip(a.named_parameters(), b.parameters()):
        if q.grad is not None and q.grad.abs().max() > 1e-6 * max(r.grad.abs().max() for r in b.parameters() if r.grad is not None):
            assert Hh.rel_err(p.grad, q.grad) < 1e-4, n
    a.eval(), b.eval()
    with torch.no_grad():
        monkeypatch.setattr(encoder, "FUSED_RESIDUAL_NORM", True)
        out = a(batch)
        assert len(seen) == 10
        assert torch.equal(out, a(batch)) and Hh.rel_err(out, b(batch)) < 1e-4


def test_whoever_looks_at_a_norm_gets_the_module(monkeypatch):
    seen = _calls(monkeypatch)
    model, batch = _model().eval(), _batch()
    with torch.no_grad():
        model(batch)
        assert len(seen) == 5
        got = []
        handle = model.encoder.layers[0].norm1.register_forward_hook(lambda m, i, o: got.append(o))
        model(batch)
        assert len(seen) == 9 and len(got) == 1
        handle.remove()
        with torch.autocast("cuda", dtype=torch.bfloat16, enabled=True):
            n = len(seen)
            x = torch.randn(5, 128, device="cuda")
            from crystalframer_amd import encoder
            assert encoder._normed(model.encoder.norm, x).dtype == torch.float32 and len(seen) == n
        model.encoder.norm = torch.nn.RMSNorm(128).cuda()
        model(batch)
        assert len(seen) == n + 4


@pytest.mark.parametrize("bits", [8, 32])
def test_training_run(bits, monkeypatch):
    """Ten steps, eager and as a captured graph, give the same parameters; against the modules with torch's clipping and AdamW the first
    step's update (the same formula, gradients to 1e-4) differs by what a gradient's error makes of it."""
    from crystalframer_amd import encoder, optim
    batch, target = _batch(), torch.linspace(-1, 1, 9, device="cuda")[:, None]
    base = _model(dropout=0.0)
    base(batch).sum().backward()
    base.zero_grad()
    loss_of = lambda m: torch.nn.functional.mse_loss(m(batch), target)  # noqa: E731

    def make():
        m = copy.deepcopy(base)
        return m, optim.AdamW(m.parameters(), lr=1e-3, weight_decay=1e-2, state_bits=bits, max_grad_norm=0.05)
    eager, opt = make()
    grads, norms = [], []
    for step in range(6):
        opt.zero_grad()
        loss_of(eager).backward()
        if step == 0:
            grads = [None if p.grad is None else p.grad.clone() for p in eager.parameters()]
        before = [p.detach().clone() for p in eager.parameters()] if step == 0 else None
        opt.step()
        norms.append(float(opt.grad_norm))
        if step == 0:
            norm = torch.sqrt(sum(g.double().square().sum() for g in grads if g is not None))
            assert abs(norms[0] - float(norm)) <= 1e-6 * float(norm)
            factor = min(1.0, 0.05 / (float(norm) + 1e-6))
            for p, b, g in zip(eager.parameters(), before, grads):
                if g is None:
                    assert torch.equal(p, b)
                    continue
                # the first step moves by lr c g / (|c g| + eps), whatever the moments are kept in afterwards
                c = g.double() * factor
                want = b.double() * (1 - 1e-5) - 1e-3 * c / (c.abs() + 1e-8)
                assert (p.double() - want).abs().max() <= 2.0 ** -24 * b.abs().max() * 4 + 1e-3 * 1e-5
    replayed, opt2 = make()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            opt2.zero_grad()
            loss_of(replayed).backward()
            opt2.step()
    torch.cuda.current_stream().wait_stream(side)
    opt2.zero_grad()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss_of(replayed).backward()
        opt2.step()
    for step in range(2, 6):
        graph.replay()
        torch.cuda.synchronize()
        assert float(opt2.grad_norm) == norms[step], step
    for p, q in zip(eager.parameters(), replayed.parameters()):
        assert torch.equal(p, q)
