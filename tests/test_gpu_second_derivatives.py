"""A backward pass that is itself recorded (``create_graph``) through the norms of the encoder's layers, as torch.nn.LayerNorm has it, and
through ``cuda_funcs.residual_norm`` where it is asked for."""
import copy

import pytest
import torch

import helpers as Hh
import training_reference as TR
from test_gpu_normed_model import _batch, _model

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


@pytest.mark.parametrize("norm_first", [False, True])
def test_penalties_on_gradients_in_the_model(norm_first, monkeypatch):
    """The gradients of the norms' own weights and biases, squared, as a penalty: the same formula as with the modules, to the 1e-4 that the model is
    held to (test_gpu_normed_model)."""
    from crystalframer_amd import encoder
    base, batch = _model(norm_first), _batch()
    base(batch).sum().backward()              # the first training pass stores the normalisation of the Gaussian widths
    base.zero_grad()
    results = []
    for fused in (True, False):
        monkeypatch.setattr(encoder, "FUSED_RESIDUAL_NORM", fused)
        model = copy.deepcopy(base)
        params = {n: p for n, p in model.named_parameters() if p.requires_grad}
        loss = model(batch).square().mean()
        last = [p for n, p in params.items() if n.startswith("encoder.norm") or (n.startswith("encoder.layers.1.norm2") and not norm_first)]
        assert len(last) == (2 if norm_first else 4)
        first = torch.autograd.grad(loss, last, create_graph=True)
        second = torch.autograd.grad(loss + 10.0 * sum(g.square().sum() for g in first), list(params.values()), allow_unused=True)
        results.append((list(params), [g.detach() for g in first], second))
    (names, first, second), (_, first_ref, second_ref) = results
    for a, b in zip(first, first_ref):
        assert Hh.rel_err(a, b) < 1e-4
    top = max(float(g.abs().max()) for g in second_ref if g is not None)
    for n, a, b in zip(names, second, second_ref):
        assert (a is None) == (b is None), n
        if b is not None and float(b.abs().max()) > 1e-6 * top:
            assert Hh.rel_err(a, b) < 1e-4, n


@pytest.mark.parametrize("shape", [(1, 1), (5, 3), (7, 130), (3, 4, 1000)], ids=str)
@pytest.mark.parametrize("block,keep", [(False, False), (False, True), (True, False), (True, True)])
def test_against_float64(shape, block, keep):
    """Gradients of a function of the gradients, in float32 from the framework's operations: 256 roundings of the largest magnitude of each
    (normed values to 4 deviations, products of five such terms)."""
    from crystalframer_amd import cuda_funcs
    gen = torch.Generator().manual_seed(1)
    D = shape[-1]
    rnd = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    t = dict(x=rnd(*shape), weight=1.0 + 0.2 * rnd(D), bias=0.1 * rnd(D), **(dict(block=rnd(*shape)) if block else {}))
    c, e = rnd(*shape), rnd(*shape)
    results = []
    for ours in (True, False):
        leaves = {k: (v.cuda() if ours else v.double()).requires_grad_() for k, v in t.items()}
        to = (lambda v: v.cuda()) if ours else (lambda v: v.double())
        if ours:
            out = cuda_funcs.residual_norm(**leaves, keep_residual=keep, twice_differentiable=True)
            h, y = out if keep else (None, out)
        else:
            h, y = TR.residual_norm(**leaves)
        loss = (y * y * to(c)).sum() + ((h * h * to(e)).sum() if keep else 0.0)
        first = torch.autograd.grad(loss, list(leaves.values()), create_graph=True)
        second = torch.autograd.grad(sum((g * g).sum() for g in first), list(leaves.values()))
        results.append(first + second)
    for k, (a, b) in enumerate(zip(*results)):
        a, b = a.detach().cpu().double(), b.detach()
        assert (a - b).abs().max() <= 256 * 2.0 ** -24 * max(1.0, float(b.abs().max())), k


def test_one_output_in_16_bits_and_without_weights():
    from crystalframer_amd import cuda_funcs
    x = torch.randn(6, 64).to(BF16).cuda().requires_grad_()
    w = torch.ones(64, device="cuda", requires_grad=True)
    h, y = cuda_funcs.residual_norm(x, None, w, twice_differentiable=True)
    g, gw = torch.autograd.grad(y.float().square().sum(), (x, w), create_graph=True)
    assert g.dtype == BF16 and gw.dtype == F32
    plain, = torch.autograd.grad(cuda_funcs.residual_norm(x, None, w)[1].float().square().sum(), w)
    assert (gw - plain).abs().max() <= 64 * 2.0 ** -24 * 6 * 16
    gg, = torch.autograd.grad(gw.sum(), x, retain_graph=True)
    assert gg.dtype == BF16 and gg.shape == x.shape and torch.isfinite(gg).all()
    gh, = torch.autograd.grad(h.float().square().sum(), x, create_graph=True)       # h alone: twice x
    assert torch.equal(gh, (2 * x).to(BF16)) and torch.autograd.grad(gh.float().sum(), x)[0].eq(2).all()
    y = cuda_funcs.residual_norm(x.detach().float().requires_grad_(), keep_residual=False, twice_differentiable=True)
    assert y.requires_grad


def test_a_pass_that_is_not_recorded_is_the_same_to_the_bit():
    from crystalframer_amd import cuda_funcs
    t = [torch.randn(9, 200, device="cuda"), torch.randn(9, 200, device="cuda"), torch.rand(200, device="cuda"), torch.randn(200, device="cuda")]
    g = torch.randn(9, 200, device="cuda")
    grads = []
    for twice in (False, True):
        leaves = [v.clone().requires_grad_() for v in t]
        grads.append(torch.autograd.grad(cuda_funcs.residual_norm(*leaves, twice_differentiable=twice)[1], leaves, g))
    assert all(torch.equal(a, b) for a, b in zip(*grads))


def test_refusals():
    from crystalframer_amd import cuda_funcs
    x = torch.zeros(4, 32, device="cuda")
    v = torch.zeros(32, device="cuda")
    for options in (dict(norm="rms"), dict(norm=None), dict(block=x, block_norm="layer"), dict(block=x, gate=v), dict(residual_scale=0.5),
                    dict(block=x, block_scale=0.5)):
        with pytest.raises(ValueError, match="second derivatives"):
            cuda_funcs.residual_norm(x, **options, twice_differentiable=True)
