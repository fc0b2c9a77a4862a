"""One training step of an encoder with layer norms through the joined norms, the clipping inside the step and AdamW's moments in 8 or 32 bits, against
the same step made of torch.nn.LayerNorm and additions, torch.nn.utils.clip_grad_norm_ and torch.optim.AdamW; and inference as it is served.

The two paths' gradients differ by rounding: 1e-4 of a tensor's largest, what the model is held to (test_gpu_normed_model).  With
d = 1e-4 max |g| per tensor the norms differ by the root of the sum of n d^2 at most.  The first step moves a parameter by
lr f(c g), f(z) = z / (|z| + eps), whose slope is eps / (|z| + eps)^2: for |g| > 2 d + the change of c the two moves differ by
lr times the slope at the smaller of the two times the distance, elsewhere by 2 lr."""
import copy

import pytest
import torch

from test_gpu_normed_model import _batch, _model

pytestmark = pytest.mark.gpu
LR, EPS, WD, MOST = 1e-3, 1e-8, 1e-2, 0.05


@pytest.mark.parametrize("norm_first", [False, True])
@pytest.mark.parametrize("bits", [8, 32])
def test_a_step_against_the_frameworks(bits, norm_first, monkeypatch):
    from crystalframer_amd import encoder, optim
    base, batch, target = _model(norm_first), _batch(), torch.linspace(-1, 1, 9, device="cuda")[:, None]
    base(batch).sum().backward()              # the first training pass stores the normalisation of the Gaussian widths
    base.zero_grad()

    def backward(fused):
        monkeypatch.setattr(encoder, "FUSED_RESIDUAL_NORM", fused)
        model = copy.deepcopy(base)
        torch.nn.functional.mse_loss(model(batch), target).backward()
        return model
    ours, theirs = backward(True), backward(False)
    before = [p.detach().clone() for p in ours.parameters()]
    grads = [None if p.grad is None else p.grad.double() for p in ours.parameters()]
    ref = [None if p.grad is None else p.grad.double() for p in theirs.parameters()]
    opt = optim.AdamW(ours.parameters(), lr=LR, eps=EPS, weight_decay=WD, state_bits=bits, max_grad_norm=MOST)
    opt.step()
    norm = float(torch.nn.utils.clip_grad_norm_(theirs.parameters(), MOST))
    torch.optim.AdamW(theirs.parameters(), lr=LR, eps=EPS, weight_decay=WD).step()
    assert norm > 2 * MOST                    # (it is clipped)
    off = sum(g.numel() * (1e-4 * float(g.abs().max())) ** 2 for g in ref if g is not None) ** 0.5
    assert abs(float(opt.grad_norm) - norm) <= off + 1e-6 * norm
    c, dc = MOST / norm, MOST / norm * (off / norm + 1e-5)
    for (n, p), q, b, g, r in zip(ours.named_parameters(), theirs.parameters(), before, grads, ref):
        assert (g is None) == (r is None), n
        if r is None:
            assert torch.equal(p, b) and torch.equal(q, b)
            continue
        d = 1e-4 * r.abs().max()
        assert (g - r).abs().max() <= d or r.abs().max() <= 1e-6 * max(x.abs().max() for x in ref if x is not None), n
        distance = c * (g - r).abs() + dc * g.abs()
        least = torch.minimum(c * r.abs(), (c - dc) * g.abs())
        same = torch.sign(g) == torch.sign(r)
        bound = torch.where(same, torch.clamp(distance * EPS / (least + EPS) ** 2, max=2.0), 2.0) * LR
        # roundings: of the parameter (each side), of the move
        assert ((p.double() - q.double()).abs() <= bound + 4 * 2.0 ** -24 * b.double().abs() + 16 * 2.0 ** -24 * LR).all(), n


@pytest.mark.parametrize("norm_first", [False, True])
def test_a_captured_pass(norm_first):
    from crystalframer_amd import encoder
    model, batch = _model(norm_first).eval(), _batch()
    with torch.no_grad():
        want = model(batch)
    norm = model.encoder.norm
    x, block = torch.randn(2, 50, 128, device="cuda")
    with torch.no_grad():
        normed = encoder._normed_sum(norm, x, block, keep_sum=True)
    with torch.inference_mode():
        assert all(torch.equal(a, b) and a.is_inference() for a, b in zip(encoder._normed_sum(norm, x, block, keep_sum=True), normed))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side), torch.no_grad():
        model(batch)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.no_grad(), torch.cuda.graph(graph):
        out = model(batch)
    for _ in range(3):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        with torch.no_grad():
            assert torch.equal(model(batch), want)
