"""optim.AdamW over as many elements as choose each form of its kernels, against float64 (training_reference): up to 512 * 2048
elements (test_gpu_adamw_moments), more, and more bytes than the last cache holds; the gradients' norm over more than 512 * 8192.
Tolerances as in test_gpu_adamw_moments."""
import numpy as np
import pytest
import torch

import training_reference as TR
from test_gpu_adamw_moments import BF16, F16, F32, HYPER, Reference, _check, _grads, _numbers, _params

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("dtype", [F32, BF16, F16, "mixed"])
def test_whole_chunks_and_odd_ends(dtype, bits):
    """1.05 M elements and a few: chunks of 2048, with 4 or 8 elements of a lane."""
    from crystalframer_amd import optim
    shapes = [(1021, 1001), (20011,), (2048,), (2049,), (4095,), (63,), (1,)]
    params = _params([(F32, BF16, F16)[k % 3] for k in range(len(shapes))] if dtype == "mixed" else dtype, shapes)
    assert sum(p.numel() for p in params) >= 512 * 2048
    opt = optim.AdamW(params, **HYPER, state_bits=bits, max_grad_norm=0.5)
    ref = Reference(params, bits)
    for step in range(2):
        _grads(params, step)
        before = [p.detach().clone() for p in params]
        grads = _numbers([p.grad for p in params])
        norm = float(np.sqrt(sum((g * g).sum() for g in grads)))
        opt.step()
        assert abs(float(opt.grad_norm) - norm) <= 2.0 ** -23 * norm
        _check(opt, params, before, ref.step(_numbers(before), grads, float(np.float32(min(1.0, 0.5 / (norm + 1e-6))))), ref, bits)


def _sampled(dtype, bits, n):
    """Two steps over a tensor of n elements and a short one; places of the long one against the reference: its begin, around a
    border of the chunks, its end.  (All of them whole blocks of 64 but for the end: a block shares a scale.)"""
    from crystalframer_amd import optim
    gen = torch.Generator(device="cuda").manual_seed(1)
    rnd = lambda k, by: (by * torch.randn(k, generator=gen, device="cuda")).to(dtype)  # noqa: E731
    params = [torch.nn.Parameter(rnd(n, 0.1)), torch.nn.Parameter(rnd(1001, 0.1))]
    middle = n // 2 // 8192 * 8192
    places = [(0, slice(0, 320)), (0, slice(middle - 128, middle + 192)), (0, slice(n // 64 * 64 - 2048, n)), (1, slice(0, 1001))]
    first = (0, -(-n // 64) * 64)
    states = [TR.State(s.stop - s.start, bits, first[k] + s.start) for k, s in places]
    opt = optim.AdamW(params, **HYPER, state_bits=bits, max_grad_norm=20.0)
    for step in (1, 2):
        for p in params:
            p.grad = rnd(p.numel(), 0.05)
            p.grad[::5] *= 2.0 ** -6
        norm = float(torch.sqrt(sum(part.double().square().sum() for p in params for part in p.grad.split(1 << 24))))
        before = _numbers([params[k][s].clone() for k, s in places])
        opt.step()
        assert abs(float(opt.grad_norm) - norm) <= 2.0 ** -23 * norm
        factor = float(np.float32(min(1.0, 20.0 / (norm + 1e-6))))
        for (k, s), st, b in zip(places, states, before):
            g, = _numbers([params[k].grad[s]])
            want = st.step(b, g, step, HYPER["lr"], HYPER["betas"], HYPER["eps"], HYPER["weight_decay"], factor)
            got, = _numbers([params[k][s]])
            tol = TR.HALF[dtype] * np.abs(want) + TR.TINY[dtype] + 8 * 2.0 ** -24 * (st.size + np.abs(b))
            assert (np.abs(got - want) <= tol).all(), (k, s, np.abs(got - want).max())
            own = opt.state[params[k]]
            if bits == 8:
                scales = slice(s.start // 64, -(-s.stop // 64))
                for name, at, codes in (("exp_avg", s, st.cm), ("exp_avg_sq", s, st.cv), ("exp_avg_scale", scales, st.sm),
                                        ("exp_avg_sq_scale", scales, st.sv)):
                    wrong = np.flatnonzero(own[name].view(torch.uint8)[at].cpu().numpy() != codes)
                    assert not len(wrong), (k, s, name, wrong[:5])
            else:       # three roundings a step, relative to what the moment has been summed from
                for name, x, terms in (("exp_avg", st.m, st.terms), ("exp_avg_sq", st.v, st.v)):
                    got, = _numbers([own[name][s]])
                    assert (np.abs(got - x) <= 8 * step * 2.0 ** -24 * (np.abs(x) + terms)).all(), (k, s, name)
    if bits == 8:
        (m, v), = opt.moments()
        for (k, s), st in zip(places, states):
            for got, x in zip((m, v), st.values()):
                assert np.array_equal(got[first[k] + s.start:first[k] + s.stop].cpu().numpy(), x.astype(np.float32))


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_the_norm_of_many_elements(dtype, bits):
    _sampled(dtype, bits, 512 * 8192 + 12347)


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("dtype,n", [(F32, 68_000_003), (BF16, 135_000_001), (F16, 135_000_001)])
def test_more_than_the_last_cache_holds(dtype, n, bits):
    """Tensors, moments and gradients past the caches: 256 MiB of gradients, and more than that of moments."""
    assert n * dtype.itemsize >= 256 << 20
    _sampled(dtype, bits, n)
