"""Checkpoints and copies of ``optim.AdamW`` on the device: what hooks make of a load reaches the moments that the kernels use."""
import copy
import io
import pickle

import pytest
import torch

pytestmark = pytest.mark.gpu
HYPER = dict(lr=3e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2)


def _optimizer(dtype, bits, seed=0, **options):
    from crystalframer_amd import optim
    gen = torch.Generator().manual_seed(seed)
    ps = [torch.nn.Parameter((0.1 * torch.randn(n, generator=gen)).to(dtype).cuda()) for n in (5, 70, 4097)]
    return ps, optim.AdamW(ps, **HYPER, state_bits=bits, **options)


def _steps(ps, opt, seeds):
    for seed in seeds:
        gen = torch.Generator().manual_seed(seed)
        for p in ps:
            p.grad = torch.randn(p.shape, generator=gen).to(p.dtype).cuda()
        opt.step()


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_hooks_of_a_load_reach_the_moments(dtype, bits):
    a, one = _optimizer(dtype, bits)
    b, two = _optimizer(dtype, bits)
    _steps(a, one, (1, 2)), _steps(b, two, (3, 4))
    saved, other = one.state_dict(), two.state_dict()
    c, three = _optimizer(dtype, bits)
    three.register_load_state_dict_pre_hook(lambda o, state: dict(state, state=other["state"]))

    def after(o):
        o.state[c[1]]["exp_avg"] = torch.zeros_like(o.state[c[1]]["exp_avg"].view(torch.uint8) if bits == 8 else o.state[c[1]]["exp_avg"])
        if bits == 8:
            o.state[c[1]]["exp_avg"] = o.state[c[1]]["exp_avg"].view(torch.float8_e4m3fn)
    three.register_load_state_dict_post_hook(after)
    three.load_state_dict(saved)
    names = list(three.state[c[0]])
    assert len(names) == (5 if bits == 8 else 3)
    for k, (p, q) in enumerate(zip(c, b)):
        for name in names:
            want = torch.zeros_like(two.state[q][name].view(torch.uint8)) if (k, name) == (1, "exp_avg") else two.state[q][name].view(torch.uint8)
            assert torch.equal(three.state[p][name].view(torch.uint8), want), (k, name)
    (m, v), = three.moments()
    (m2, v2), = two.moments()
    assert torch.equal(v, v2) and not m[64:64 + 70].any() and torch.equal(m[64 + 128:], m2[64 + 128:])


@pytest.mark.parametrize("bits", [8, 32])
def test_copies_go_on_clipping(bits):
    a, one = _optimizer(torch.float32, bits, max_grad_norm=0.1)
    _steps(a, one, (1, 2))
    file = io.BytesIO()
    torch.save(one, file)
    file.seek(0)
    copies = [copy.deepcopy(one), pickle.loads(pickle.dumps(one)), torch.load(file, weights_only=False)]
    for two in copies:
        assert torch.equal(two.grad_norm, one.grad_norm)
    _steps(a, one, (3, 4))
    for two in copies:
        b = two.param_groups[0]["params"]
        _steps(b, two, (3, 4))
        assert all(torch.equal(p, q) for p, q in zip(a, b)) and torch.equal(two.grad_norm, one.grad_norm)
