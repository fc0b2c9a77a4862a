"""Attention between sequences of tensors in other orders than (batch, positions, heads, channels): results and gradients have the bits of
the same tensors laid out in that order."""
import pytest
import torch

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _call(query, key, value, packed, **kw):
    from crystalframer_amd import cuda_funcs
    if packed:
        kw.update(query_starts=torch.tensor([0, 4, 9], device="cuda"), key_starts=torch.tensor([0, 7, 40], device="cuda"))
    return cuda_funcs.cross_attention(query, key, value, **kw)


def _equal(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b))


# channels do not fill their last 16 bytes in the first of each type, and do in the last
SIZES = [(F32, 7), (F32, 42), (F32, 32), (BF16, 20), (BF16, 100), (BF16, 32), (F16, 42), (F16, 3), (F16, 32)]
# the order of (batch, positions, heads, channels) in memory, from the outermost on
ORDERS = [(0, 2, 3, 1), (0, 3, 1, 2), (1, 0, 2, 3), (0, 1, 3, 2), (3, 2, 1, 0), (2, 3, 0, 1)]


def _laid_out(t, order):
    """t with its dimensions in memory in this order (packed tensors: without the first of them)."""
    order = [n - (4 - t.dim()) for n in order if n >= 4 - t.dim()]
    return t.permute(order).contiguous().permute([order.index(n) for n in range(t.dim())])


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("order", ORDERS, ids=str)
@pytest.mark.parametrize("dtype,dim", SIZES, ids=str)
def test_inputs_and_gradients_in_any_order(dtype, dim, order, packed):
    gen = torch.Generator().manual_seed(dim)
    rows = ((9,), (40,)) if packed else ((2, 5), (2, 21))
    x = [torch.randn(*rows[n > 0], 6 if n == 0 else 3, dim, generator=gen).to(dtype).cuda() for n in range(3)]
    go = torch.randn(x[0].shape, generator=gen).to(dtype).cuda()

    def both(place, place_go):
        t = [place(u).detach().requires_grad_() for u in x]
        out = _call(*t, packed)
        return (out.detach(), *torch.autograd.grad(out, t, place_go(go)))
    plain = both(lambda u: u, lambda u: u)
    other = lambda u: _laid_out(u, order)  # noqa: E731
    assert _equal(plain, both(other, other))
    assert _equal(plain, both(lambda u: u, other))
    assert _equal(plain, both(other, lambda u: u))


@pytest.mark.parametrize("dtype,dim", [(F32, 7), (BF16, 20)])
def test_a_convolution_over_positions_behind_an_attention(dtype, dim):
    """Its gradient comes back with the positions next to one another."""
    torch.manual_seed(0)
    x = [torch.randn(2, n, 3, dim).to(dtype).cuda().requires_grad_() for n in (28, 31, 31)]
    conv = torch.nn.Conv1d(3 * dim, 5, 3).to(dtype).cuda()
    out = _call(*x, False)
    seen = []
    out.register_hook(seen.append)
    conv(out.flatten(2).transpose(1, 2)).float().square().sum().backward()
    want = torch.autograd.grad(_call(*x, False), x, seen[0].contiguous())
    assert _equal([t.grad for t in x], want)
