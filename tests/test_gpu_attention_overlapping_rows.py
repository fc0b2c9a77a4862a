"""Attention between sequences whose rows share their memory (a row expanded over positions) or are a single one: what is there
counts as often as it is there, infinities among it."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
INF = math.inf


def _run(x, go, **kw):
    from crystalframer_amd import cuda_funcs
    t = [u.detach().requires_grad_() for u in x]
    out = cuda_funcs.cross_attention(*t, **kw)
    return (out.detach(), *torch.autograd.grad(out, t, go))


def _same(a, b):
    for x, y in zip(a, b):
        torch.testing.assert_close(x, y, rtol=0, atol=0, equal_nan=True)


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=str)
@pytest.mark.parametrize("tq,tk", [(1, 45), (45, 45), (150, 300)])
@pytest.mark.parametrize("infinite", [False, True])
def test_one_row_for_all_positions(tq, tk, infinite, dtype):
    """Lengths end inside tiles; the rows behind them are in the same memory."""
    torch.manual_seed(tq)
    B, H, D = 3, 4, 64
    q, k, v, go = (torch.randn(B, 1, H, D).to(dtype).cuda() for _ in range(4))
    if infinite:
        v[:, :, :, 5], go[:, :, :, 9] = INF, -INF
    x = [q.expand(B, tq, H, D), k.expand(B, tk, H, D), v.expand(B, tk, H, D)]
    sizes = dict(query_sizes=torch.tensor([tq, max(1, tq - 7), 0], device="cuda"), key_sizes=torch.tensor([tk - 1, 0, 33], device="cuda"))
    _same(_run(x, go.expand(B, tq, H, D), **sizes), _run([u.contiguous() for u in x], go.expand(B, tq, H, D).contiguous(), **sizes))


@pytest.mark.parametrize("dtype", [BF16, F16], ids=str)
@pytest.mark.parametrize("B", [1, 70])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("tq", [1, 3, 130])
def test_a_single_key_of_infinite_value(tq, D, B, dtype):
    """The probability of an only key is 1, so that its value is the output, and the sum of the outputs' gradients its gradient."""
    torch.manual_seed(0)
    q, k, v, go = (torch.randn(B, n, 4, D).to(dtype).cuda() for n in (tq, 1, 1, tq))
    v[..., 3], v[..., 4] = INF, -INF
    out = _run([q, k, v], torch.zeros_like(go))[0]
    assert torch.equal(out, v.expand_as(out))
    one = go[:, :1].clone()
    one[..., 7] = INF
    v[..., 3], v[..., 4] = 1.0, 2.0
    dv = _run([q[:, :1], k, v], one)[3]
    assert torch.equal(dv, one)
