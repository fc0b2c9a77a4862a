"""Attention between sequences whose inputs are shared along a batch or along heads, have no entries, or scores of no size."""
import pytest
import torch

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _run(x, go, table=None, **kw):
    from crystalframer_amd import cuda_funcs
    t = [u.detach().requires_grad_() for u in (*x, *([] if table is None else [table]))]
    if table is None:
        out = cuda_funcs.cross_attention(*t, **kw)
    else:
        out = cuda_funcs.relative_attention(*t, cuda_funcs.position_buckets(8, 20, device="cuda"), **kw)
    return (out.detach(), *torch.autograd.grad(out, t, go))


def _equal(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=str)
@pytest.mark.parametrize("D", [20, 64])
@pytest.mark.parametrize("relative", [False, True])
def test_states_shared_by_a_batch_and_by_heads(relative, D, dtype):
    """Strides of 0 along the batch and the heads, windows that overlap, and gradients of what they were made from."""
    torch.manual_seed(D)
    B, Tq, Tk, H, G = 3, 33, 70, 4, 2
    rnd = lambda *s: torch.randn(*s).to(dtype).cuda()  # noqa: E731
    q, k, v, go = rnd(B, Tq, H, D), rnd(1, Tk, G, D), rnd(B, Tk, 1, D), rnd(B, 1, H, D)
    table = rnd(8, H) if relative else None
    x = [q, k.expand(B, Tk, G, D), v.expand(B, Tk, G, D)]
    assert _equal(_run(x, go.expand(B, Tq, H, D), table), _run([t.contiguous() for t in x], go.expand(B, Tq, H, D).contiguous(), table))
    long = rnd(2 * Tk, G, D)
    windows = long.unfold(0, Tk, 10).movedim(-1, 1)[:B]                  # (B, Tk, G, D) of rows that lie in several of them
    x = [q, windows, windows]
    assert _equal(_run(x, go.expand(B, Tq, H, D), table), _run([t.contiguous() for t in x], go.expand(B, Tq, H, D).contiguous(), table))


@pytest.mark.parametrize("dtype", [F32, BF16], ids=str)
@pytest.mark.parametrize("B,Tq,Tk", [(0, 5, 7), (2, 0, 7), (2, 5, 0), (2, 0, 0), (0, 0, 0)])
@pytest.mark.parametrize("relative", [False, True])
def test_nothing_to_do(relative, B, Tq, Tk, dtype):
    rnd = lambda *s: torch.randn(*s).to(dtype).cuda()  # noqa: E731
    table = rnd(8, 4) if relative else None
    for D in (16, 20):
        got = _run([rnd(B, Tq, 4, D), rnd(B, Tk, 2, D), rnd(B, Tk, 2, D)], rnd(B, Tq, 4, D), table)
        assert [tuple(g.shape[:2]) for g in got[:4]] == [(B, Tq), (B, Tq), (B, Tk), (B, Tk)]
        assert all((g == 0).all() for g in got)


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=str)
@pytest.mark.parametrize("scale", [1e-45, 1e-40, 2.0 ** -130, 1e-30])
def test_scales_that_leave_a_mean(scale, dtype):
    """Scores of 0 but for 2^-60: outputs are means of the visible keys' whole numbers of up to 4, off by one rounding of the result and some
    of float32."""
    torch.manual_seed(0)
    for B, Tq, Tk in ((2, 3, 64), (24, 150, 256)):
        q, k = torch.randn(B, Tq, 4, 64).to(dtype).cuda(), torch.randn(B, Tk, 4, 64).to(dtype).cuda()
        v = torch.randint(-4, 5, (B, Tk, 4, 64)).to(dtype).cuda()
        mask = torch.zeros(B, Tk, dtype=torch.bool)
        mask[:, 5:37] = True
        got = _run([q, k, v], torch.ones(B, Tq, 4, 64, dtype=dtype, device="cuda"), scale=scale, key_mask=mask.cuda())
        want = v[:, 5:37].double().mean(1, keepdim=True)
        assert (got[0].double() - want).abs().max() <= 4 * torch.finfo(dtype).eps / 2 + 2.0 ** -20
        assert all(g.isfinite().all() for g in got)
