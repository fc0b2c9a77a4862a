"""Attention between sequences where a rule on sizes takes a kernel of its own: reaches that leave a workgroup one wavefront, caches that
go past the processor's, rows that are laid out again under capture.  Tolerances: see attention_reference."""
import pytest
import torch

import attention_reference as AR

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _random(seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return lambda *s: torch.randn(*s, generator=gen, device="cuda")


@pytest.mark.parametrize("dim", [65, 96, 128])
@pytest.mark.parametrize("reach", [809, 810, 1024])
def test_long_reaches_of_wide_heads_in_float32(reach, dim):
    """Biases and their sums beside tiles of 24 KB: up to a reach of 809 there is room for four wavefronts' sums."""
    from crystalframer_amd import cuda_funcs
    rnd = _random(reach + dim)
    Tq, Tk, H, G, buckets = 130, 1100, 2, 1, 24
    x = [t.requires_grad_() for t in (rnd(1, Tq, H, dim), rnd(1, Tk, G, dim), rnd(1, Tk, G, dim), rnd(buckets, H))]
    go = rnd(1, Tq, H, dim)
    of = cuda_funcs.position_buckets(buckets, reach, True)
    out = cuda_funcs.relative_attention(*x, of.cuda(), queries_last=True)
    got = dict(zip(("out", "dq", "dk", "dv", "dtable"), (out.detach(), *torch.autograd.grad(out, x, go))))
    q, k, v, table = (t.detach().cpu() for t in x)
    bucket, side, _ = AR.relative(Tq, Tk, True, of, reach)
    want, tol = AR.attention(q[0], k[0], v[0], torch.ones(Tq, Tk, dtype=torch.bool), bias=table.double()[bucket].permute(2, 0, 1),
                             go=go[0].cpu(), bucket=bucket, buckets=buckets, reach_index=side)
    for name, a in got.items():
        a = a.cpu().double() if name == "dtable" else a[0].cpu().double()
        bound = tol[name] + (AR.HALF[F32] * want[name].abs() + AR.TINY[F32] if name == "dtable" else 0.0)
        assert bool(((a - want[name]).abs() <= bound).all()), name


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=str)
@pytest.mark.parametrize("relative", [False, True])
@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("dim", [20, 64, 128])
def test_long_caches(dim, packed, relative, dtype):
    """Single tokens, 128 MB of keys and values and more: some of the sequences and heads against float64, masked and of their own lengths,
    with NaN in the place of what is not there."""
    from crystalframer_amd import cuda_funcs
    rnd = _random(dim)
    B, H, G = 4, 16, 8
    T = (1 << 27) // (2 * dtype.itemsize * B * G * dim) + 33
    assert 2 * B * T * G * dim * dtype.itemsize >= 1 << 27
    q, k, v = (rnd(B, n, h, dim).to(dtype) for n, h in ((1, H), (T, G), (T, G)))
    sizes = [T, 1, T - 700, 2000]
    mask = torch.rand(B, T, generator=torch.Generator().manual_seed(1)) < 0.9
    mask[1, 0] = True
    keep = mask & (torch.arange(T) < torch.tensor(sizes)[:, None])
    for t in (k, v):
        t[~keep.cuda()] = float("nan")
    kw = dict(key_mask=mask.cuda(), key_sizes=torch.tensor(sizes, device="cuda"))
    if packed:
        ends = torch.tensor([0, T, 2 * T, 3 * T, 4 * T], device="cuda")
        kw = dict(key_mask=keep.flatten().cuda(), query_starts=torch.arange(B + 1, device="cuda"), key_starts=ends)
        sizes = [T] * B
    extra = {}
    call = [t.flatten(0, 1) if packed else t for t in (q, k, v)]
    if relative:
        of, table = cuda_funcs.position_buckets(32, 128, False), rnd(32, H).to(dtype)
        out = cuda_funcs.relative_attention(*call, table, of.cuda(), causal=True, queries_last=True, **kw)
    else:
        out = cuda_funcs.cross_attention(*call, **kw)
    out = out.view(B, 1, H, dim)
    for b, h in ((0, 0), (0, 15), (1, 3), (2, 8), (3, 15)):
        n = sizes[b]
        if relative:
            bucket, _, _ = AR.relative(1, n, True, of, 128)
            extra = dict(bias=table[:, h:h + 1].cpu().double()[bucket].permute(2, 0, 1))
        g = slice(h // 2, h // 2 + 1)
        want, tol = AR.attention(q[b, :, h:h + 1].cpu(), k[b, :n, g].cpu(), v[b, :n, g].cpu(), keep[b, :n][None], **extra)
        assert bool(((out[b, :, h:h + 1].cpu().double() - want["out"]).abs() <= tol["out"]).all()), (b, h)


@pytest.mark.parametrize("dtype,dim", [(F32, 7), (BF16, 20), (F16, 33)], ids=str)
def test_rows_laid_out_again_under_capture(dtype, dim):
    from crystalframer_amd import cuda_funcs
    rnd = _random(dim)
    x = [rnd(2, n, 3, dim).to(dtype).requires_grad_() for n in (28, 61, 61)]
    go = rnd(2, 3, dim, 28).to(dtype).permute(0, 3, 1, 2)

    def run():
        out = cuda_funcs.cross_attention(*x)
        return (out.detach(), *torch.autograd.grad(out, x, go))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run()
    for n in range(4):
        with torch.no_grad():
            for t in x:
                t.copy_(rnd(*t.shape).to(dtype))
            for t in got:
                t.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, run())), n


def test_compiled_programs_call_it_as_it_is():
    """torch.compile breaks its graph at the call and goes on behind it."""
    from crystalframer_amd import cuda_funcs
    rnd = _random(0)
    x = [rnd(2, n, 4, 16).requires_grad_() for n in (9, 20, 20)]

    def run(q, k, v):
        return (cuda_funcs.cross_attention(q * 2.0, k, v) + 1.0).square()
    want = run(*x)
    got = torch.compile(run, backend="eager")(*x)
    assert torch.equal(got, want)
    for a, b in zip(torch.autograd.grad(got.sum(), x), torch.autograd.grad(want.sum(), x)):
        assert torch.equal(a, b)
