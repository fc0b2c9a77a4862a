"""Causal attention over more keys than any query sees: what memory holds in their place does not matter, and their gradients are 0."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _run(x, go, of, **kw):
    from crystalframer_amd import cuda_funcs
    t = [u.detach().requires_grad_() for u in x]
    out = cuda_funcs.relative_attention(*t, of, causal=True, **kw)
    return (out.detach(), *torch.autograd.grad(out, t, go))


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=str)
@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("B,tq,tk", [(1, 1, 40), (2, 5, 64), (3, 40, 45), (1, 130, 300), (24, 150, 170)])
@pytest.mark.parametrize("bad", [math.inf, math.nan])
def test_keys_that_no_query_sees(bad, B, tq, tk, packed, dtype):
    from crystalframer_amd import cuda_funcs
    gen = torch.Generator().manual_seed(tk)
    rnd = lambda *s: torch.randn(*s, generator=gen).to(dtype).cuda()  # noqa: E731
    q, k, v, go, table = rnd(B, tq, 4, 64), rnd(B, tk, 2, 64), rnd(B, tk, 2, 64), rnd(B, tq, 4, 64), rnd(8, 4)
    of = cuda_funcs.position_buckets(8, 20, False, device="cuda")
    kw = {}
    place = lambda t: t  # noqa: E731
    if packed:
        place = lambda t: t.flatten(0, 1)  # noqa: E731
        kw = {n: torch.arange(B + 1, device="cuda") * each for n, each in (("query_starts", tq), ("key_starts", tk))}
    results = []
    for fill in (0.0, bad):
        k[:, tq:], v[:, tq:] = fill, fill
        results.append(_run((place(q), place(k), place(v), table), place(go), of, **kw))
    for name, a, b in zip(("out", "query", "key", "value", "table"), *results):
        assert a.isfinite().all() and torch.equal(a, b), name
    for g in results[1][2:4]:
        assert (g.view(B, tk, 2, 64)[:, tq:] == 0).all()
