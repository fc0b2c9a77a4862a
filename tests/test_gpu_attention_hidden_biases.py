"""Biases by relative position that no visible key has: plus infinity or NaN in their entries of the table changes nothing.  A row that
sees such a key is NaN, as its softmax is."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
BEHIND, HERE, AHEAD = 1, 0, 2


def _map(reach):
    of = torch.zeros(2 * reach + 1, dtype=torch.int32)
    of[:reach], of[reach + 1:] = BEHIND, AHEAD
    return of.cuda()


def _run(x, table, go, of, **kw):
    from crystalframer_amd import cuda_funcs
    t = [u.detach().requires_grad_() for u in (*x, table)]
    out = cuda_funcs.relative_attention(*t, of, **kw)
    return (out.detach(), *torch.autograd.grad(out, t, go))


def _check(B, tq, tk, H, G, D, dtype, reach, bucket, bad, **kw):
    gen = torch.Generator().manual_seed(tq)
    rnd = lambda *s: torch.randn(*s, generator=gen).to(dtype).cuda()  # noqa: E731
    x, go, of = (rnd(B, tq, H, D), rnd(B, tk, G, D), rnd(B, tk, G, D)), rnd(B, tq, H, D), _map(reach)
    table = rnd(3, H)
    table[bucket] = 0.0
    want = _run(x, table, go, of, **kw)
    odd = table.clone()
    odd[bucket] = bad
    got = _run(x, odd, go, of, **kw)
    for name, a, b in zip(("out", "query", "key", "value", "table"), got, want):
        assert b.isfinite().all() and torch.equal(a, b), name
    assert (got[4][bucket] == 0).all()


SHAPES = [(1, 3, 300), (2, 40, 70), (1, 150, 400), (24, 150, 290)]      # few queries and tiles of them, with and without parts


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=str)
@pytest.mark.parametrize("B,tq,tk", SHAPES)
@pytest.mark.parametrize("reach", [1, 4, 200])
@pytest.mark.parametrize("bad", [math.inf, math.nan])
def test_masked_keys(bad, reach, B, tq, tk, dtype):
    """Queries are the last positions; keys ahead of the first of them are masked."""
    mask = (torch.arange(tk, device="cuda") <= tk - tq).expand(B, tk)
    _check(B, tq, tk, 4, 2, 64, dtype, reach, AHEAD, bad, queries_last=True, key_mask=mask)


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=str)
@pytest.mark.parametrize("B,tq,tk", SHAPES)
@pytest.mark.parametrize("reach", [1, 4, 200])
@pytest.mark.parametrize("bad", [math.inf, math.nan])
def test_keys_behind_a_causal_query(bad, reach, B, tq, tk, dtype):
    _check(B, tq, tk, 4, 2, 64, dtype, reach, AHEAD, bad, causal=True, queries_last=True)


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=str)
@pytest.mark.parametrize("B,tq,tk", SHAPES)
@pytest.mark.parametrize("reach", [1, 4, 200])
@pytest.mark.parametrize("bad", [math.inf, math.nan])
def test_rows_behind_the_lengths(bad, reach, B, tq, tk, dtype):
    """One query at position 0: what a row behind it would see further back, or a key behind the last one ahead, is not there."""
    one = torch.ones(B, dtype=torch.int64, device="cuda")
    _check(B, tq, tk, 4, 2, 64, dtype, reach, BEHIND, bad, query_sizes=one)
    _check(B, tq, tk, 4, 2, 64, dtype, reach, AHEAD, bad, key_sizes=one)
    _check(B, tq, tk, 4, 2, 64, dtype, reach, BEHIND, bad, query_sizes=one, key_sizes=one)


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=str)
@pytest.mark.parametrize("B,tq,tk", SHAPES)
@pytest.mark.parametrize("reach", [1, 4, 200])
@pytest.mark.parametrize("bad", [math.inf, math.nan])
def test_rows_that_see_them(bad, reach, B, tq, tk, dtype):
    """Only the first query has no key behind it."""
    from crystalframer_amd import cuda_funcs
    torch.manual_seed(0)
    q, k, v = (torch.randn(B, n, 4, 64).to(dtype).cuda() for n in (tq, tk, tk))
    table = torch.zeros(3, 4, dtype=dtype, device="cuda")
    want = cuda_funcs.relative_attention(q, k, v, table, _map(reach))
    table[BEHIND] = bad
    got = cuda_funcs.relative_attention(q, k, v, table, _map(reach))
    assert torch.equal(got[:, :1], want[:, :1]) and got[:, 1:].isnan().all()
