"""The table's gradient where one bucket takes most of a row's probability.

Its entry b is the sum over rows of P_ib (a_ib - D_i), with P_ib the probability of the row's keys in b, a_ib the mean of do_i . v_j over them and
D_i that over all keys: what is off in a_ib against D_i in the same way in every row stays, and is large against a gradient that is
small where P_ib is near 1."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T, D, buckets, distance", [(551, 96, 10, 383), (551, 128, 10, 383), (78, 16, 12, 70), (1030, 40, 6, 1000)])
def test_gradient_of_a_wide_bucket_float32(T, D, buckets, distance):
    from crystalframer_amd import cuda_funcs
    B, H = 6, 4
    gen = torch.Generator().manual_seed(T + D)
    rnd = lambda *s: torch.randn(*s, generator=gen).cuda()  # noqa: E731
    q, k, v, go, table = rnd(B, T, H, D), rnd(B, T, H, D) * 0.5, rnd(B, T, H, D), rnd(B, T, H, D), rnd(buckets, H) * 0.7
    of = cuda_funcs.position_buckets(buckets, distance, bidirectional=False, device="cuda")      # half of all pairs: bucket 0
    leaf = table.clone().requires_grad_()
    got = torch.autograd.grad(cuda_funcs.relative_attention(q.requires_grad_(), k, v, leaf, of), leaf, go)[0]

    at = torch.arange(T, device="cuda")
    bucket = of.long()[(at[None] - at[:, None]).clamp(-distance, distance) + distance]
    want, size = torch.zeros(buckets, H, dtype=torch.float64, device="cuda"), torch.zeros(buckets, H, dtype=torch.float64, device="cuda")
    for b in range(B):
        for h in range(H):
            x = {n: t[b, :, h].detach().double() for n, t in dict(q=q, k=k, v=v, go=go).items()}
            P = torch.softmax(x["q"] @ x["k"].T / D ** 0.5 + table[:, h].double()[bucket], 1)
            dp = x["go"] @ x["v"].T
            D_i = (P * dp).sum(1, keepdim=True)
            flat = bucket.flatten()
            each = lambda y: torch.zeros(buckets, dtype=torch.float64, device="cuda").index_add_(0, flat, y.flatten())  # noqa: E731
            want[:, h] += each(P * (dp - D_i))
            # the two sums that a relative error common to all rows enters
            size[:, h] += each(P * dp).abs() + each(P * D_i).abs()
    # A matrix instruction may cut its sum below the last place: ceil(D / 16) additions into the sum and one of the small products' own, each less
    # than 2^-23 of it; D and the output as many roundings again.  What has no common sign, 2^-24 of terms sqrt(rows) times as small, is in that.
    steps = (D + 15) // 16 + 1
    bound = 2 * steps * 2.0 ** -24 * size.norm() + 8 * 2.0 ** -24 * want.norm()
    off = (got.double() - want).norm()
    print(f"off {off / want.norm():.2e}, bound {bound / want.norm():.2e}")
    assert off <= bound
