"""``cuda_funcs.cross_attention`` and ``cuda_funcs.relative_attention`` against float64: values and all gradients, over types, lengths,
heads, channels, masks, layouts and strides.  Tolerances: see attention_reference."""
import random

import pytest
import torch

import attention_reference as AR

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TYPES = [F32, BF16, F16]


def _starts(sizes):
    return torch.tensor([sum(sizes[:n]) for n in range(len(sizes) + 1)], dtype=torch.int64)


def _run(sizes, H, G, D, dtype, *, packed=True, mask=0.0, relative=None, causal=False, last=False, train=True, scale=None, seed=0, tail=(0, 0),
         capacity=(0, 0), q_sizes=False, table_type=None, spread=1.0, place=None, garbage=True, need=("query", "key", "value", "table")):
    """sizes: [(queries, keys)]; relative: (buckets tensor, number of buckets)."""
    from crystalframer_amd import cuda_funcs
    gen = torch.Generator().manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    B = len(sizes)
    tq, tk = [s[0] for s in sizes], [s[1] for s in sizes]
    rows_q = (sum(tq) + tail[0],) if packed else (B, max(tq + [capacity[0]]))
    rows_k = (sum(tk) + tail[1],) if packed else (B, max(tk + [capacity[1]]))
    q, go = (rnd(*rows_q, H, D) * spread).to(dtype), rnd(*rows_q, H, D).to(dtype)
    k, v = ((rnd(*rows_k, G, D) * f + 0.2).to(dtype) for f in (spread, 1.0))
    keep = torch.rand(rows_k, generator=gen) >= mask if mask else torch.ones(rows_k, dtype=torch.bool)
    there = torch.zeros(rows_k, dtype=torch.bool)
    at = []
    for b in range(B):
        at.append((slice(sum(tq[:b]), sum(tq[:b + 1])), slice(sum(tk[:b]), sum(tk[:b + 1]))) if packed else
                  ((b, slice(0, tq[b])), (b, slice(0, tk[b]))))
        there[at[b][1]] = True
    if garbage:      # in the place of keys that are not there
        bad = ~(there & keep)
        for x, what in ((k, float("nan")), (v, float("inf"))):
            x[bad] = what
        if packed or q_sizes:      # and of queries
            real = torch.zeros(rows_q, dtype=torch.bool)
            for b in range(B):
                real[at[b][0]] = True
            q[~real], go[~real] = float("inf"), float("nan")
    table = of = None
    reach = 0
    if relative is not None:
        of, buckets = relative
        reach = len(of) // 2
        table = (rnd(buckets, H) * 0.8).to(table_type or dtype)
    place = place or (lambda name, t: t.cuda())
    dev = {n: place(n, t) for n, t in (("query", q), ("key", k), ("value", v)) + ((("table", table),) if table is not None else ())}
    for n in dev:
        if train and n in need:
            dev[n].requires_grad_(True)
    opts = dict(scale=scale)
    if packed:
        opts.update(query_starts=_starts(tq).cuda(), key_starts=_starts(tk).cuda())
    else:
        opts.update(key_sizes=torch.tensor(tk).cuda(), query_sizes=torch.tensor(tq).cuda() if q_sizes else None)
    if mask:
        opts.update(key_mask=keep.cuda())
    if table is None:
        out = cuda_funcs.cross_attention(dev["query"], dev["key"], dev["value"], **opts)
    else:
        out = cuda_funcs.relative_attention(dev["query"], dev["key"], dev["value"], dev["table"], of.cuda(), causal=causal, queries_last=last, **opts)
    assert out.dtype == dtype and out.shape == q.shape
    got = dict(out=out.detach())
    names = dict(query="dq", key="dk", value="dv", table="dtable")
    if train:
        leaves = [n for n in dev if dev[n].requires_grad]
        got.update({names[n]: g for n, g in zip(leaves, torch.autograd.grad(out, [dev[n] for n in leaves], go.cuda()))})
    want = {n: torch.zeros(x.shape, dtype=torch.float64) for n, x in got.items()}
    tol = {n: torch.zeros(x.shape, dtype=torch.float64) for n, x in got.items()}
    for b in range(B):
        Q, K = at[b]
        # (padded queries that no size cuts off are rows like the others, against the same keys)
        Tq = tq[b] if packed or q_sizes else rows_q[1]
        if not packed and not q_sizes:
            Q = (b, slice(0, Tq))
        visible = keep[K][None].expand(Tq, tk[b])
        extra = {}
        if table is not None:
            bucket, side, r = AR.relative(Tq, tk[b], last, of, reach)
            if causal:
                visible = visible & (r <= 0)
            value = torch.cat([table.double(), torch.zeros(1, H, dtype=torch.float64)])
            extra = dict(bias=value[torch.where((bucket >= 0) & (bucket < buckets), bucket, buckets)].permute(2, 0, 1), bucket=bucket, buckets=buckets, reach_index=side)
        res, bound = AR.attention(q[Q], k[K], v[K], visible, scale=scale, go=go[Q] if train else None, **extra)
        for name in got:
            where = dict(out=Q, dq=Q, dk=K, dv=K, dtable=Ellipsis)[name]
            want[name][where] += res[name]
            tol[name][where] += bound[name]
    for name, x in got.items():
        x = x.cpu()
        if name == "dtable":
            assert x.dtype == table.dtype
            tol[name] += AR.HALF[x.dtype] * want[name].abs() + AR.TINY[x.dtype]
        else:
            assert x.dtype == dtype
        off = (x.double() - want[name]).abs()
        assert x.shape == want[name].shape and bool((off <= tol[name]).all()), (
            name, "largest error over its bound", float((off / tol[name].clamp_min(1e-300)).nan_to_num(1e9).max()))
    return got


def _buckets(n, distance, both):
    from crystalframer_amd import cuda_funcs
    return cuda_funcs.position_buckets(n, distance, both), n


LENGTHS = [(1, 1), (1, 2), (2, 1), (1, 31), (5, 33), (31, 32), (33, 64), (65, 63), (1, 257), (129, 130), (200, 7), (3, 700)]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("tq,tk", LENGTHS)
def test_lengths(tq, tk, dtype):
    _run([(tq, tk)], 2, 2, 16, dtype, seed=1)
    _run([(tq, tk)], 2, 1, 64, dtype, packed=False, mask=0.3, seed=2)
    _run([(tq, tk)], 2, 2, 32, dtype, relative=_buckets(8, 20, True), seed=3)
    _run([(tq, tk)], 2, 2, 64, dtype, packed=False, relative=_buckets(6, 9, False), causal=True, last=True, seed=4)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("dim", [1, 2, 3, 7, 8, 15, 16, 17, 24, 33, 40, 63, 64, 65, 80, 96, 100, 127, 128])
def test_channels(dim, dtype):
    _run([(37, 70)], 2, 1, dim, dtype, seed=dim)
    _run([(3, 70)], 2, 2, dim, dtype, relative=_buckets(8, 20, True), seed=dim)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("H,G", [(1, 1), (5, 5), (6, 3), (4, 1), (7, 1), (32, 1), (33, 1), (40, 2), (12, 12)])
def test_heads(H, G, dtype):
    for tq in (1, 3, 50):
        _run([(tq, 90), (2, 20)], H, G, 24, dtype, seed=H, mask=0.2)
    _run([(40, 45)], H, G, 16, dtype, relative=_buckets(9, 30, False), causal=True, seed=H)


RAGGED = [[(3, 40), (0, 5), (17, 0), (1, 1), (0, 0), (70, 90), (64, 33)], [(0, 0)], [(5, 0), (0, 5)], [(1, n) for n in range(1, 40)],
          [(n % 5, n % 7) for n in range(150)], []]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("sizes", RAGGED, ids=lambda s: str(len(s)))
def test_ragged(sizes, dtype):
    """Packed sequences, empty ones among them, with rows behind the last one: those are 0."""
    _run(sizes, 2, 1, 32, dtype, tail=(5, 3), seed=1)
    _run(sizes, 2, 2, 16, dtype, tail=(0, 70), seed=2, mask=0.5)
    _run(sizes, 2, 2, 16, dtype, tail=(33, 0), seed=3, relative=_buckets(8, 16, True))
    _run(sizes, 2, 2, 40, dtype, tail=(1, 1), seed=4, relative=_buckets(4, 6, False), causal=True, last=True)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("q_sizes", [False, True])
def test_padded(q_sizes, dtype):
    sizes = [(7, 40), (9, 1), (3, 0), (9, 64)]
    for kw in (dict(), dict(mask=0.6), dict(relative=_buckets(8, 16, True)), dict(relative=_buckets(8, 16, False), causal=True)):
        _run(sizes, 4, 2, 48, dtype, packed=False, q_sizes=q_sizes, capacity=(50, 70), seed=5, **kw)
    _run([(1, n) for n in (5, 800, 31, 0)], 4, 1, 64, dtype, packed=False, capacity=(1, 900), seed=6, relative=_buckets(32, 128, False),
         causal=True, last=True, train=False)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_rows_that_the_mask_leaves_empty(dtype):
    _run([(20, 30), (130, 140)], 2, 2, 32, dtype, mask=1.0, seed=1)
    _run([(40, 20), (140, 9)], 2, 1, 32, dtype, relative=_buckets(8, 16, False), causal=True, last=True, seed=2)      # rows before the first key
    _run([(1, 20)] * 3, 2, 1, 32, dtype, mask=0.97, seed=3)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("n,distance,both", [(4, 3, True), (32, 128, True), (32, 128, False), (47, 77, True), (128, 600, False), (2, 1024, False)])
def test_buckets(n, distance, both, dtype):
    if n // (2 if both else 1) // 2 >= distance:
        pytest.skip("no such map")
    _run([(150, 300)], 2, 2, 32, dtype, relative=_buckets(n, distance, both), seed=n)
    _run([(300, 300)], 1, 1, 64, dtype, relative=_buckets(n, distance, both), seed=n, causal=not both, table_type=F32)
    _run([(2, 1500)], 2, 1, 16, dtype, relative=_buckets(n, distance, both), seed=n, last=True)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_maps_of_any_kind(dtype):
    """One bucket for all, a bucket for each position in no order, and numbers that are no rows of the table."""
    _run([(40, 50)], 2, 2, 32, dtype, relative=(torch.zeros(1, dtype=torch.int32), 1), seed=1)
    gen = torch.Generator().manual_seed(0)
    _run([(140, 150)], 2, 2, 32, dtype, relative=(torch.randperm(41, generator=gen).int(), 41), seed=2)
    _run([(140, 150), (1, 90)], 2, 2, 32, dtype, relative=(torch.randint(-3, 9, (61,), generator=gen).int(), 5), seed=3)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_large_and_small_scores(dtype):
    _run([(40, 150)], 2, 2, 64, dtype, spread=4.0, seed=1)
    _run([(40, 150)], 2, 2, 64, dtype, scale=1e-3, seed=2)
    _run([(200, 150)], 2, 2, 32, dtype, scale=2.5, seed=3, relative=_buckets(8, 20, True))


def _strided(kind):
    def place(name, t):
        if name == "table":
            return t.t().contiguous().cuda().t() if kind == "transposed" else t.cuda()
        *rows, H, D = t.shape
        if kind == "one projection":                 # part of a wider row, aligned
            wide = torch.full((*rows, 3, H, D), float("nan"), dtype=t.dtype).cuda()
            x = wide[..., 1, :, :]
        elif kind == "heads first":
            x = torch.empty((H, *rows, D), dtype=t.dtype).cuda().movedim(0, -2)
        elif kind == "unaligned":
            flat = torch.full((t.numel() + 1,), float("nan"), dtype=t.dtype).cuda()
            x = flat[1:].view(t.shape)
        elif kind == "odd rows":
            wide = torch.full((*rows, H, D + 3), float("nan"), dtype=t.dtype).cuda()
            x = wide[..., :D]
        elif kind == "transposed":                   # channels apart
            x = torch.empty((*rows, D, H), dtype=t.dtype).cuda().transpose(-1, -2)
        elif kind == "one row for all":
            x = t.cuda()
            return x
        x.copy_(t)
        return x.detach()
    return place


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("kind", ["one projection", "heads first", "unaligned", "odd rows", "transposed"])
@pytest.mark.parametrize("packed", [True, False])
def test_strides(kind, packed, dtype):
    _run([(37, 70), (2, 90)], 4, 2, 32, dtype, packed=packed, place=_strided(kind), seed=1, mask=0.2)
    _run([(137, 170)], 2, 2, 64, dtype, packed=packed, place=_strided(kind), seed=2, relative=_buckets(8, 20, True))


def test_gradients_that_are_wanted():
    for need in (("query",), ("key",), ("value", "query"), ("table",), ("query", "table")):
        got = _run([(37, 70), (2, 90)], 4, 2, 32, BF16, need=need, seed=1, relative=_buckets(8, 20, True))
        assert len(got) == 1 + len(need)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_random_cases(dtype):
    rng = random.Random(7)
    for n in range(40):
        B = rng.choice([1, 1, 2, 5])
        top = rng.choice([3, 40, 150, 300])
        sizes = [(rng.randint(0, top), rng.randint(0, top)) for _ in range(B)]
        G = rng.choice([1, 2, 3])
        kw = dict(mask=rng.choice([0.0, 0.3]), packed=rng.random() < 0.5, tail=(rng.randint(0, 3), rng.randint(0, 3)), q_sizes=rng.random() < 0.5)
        if rng.random() < 0.6:
            both = rng.random() < 0.5
            kw.update(relative=_buckets(rng.choice([4, 9, 32]), rng.choice([20, 33, 140]), both), causal=not both and rng.random() < 0.7,
                      last=rng.random() < 0.5)
        _run(sizes, G * rng.choice([1, 2, 4]), G, rng.choice([8, 16, 20, 64, 72, 128]), dtype, seed=n, **kw)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_many_tiles(dtype):
    """More workgroups than processors, keys in parts, and both sides long."""
    _run([(700, 900), (1000, 300)], 4, 2, 64, dtype, seed=1, mask=0.1)
    _run([(1030, 1030)], 3, 3, 64, dtype, seed=2, relative=_buckets(32, 128, False), causal=True)
    _run([(1, 5000), (2, 3000)], 4, 1, 128, dtype, seed=3)
    _run([(3000, 3)], 2, 1, 32, dtype, seed=4)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("reach", [4, 200])
def test_buckets_that_take_keys_away(reach, dtype):
    """Minus infinity in the table takes a bucket's keys away, as a mask does, and so does the type's lowest value where a row has others;
    a row that has only such keys stays a mean of their values."""
    from crystalframer_amd import cuda_funcs
    gen = torch.Generator().manual_seed(0)
    for tq, tk in ((150, 170), (3, 300)):
        q, k, v, go = (torch.randn(1, n, 2, 32, generator=gen).to(dtype).cuda() for n in (tq, tk, tk, tq))
        of = torch.zeros(2 * reach + 1, dtype=torch.int32)
        of[:reach], of[reach + 1:] = 1, 2                # behind, here, ahead
        for low in (-float("inf"), torch.finfo(dtype).min):
            x = [t.clone().requires_grad_() for t in (q, k, v)]
            y = [t.clone().requires_grad_() for t in (q, k, v)]
            table = torch.tensor([[0.5, -0.5], [0.25, 1.0], [low, low]], dtype=dtype).cuda()
            a = cuda_funcs.relative_attention(*x, table, of.cuda())
            b = cuda_funcs.relative_attention(*y, torch.where(table == low, 0.0, table), of.cuda(), causal=True)      # (a row's own key is always there)
            assert torch.equal(a, b)
            for g, w in zip(torch.autograd.grad(a, x, go), torch.autograd.grad(b, y, go)):
                assert torch.equal(g, w)
            only = cuda_funcs.relative_attention(q, k, v, torch.full((3, 2), low, dtype=dtype).cuda(), of.cuda())
            if low == -float("inf"):
                assert (only == 0).all()
            else:
                assert (only <= v.amax(1, keepdim=True)).all() and (only >= v.amin(1, keepdim=True)).all() and only.isfinite().all()
