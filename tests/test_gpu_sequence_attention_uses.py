"""Attention between sequences as programs use it: refusals, autograd, graphs, streams, threads, caches, long tensors, and a decoder
over an encoder's states."""
import math
import threading

import pytest
import torch
from torch.utils.checkpoint import checkpoint

import attention_reference as AR

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _leaves(dtype=F32, B=2, Tq=40, Tk=70, H=4, G=2, D=32, seed=0, table=True):
    gen = torch.Generator().manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    t = dict(query=rnd(B, Tq, H, D), key=rnd(B, Tk, G, D), value=rnd(B, Tk, G, D))
    if table:
        t["table"] = rnd(8, H)
    return {k: v.to(dtype).cuda().requires_grad_() for k, v in t.items()}


def _of():
    from crystalframer_amd import cuda_funcs
    return cuda_funcs.position_buckets(8, 20, device="cuda")


def _call(leaves, **kw):
    from crystalframer_amd import cuda_funcs
    if "table" in leaves:
        of = kw.pop("of") if "of" in kw else _of()
        return cuda_funcs.relative_attention(leaves["query"], leaves["key"], leaves["value"], leaves["table"], of, **kw)
    return cuda_funcs.cross_attention(leaves["query"], leaves["key"], leaves["value"], **kw)


def _grads(out, leaves, seed=5):
    go = torch.randn(out.shape, generator=torch.Generator().manual_seed(seed)).to(out.dtype).cuda()
    return torch.autograd.grad(out, list(leaves.values()), go)


def _equal(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b))


# ------------------------------------------------------------------------------------------------ refusals
def test_refusals():
    from crystalframer_amd import cuda_funcs
    q, k, t = torch.zeros(2, 5, 4, 16, device="cuda"), torch.zeros(2, 7, 2, 16, device="cuda"), torch.zeros(8, 4, device="cuda")
    of = _of()
    n = torch.tensor([5, 3], device="cuda")
    starts = torch.tensor([0, 2, 5], device="cuda")
    cross, rel = cuda_funcs.cross_attention, cuda_funcs.relative_attention
    p, s = q[0], k[0]
    for call, error, word in (
            (lambda: cross(q.double(), k.double(), k.double()), TypeError, "float32"), (lambda: cross(q.half(), k, k), TypeError, "one type"),
            (lambda: cross(q, k, k.half()), TypeError, "one type"), (lambda: cross(q[0, 0], k, k), ValueError, "shape"), (lambda: cross(q, k, k[:, :6]), ValueError, "shape"),
            (lambda: cross(q, k[..., :8], k[..., :8]), ValueError, "channels"), (lambda: cross(q[:, :, :3], k, k), ValueError, "heads"),
            (lambda: cross(q[:, :, :0], k, k), ValueError, "heads"), (lambda: cross(q[..., :0], k[..., :0], k[..., :0]), ValueError, "channels"),
            (lambda: cross(torch.zeros(1, 1, 1, 129, device="cuda"), *[torch.zeros(1, 1, 1, 129, device="cuda")] * 2), ValueError, "channels"),
            (lambda: cross(q[:1], k, k), ValueError, "batches"), (lambda: cross(p, s, s), ValueError, "query_starts"),
            (lambda: cross(p, s, s, query_starts=starts), ValueError, "query_starts"), (lambda: cross(q, k, k, query_starts=starts, key_starts=starts), ValueError, "packed"),
            (lambda: cross(p, s, s, query_starts=starts, key_starts=starts[:2]), ValueError, "begins"),
            (lambda: cross(p, s, s, query_starts=starts[:0], key_starts=starts[:0]), ValueError, "begins"),
            (lambda: cross(p, s, s, query_starts=starts.int(), key_starts=starts.int()), TypeError, "int64"),
            (lambda: cross(p, s, s, query_starts=starts, key_starts=starts, key_sizes=n), ValueError, "sizes"),
            (lambda: cross(q, k, k, key_sizes=n[:1]), ValueError, "key_sizes"), (lambda: cross(q, k, k, key_sizes=n.float()), TypeError, "int64"),
            (lambda: cross(q, k, k, key_mask=torch.ones(2, 7, device="cuda")), TypeError, "bool"),
            (lambda: cross(q, k, k, key_mask=torch.ones(7, dtype=torch.bool, device="cuda")), ValueError, "key_mask"),
            (lambda: cross(q, k, k, scale=math.inf), ValueError, "scale"), (lambda: cross(q, k, k, key_sizes=n.cpu()), RuntimeError, "HIP device"),
            (lambda: rel(q, k, k, t.double(), of), TypeError, "table"), (lambda: rel(q, k, k, t[:, :3], of), ValueError, "table"),
            (lambda: rel(q, k, k, t[:0], of), ValueError, "table"), (lambda: rel(q, k, k, t, of.long()), TypeError, "int32"),
            (lambda: rel(q, k, k, t, of[:-1]), ValueError, "buckets"), (lambda: rel(q, k, k, t, of[None]), ValueError, "buckets"),
            (lambda: rel(q, k, k, t, torch.zeros(2051, dtype=torch.int32, device="cuda")), ValueError, "buckets")):
        with pytest.raises(error, match=word):
            call()
    with torch.autograd.forward_ad.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
        cross(q, k, k)
    with pytest.raises(RuntimeError, match="traced or transformed"):
        torch.func.vmap(lambda a: cross(a, k, k))(q[None])


def test_starts_and_sizes_are_cut_to_the_rows_that_are_there():
    """Values that point elsewhere read and write nothing outside; sequences that they leave are right."""
    from crystalframer_amd import cuda_funcs
    x = torch.randn(10, 2, 16, device="cuda")
    wild = torch.tensor([0, 4, 1 << 40], device="cuda")
    a = cuda_funcs.cross_attention(x, x, x, query_starts=wild, key_starts=wild)
    b = cuda_funcs.cross_attention(x, x, x, query_starts=torch.tensor([0, 4, 10], device="cuda"), key_starts=torch.tensor([0, 4, 10], device="cuda"))
    assert torch.equal(a, b)
    for starts in ([0, -5, 7], [0, 9, 3], [0, 1 << 62, -(1 << 62)]):
        s = torch.tensor(starts, device="cuda")
        y = x.clone().requires_grad_()
        cuda_funcs.cross_attention(y, y, y, query_starts=s, key_starts=s).sum().backward()
    p = torch.randn(2, 10, 2, 16, device="cuda")
    for sizes in ([-3, 11], [1 << 40, 10]):
        a = cuda_funcs.cross_attention(p, p, p, key_sizes=torch.tensor(sizes, device="cuda"))
        b = cuda_funcs.cross_attention(p, p, p, key_sizes=torch.tensor([max(0, min(10, n)) for n in sizes], device="cuda"))
        assert torch.equal(a, b)
    torch.cuda.synchronize()


# ------------------------------------------------------------------------------------------------ autograd
@pytest.mark.parametrize("table", [False, True])
def test_gradients_against_differences(table):
    """Central differences along a direction, at two steps: what the smaller one leaves is a third of what they differ by, and 2^-20
    (a score's sums, powers and sums of P, each some units of 2^-24) of the sum's terms over the step."""
    leaves = _leaves(table=table)
    gen = torch.Generator().manual_seed(1)
    go = torch.randn(2, 40, 4, 32, generator=gen).cuda()
    out = _call(leaves, scale=0.2)
    grads = torch.autograd.grad(out, list(leaves.values()), go)
    for name, g in zip(leaves, grads):
        d = torch.randn(leaves[name].shape, generator=gen).cuda()

        def value(h):
            with torch.no_grad():
                y = _call({**leaves, name: leaves[name] + h * d}, scale=0.2)
            return float((y.double() * go.double()).sum())
        h = 2.0 ** -7
        big, small = ((value(s) - value(-s)) / (2 * s) for s in (h, h / 2))
        want = float((g.double() * d.double()).sum())
        noise = 2.0 ** -20 * float((out.detach().double() * go.double()).square().sum().sqrt()) * 4 / (h / 2)
        assert abs(small - want) <= abs(big - small) + noise, (name, small, big, want, noise)


def test_gradients_of_gradients_and_second_passes_are_refused():
    leaves = _leaves()
    out = _call(leaves)
    g, = torch.autograd.grad(out.square().sum(), [leaves["query"]], create_graph=True)
    with pytest.raises(RuntimeError, match="not differentiable"):
        g.sum().backward()
    out = _call(leaves)
    first = torch.autograd.grad(out.sum(), list(leaves.values()), retain_graph=True)
    assert _equal(first, torch.autograd.grad(out.sum(), list(leaves.values())))
    with pytest.raises(RuntimeError, match="second time"):
        out.sum().backward()


@pytest.mark.parametrize("dtype", [F32, F16])
def test_kept_on_the_host_and_made_again(dtype):
    leaves = _leaves(dtype)
    want = _grads(_call(leaves), leaves)
    with torch.autograd.graph.save_on_cpu():
        out = _call(leaves)
    assert _equal(_grads(out, leaves), want)
    out = checkpoint(lambda *a: _call(dict(zip(leaves, a))), *leaves.values(), use_reentrant=False)
    assert _equal(_grads(out, leaves), want)
    with torch.autograd.set_detect_anomaly(True):
        assert _equal(_grads(_call(leaves), leaves), want)


@pytest.mark.parametrize("what", ["query", "key", "table", "out", "mask", "sizes"])
def test_what_is_kept_must_not_change(what):
    leaves = _leaves()
    mask, sizes = torch.ones(2, 70, dtype=torch.bool, device="cuda"), torch.tensor([70, 50], device="cuda")
    out = _call(leaves, key_mask=mask, key_sizes=sizes)
    with torch.no_grad():
        if what == "out":
            out.mul_(2.0)
        elif what in leaves:
            leaves[what].mul_(2.0)
        elif what == "mask":
            mask[0, 0] = False
        else:
            sizes.sub_(1)
    with pytest.raises(RuntimeError, match="inplace|in-place|in place"):
        _grads(out, leaves)


def test_one_leaf_in_several_places_and_gradients_of_odd_layouts():
    from crystalframer_amd import cuda_funcs
    x = torch.randn(2, 33, 3, 16, device="cuda", requires_grad=True)
    a, b, c = (x.detach().clone().requires_grad_() for _ in range(3))
    cuda_funcs.cross_attention(x, x, x).sum().backward()          # (an expanded gradient)
    cuda_funcs.cross_attention(a, b, c).sum().backward()
    assert (x.grad - (a.grad + b.grad + c.grad)).abs().max() <= 2 * 2.0 ** -24 * (a.grad.abs() + b.grad.abs() + c.grad.abs()).max()
    go = torch.randn(2, 33, 16, 3, device="cuda").transpose(-1, -2)
    one = torch.autograd.grad(cuda_funcs.cross_attention(a, b, c), [a, b, c], go)
    assert _equal(one, torch.autograd.grad(cuda_funcs.cross_attention(a, b, c), [a, b, c], go.contiguous()))


# ------------------------------------------------------------------------------------------------ graphs, streams, threads
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_equal_runs_give_equal_bits_and_graphs_replay_them(dtype):
    """Forward and backward captured, keys in parts among it, two graphs in turn with eager work between the replays."""
    shapes = [dict(B=3, Tq=130, Tk=200), dict(B=1, Tq=2, Tk=3000, G=1), dict(B=1, Tq=3000, Tk=5, G=1)]
    for shape in shapes:
        sets = []
        for seed in (0, 1):
            leaves = _leaves(dtype, seed=seed, **shape)
            go = torch.randn(leaves["query"].shape, generator=torch.Generator().manual_seed(9)).to(dtype).cuda()
            of = _of()
            run = lambda l=leaves, g=go, of=of: (lambda o: (o.detach(), *torch.autograd.grad(o, list(l.values()), g)))(_call(l, of=of))  # noqa: E731
            want = run()
            assert _equal(want, run())
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                run()
            torch.cuda.current_stream().wait_stream(side)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                got = run()
            sets.append((graph, got, want, run, leaves))
        for k in range(4):
            for graph, got, want, run, leaves in sets:
                with torch.no_grad():
                    leaves["query"].add_(1.0).sub_(1.0).copy_(leaves["query"])
                    for g in got:
                        g.fill_(float("nan"))
                graph.replay()
                torch.cuda.synchronize()
                fresh = run()
                torch.cuda.synchronize()
                assert _equal(got, fresh), k


def test_capture_beside_an_eager_graph_of_the_same_leaves_is_refused():
    leaves = _leaves()
    of = _of()
    kept = _call(leaves, of=of)
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="let go"):
        with torch.cuda.graph(graph):
            _call(leaves, of=of).sum().backward()
    graph, y = torch.cuda.CUDAGraph(), []
    with torch.cuda.graph(graph):
        y.append(_call(leaves, of=of).detach())
    graph.replay()
    assert torch.equal(y[0], kept.detach())
    del kept


def test_streams():
    from crystalframer_amd import cuda_funcs
    leaves = _leaves(BF16, B=4, Tq=300, Tk=500)
    want = _grads(_call(leaves), leaves)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        x = [torch.zeros_like(v) for v in leaves.values()]
        torch.cuda._sleep(10_000_000)
        for a, b in zip(x, leaves.values()):      # (only behind the wait are the inputs there)
            a.copy_(b.detach())
        made = dict(zip(leaves, (a.requires_grad_() for a in x)))
        out = _call(made)
        got = _grads(out, made)
    side.synchronize()
    assert _equal(got, want) and cuda_funcs is not None


def test_threads():
    sets = [_leaves(BF16, seed=s, Tq=100, Tk=150) for s in range(4)]
    want = [_grads(_call(s), s) for s in sets]
    got = [None] * 4

    def work(n):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(10):
                got[n] = _grads(_call(sets[n]), sets[n])
            torch.cuda.current_stream().synchronize()
    torch.cuda.synchronize()
    threads = [threading.Thread(target=work, args=(n,)) for n in range(4)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert all(_equal(g, w) for g, w in zip(got, want))


# ------------------------------------------------------------------------------------------------ long and many
def test_offsets_beyond_32_bits():
    """A cache of more than 2^32 bytes and 2^31 elements in each of key and value: the last positions of the last sequence count."""
    from crystalframer_amd import cuda_funcs
    T, G, D = 140000, 64, 128
    k = torch.empty(2, T, G, D, dtype=BF16, device="cuda")
    v = torch.empty(2, T, G, D, dtype=BF16, device="cuda")
    for x in (k, v):
        for b in range(2):
            for h in range(0, G, 8):
                x[b, :, h:h + 8] = torch.randn(T, 8, D, device="cuda").to(BF16)
    q = torch.randn(2, 1, G, D, device="cuda").to(BF16)
    sizes = torch.tensor([T - 3, T], device="cuda")
    out = cuda_funcs.cross_attention(q, k, v, key_sizes=sizes)
    starts = torch.tensor([0, T - 3, 2 * T - 3], device="cuda")
    packed = cuda_funcs.cross_attention(q.view(2, G, D), k.view(2 * T, G, D)[:2 * T - 3], v.view(2 * T, G, D)[:2 * T - 3],
                                        query_starts=torch.tensor([0, 1, 2], device="cuda"), key_starts=starts)
    for b, h in ((0, 0), (1, 0), (1, 63)):
        n = int(sizes[b])
        res, tol = AR.attention(q[b, :, h:h + 1].cpu(), k[b, :n, h:h + 1].cpu(), v[b, :n, h:h + 1].cpu(), torch.ones(1, n, dtype=torch.bool))
        assert ((out[b, :, h:h + 1].cpu().double() - res["out"]).abs() <= tol["out"]).all(), (b, h)
        if b == 0:
            assert ((packed[b, h].cpu().double() - res["out"][0, 0]).abs() <= tol["out"][0, 0]).all()


def test_many_sequences():
    from crystalframer_amd import cuda_funcs
    gen = torch.Generator().manual_seed(3)
    sizes = torch.randint(0, 4, (9000,), generator=gen)
    starts = torch.nn.functional.pad(sizes.cumsum(0), (1, 0))
    N = int(starts[-1])
    x = [torch.randn(N, 2, 16, generator=gen).requires_grad_() for _ in range(3)]
    d = [t.detach().cuda().requires_grad_() for t in x]
    out = cuda_funcs.cross_attention(*d, query_starts=starts.cuda(), key_starts=starts.cuda())
    got = (out, *_grads(out, dict(enumerate(d))))
    of = torch.repeat_interleave(torch.arange(9000), sizes)
    go = torch.randn(out.shape, generator=torch.Generator().manual_seed(5)).double()
    w = [t.detach().double() for t in x]
    at = torch.arange(N)
    near = [at + s for s in range(-3, 4)]      # a sequence has up to three positions
    same = torch.stack([(n >= 0) & (n < N) & (of[n.clamp(0, N - 1)] == of) for n in near], 1)
    near = torch.stack([n.clamp(0, N - 1) for n in near], 1)
    r = [t.requires_grad_() for t in w]
    s = (r[0][:, None] * r[1][near]).sum(-1) / 4.0
    P = torch.softmax(s.masked_fill(~same[..., None], -math.inf), 1)
    ref = (P[..., None] * r[2][near]).sum(1)
    want = (ref, *torch.autograd.grad(ref, r, go))
    for a, b in zip(got, want):      # three keys, sixteen channels: some dozens of roundings of values of a few units each
        assert (a.detach().cpu().double() - b.detach()).abs().max() <= 64 * 2.0 ** -24 * 8 * float(b.detach().abs().max().clamp_min(1.0))


# ------------------------------------------------------------------------------------------------ together
class _Decoder(torch.nn.Module):
    """A layer over an encoder's states: causal attention with a bias by relative position, cross attention, norms between them."""

    def __init__(self, width, heads, buckets):
        super().__init__()
        self.H = heads
        self.qkv, self.o1 = torch.nn.Linear(width, 3 * width), torch.nn.Linear(width, width)
        self.q, self.kv, self.o2 = torch.nn.Linear(width, width), torch.nn.Linear(width, 2 * width), torch.nn.Linear(width, width)
        self.n1, self.n2 = (torch.nn.Parameter(torch.ones(width)) for _ in range(2))
        self.table = torch.nn.Parameter(0.3 * torch.randn(buckets, heads))

    def forward(self, x, states, starts, state_starts, relative, cross, norm):
        split = lambda t, n: t.unflatten(-1, (n, self.H, -1)).unbind(-3)  # noqa: E731
        q, k, v = split(self.qkv(x), 3)
        h, y = norm(x, self.o1(relative(q, k, v, self.table, starts).flatten(-2)), self.n1)
        k, v = split(self.kv(states), 2)
        h, y = norm(h, self.o2(cross(self.q(y).unflatten(-1, (self.H, -1)), k, v, starts, state_starts).flatten(-2)), self.n2)
        return y


def test_a_decoder_over_the_encoders_states():
    """Tokens of a batch of crystals read the atoms' states of the model's own encoder; outputs and gradients of all parameters against
    the same layer in float64 on the CPU, with a step of the optimizer behind it."""
    from crystalframer_amd import cuda_funcs, latticeformer, optim, params, synthetic
    torch.manual_seed(0)
    model = latticeformer.Latticeformer(params.ModelParams(num_layers=1)).cuda()
    batch = synthetic.make_batch(5, atoms="uniform", atoms_lo=1, atoms_hi=9, len_lo=3.0, len_hi=8.0, ang_lo=70.0, ang_hi=110.0, seed=3)
    data = batch.to("cuda")
    with torch.no_grad():
        states = model.encoder(model.input_embeddings(data.x), data.pos, data.batch, data.trans_vec, data.sizes)
    state_starts = torch.nn.functional.pad(data.sizes.cumsum(0), (1, 0))
    lengths = torch.tensor([3, 1, 40, 7, 12])
    starts = torch.nn.functional.pad(lengths.cumsum(0), (1, 0)).cuda()
    layer = _Decoder(128, 8, 12)
    x = torch.randn(int(lengths.sum()), 128)
    of = cuda_funcs.position_buckets(12, 25, False, device="cuda")
    exact = _Decoder(128, 8, 12).double()
    exact.load_state_dict({k: v.double() for k, v in layer.state_dict().items()})
    layer = layer.cuda()
    opt = optim.AdamW(layer.parameters(), lr=1e-3)
    out = layer(x.cuda(), states, starts, state_starts,
                lambda q, k, v, t, s: cuda_funcs.relative_attention(q, k, v, t, of, causal=True, query_starts=s, key_starts=s),
                lambda q, k, v, s, z: cuda_funcs.cross_attention(q, k, v, query_starts=s, key_starts=z),
                lambda h, b, w: cuda_funcs.residual_norm(h, b, w, norm="rms"))
    go = torch.randn(out.shape, generator=torch.Generator().manual_seed(2))
    out.backward(go.cuda())

    def plain(q, k, v, visible, bias=None):
        o = torch.zeros_like(q)
        t = torch.einsum("ihd,jhd->hij", q, k) / 4.0
        t = t if bias is None else t + bias
        P = torch.softmax(t.masked_fill(~visible, -math.inf), -1)
        return o + torch.einsum("hij,jhd->ihd", P, v)

    token = torch.repeat_interleave(torch.arange(5), lengths)
    place = torch.arange(len(token)) - starts.cpu()[token]
    r = place[None] - place[:, None]
    same = token[None] == token[:, None]
    bucket = of.cpu().long()[torch.clamp(r, -25, 25) + 25]
    atoms = torch.repeat_interleave(torch.arange(5), batch.sizes.cpu())
    ref = exact(x.double(), states.detach().cpu().double(), None, None,
                lambda q, k, v, t, s: plain(q, k, v, same & (r <= 0), t[bucket].permute(2, 0, 1)),
                lambda q, k, v, s, z: plain(q, k, v, token[:, None] == atoms[None]),
                lambda h, b, w: (h + b, (h + b) / ((h + b).square().mean(-1, keepdim=True) + 1e-5).sqrt() * w))
    ref.backward(go.double())
    # float32 through products of 128 terms, two attentions and two norms: errors of some hundred units of the largest magnitudes
    assert (out.detach().cpu().double() - ref.detach()).abs().max() <= 2.0 ** -24 * 512 * float(ref.detach().abs().max())
    for (name, a), b in zip(layer.named_parameters(), exact.parameters()):
        assert (a.grad.cpu().double() - b.grad).abs().max() <= 2.0 ** -24 * 2048 * float(b.grad.abs().max().clamp_min(1e-2)), name
    before = layer.table.detach().clone()
    opt.step()
    assert not torch.equal(before, layer.table)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("G", [4, 1])
def test_tokens_one_by_one_and_all_at_once(dtype, G):
    """A cache filled step by step, and in pieces, against the causal pass over the whole sequence: the same products, so that they
    differ by their bounds against float64 at the most."""
    from crystalframer_amd import cuda_funcs
    B, T, H, D = 3, 70, 4, 32
    leaves = {k: v.detach() for k, v in _leaves(dtype, B=B, Tq=T, Tk=T, H=H, G=G, D=D).items()}
    q, k, v, table = leaves.values()
    of = cuda_funcs.position_buckets(8, 20, False, device="cuda")
    whole = cuda_funcs.relative_attention(q, k, v, table, of, causal=True)
    bucket, _, r = AR.relative(T, T, False, of.cpu(), 20)
    bias = table.cpu().double()[bucket].permute(2, 0, 1)
    bounds = [AR.attention(q[b].cpu(), k[b].cpu(), v[b].cpu(), r <= 0, bias=bias) for b in range(B)]
    exact, tol = (torch.stack([x[n]["out"] for x in bounds]) for n in (0, 1))
    assert ((whole.cpu().double() - exact).abs() <= tol).all()
    ck, cv = (torch.full((B, 90, G, D), float("nan"), dtype=dtype, device="cuda") for _ in range(2))
    sizes = torch.zeros(B, dtype=torch.int64, device="cuda")
    at = 0
    for n in [1] * 20 + [13, 1, 30, 6]:
        ck[:, at:at + n], cv[:, at:at + n] = k[:, at:at + n], v[:, at:at + n]
        sizes += n
        y = cuda_funcs.relative_attention(q[:, at:at + n], ck, cv, table, of, causal=True, queries_last=True, key_sizes=sizes)
        assert ((y.cpu().double() - exact[:, at:at + n]).abs() <= tol[:, at:at + n]).all(), at
        at += n
