"""Attention between sequences of their own lengths, as programs use it that read an encoder's states.

    listed()             the cases
    draw(rng)            one more case of the same ranges
    prepare(case, seed)  inputs on the GPU, and the map of buckets that a program keeps
    run(state)           one pass: in plain torch operations, or (``own``) through the framework's entry points
    work(case)           bytes and flop that the pass cannot do without
    exact(case, seed)    what run() returns for these inputs, from the definition in 64 bits

Two kinds of case, forward, or forward and backward:

cross     ``cuda_funcs.cross_attention``: queries of one set of sequences read keys and values of another,
              o_i = sum_j P_ij v_j,    P_i. = softmax_j(q_i . k_j / sqrt(Dh))
          over the keys of the same index in the batch which the mask keeps.  Without any, the row is 0.
relative  ``cuda_funcs.relative_attention``: the same with a learned bias by the bucket of the relative position,
              P_i. = softmax_j(q_i . k_j / sqrt(Dh) + table[bucket(j - i - shift), head]),
          shift = keys - queries where the queries are the last positions, else 0; "causal": j <= i + shift only.

Buckets of r = j - i - shift: of n per direction the first e = n / 2 (rounded down) hold one distance each; distance d >= e is in
bucket min(n - 1, e + floor((n - e) log(d / e) / log(distance / e))).  "both": half of the buckets are for r > 0; otherwise r > 0 counts
as 0.  A layout is "packed" (sequences behind one another, their starts in a tensor) or "padded" ((batch, positions, heads, Dh), the
keys' lengths in a tensor if they differ).  Key and value heads may each serve several query heads.
"""
import math
import random

import torch

own = False

F32, F64 = torch.float32, torch.float64
DTYPE = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


def listed():
    cross = dict(kind="cross", layout="packed", batch=1, queries=1, keys=1, ragged="", heads=8, kv_heads=8, dim=16, dtype="float32",
                 mask=0.0, train=False, buckets=0, distance=0, both=False, causal=False, last=False)
    relative = dict(cross, kind="relative", buckets=32, distance=128, both=True)
    return [
        # four property queries read one crystal of 13 atoms with the heads of the default model: launches and host time alone
        dict(cross, name="cross_infer_13", queries=4, keys=13),
        # 16 queries to each of 256 crystals of 1 to 60 atoms, the default training batch, forward and backward
        dict(cross, name="cross_train_crystals", batch=256, queries=16, keys=60, ragged="keys", train=True),
        # a prompt's cross attention in serving: 8 sequences of 512 tokens, states of 1500 positions
        dict(cross, name="cross_infer_prompt", layout="padded", batch=8, queries=512, keys=1500, heads=16, kv_heads=16, dim=64,
             dtype="bfloat16"),
        # one token of each of 64 sequences reads states of 1 to 4096 positions, four heads to a key head
        dict(cross, name="cross_infer_token", layout="padded", batch=64, queries=1, keys=4096, ragged="keys", heads=32, kv_heads=8, dim=128,
             dtype="bfloat16"),
        # the largest training step of the range, a tenth of the states masked
        dict(cross, name="cross_train_wide", layout="padded", batch=4, queries=2048, keys=4096, heads=32, kv_heads=8, dim=128,
             dtype="bfloat16", mask=0.1, train=True),
        # odd lengths and heads of 80 channels, half of the states masked, sequences with no states at all
        dict(cross, name="cross_train_odd", batch=7, queries=389, keys=701, ragged="all", heads=6, kv_heads=3, dim=80, dtype="float16",
             mask=0.5, train=True),
        # a sequence of 37 tokens attends to itself: the smallest call with a bias
        dict(relative, name="relative_infer_37", queries=37, keys=37),
        # one token each of 16 sequences, caches of 1 to 8192 positions
        dict(relative, name="relative_infer_token", layout="padded", batch=16, queries=1, keys=8192, ragged="keys", heads=16, kv_heads=16,
             dim=64, dtype="bfloat16", both=False, causal=True, last=True),
        # an encoder's training batch: 32 sequences of 512 tokens
        dict(relative, name="relative_train_512", layout="padded", batch=32, queries=512, keys=512, heads=12, kv_heads=12, dim=64,
             dtype="bfloat16", train=True),
        # a decoder's training batch of long sequences
        dict(relative, name="relative_train_causal", layout="padded", batch=2, queries=4096, keys=4096, heads=16, kv_heads=16, dim=128,
             dtype="bfloat16", both=False, causal=True, train=True),
        # one long document through an encoder
        dict(relative, name="relative_infer_long", queries=12000, keys=12000, dim=64, dtype="float16"),
        # odd lengths, heads and buckets in float32, one key head for all
        dict(relative, name="relative_train_odd", batch=6, queries=1001, keys=1001, ragged="same", heads=5, kv_heads=1, dim=40, buckets=47,
             distance=77, train=True),
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, spread over the logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    case = dict(kind=rng.choice(["cross", "relative"]), layout=rng.choice(["packed", "padded"]))
    kv_heads = rng.choice([1, 2, 4, 8, 16, 3, 5, 12])
    case.update(heads=kv_heads * rng.choice([1, 1, 2, 4]), kv_heads=kv_heads, dim=rng.choice([16, 24, 32, 40, 64, 64, 80, 96, 128, 128]),
                dtype=rng.choice(["float32", "bfloat16", "bfloat16", "float16"]))
    form = rng.choice(["token", "same", "other", "other"])
    case["train"] = form != "token" and rng.random() < 0.6
    keys = _spread(rng, 16 if case["train"] else 1, 16384 if form == "token" else 8192)
    queries = rng.choice([1, 1, 1, 2, 4]) if form == "token" else keys if form == "same" else _spread(rng, 1, 4096)
    # a pair of a head costs its products; float32 costs about 8 times a 16-bit type's
    each = case["heads"] * case["dim"] * (7 if case["train"] else 2) * (8 if case["dtype"] == "float32" else 1)
    each, limit = max(each, case["heads"] << 9), 1 << 39      # (2^30 scores at the most)
    while each * queries * keys > limit:
        queries, keys = max(1, queries // 2), max(16, keys // 2)
    most = limit // (each * queries * keys) if form != "token" else max(1, (1 << 28) // (kv_heads * case["dim"] * keys))
    batch = _spread(rng, 1, min(most, 256))
    ragged = "" if batch == 1 else rng.choice(["", "keys"] if case["layout"] == "padded" else ["", "keys", "same" if form == "same" else "all"])
    case.update(batch=batch, queries=queries, keys=keys, ragged=ragged, mask=rng.choice([0.0, 0.0, 0.1, 0.7]))
    case.update(buckets=0, distance=0, both=False, causal=False, last=False)
    if case["kind"] == "relative":
        buckets = _spread(rng, 4, 128)
        case.update(buckets=buckets, distance=_spread(rng, buckets, 600), both=rng.random() < 0.5, last=form == "token" or rng.random() < 0.3)
        case["causal"] = not case["both"] and rng.random() < 0.7
    return case


# ------------------------------------------------------------------------------------------------ inputs
def _sizes(case):
    """Lengths of the sequences: (queries, keys)."""
    B, rng = case["batch"], random.Random(f"{case['batch']} {case['queries']} {case['keys']} {case['ragged']}")
    tq, tk = [case["queries"]] * B, [case["keys"]] * B
    if case["ragged"] in ("keys", "all"):
        tk = [rng.randint(1, case["keys"]) for _ in range(B)]
    if case["ragged"] == "all":
        tq = [rng.randint(1, case["queries"]) for _ in range(B)]
        tk[0] = 0
    if case["ragged"] == "same":
        tq = tk = [rng.randint(1, case["keys"]) for _ in range(B)]
    return tq, tk


def _starts(sizes):
    at = [0]
    for n in sizes:
        at.append(at[-1] + n)
    return at


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    dt, B, H, G, D = DTYPE[case["dtype"]], case["batch"], case["heads"], case["kv_heads"], case["dim"]
    normal = lambda *shape: torch.randn(*shape, generator=gen, device=dev)  # noqa: E731
    tq, tk = _sizes(case)
    packed = case["layout"] == "packed"
    rows_q, rows_k = ((sum(tq),), (sum(tk),)) if packed else ((B, case["queries"]), (B, case["keys"]))
    # keys have something in common, and channels differ in size; key and value come out of one projection
    channel = torch.exp(0.3 * normal(G, D))
    kv = normal(*rows_k, 2, G, D)
    kv[..., 0, :, :].add_(0.5 * normal(G, D)).mul_(channel)
    kv = kv.to(dt)
    s = dict(case=case, q=(normal(*rows_q, H, D) * 1.2).to(dt), k=kv[..., 0, :, :], v=kv[..., 1, :, :], table=None, buckets=None,
             query_starts=None, key_starts=None, key_sizes=None, mask=None, most_q=max(tq), most_k=max(max(tk), 1))
    long = lambda x: torch.tensor(x, dtype=torch.int64, device=dev)  # noqa: E731
    if packed:
        s["query_starts"], s["key_starts"] = long(_starts(tq)), long(_starts(tk))
    elif case["ragged"]:
        s["key_sizes"] = long(tk)
    if case["mask"]:
        s["mask"] = torch.rand(rows_k, generator=gen, device=dev) >= case["mask"]
    if case["kind"] == "relative":
        s["table"] = (normal(case["buckets"], H) * 0.7).to(dt)
        if own:
            from crystalframer_amd import cuda_funcs
            s["buckets"] = cuda_funcs.position_buckets(case["buckets"], case["distance"], bidirectional=case["both"], device=dev)
        else:
            s["borders"] = long(_borders(case))
    if case["train"]:
        s["go"] = (normal(*rows_q, H, D) * 0.5).to(dt)
        for k in _leaves(case):
            s[k] = s[k].detach().requires_grad_(True)
    return s


def _leaves(case):
    return ("q", "k", "v", "table") if case["kind"] == "relative" else ("q", "k", "v")


def _borders(case):
    """The first distance of each bucket of a direction but the first, in whole numbers: floor(x) >= t for a logarithm x is a
    comparison of powers."""
    n = case["buckets"] // 2 if case["both"] else case["buckets"]
    e, M = n // 2, case["distance"]
    first = list(range(1, e + 1))
    for t in range(1, n - e):
        d = first[-1]
        while d ** (n - e) * e ** t < M ** t * e ** (n - e):
            d += 1
        first.append(d)
    return first


# ------------------------------------------------------------------------------------------------ passes
def run(state):
    return _own(state) if own else _plain(state)


def _own(s):
    from crystalframer_amd import cuda_funcs
    case = s["case"]
    where = dict(query_starts=s["query_starts"], key_starts=s["key_starts"], key_sizes=s["key_sizes"], key_mask=s["mask"])
    if case["kind"] == "cross":
        call = lambda: cuda_funcs.cross_attention(s["q"], s["k"], s["v"], **where)  # noqa: E731
    else:
        call = lambda: cuda_funcs.relative_attention(s["q"], s["k"], s["v"], s["table"], s["buckets"], causal=case["causal"],  # noqa: E731
                                                     queries_last=case["last"], **where)
    if not case["train"]:
        with torch.no_grad():
            return dict(out=call())
    out = call()
    leaves = _leaves(case)
    grads = torch.autograd.grad(out, [s[k] for k in leaves], s["go"])
    return dict(out=out.detach(), **{"grad_" + k: g for k, g in zip(leaves, grads)})


def _padded(x, starts, most):
    """Packed rows as (batch, most, ...), and which of these are rows; the last row where there is none."""
    at = starts[:-1, None] + torch.arange(most, device=x.device)
    real = at < starts[1:, None]
    if x.shape[0] == 0:
        return x.new_zeros(at.shape + x.shape[1:]), real
    return x[torch.clamp_max(at, x.shape[0] - 1)], real


def _plain(s):
    case, dt = s["case"], s["q"].dtype
    q, k, v = (s[n].detach().to(F32) for n in ("q", "k", "v"))
    go = s["go"].float() if case["train"] else None
    rows, mask = None, s["mask"]
    if s["query_starts"] is not None:
        q, rows = _padded(q, s["query_starts"], s["most_q"])
        go = None if go is None else torch.where(rows[..., None, None], _padded(go, s["query_starts"], s["most_q"])[0], 0.0)
        (k, keep), (v, _) = (_padded(x, s["key_starts"], s["most_k"]) for x in (k, v))
        tq, tk = s["query_starts"].diff(), s["key_starts"].diff()
        mask = None if mask is None else _padded(mask, s["key_starts"], s["most_k"])[0]
    else:
        tq = torch.full((q.shape[0],), q.shape[1], device=q.device)
        tk = s["key_sizes"] if s["key_sizes"] is not None else torch.full_like(tq, k.shape[1])
        keep = torch.arange(k.shape[1], device=q.device) < tk[:, None]
    B, Tq, Tk, H, share = q.shape[0], q.shape[1], k.shape[1], case["heads"], case["heads"] // case["kv_heads"]
    keep = (keep if mask is None else keep & mask)[:, None, None, :]
    line = r = bucket = None
    if case["kind"] == "relative":
        # biases by relative position: row i of a matrix is a window of this line, the last row the first window
        shift = (tk - tq if case["last"] else torch.zeros_like(tk))[:, None]
        r = torch.arange(Tq + Tk - 1, device=q.device) - (Tq - 1) - shift
        far = r.abs() if case["both"] else torch.clamp_min(-r, 0)
        bucket = torch.bucketize(far, s["borders"], right=True)
        if case["both"]:
            bucket = bucket + (r > 0) * (case["buckets"] // 2)
        line = s["table"].detach().float()[bucket].transpose(1, 2)
    q, k, v = (x.transpose(1, 2) for x in (q.flip(1), k, v))
    go = None if go is None else go.flip(1).transpose(1, 2)
    o = torch.empty_like(q)
    grads = [torch.zeros_like(x) for x in (q, k, v)] if case["train"] else None
    lines = torch.zeros(B, H, Tq + Tk - 1, dtype=F64, device=q.device) if case["train"] and line is not None else None
    # as many sequences and heads at once as have 2^28 scores
    heads = max(1, min(H, _AT_ONCE // (Tq * Tk)))
    heads = heads // share * share if heads >= share else max(n for n in range(1, heads + 1) if share % n == 0)
    some = max(1, _AT_ONCE // (Tq * Tk * heads))
    for b in range(0, B, some):
        for h in range(0, H, heads):
            at = (slice(b, b + some), slice(h, h + heads))
            kv = (at[0], slice(h // share, max(h // share + 1, (h + heads) // share)))
            leaves = [x.clone().requires_grad_(case["train"]) for x in (q[at], k[kv], v[kv])]
            each = min(share, heads)
            wide = [x.repeat_interleave(each, 1) if each > 1 else x for x in leaves[1:]]
            S = torch.matmul(leaves[0] / math.sqrt(case["dim"]), wide[0].transpose(-1, -2))
            visible = keep[at[0]]
            if line is not None:
                S = S + line[at].unfold(-1, Tk, 1)
                if case["causal"]:
                    visible = visible & (r[at[0]] <= 0)[:, None].unfold(-1, Tk, 1)
            S = torch.where(visible, S, -math.inf)
            top = S.detach().amax(-1, keepdim=True)
            e = torch.exp(S - torch.where(top > -math.inf, top, 0.0))
            total = e.sum(-1, keepdim=True)
            part = torch.matmul(e / torch.where(total > 0, total, 1.0), wide[1])
            o[at] = part.detach()
            if case["train"]:
                got = torch.autograd.grad(part, leaves + ([S] if line is not None else []), go[at])
                for place, where, g in zip(grads, (at, kv, kv), got):
                    place[where] += g
                if line is not None:      # (no gradient reaches a score that is not visible)
                    lines[at] = _diagonals(torch.where(visible, got[3], 0.0))
    back = lambda x: x.transpose(1, 2).flip(1)  # noqa: E731
    out = dict(out=back(o) if rows is None else back(o)[rows])
    if case["train"]:
        out["grad_q"] = back(grads[0]) if rows is None else back(grads[0])[rows]
        for n, g in zip("kv", grads[1:]):
            g = g.transpose(1, 2)
            out["grad_" + n] = g if rows is None else g[torch.arange(Tk, device=q.device) < tk[:, None]]
        if line is not None:              # sums of many terms of either sign, in 64 bits
            out["grad_table"] = torch.zeros(s["table"].shape, dtype=F64, device=q.device).index_add_(
                0, bucket.reshape(-1), lines.transpose(1, 2).reshape(-1, H))
    return {n: x.to(dt) for n, x in out.items()}


_AT_ONCE = 1 << 28


def _diagonals(x):
    """Sums of (..., i, j) over the pairs of one i + j: rows behind one another, each a place further right."""
    m, n = x.shape[-2:]
    x = torch.nn.functional.pad(x, (0, m)).flatten(-2)[..., :m * (m + n - 1)]
    return x.unflatten(-1, (m, m + n - 1)).sum(-2, dtype=F64)


# ------------------------------------------------------------------------------------------------ what a pass needs
def _pairs(case):
    """Pairs of a query and a key that reach the softmax, over the batch."""
    n = 0
    for tq, tk in zip(*_sizes(case)):
        if not case["causal"]:
            n += tq * tk
            continue
        shift = tk - tq if case["last"] else 0
        lo, hi = max(0, -shift), max(0, min(tq, tk - shift))       # rows whose last key is inside
        n += (max(0, hi - lo) * (lo + shift + 1 + hi + shift)) // 2 + (tq - max(hi, lo)) * tk
    return n * (1 - case["mask"])


def work(case):
    tq, tk = _sizes(case)
    H, G, D, size = case["heads"], case["kv_heads"], case["dim"], DTYPE[case["dtype"]].itemsize
    ways = 2 if case["train"] else 1
    kept = (1 - case["mask"]) * sum(tk)
    rows = sum(tq) * H * D * size * (2 if not case["train"] else 4)               # q, o; go, dq
    keys = 2 * G * D * size * (kept + (sum(tk) if case["train"] else 0))          # k, v; dk, dv
    return {"bytes": int(rows + keys + (sum(tk) if case["mask"] else 0) + ways * case["buckets"] * H * size),
            "flops": int(_pairs(case) * H * D * (14 if case["train"] else 4))}


# ------------------------------------------------------------------------------------------------ the definition in 64 bits
def _exact_bucket(case, r):
    """Bucket of a relative position, from the formula: the logarithms' ratio is a whole number or clearly none in 200 bits."""
    n = case["buckets"] // 2 if case["both"] else case["buckets"]
    first = n if case["both"] and r > 0 else 0
    d = abs(r) if case["both"] else max(0, -r)
    e, M = n // 2, case["distance"]
    if d < e:
        return first + d
    t = 0
    while t + 1 < n - e and (d / e) ** (n - e) >= (M / e) ** (t + 1) * (1 - 1e-9) and d ** (n - e) * e ** (t + 1) >= M ** (t + 1) * e ** (n - e):
        t += 1
    return first + min(n - 1 - e, t) + e


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return _exact(s)


def _exact(s):
    case = s["case"]
    dev, share, root = s["q"].device, case["heads"] // case["kv_heads"], math.sqrt(case["dim"])
    tq, tk = _sizes(case)
    sq, sk = _starts(tq), _starts(tk)
    names = _leaves(case)
    x = {n: s[n].detach() for n in names}
    out = {"out": torch.zeros(x["q"].shape, dtype=F64, device=dev)}
    if case["train"]:
        out.update({"grad_" + n: torch.zeros(x[n].shape, dtype=F64, device=dev) for n in names})
    packed = s["query_starts"] is not None
    M = case["distance"]
    if case["kind"] == "relative":
        of = torch.tensor([_exact_bucket(case, r) for r in range(-M, M + 1)], device=dev)
    for b in range(case["batch"]):
        mine = (slice(sq[b], sq[b + 1]), slice(sk[b], sk[b + 1])) if packed else ((b, slice(0, tq[b])), (b, slice(0, tk[b])))
        if tk[b] == 0 or tq[b] == 0:
            continue
        keep = torch.ones(1, tk[b], dtype=torch.bool, device=dev) if s["mask"] is None else s["mask"][mine[1]][None]
        if case["kind"] == "relative":
            shift = tk[b] - tq[b] if case["last"] else 0
            r = torch.arange(tk[b], device=dev)[None] - torch.arange(tq[b], device=dev)[:, None] - shift
            bucket = of[r.clamp(-M, M) + M]
            if case["causal"]:
                keep = keep & (r <= 0)
        for g in range(case["kv_heads"]):
            k, v = x["k"][mine[1]][:, g].to(F64), x["v"][mine[1]][:, g].to(F64)
            for h in range(g * share, (g + 1) * share):
                q = x["q"][mine[0]][:, h].to(F64)
                score = q @ k.T / root
                if case["kind"] == "relative":
                    score = score + x["table"].to(F64)[:, h][bucket]
                score = score.masked_fill(~keep, -math.inf)
                P = torch.nan_to_num(torch.softmax(score, -1), nan=0.0) if s["mask"] is not None or case["causal"] else torch.softmax(score, -1)
                o = P @ v
                out["out"][mine[0]][:, h] = o
                if not case["train"]:
                    continue
                go = s["go"][mine[0]][:, h].to(F64)
                dS = P * (go @ v.T - (go * o).sum(-1, keepdim=True))
                out["grad_q"][mine[0]][:, h] = dS @ k / root
                out["grad_k"][mine[1]][:, g] += dS.T @ q / root
                out["grad_v"][mine[1]][:, g] += P.T @ go
                if case["kind"] == "relative":
                    out["grad_table"][:, h] += torch.bincount(bucket.view(-1), dS.reshape(-1), case["buckets"])
    return out
