"""Attention between sequences in float64 on the CPU, with its gradients, and how far float32 arithmetic with roundings to a type may
be from it.

Bounds.  u: half a unit of the type, e: 2^-24.  With A_i the largest of scale sum_d |q_d k_d| + |bias| over a row, a score has an error of
up to (D + 24) e A_i (its products' sum, scale, bias, maximum and the change of base), and a probability relative to its sum one of
twice that and of the sum's own additions: E_i = e (2 (D + 24) A_i + keys + 64).
    o:      u |o| + (u + E_i) sum_j P |v|                                       (P rounded to the type before its product)
    D_i:    sum_d |do| (error of o, where u |o| is u^2 |o| in 16 bits: the output is kept in two parts) + e (D + 8) sum_d |do o|  =: Z_i
    ds:     P (2 E_i (W + |D|) + Z_i), W_ij = sum_d |do v|                      (W's own sum in it: D + 8 < what E_i holds, W e each)
    dq:     u |dq| + scale sum_j (error of ds + (u + e keys) |ds|) |k|          (ds rounded to the type before its product)
    dk:     u |dk| + scale sum_i (error of ds + (u + e rows) |ds|) |q|
    dv:     u |dv| + sum_i (u + E_i + e rows) P |do|
    dtable: u |dtable| + sum over the bucket of (error of ds + e (rows + keys) |ds|), and, for what lies beyond the reach, the row's own
            sum of ds (0, but for the errors of its terms) times its P: bounded by the errors of all ds of the row times that P
float16 loses in those roundings what is below half of its smallest step, 2^-25, behind the powers of two that terms are multiplied by:
2^-31 of a row's largest probability (o: 2^-31 sum_j |v|), 2^-40 of a probability (dv: 2^-40 sum_i |do|), 2^-39 of the largest ds of the
column (dq: of the row) that they are summed for.
For float32 the roundings to the type before a product are none.  16-bit results may be denormal: half the smallest step is added."""
import math

import torch

HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -150, torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}


def attention(q, k, v, keep, bias=None, scale=None, go=None, bucket=None, buckets=0, reach_index=None):
    """One sequence: q (Tq, H, D), k, v (Tk, G, D) of their type, keep (Tq, Tk) bool, bias (H, Tq, Tk) float64 or None, go as q.
    bucket (Tq, Tk): of the pairs; far (Tq, Tk) = reach_index: -1, 0, 1 (beyond the reach on a side).  Returns (results, bounds)."""
    u, dtype = HALF[q.dtype], q.dtype
    before = 0.0 if dtype == torch.float32 else u
    narrow = 1.0 if dtype == torch.float16 else 0.0
    e = 2.0 ** -24
    q, k, v = q.double(), k.double(), v.double()
    go = None if go is None else go.double()
    Tq, H, D = q.shape
    Tk, G = k.shape[:2]
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    names = ["out"] + ([] if go is None else ["dq", "dk", "dv"]) + ([] if go is None or bucket is None else ["dtable"])
    shape = dict(out=q.shape, dq=q.shape, dk=k.shape, dv=k.shape, dtable=(buckets, H))
    res = {n: torch.zeros(shape[n], dtype=torch.float64) for n in names}
    tol = {n: torch.zeros(shape[n], dtype=torch.float64) for n in names}
    any_key = keep.any(0)      # what is in the place of a key that is not there does not matter
    k = torch.where(any_key[:, None, None], k, 0.0)
    v = torch.where(any_key[:, None, None], v, 0.0)
    for h in range(H):
        g = h // (H // G)
        qh, kh, vh = q[:, h], k[:, g], v[:, g]
        t = scale * qh @ kh.T
        size = scale * qh.abs() @ kh.abs().T
        if bias is not None:
            t, size = t + bias[h], size + bias[h].abs()
        t = t.masked_fill(~keep, -math.inf)
        A = size.masked_fill(~keep, 0.0).amax(1, keepdim=True) if Tk else torch.zeros(Tq, 1, dtype=torch.float64)
        E = e * (2 * (D + 24) * A + Tk + 64)
        if Tk:
            top = t.amax(1, keepdim=True)
            p = torch.exp(t - torch.where(top > -math.inf, top, 0.0))
            s = p.sum(1, keepdim=True)
            P = p / torch.where(s > 0, s, 1.0)
        else:
            P = torch.zeros(Tq, 0, dtype=torch.float64)
        o = P @ vh
        err_o = u * o.abs() + (before + E) * (P @ vh.abs()) + narrow * 2.0 ** -31 * vh.abs().sum(0)
        res["out"][:, h], tol["out"][:, h] = o, err_o + TINY[dtype]
        if go is None:
            continue
        gh = go[:, h]
        dp, W = gh @ vh.T, gh.abs() @ vh.abs().T
        Di = (gh * o).sum(1, keepdim=True)
        Z = (gh.abs() * (err_o + ((u * u - u) * o.abs() + TINY[dtype] if dtype != torch.float32 else 0.0))).sum(1, keepdim=True) + e * (D + 8) * (gh * o).abs().sum(1, keepdim=True)
        ds = P * (dp - Di)
        err = P * (2 * E * (W + Di.abs()) + Z)
        lost = [narrow * 2.0 ** -39 * (ds.abs().amax(n, keepdim=True) if ds.numel() else 0.0) * torch.ones_like(ds) for n in (1, 0)]
        res["dq"][:, h] = scale * ds @ kh
        tol["dq"][:, h] = u * res["dq"][:, h].abs() + scale * (err + (before + e * Tk) * ds.abs() + lost[0]) @ kh.abs() + TINY[dtype]
        res["dk"][:, g] += scale * ds.T @ qh
        tol["dk"][:, g] += scale * (err + (before + e * (H // G) * Tq) * ds.abs() + lost[1]).T @ qh.abs()
        res["dv"][:, g] += P.T @ gh
        tol["dv"][:, g] += ((before + E + e * (H // G) * Tq) * P + narrow * 2.0 ** -40).T @ gh.abs()
        if bucket is not None:
            flat = bucket.reshape(-1)
            at = torch.clamp(flat, 0, buckets - 1)
            real = ((flat >= 0) & (flat < buckets)).double()
            res["dtable"][:, h].index_add_(0, at, ds.reshape(-1) * real)
            more = err + e * (Tq + Tk) * ds.abs()
            more = more + (reach_index != 0) * P * more.sum(1, keepdim=True)
            tol["dtable"][:, h].index_add_(0, at, more.reshape(-1) * real)
    if go is not None:
        for n in ("dk", "dv"):
            tol[n] += u * res[n].abs() + TINY[dtype]
    return res, tol


def relative(Tq, Tk, last, buckets, reach):
    """Relative positions' buckets (Tq, Tk), on which side they are beyond the reach, and j - i - shift."""
    r = torch.arange(Tk)[None] - torch.arange(Tq)[:, None] - (Tk - Tq if last else 0)
    side = (r >= reach).int() - (r <= -reach).int()
    return buckets[torch.clamp(r, -reach, reach) + reach].long(), side, r
