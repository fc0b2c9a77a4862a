"""Plain implementations in float64, on the CPU: the joined residual norm with its gradients, and one AdamW step with
moments in 32 or 8 bits (the formats as include/crystalframer_hip.h defines them)."""
import math

import numpy as np
import torch

HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}      # of one rounding, relative
TINY = {torch.float32: 2.0 ** -150, torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}   # half the smallest denormal


# ------------------------------------------------------------------------------------------------ residual norm
def norm_forward(v, kind, w, b, eps):
    """(y, normed rows, one over the deviation)."""
    if kind is None:
        return None, None, None
    c = v - v.mean(-1, keepdim=True) if kind == "layer" else v
    r = 1.0 / torch.sqrt((c * c).mean(-1, keepdim=True) + eps)
    y = c * r
    return (y if w is None else y * w) + (0.0 if b is None else b), y, r


def residual_norm(x, block=None, weight=None, bias=None, norm="layer", eps=1e-5, gate=None, residual_scale=1.0, block_scale=1.0,
                  block_norm=None, block_weight=None, block_bias=None, block_eps=1e-5):
    """h, y for float64 tensors (differentiable), and the largest magnitudes that roundings are relative to."""
    h = residual_scale * x
    if block is not None:
        a, _, ra = norm_forward(block, block_norm, block_weight, block_bias, block_eps) if block_norm else (block, None, None)
        h = h + block_scale * (a if gate is None else gate * a)
    y, _, r = norm_forward(h, norm, weight, bias, eps)
    return h, y


def tolerance(ref, dtype, size, roundings=64):
    """Half a unit of the result's type, and so many float32 roundings of terms of magnitude ``size``."""
    return HALF[dtype] * ref.abs() + TINY[dtype] + roundings * 2.0 ** -24 * size


# ------------------------------------------------------------------------------------------------ AdamW
M_VALUES = np.array([(c % 8 + 8 * (c >= 8)) * 2.0 ** (max(c // 8, 1) - 10) for c in range(127)])       # e4m3 without its sign
V_VALUES = np.array([(c % 8 + 8 * (c >= 8)) * 2.0 ** (max(c // 8, 1) - 33) for c in range(255)])


def rounding(step, elements):
    """(of exp_avg, of exp_avg_sq): the fractions that are added before the cut, per element."""
    u32 = lambda a: np.asarray(a, dtype=np.uint64) & np.uint64(0xffffffff)  # noqa: E731
    k = int(step) * 0x6A09E667 & 0xffffffff
    k = (k ^ k >> 15) * 0x9E3779B1 & 0xffffffff
    k ^= k >> 16
    x = u32(u32(elements) * np.uint64(0x9E3779B1) + np.uint64(k))
    x = u32((x ^ (x >> np.uint64(16))) * np.uint64(0xBB67AE85))
    x = x ^ (x >> np.uint64(15))
    return (x % 65536 + 0.5) / 65536, (x // 65536 + 0.5) / 65536


def encode(x, values, top, u):
    """Codes (without sign) and scale bytes of blocks of 64: x (n,) >= 0, what is not finite gets code len(values)."""
    n = len(x)
    codes, scales = np.zeros(n, dtype=np.int64), np.zeros(-(-n // 64), dtype=np.int64)
    for b in range(len(scales)):
        s = slice(64 * b, min(64 * b + 64, n))
        fine = np.isfinite(x[s])
        largest = x[s][fine].max() if fine.any() else 0.0
        e = 0 if largest == 0 else min(max(math.frexp(largest)[1] - 1 - top, -127), 127)
        scales[b] = 0 if largest == 0 else e + 127
        t = np.where(fine, x[s], 0.0) * 2.0 ** (127 - int(scales[b]))
        low = np.searchsorted(values, t, side="right") - 1
        up = np.minimum(low + 1, len(values) - 1)
        step = np.where(up > low, values[up] - values[low], 1.0)
        codes[s] = np.where(fine, low + ((t - values[low]) / step + u[s] >= 1.0), len(values))
    return codes, scales


class State:
    """Moments of one tensor whose elements begin at ``first`` of the flat moments."""

    def __init__(self, n, bits, first=0):
        self.n, self.bits, self.first = n, bits, first
        self.m, self.v = np.zeros(n), np.zeros(n)
        self.terms = np.zeros(n)      # magnitude of what exp_avg has been summed from: what its float32 roundings are relative to
        self.size = np.zeros(n)       # of the last update, with that in the place of exp_avg
        if bits == 8:
            blocks = -(-n // 64)
            self.cm, self.cv = np.zeros(n, dtype=np.int64), np.zeros(n, dtype=np.int64)
            self.sm, self.sv = np.zeros(blocks, dtype=np.int64), np.zeros(blocks, dtype=np.int64)

    def step(self, p, g, t, lr, betas, eps, wd, factor=1.0):
        """The parameter (float64) after step ``t`` with gradient ``g``; moves the moments."""
        b1, b2 = betas
        c = g * factor
        with np.errstate(all="ignore"):
            m, v = b1 * self.m + (1 - b1) * c, b2 * self.v + (1 - b2) * c * c
            self.terms = np.maximum(b1 * self.terms + (1 - b1) * np.abs(c), b1 * np.abs(self.m) + (1 - b1) * np.abs(c))
            held = np.where(v < 2.0 ** 128, v, np.inf)      # 32 bits hold no more
            over = lr / (1 - b1 ** t) / (np.sqrt(held / (1 - b2 ** t)) + eps)
            update, self.size = m * over, self.terms * over
            if self.bits == 8:
                um, uv = rounding(t, self.first + np.arange(self.n))
                self.cm, self.sm = encode(np.abs(m), M_VALUES, 7, um)
                self.cm += 128 * np.signbit(m)
                self.cv, self.sv = encode(held, V_VALUES, 0, uv)
                self.cv = np.where((v > 0) & (self.cv == 0), 1, self.cv)
                self.m, self.v = self.values()
            else:
                self.m, self.v = m, held
            return p * (1 - lr * wd) - update

    def values(self):
        block = np.arange(self.n) // 64
        table = np.append(M_VALUES, np.nan)
        m = table[self.cm % 128] * 2.0 ** (self.sm[block] - 127) * np.where(self.cm > 127, -1.0, 1.0)
        return m, np.append(V_VALUES, np.inf)[self.cv] * 2.0 ** (self.sv[block] - 127)
