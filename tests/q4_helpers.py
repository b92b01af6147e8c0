"""The four-bit format in numpy, in 64 bits where it is exact, and bounds of the products' errors."""
import math

import numpy as np
import torch

HALF_BF16 = 2.0 ** -8    # a rounding to bfloat16, relative


def to_bf16(x):
    """float64 values rounded to bfloat16 (ties to even), by integer arithmetic on the float32 that holds them exactly or nearly."""
    return torch.from_numpy(np.ascontiguousarray(x, dtype=np.float64)).to(torch.float32).to(torch.bfloat16).to(torch.float64).numpy()


def quantise(w, group):
    """(codes, scales, offsets) of a float32 array [N, K]: every step in float32, rounded once."""
    n, k = w.shape
    g = w.astype(np.float32).reshape(n, k // group, group)
    with np.errstate(all="ignore"):
        lo, hi = g.min(2), g.max(2)
        s = to_bf16(((hi - lo) / np.float32(15)).astype(np.float64)).astype(np.float32)
        b = to_bf16(lo.astype(np.float64)).astype(np.float32)
        bad = ~(np.isfinite(g).all(2) & np.isfinite(s) & np.isfinite(b))
        t = (g - b[:, :, None]) / s[:, :, None]
        q = np.where(s[:, :, None] > 0, np.clip(np.rint(t), 0, 15), 0)
    q[np.repeat(bad[:, :, None], group, 2)] = 0
    s[bad], b[bad] = np.nan, np.nan
    return q.astype(np.int64).reshape(n, k), s, b


def matrix(q, s, b, group):
    """What codes, scales and offsets stand for: q s + b (exact in 64 bits for the sizes of these tests), rounded once to bfloat16."""
    return to_bf16(q * np.repeat(s, group, 1).astype(np.float64) + np.repeat(b, group, 1).astype(np.float64))


def unpack(m):
    """(codes, scales, offsets) of an `ops.Q4Matrix`, element by element from its layout."""
    codes = m.codes.cpu().numpy().astype(np.int64) & 0xffffffff
    affine = m.affine.to(torch.float32).cpu().numpy()
    n, k = m.shape
    rows, cols = np.arange(n)[:, None], np.arange(k)[None, :]
    word = codes[rows // 16, cols // 64, cols // 16 % 4, rows % 8, rows // 8 % 2, cols // 8 % 2]
    q = (word >> (4 * (4 * (cols % 2) + cols // 2 % 4))) & 15
    groups = np.arange(k // m.group)[None, :]
    pairs = affine[rows // 16, groups, rows % 8, rows // 8 % 2]
    return q, pairs[..., 0], pairs[..., 1]


def sum_bound(x, w):
    """Bound on the error of float32 sums x w^T.  A tensor-core product adds its 16 (or twice 8) exact terms to the sum with an error of at
    most 2^-23 of the terms' absolute sum a step; the joins of partial sums are a few dozen additions more."""
    steps = x.shape[1] / 8 + 32
    return steps * 2.0 ** -23 * (np.abs(x) @ np.abs(w).T)


def run_bound(x, w):
    """The same for deep products, where the bound above says little: a step's error is at most 2^-23 of the sum that it adds to and of its own terms'
    absolute sum.  What a step adds to is the sum of a run of neighbouring blocks of 64 k and of part of a block (both kernels cut k so): no larger
    than the range of the sums up to a block, and the largest block's absolute sum."""
    m, n, blocks = x.shape[0], w.shape[0], -(-x.shape[1] // 64)
    at, low, high, most = np.zeros((m, n)), np.zeros((m, n)), np.zeros((m, n)), np.zeros((m, n))
    for i in range(blocks):
        a, b = x[:, 64 * i:64 * i + 64], w[:, 64 * i:64 * i + 64]
        at = at + a @ b.T
        low, high = np.minimum(low, at), np.maximum(high, at)
        most = np.maximum(most, np.abs(a) @ np.abs(b).T)
    return 2.0 ** -23 * ((x.shape[1] / 8 + 32) * (high - low + most) + np.abs(x) @ np.abs(w).T)


def act(z, name):
    if name == "silu":
        return z / (1 + np.exp(-z))
    if name == "gelu":
        return 0.5 * z * (1 + np.vectorize(math.erf)(z / math.sqrt(2)))
    if name == "gelu_pytorch_tanh":
        return 0.5 * z * (1 + np.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))
    return np.maximum(z, 0) ** (2 if name == "relu2" else 1)


def gated(x, wg, wu, name, of_sums=sum_bound):
    """(act(x wg^T) * (x wu^T), a bound on the error of the float32 values behind the result's rounding)."""
    g, u = x @ wg.T, x @ wu.T
    dg, du = of_sums(x, wg), of_sums(x, wu)
    a = act(g, name)
    slope = 1.13 if name != "relu2" else 2 * (np.abs(g) + dg)   # (the largest slope of silu and gelu is below 1.13)
    # the activation itself: a few roundings of terms up to |g| (1 + erf and the like cancel for negative g)
    own = 16 * 2.0 ** -24 * (np.abs(g) + np.abs(a))
    return a * u, (slope * dg + own) * (np.abs(u) + du) + np.abs(a) * du


def close(got, want, bound, dtype):
    """Asserts |got - want| <= bound, and the rounding of the result to `dtype`."""
    got = got.to(torch.float64).cpu().numpy()
    half = HALF_BF16 if dtype == torch.bfloat16 else 2.0 ** -24
    limit = bound + half * (np.abs(want) + bound) + 1e-38
    off = np.abs(got - want)
    assert got.shape == want.shape
    assert (off <= limit).all(), "worst %.3g times its limit at %s" % ((off / limit).max(), np.unravel_index((off / limit).argmax(), off.shape))
