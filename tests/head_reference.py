"""A language model head's operators in 64 bits, and operands in every layout for their tests.

Numbers are numpy arrays of f64; bf16 and e4m3 travel as their bits. Quantization is restated
operation by operation in f32, as its definition has it, so its results are compared bit for bit.
"""
from __future__ import annotations

import numpy as np

from linalg_hip import backend as B

F32, F16, BF16 = B.DType.F32, B.DType.F16, B.DType.BF16
E4M3, E8M0, I32 = B.DType.E4M3, B.DType.E8M0, B.DType.I32
STORED = {F32: np.float32, F16: np.float16, BF16: np.uint16, E4M3: np.uint8, E8M0: np.uint8, I32: np.int32}
# Half a unit in the last place over the value, and the smallest normal number, of a result's type.
ROUNDING = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}
SMALL = {F32: 2.0 ** -126, F16: 2.0 ** -14, BF16: 2.0 ** -126}


# ------------------------------------------------------------------------------- the types


def to_bits(x, dtype):
    """f64 or f32 numbers rounded to the type, to nearest, ties to even, as they are stored."""
    if dtype is not BF16:
        with np.errstate(over="ignore"):
            return np.asarray(x).astype(STORED[dtype])
    b = np.ascontiguousarray(np.asarray(x, dtype=np.float32)).view(np.uint32).astype(np.uint64)
    r = ((b + 0x7fff + ((b >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where((b & 0x7fffffff) > 0x7f800000, np.uint16(0x7fc0), r)


def values(bits, dtype):
    """What stored elements stand for, as f64."""
    if dtype is BF16:
        return (bits.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    if dtype is E4M3:
        return E4M3_VALUES[bits]
    if dtype is E8M0:
        return np.where(bits == 255, np.nan, np.exp2(bits.astype(np.float64) - 127))
    return bits.astype(np.float64)


def _e4m3_values():
    b = np.arange(256)
    e, f = (b >> 3) & 15, b & 7
    v = np.where(e == 0, f * 2.0 ** -9, (8 + f) * np.exp2(e - 10.0))
    v = np.where((b & 127) == 127, np.nan, v)
    return np.where(b > 127, -v, v)


E4M3_VALUES = _e4m3_values()


def to_e4m3(x):
    """Numbers of at most 448 (or NaN) rounded to e4m3, to nearest, ties to even: bits."""
    grid = E4M3_VALUES[:127]
    a = np.abs(np.asarray(x, dtype=np.float64))
    hi = np.searchsorted(grid, np.where(np.isnan(a), 0.0, a)).clip(0, 126)
    lo = np.maximum(hi - 1, 0)
    up, down = grid[hi] - a, a - grid[lo]
    code = np.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
    code = np.where(np.isnan(a), 127, code)
    return np.where(np.signbit(x) & ~np.isnan(a), code + 128, code).astype(np.uint8)


def quantize(x, block, scales):
    """(e4m3 bits, scales as stored) of x, f32 numbers [R, C]."""
    r, c = x.shape
    pr, pc = -(-r // block) * block, -(-c // 128) * 128
    p = np.zeros((pr, pc), np.float32)
    p[:r, :c] = x
    p = p.reshape(pr // block, block, pc // 128, 128)
    a = np.abs(p).max(axis=(1, 3))
    fine = np.isfinite(a)
    a = np.where(fine, np.maximum(a, np.float32(2.0 ** -100)), np.float32(np.nan)).astype(np.float32)
    if scales is F32:
        with np.errstate(invalid="ignore"):
            s, inverse = a / np.float32(448), np.float32(448) / a
    else:
        e = np.ceil(np.log2(np.where(fine, a, 1).astype(np.float64) / 448.0) - 1e-12).astype(int)
        e += np.where(fine, a, 1).astype(np.float64) > 448.0 * np.exp2(e.astype(np.float64))
        s = np.where(fine, e + 127, 255).astype(np.uint8)
        inverse = np.where(fine, np.exp2(-e.astype(np.float64)), np.nan).astype(np.float32)
    with np.errstate(invalid="ignore", over="ignore", under="ignore"):
        y = p * inverse[:, None, :, None]
    return to_e4m3(y).reshape(pr, pc)[:r, :c], s


def unquantized(q, s, block, scales):
    """The f64 numbers that quantized elements and their scales stand for."""
    r, c = q.shape
    s = np.repeat(np.repeat(values(s, scales), block, 0)[:r], 128, 1)[:, :c]
    return values(q, E4M3) * s


# -------------------------------------------------------------------------------- softmax


def _row(x, t):
    """(kind, log probabilities, p) of one row of logits."""
    if np.isnan(x).any() or (x == np.inf).any():
        return "bad", None, None
    if (x == -np.inf).all():
        return "empty", None, None
    with np.errstate(divide="ignore"):
        d = (x - x.max()) / t
        lp = d - np.log(np.exp(d).sum())
    return "fine", lp, np.exp(lp)


def logprobs(x, tokens, k, t):
    """token_logprobs of f64 logits: (logprobs, entropy, stats, top log probabilities, ids)."""
    r, v = x.shape
    lp, h, st = np.zeros(r), np.zeros(r), np.zeros((r, 2))
    top, ids = np.full((r, k), -np.inf), np.full((r, k), -1, np.int32)
    for i in range(r):
        kind, logs, p = _row(x[i], t)
        named = 0 <= tokens[i] < v
        if kind == "bad":
            lp[i], h[i], st[i], top[i] = (np.nan if named else 0), np.nan, np.nan, np.nan
        elif kind == "empty":
            lp[i], h[i], st[i] = (-np.inf if named else 0), 0, -np.inf
        else:
            lp[i] = logs[tokens[i]] if named else 0
            h[i] = -(p[p > 0] * logs[p > 0]).sum()
            m = x[i].max()
            st[i] = m, np.log(np.exp((x[i] - m) / t).sum())
            best = np.argsort(-x[i], kind="stable")[:k]
            best = best[x[i][best] > -np.inf]
            top[i, :len(best)], ids[i, :len(best)] = logs[best], best
    return lp, h, st, top, ids


def logprobs_backward(x, tokens, t, g, gh):
    r, v = x.shape
    dx = np.zeros((r, v))
    for i in range(r):
        kind, logs, p = _row(x[i], t)
        if kind == "bad":
            dx[i] = np.nan
        elif kind == "fine":
            named = 0 <= tokens[i] < v
            gi = g[i] if named else 0.0
            dx[i] = -gi * p
            if named:
                dx[i, tokens[i]] += gi
            live = p > 0
            h = -(p[live] * logs[live]).sum()
            dx[i, live] -= gh[i] * p[live] * (logs[live] + h)
    return dx / t


def distill(x, ids, lists, weights, t, normalize):
    """(losses, dlogits)."""
    r, v = x.shape
    losses, dx = np.zeros(r), np.zeros((r, v))
    for i in range(r):
        named = (ids[i] >= 0) & (ids[i] < v) & (lists[i] != -np.inf)
        kind, logs, q = _row(x[i], t)
        if weights[i] == 0 or not named.any() or kind == "empty":
            continue
        if kind == "bad":
            losses[i], dx[i] = np.nan, np.nan
            continue
        at, lp = ids[i][named], lists[i][named].astype(np.float64)
        if normalize:
            lp = lp - lp.max() - np.log(np.exp(lp - lp.max()).sum())
        p = np.exp(lp)
        live = p > 0
        losses[i] = weights[i] * t * t * (p[live] * (lp[live] - logs[at[live]])).sum()
        dx[i] = p.sum() * q
        np.subtract.at(dx[i], at, p)
        dx[i] *= weights[i] * t
    return losses, dx


# ------------------------------------------------------------------------------- operands


class Window:
    """An [R, C] operand inside a larger allocation: `pad` elements between rows, `offset` before
    the first; what lies around it keeps a pattern that a test can look at afterwards."""

    def __init__(self, hb, dtype, data=None, shape=None, pad=0, offset=0, tail=0):
        shape = list(data.shape if data is not None else shape)
        self.hb, self.dtype, self.shape = hb, dtype, shape
        rows, cols = (shape[0], shape[1]) if len(shape) == 2 else (1, shape[0])
        self.pitch, self.offset = cols + pad, offset
        n = offset + max(0, rows - 1) * self.pitch + cols + tail
        self.around = np.arange(n, dtype=np.int64).astype(np.uint8) | 1
        host = np.repeat(self.around, dtype.size_of()).view(STORED[dtype]).copy()
        self.index = (offset + np.arange(rows)[:, None] * self.pitch + np.arange(cols)[None]).reshape(shape)
        if data is not None:
            host[self.index] = data
        self.host = host
        base = hb.upload(dtype, [n], host.tobytes())
        strides = [self.pitch, 1] if len(shape) == 2 else [1]
        self.t = B.Tensor(base.storage, dtype, shape, strides, offset)
        self.whole = base

    def read(self):
        """The operand's elements; everything around them has to be untouched."""
        got = np.frombuffer(self.hb.download(self.whole), STORED[self.dtype])
        outside = np.ones(got.size, bool)
        outside[self.index] = False
        assert np.array_equal(got[outside].view(np.uint8), self.host[outside].view(np.uint8)), "wrote outside its operand"
        return got[self.index]


def close(got, want, atol, rtol, what):
    """Equal where `want` is not finite, within atol + rtol |want| elsewhere."""
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    fine = np.isfinite(want)
    assert np.array_equal(np.isnan(got), np.isnan(want)), f"{what}: NaN in other places"
    assert np.array_equal(got[~fine & ~np.isnan(want)], want[~fine & ~np.isnan(want)]), f"{what}: infinities differ"
    with np.errstate(invalid="ignore"):
        over = np.abs(got - want) - (np.broadcast_to(atol, want.shape) + rtol * np.abs(want))
    over = np.where(fine, over, -1.0)
    if over.size:
        i = np.unravel_index(np.argmax(over), over.shape)
        assert over[i] <= 0, f"{what}: {got[i]} for {want[i]} at {i}, {over[i]:.3g} past the bound"
