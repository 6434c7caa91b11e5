"""Plain 64-bit restatement of the 4-bit page format and of windowed attention with sinks, for the tests.

All quotients and sums below are of f32 inputs in f64, where they are off by at most 2^-53 relative; the
borders they are compared with are multiples of 2^-24 relative to them, so every decision is the exact one.
"""
import numpy as np

GROUP = 32


def bf16_nearest(x):
    """Nearest bf16 value of f64 values (ties to even), as f64."""
    bits = np.ascontiguousarray(x, np.float64).view(np.uint64)
    bits = bits + np.uint64((1 << 44) - 1) + ((bits >> np.uint64(45)) & np.uint64(1))
    return (bits >> np.uint64(45) << np.uint64(45)).view(np.float64)


def bf16_bits(x):
    """Bit pattern of f64 values that are bf16 values."""
    return (np.asarray(x, np.float64).astype(np.float32).view(np.uint32) >> 16).astype(np.uint16)


def quantize(x, row0, hd):
    """Rows x [n][kv_dim] (f32) written from position row0 on -> codes [n][kv_dim], signed scale and bias [n][kv_dim/32]
    (f64). Groups with values that are not finite: code 0, scale NaN, bias 0."""
    n, kv_dim = x.shape
    sign = np.where((np.arange(n) + row0) % 2 == 1, -1.0, 1.0)[:, None, None, None]
    y = x.astype(np.float64).reshape(n, kv_dim // hd, hd // GROUP, GROUP) * sign
    bad = ~np.isfinite(y).all(-1, keepdims=True)
    y = np.where(bad, 0.0, y)
    bias = bf16_nearest(y.min(-1, keepdims=True))
    width = y.max(-1, keepdims=True) - bias
    bad |= (np.abs(bias) > 3.39e38) | (width >= 2.0 ** 128 - 2.0 ** 103)
    bias, width = np.where(bad, 0.0, bias), np.where(bad, 0.0, width)
    widest = np.maximum((width / 15).max(2, keepdims=True), 2.0 ** -40)
    floor = np.ldexp(1.0, np.frexp(widest)[1] - 17)
    step = bf16_nearest(np.maximum(np.maximum(width / 15, floor), 2.0 ** -40))
    code = np.clip(np.rint((y - bias) / step), 0, 15)
    code = np.where(bad, 0, code)
    scale = np.where(bad, np.nan, sign * step)
    bias = np.where(bad, 0.0, sign * bias)
    return code.astype(np.uint8).reshape(n, kv_dim), scale.reshape(n, -1), bias.reshape(n, -1)


def dequantize(code, scale, bias):
    """f64 values; rounded to f32 they are what the row reads back as."""
    return code.astype(np.float64) * np.repeat(scale, GROUP, -1) + np.repeat(bias, GROUP, -1)


def read_back(x, row0, hd):
    return dequantize(*quantize(x, row0, hd)).astype(np.float32)


def stored(x, row0, hd, dtype):
    """What rows x read back as from pages of `dtype` (0 f32, 1 bf16, 3 u4), f64."""
    if dtype == 3:
        return read_back(x, row0, hd).astype(np.float64)
    return bf16_nearest(x.astype(np.float64)) if dtype == 1 else x.astype(np.float64)


def attention(q, k, v, kv_heads, start=0, sinks=0, scalar=0.0):
    """q [q_heads][hd], k and v [rows][kv_heads * hd] f64 -> (out [q_heads][hd], bound): softmax(q.k / sqrt(scalar)).v over
    the rows r < sinks or r >= start.

    bound: how far a kernel may be that forms every product of codes, steps and biases with f32 sums. With S the
    largest over the rows of sum |q| (|k| + 2 spread) / sqrt(hd), spread = the values' largest magnitude (a code's
    share and the bias are each at most that large), the scores are off by at most (hd / 8 + 16) 2^-23 S, which moves a
    weight by that share; the sums over rows / 16 pages add (rows / 16 + 64) 2^-23 of the weighted magnitudes."""
    q_heads, hd = q.shape
    rows = np.arange(len(k))
    seen = (rows < sinks) | (rows >= start)
    k, v = (x.reshape(len(rows), kv_heads, hd)[seen] for x in (k, v))
    gqa = q_heads // kv_heads
    scalar = scalar if scalar > 0 else hd
    out, bound = np.empty((q_heads, hd)), np.empty((q_heads, 1))
    for h in range(q_heads):
        kh, vh = k[:, h // gqa], v[:, h // gqa]
        s = kh @ q[h].astype(np.float64) / np.sqrt(scalar)
        p = np.exp(s - s.max())
        p /= p.sum()
        out[h] = p @ vh
        size = np.sum(np.abs(q[h])) * 3 * np.abs(kh).max() / np.sqrt(scalar)
        bound[h] = (2 * (hd / 8 + 16) * size + len(kh) / 16 + 64) * 2.0 ** -23 * 3 * np.abs(vh).max()
    return out, bound


def close(got, want_bound, rel=1e-5):
    """Every value within the bound, and the whole row within `rel` in the 2-norm: the roundings are independent, so
    scores are typically off by sqrt(hd / 8 + 16) 2^-24 of their largest partial sum (about 1e-6) and the sums over the
    pages by as much again; 1e-5 leaves a factor of five."""
    want, bound = want_bound
    got = np.asarray(got, np.float64).reshape(want.shape)
    err = np.abs(got - want)
    norm = np.linalg.norm(want)
    return bool(np.all(err <= bound)) and np.linalg.norm(got - want) <= rel * norm, (err.max(), np.linalg.norm(got - want) / norm)
