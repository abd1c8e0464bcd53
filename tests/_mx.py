"""Microscaled blocks restated in numpy, in 64 bits: the value tables, the
block scale and the rounding, from the format's definition."""

from __future__ import annotations

import math

import numpy as np

# mantissa bits, exponent of the smallest normal number, largest value, bits of a code
FORMATS = {"e4m3": (3, -6, 448.0, 8), "e5m2": (2, -14, 57344.0, 8), "e2m1": (1, 0, 6.0, 4)}
U32 = 2.0 ** -24  # half a step of float32, relative


def magnitudes(fmt: str) -> np.ndarray:
    """The format's values >= 0, by code."""
    mant, emin, top, bits = FORMATS[fmt]
    out = []
    for c in range(1 << (bits - 1)):
        field, frac = c >> mant, c & ((1 << mant) - 1)
        v = math.ldexp(frac / (1 << mant), emin) if field == 0 else math.ldexp(1 + frac / (1 << mant), field - 1 + emin)
        if v > top:
            break
        out.append(v)
    return np.array(out)


def scale_exponents(blocks: np.ndarray, fmt: str) -> np.ndarray:
    """[..., 32] -> the smallest e in -127.. with max|x| <= top * 2^e; 128 for
    a block with an infinity or a NaN."""
    top = FORMATS[fmt][2]
    out = np.full(blocks.shape[:-1], -127)
    flat, res = blocks.reshape(-1, blocks.shape[-1]), out.reshape(-1)
    for i, b in enumerate(flat):
        if not np.isfinite(b).all():
            res[i] = 128
            continue
        a = float(np.abs(b).max()) if b.size else 0.0
        if a > 0:
            e = math.frexp(a)[1] - math.frexp(top)[1] - 1
            while a > math.ldexp(top, e):
                e += 1
            res[i] = max(e, -127)
    return out


def pad_blocks(x: np.ndarray) -> np.ndarray:
    n, b = x.shape
    nb = -(-b // 32)
    return np.pad(x.astype(np.float64), ((0, 0), (0, nb * 32 - b))).reshape(n, nb, 32)


def quantize(x: np.ndarray, fmt: str, keep: bool = False):
    """[N, B] -> (codes as the framework lays them out, scale bytes)."""
    bits = FORMATS[fmt][3]
    mags = magnitudes(fmt)
    blk = pad_blocks(x)
    e = scale_exponents(blk, fmt)
    bad = e == 128
    with np.errstate(all="ignore"):
        z = np.abs(np.ldexp(blk, -np.where(bad, 0, e)[..., None]))
    z = np.where(bad[..., None], 0.0, z)
    i = np.clip(np.searchsorted(mags, z), 1, len(mags) - 1)
    lo, hi = z - mags[i - 1], mags[i] - z
    code = np.where((lo > hi) | ((lo == hi) & (i % 2 == 0)), i, i - 1)
    if keep:
        code = np.where((z != 0) & (code == 0), 1, code)
    code = code | (np.signbit(blk) & ~bad[..., None]).astype(np.int64) << (bits - 1)
    n, nb, _ = blk.shape
    code = code.astype(np.uint8)
    if bits == 4:
        code = code[..., 0::2] | (code[..., 1::2] << 4)
    return code.reshape(n, nb * code.shape[-1]), (e + 127).astype(np.uint8)


def values(codes: np.ndarray, scales: np.ndarray, fmt: str, batch: int) -> np.ndarray:
    """Codes and scale bytes -> [N, batch] float64."""
    bits = FORMATS[fmt][3]
    c = codes.astype(np.int64)
    if bits == 4:
        c = np.stack([c & 15, c >> 4], axis=-1).reshape(codes.shape[0], 2 * codes.shape[1])
    mags = magnitudes(fmt)
    mags = np.concatenate([mags, np.full((1 << (bits - 1)) - len(mags), np.nan)])
    v = mags[c & ((1 << (bits - 1)) - 1)] * np.where(c >> (bits - 1), -1.0, 1.0)
    s = np.where(scales == 255, np.nan, np.ldexp(1.0, scales.astype(np.int64) - 127))
    return (v * np.repeat(s, 32, axis=1))[:, :batch]


def half_step(y: np.ndarray, err: np.ndarray, fmt: str) -> np.ndarray:
    """Half the distance between elements around [N, B] values known within
    `err`, at the largest scale their block may take."""
    mant, emin, _, _ = FORMATS[fmt]
    blk, eb = pad_blocks(np.abs(y)), pad_blocks(err)
    e = scale_exponents(blk + eb, fmt)
    z = np.ldexp(blk + eb, -e[..., None])
    ex = np.where(z > 0, np.frexp(z)[1] - 1, emin)
    step = np.ldexp(1.0, np.maximum(ex, emin) - mant + e[..., None])
    return (step / 2).reshape(y.shape[0], -1)[:, :y.shape[1]]


def act(kind: str, x: np.ndarray) -> np.ndarray:
    with np.errstate(over="ignore"):
        return {"tanh": np.tanh, "relu": lambda v: np.maximum(v, 0.0), "sigmoid": lambda v: 1 / (1 + np.exp(-v)),
                "identity": lambda v: v}[kind](x)


def act_prime(kind: str, a: np.ndarray) -> np.ndarray:
    return {"tanh": lambda v: 1 - v * v, "relu": lambda v: (v > 0).astype(np.float64), "sigmoid": lambda v: v - v * v,
            "identity": np.ones_like}[kind](a)


def product(off, src, w, x, units, rows: int, kind: str, num_src: int):
    """The grouped product and a bound of a float32 evaluation's error:
    (n + 2) roundings of every term for a sum of n (each term takes one for
    its product, one for its scale at most, and one per addition), through an
    activation of slope at most 1, whose own evaluation is off by at most 8
    roundings of the result (4 units in the last place)."""
    y, err = np.zeros((rows, x.shape[1])), np.zeros((rows, x.shape[1]))
    for i, u in enumerate(units):
        if not 0 <= u < rows:
            continue
        e = np.arange(off[i], off[i + 1])
        e = e[(src[e] >= 0) & (src[e] < num_src)]
        t = w[e, None] * x[src[e]]
        y[u] = act(kind, t.sum(axis=0))
        err[u] = (len(e) + 2) * U32 * np.abs(t).sum(axis=0) * 1.01 + 8 * U32 * np.abs(y[u])
    return y, err
