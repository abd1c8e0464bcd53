"""The microscaled row operators on the GPU against their numpy restatement in
64 bits (tests/_mx.py): codes and scales bit for bit, sums within the bound of
a float32 evaluation (every rounding at most half a step, 2^-24 of the value).
"""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

import plastax_b200 as px
from plastax_b200 import kernels as K
from plastax_b200 import mx

from tests import _mx

pytestmark = pytest.mark.gpu

SIZES = [(1, 1), (3, 7), (5, 31), (5, 32), (7, 33), (64, 250), (33, 256), (9, 1000), (300, 4)]
FMTS = sorted(_mx.FORMATS)
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def _values(rng, n, b):
    """Rows over many sizes, with silent rows, values next to the borders of
    the scale and the elements, zeros of both signs and tiny ones."""
    x = rng.standard_normal((n, b)) * np.exp(rng.standard_normal((n, 1)) * 6)
    x[rng.random((n, b)) < 0.1] = 0.0
    x[rng.random((n, b)) < 0.05] *= 1e-7
    x[rng.random((n, b)) < 0.05] *= -0.0
    tie = rng.random((n, b)) < 0.2  # few mantissa bits: many ties and maxima on the scale's border
    m, e = np.frexp(x)
    x[tie] = np.ldexp(np.round(m * 32) / 32, e)[tie]
    x[n // 3] = 0.0
    return x.astype(np.float32)


def _rows(x, fmt, keep, dev):
    codes, scales = _mx.quantize(x, fmt, keep)
    return px.MxRows(torch.from_numpy(codes).to(dev), torch.from_numpy(scales).to(dev), fmt, x.shape[1])


def _same(rows, codes, scales, msg=""):
    np.testing.assert_array_equal(rows.scales.cpu().numpy(), scales, err_msg=msg)
    np.testing.assert_array_equal(rows.codes.cpu().numpy(), codes, err_msg=msg)


def _within(got, want, err, msg=""):
    """|got - want| <= err, and NaN where want has one."""
    got = got.astype(np.float64)
    np.testing.assert_array_equal(np.isnan(got), np.isnan(want), err_msg=msg)
    ok = ~np.isnan(want)
    off = np.abs(got - want)[ok] - err[ok]
    assert off.size == 0 or off.max() <= 0, f"{msg}: past the bound by {off.max()}"


# ---------------------------------------------------------------------------
# quantisation and reading back
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("n,b", SIZES)
def test_quantize_is_bit_exact(cuda, fmt, dtype, n, b):
    rng = np.random.default_rng(n * 1000 + b)
    x = torch.from_numpy(_values(rng, n, b)).clamp(-6e4, 6e4).to(DTYPES[dtype]).to(cuda)
    host = x.float().cpu().numpy()
    wide = torch.full((n, b + 3), 9.0, dtype=x.dtype, device=cuda)
    wide[:, 1:b + 1] = x
    flat = torch.full((n * b + 1,), 9.0, dtype=x.dtype, device=cuda)
    flat[1:] = x.reshape(-1)
    forms = {"rows": x, "by sample": x.t().contiguous().t(), "wide rows": wide[:, 1:b + 1],
             "off the boundary": flat[1:].view(n, b), "every other": x.repeat_interleave(2, dim=1)[:, ::2]}
    for keep in (False, True):
        want = _mx.quantize(host, fmt, keep)
        for name, v in forms.items():
            _same(px.mx_quantize(v, fmt, keep_nonzero=keep), *want, msg=f"{name} keep={keep}")


@pytest.mark.parametrize("fmt", FMTS)
def test_quantize_special_values(cuda, fmt):
    top = _mx.FORMATS[fmt][2]
    x = np.zeros((10, 40), np.float32)
    x[0, 3] = np.nan
    x[1, 35] = np.inf
    x[2, 0] = -np.inf
    x[3, :] = 3.4e38
    x[4, :] = -1e-45  # the smallest subnormal
    x[5, 1:] = 1e-40
    x[5, 0] = 2.0 ** -126
    x[6, :] = top
    x[7, :] = np.nextafter(np.float32(top), np.float32(np.inf))
    x[8, 0] = 3e38
    x[8, 1:] = 1e-38
    x[0, 4:] = 5.0
    t = torch.from_numpy(x).to(cuda)
    for keep in (False, True):
        want = _mx.quantize(x, fmt, keep)
        rows = px.mx_quantize(t, fmt, keep_nonzero=keep)
        _same(rows, *want)
        # read in float32: the element nearest 3.4e38 in e2m1 is 4 * 2^126 = 2^128, past float32's largest, so infinite
        with np.errstate(over="ignore"):
            held = _mx.values(*want, fmt, 40).astype(np.float32).astype(np.float64)
        got = px.mx_dequantize(rows).cpu().numpy().astype(np.float64)
        np.testing.assert_array_equal(got, held)
        if keep:
            fine = np.isfinite(got)
            np.testing.assert_array_equal(np.sign(got)[fine], np.sign(x)[fine])
    # a block next to a poisoned one is untouched
    assert np.isnan(got[0, :32]).all() and np.isfinite(got[0, 32:]).all()


def test_quantize_into_rows(cuda):
    """`ids` scatters; out-of-range ids are skipped; other rows stay."""
    rng = np.random.default_rng(5)
    x = _values(rng, 6, 45)
    out = px.MxRows.empty(20, 45, "e2m1", cuda)
    out.codes.fill_(7), out.scales.fill_(9)
    ids = torch.tensor([3, 19, -1, 0, 20, 11], device=cuda)
    px.mx_quantize(torch.from_numpy(x).to(cuda), "e2m1", ids=ids, out=out)
    codes, scales = np.full((20, 32), 7, np.uint8), np.full((20, 2), 9, np.uint8)
    c, s = _mx.quantize(x, "e2m1")
    for i, u in ((0, 3), (1, 19), (3, 0), (5, 11)):
        codes[u], scales[u] = c[i], s[i]
    _same(out, codes, scales)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("n,b", SIZES)
def test_dequantize(cuda, fmt, dtype, n, b):
    rng = np.random.default_rng(n * 100 + b)
    rows = _rows(np.clip(_values(rng, n, b), -6e4, 6e4), fmt, False, cuda)
    want = torch.from_numpy(_mx.values(rows.codes.cpu().numpy(), rows.scales.cpu().numpy(), fmt, b))
    want = want.to(torch.float32).to(DTYPES[dtype])  # the first step is exact
    assert torch.equal(px.mx_dequantize(rows, dtype=DTYPES[dtype]).cpu(), want)
    wide = torch.full((n, b + 5), 9.0, dtype=DTYPES[dtype], device=cuda)
    px.mx_dequantize(rows, out=wide[:, 2:b + 2])
    assert torch.equal(wide[:, 2:b + 2].cpu(), want)
    assert bool((wide[:, :2] == 9).all()) and bool((wide[:, b + 2:] == 9).all())


def test_every_code_reads_its_value(cuda):
    for fmt in FMTS:
        for scale in (0, 1, 100, 127, 200, 254, 255):
            codes = np.arange(256, dtype=np.uint8).reshape(8 if fmt != "e2m1" else 16, -1)
            scales = np.full((codes.shape[0], 1), scale, np.uint8)
            rows = px.MxRows(torch.from_numpy(codes).to(cuda), torch.from_numpy(scales).to(cuda), fmt, 32)
            want = _mx.values(codes, scales, fmt, 32)
            if fmt == "e5m2":  # its infinities (0x7c, 0xfc) are never written; they read as they are
                inf = (codes & 0x7f) == 0x7c
                want[inf] = np.where(codes[inf] & 0x80, -np.inf, np.inf) * (1.0 if scale != 255 else np.nan)
            with np.errstate(over="ignore"):
                want = want.astype(np.float32)
            np.testing.assert_array_equal(px.mx_dequantize(rows).cpu().numpy(), want)


# ---------------------------------------------------------------------------
# the checkpoint: forward apply, unit gradient, edge gradient, update
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("fmt", mx.CHECKPOINT_FORMATS)
@pytest.mark.parametrize("kind", ["identity", "tanh", "relu", "sigmoid"])
@pytest.mark.parametrize("n,b", [(1, 1), (50, 7), (33, 32), (40, 100), (12, 260)])
def test_unit_apply_and_grad(cuda, fmt, kind, n, b):
    rng = np.random.default_rng(n + b)
    level = rng.integers(0, 3, n).astype(np.int32)
    roles = rng.integers(0, 3, n).astype(np.uint8)
    z = _values(rng, n, b).clip(-30, 30)
    d = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(cuda)  # noqa: E731
    rows = d(z)
    ck = px.MxRows.empty(n, b, fmt, cuda)
    ck.codes.fill_(3), ck.scales.fill_(5)
    px.mx_unit_apply(rows, ck, (kind, "identity"), level=d(level), target_level=1, roles=d(roles))
    got = rows.cpu().numpy()
    here = level == 1
    np.testing.assert_array_equal(got[~here], z[~here])
    np.testing.assert_array_equal(got[here & (roles == 1)], z[here & (roles == 1)])
    plain = here & (roles == 0)
    y = _mx.act(kind, z[plain].astype(np.float64))
    _within(got[plain], y, 8 * _mx.U32 * np.abs(y))
    np.testing.assert_array_equal(got[here & (roles == 2)], z[here & (roles == 2)])  # identity outputs
    codes, scales = _mx.quantize(got, fmt, True)  # of the float32 results: bit for bit
    codes[~here], scales[~here] = 3, 5
    _same(ck, codes, scales)
    # the gradient from the checkpoint, in place, under the same mask
    ck = px.mx_quantize(rows, fmt, keep_nonzero=True)
    a = px.mx_dequantize(ck).cpu().numpy().astype(np.float64)
    acc, seed = rng.standard_normal((n, b)).astype(np.float32), rng.standard_normal((n, b)).astype(np.float32)
    on = here & (roles != 1)
    p = np.where((roles == 2)[:, None], 1.0, _mx.act_prime(kind, a))
    for s in (None, seed):
        up = acc.astype(np.float64) + (0 if s is None else s.astype(np.float64))
        # a * a, 1 - a * a (or 1 - a, a * ..), the sum and the product each round once
        err = 1.01 * _mx.U32 * np.abs(up) * (2 * (a * a + np.abs(a) + np.abs(p)) + 2 * np.abs(p))
        want = np.where(on[:, None], up * p, acc)
        buf = d(acc)
        out = px.mx_unit_grad(buf, ck, (kind, "identity"), seed=None if s is None else d(s), level=d(level),
                              target_level=1, roles=d(roles), out=buf)
        assert out is buf
        _within(out.cpu().numpy(), want, np.where(on[:, None], err, 0))
        new = px.mx_unit_grad(d(acc), ck, (kind, "identity"), seed=None if s is None else d(s), level=d(level),
                              target_level=1, roles=d(roles)).cpu().numpy()
        np.testing.assert_array_equal(new, np.where(on[:, None], out.cpu().numpy(), 0))


def test_unit_grad_against_differences(cuda):
    """From checkpoint values inside the activation's range, the derivative
    equals the central difference of the activation at its preimage."""
    rng = np.random.default_rng(2)
    a32 = (rng.random((20, 64)) * 0.9 + 0.05).astype(np.float32)
    ck = px.mx_quantize(torch.from_numpy(a32).to(cuda), "e4m3", keep_nonzero=True)
    a = px.mx_dequantize(ck).cpu().numpy().astype(np.float64)
    acc = torch.ones((20, 64), device=cuda)
    for kind, pre in (("tanh", np.arctanh(a)), ("sigmoid", np.log(a / (1 - a)))):
        h = 1e-5
        diff = (_mx.act(kind, pre + h) - _mx.act(kind, pre - h)) / (2 * h)
        got = px.mx_unit_grad(acc, ck, kind).cpu().numpy()
        # the difference is off by h^2 / 6 times the third derivative (at most 2) and its own rounding
        assert np.abs(got - diff).max() <= h * h + 1e-10 / h * 1e-5 + 4 * _mx.U32


def _bucket(rng, n, cap, dev, dead=0.3, bad=True):
    f, t = rng.integers(0, n, cap).astype(np.int32), rng.integers(0, n, cap).astype(np.int32)
    f[:cap // 2].sort()
    dd = (rng.random(cap) < dead).astype(np.uint8)
    if bad and cap > 8:
        f[1], t[2], f[3], t[4] = -1, n, n + 5, -(1 << 31)
    b = {"from_id": f, "to_id": t, "dead": dd}
    return b, {k: torch.from_numpy(v).to(dev) for k, v in b.items()}


def _edge_reference(b, g, a, n):
    f, t = b["from_id"].astype(np.int64), b["to_id"].astype(np.int64)
    live = (b["dead"] == 0) & (f >= 0) & (f < n) & (t >= 0) & (t < n)
    prod = g[np.where(live, t, 0)].astype(np.float64) * a[np.where(live, f, 0)]
    batch = g.shape[1]
    want = np.where(live, prod.sum(1) / batch, 0.0)
    # a term rounds once as a product, once with its scale, and once per addition it takes part in
    err = np.where(live, (batch + 4) * _mx.U32 * np.abs(prod).sum(1) / batch * 1.01, 0.0)
    return live, want, err


@pytest.mark.parametrize("fmt", mx.CHECKPOINT_FORMATS)
@pytest.mark.parametrize("n,cap,batch", [(1, 1, 1), (5, 31, 3), (40, 33, 4), (17, 1000, 32), (90, 700, 33),
                                         (64, 4096, 64), (50, 3001, 256), (30, 400, 1001), (1200, 20000, 96)])
def test_edge_grad(cuda, fmt, n, cap, batch):
    rng = np.random.default_rng(cap + batch)
    b, dev = _bucket(rng, n, cap, cuda)
    g = rng.standard_normal((n, batch)).astype(np.float32)
    ck = _rows(_values(rng, n, batch).clip(-100, 100), fmt, True, cuda)
    a = _mx.values(ck.codes.cpu().numpy(), ck.scales.cpu().numpy(), fmt, batch)
    _, want, err = _edge_reference(b, g, a, n)
    out = px.mx_edge_grad(dev, torch.from_numpy(g).to(cuda), ck)
    _within(out.cpu().numpy(), want, err)
    again = px.mx_edge_grad(dev, torch.from_numpy(g).to(cuda), ck, out=torch.full_like(out, 5.0))
    assert torch.equal(out, again)  # no order of summation to chance


@pytest.mark.parametrize("fmt", mx.CHECKPOINT_FORMATS)
@pytest.mark.parametrize("n,cap,batch", [(1, 1 << 21, 32), (64, 70001, 1001), (130, 262200, 256), (1000, 300000, 260),
                                         (200, 2040000, 33)])
def test_edge_grad_of_a_small_net_with_many_slots(cuda, fmt, n, cap, batch):
    """The sizes that take one matrix product of all touched pairs: every
    pair's sum in 64 bits, gathered; odd batches, edge tiles, bad ids, a NaN and
    an infinity that reach their own row's slots only."""
    assert mx.edge_grad_scratch_bytes(cap, batch, n) > 0
    rng = np.random.default_rng(cap)
    b, dev = _bucket(rng, n, cap, cuda)
    g = (rng.standard_normal((n, batch)) * np.exp(rng.standard_normal((n, 1)) * 4)).astype(np.float32)
    x = _values(rng, n, batch).clip(-100, 100)
    if n > 5:
        x[3, batch // 2] = np.nan
        g[5, 1] = np.inf
    ck = px.mx_quantize(torch.from_numpy(x).to(cuda), fmt, keep_nonzero=True)
    a = _mx.values(ck.codes.cpu().numpy(), ck.scales.cpu().numpy(), fmt, batch)
    f, t = b["from_id"].astype(np.int64), b["to_id"].astype(np.int64)
    live = (b["dead"] == 0) & (f >= 0) & (f < n) & (t >= 0) & (t < n)
    f, t = np.where(live, f, 0), np.where(live, t, 0)
    with np.errstate(invalid="ignore"):
        pairs, size = g.astype(np.float64) @ a.T / batch, np.abs(g).astype(np.float64) @ np.abs(a).T / batch
    want, err = np.where(live, pairs[t, f], 0.0), np.where(live, size[t, f] * (batch + 4) * _mx.U32 * 1.01, 0.0)
    got = px.mx_edge_grad(dev, torch.from_numpy(g).to(cuda), ck).cpu().numpy()
    odd = ~np.isfinite(want)
    if n > 5:  # the row with the infinity: infinite, or not a number where it meets a 0
        np.testing.assert_array_equal(np.isnan(got), np.isnan(want))
        np.testing.assert_array_equal(got[np.isinf(want)], want[np.isinf(want)].astype(np.float32))
        assert odd.any()
    _within(got[~odd], want[~odd], err[~odd])
    again = px.mx_edge_grad(dev, torch.from_numpy(g).to(cuda), ck, out=torch.full((cap,), 3.0, device=cuda)).cpu().numpy()
    np.testing.assert_array_equal(got, again)


def test_update_of_a_small_net_with_many_slots(cuda):
    rng = np.random.default_rng(10)
    n, cap, batch = 150, 262144, 256
    b, dev = _bucket(rng, n, cap, cuda)
    g = torch.from_numpy(rng.standard_normal((n, batch)).astype(np.float32)).to(cuda)
    ck = px.mx_quantize(torch.from_numpy(rng.standard_normal((n, batch)).astype(np.float32)).to(cuda), "e4m3")
    dw = px.mx_edge_grad(dev, g, ck)
    w = torch.from_numpy(rng.standard_normal(cap).astype(np.float32)).to(cuda)
    col = {**dev, "weight": w.clone()}
    px.mx_update(col, g, ck, px.optim.sgd(0.25).struct())
    assert torch.equal(col["weight"], w - 0.25 * dw)  # 0.25 dw is exact: one rounding on both sides


def test_edge_grad_all_dead_empty_and_poisoned(cuda):
    rng = np.random.default_rng(8)
    b, dev = _bucket(rng, 10, 300, cuda, dead=0.0, bad=False)
    g = rng.standard_normal((10, 40)).astype(np.float32)
    x = _values(rng, 10, 40)
    x[4, 2] = np.inf  # poisons unit 4's first block
    g[6, 1] = np.nan
    ck = px.mx_quantize(torch.from_numpy(x).to(cuda), "e4m3", keep_nonzero=True)
    out = px.mx_edge_grad(dev, torch.from_numpy(g).to(cuda), ck).cpu().numpy()
    np.testing.assert_array_equal(np.isnan(out), (b["from_id"] == 4) | (b["to_id"] == 6))
    dev["dead"].fill_(1)
    assert not px.mx_edge_grad(dev, torch.from_numpy(g).to(cuda), ck).any()
    none = {k: v[:0] for k, v in dev.items()}
    assert px.mx_edge_grad(none, torch.from_numpy(g).to(cuda), ck).numel() == 0


def test_edge_grad_against_differences(cuda):
    """dw of L(w) = 1/B sum_b sum_u (sum_e w_e a[src, b])^2 / 2 (g = the unit
    sums) against central differences in 64 bits."""
    rng = np.random.default_rng(4)
    n, cap, batch = 12, 60, 40
    b, dev = _bucket(rng, n, cap, cuda, bad=False)
    ck = _rows(rng.standard_normal((n, batch)).astype(np.float32), "e4m3", True, cuda)
    a = _mx.values(ck.codes.cpu().numpy(), ck.scales.cpu().numpy(), "e4m3", batch)
    w = rng.standard_normal(cap)

    def sums(w):
        y = np.zeros((n, batch))
        live = b["dead"] == 0
        np.add.at(y, b["to_id"][live], w[live, None] * a[b["from_id"][live]])
        return y

    g = sums(w).astype(np.float32)
    got = px.mx_edge_grad(dev, torch.from_numpy(g).to(cuda), ck).cpu().numpy()
    _, _, err = _edge_reference(b, g, a, n)
    h = 1e-4
    for s in range(cap):
        e = np.zeros(cap)
        e[s] = h
        diff = ((sums(w + e) ** 2).sum() - (sums(w - e) ** 2).sum()) / (2 * batch) / (2 * h)
        # L is quadratic: the difference is exact but for its rounding; g itself was rounded once
        assert abs(diff - got[s]) <= 2 * err[s] + 1e-9


@pytest.mark.parametrize("kind", ["sgd", "momentum", "adam", "adamw", "rmsprop"])
def test_update_steps_as_the_float32_update(cuda, kind):
    """mx_update against pxb_batched_update on the read-back activations: the
    same optimizer step from gradients that differ by their sums' rounding."""
    rng = np.random.default_rng(9)
    n, cap, batch = 70, 2000, 64
    opt = {"sgd": px.optim.sgd(0.1), "momentum": px.optim.momentum(0.1), "adam": px.optim.adam(0.01),
           "adamw": px.optim.adamw(0.01), "rmsprop": px.optim.rmsprop(0.01, eps=1e-3)}[kind]
    b, dev = _bucket(rng, n, cap, cuda)
    d = lambda a: torch.from_numpy(a).to(cuda)  # noqa: E731
    cols = {"weight": rng.standard_normal(cap).astype(np.float32)}
    for name, v in (("opt/m", rng.standard_normal(cap)), ("opt/v", rng.random(cap) + 1.0), ("opt/t", np.full(cap, 3.0))):
        if name in [f.name for f in opt.state_fields]:
            cols[name] = v.astype(np.float32)
    one = {**dev, **{k: d(v) for k, v in cols.items()}}
    two = {**dev, **{k: d(v) for k, v in cols.items()}}
    g = d(rng.standard_normal((n, batch)).astype(np.float32))
    ck = px.mx_quantize(d(rng.standard_normal((n, batch)).astype(np.float32)), "e4m3", keep_nonzero=True)
    px.mx_update(one, g, ck, opt.struct())
    K.batched_update(two, g, px.mx_dequantize(ck), opt.struct())
    _, want, err = _edge_reference(b, g.cpu().numpy(), px.mx_dequantize(ck).cpu().numpy().astype(np.float64), n)
    eg = 2 * err.max()  # between the two gradients
    gmax = np.abs(want).max()
    for name in cols:
        p, q = one[name].cpu().numpy().astype(np.float64), two[name].cpu().numpy().astype(np.float64)
        # a column moves by at most eg times its slope in the gradient (all below 2 + 2 |g| with v >= 0.5, lr <= 0.1)
        # plus a handful of roundings of its own size
        bound = (2 + 2 * gmax) * eg + 8 * _mx.U32 * (np.abs(q) + np.abs(cols[name]) + 1)
        assert (np.abs(p - q) <= bound).all(), name
        dead = (b["dead"] == 1)
        np.testing.assert_array_equal(one[name].cpu().numpy()[dead], cols[name][dead])


# ---------------------------------------------------------------------------
# the product
# ---------------------------------------------------------------------------
def _graph(rng, degrees, num_src, weights, dev):
    """Grouped in-edges with the given in-degrees: the device form and numpy's (weights as held)."""
    deg = np.asarray(degrees)
    off = np.concatenate([[0], deg.cumsum()]).astype(np.int64)
    src = rng.integers(0, num_src, off[-1]).astype(np.int32)
    w = (rng.standard_normal(off[-1]) * np.exp(rng.standard_normal(off[-1]))).astype(np.float32)
    units = rng.permutation(len(deg) + 3)[:len(deg)].astype(np.int32)
    d = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(dev)  # noqa: E731
    if weights == "f32":
        return px.MxConns(d(units), d(off), d(src), "f32", weight=d(w)), off, src, w.astype(np.float64), units
    blk = np.concatenate([[0], ((deg + 31) // 32).cumsum()]).astype(np.int64)
    padded = np.zeros((blk[-1], 32), np.float32)
    for i in range(len(deg)):
        padded.reshape(-1)[blk[i] * 32:blk[i] * 32 + deg[i]] = w[off[i]:off[i + 1]]
    codes, scales = _mx.quantize(padded, weights)
    v = _mx.values(codes, scales, weights, 32)
    held = np.concatenate([v.reshape(-1)[blk[i] * 32:blk[i] * 32 + deg[i]] for i in range(len(deg))] + [np.zeros(0)])
    conns = px.MxConns(d(units), d(off), d(src), weights, block_offsets=d(blk), codes=d(codes),
                       scales=d(scales.reshape(-1)))
    return conns, off, src, held, units


DEGREES = {"ragged": [0, 1, 31, 32, 33, 0, 64, 65, 7, 100], "one": [5], "long": [3000, 0, 2, 9000], "none": [0, 0],
           "many": [12] * 700}


@pytest.mark.parametrize("rows", [*FMTS, "f32"])
@pytest.mark.parametrize("weights", [*FMTS, "f32"])
@pytest.mark.parametrize("degrees,batch", [("ragged", 1), ("ragged", 7), ("ragged", 64), ("ragged", 250), ("one", 3),
                                           ("long", 1), ("long", 33), ("long", 300), ("none", 5), ("many", 16),
                                           ("many", 2), ("many", 128), ("ragged", 520)])
def test_product(cuda, rows, weights, degrees, batch):
    rng = np.random.default_rng(batch + len(degrees))
    num_src = 90
    conns, off, src, w, units = _graph(rng, DEGREES[degrees], num_src, weights, cuda)
    x = _values(rng, num_src, batch).clip(-50, 50)
    if rows == "f32":
        xd, xv = torch.from_numpy(x).to(cuda), x.astype(np.float64)
    else:
        xd = _rows(x, rows, False, cuda)
        xv = _mx.values(xd.codes.cpu().numpy(), xd.scales.cpu().numpy(), rows, batch)
    total = len(units) + 4
    kind = ["identity", "tanh", "relu", "sigmoid"][batch % 4]
    y, err = _mx.product(off, src, w, xv, units, total, kind, num_src)
    left = np.ones(total, bool)
    left[units] = False
    out = torch.full((total, batch), 7.0, device=cuda)
    px.mx_product(conns, xd, activation=kind, out=out)
    got = out.cpu().numpy()
    assert (got[left] == 7).all()
    _within(got[~left], y[~left], err[~left])
    for fmt in FMTS:
        q = px.MxRows.empty(total, batch, fmt, cuda)
        q.codes.fill_(1), q.scales.fill_(2)
        px.mx_product(conns, xd, activation=kind, out=q)
        _same(q, *[np.where(left[:, None], v, r) for v, r in zip((1, 2), _mx.quantize(got, fmt))])


@pytest.mark.parametrize("weights", [*FMTS, "f32"])
@pytest.mark.parametrize("batch", [1, 2, 3, 4, 5, 8, 13, 16, 17])
def test_product_of_many_short_destinations(cuda, weights, batch):
    """Float32 rows of few samples and enough destinations that several share
    a warp (17 samples: the form beside it)."""
    rng = np.random.default_rng(batch)
    degrees = rng.integers(0, 75, 11003)
    degrees[rng.random(degrees.size) < 0.2] = 0
    num_src = 300
    conns, off, src, w, units = _graph(rng, degrees, num_src, weights, cuda)
    src[::97] = -5
    src[50::101] = num_src
    conns.src.copy_(torch.from_numpy(src))
    x = _values(rng, num_src, batch).clip(-50, 50)
    total = len(units) + 4
    kind = ["identity", "tanh", "relu", "sigmoid"][batch % 4]
    y, err = _mx.product(off, src, w, x.astype(np.float64), units, total, kind, num_src)
    left = np.ones(total, bool)
    left[units] = False
    out = torch.full((total, batch), 7.0, device=cuda)
    px.mx_product(conns, torch.from_numpy(x).to(cuda), activation=kind, out=out)
    got = out.cpu().numpy()
    assert (got[left] == 7).all()
    _within(got[~left], y[~left], err[~left])
    for fmt in FMTS:
        q = px.MxRows.empty(total, batch, fmt, cuda)
        q.codes.fill_(1), q.scales.fill_(2)
        px.mx_product(conns, torch.from_numpy(x).to(cuda), activation=kind, out=q)
        _same(q, *[np.where(left[:, None], v, r) for v, r in zip((1, 2), _mx.quantize(got, fmt))])


def test_rows_past_four_gigabytes(cuda):
    """Row offsets that do not fit 32 bits: the last rows of float32 rows and of
    8-bit rows that end past 4 GiB, through every operator that indexes rows."""
    rng = np.random.default_rng(2)
    batch, n = 1024, (1 << 20) + 4096  # 4.3 GB of float32
    pick = np.array([0, 5, n - 2, n - 1])
    few = rng.standard_normal((4, batch)).astype(np.float32)
    x = torch.zeros((n, batch), device=cuda)
    ids = torch.from_numpy(pick).to(cuda)
    x[ids] = torch.from_numpy(few).to(cuda)
    conns = px.MxConns(torch.tensor([n - 3, 1], dtype=torch.int32, device=cuda), torch.tensor([0, 3, 4], device=cuda),
                       torch.tensor([5, n - 1, n - 2, n - 1], dtype=torch.int32, device=cuda), "f32",
                       weight=torch.tensor([1.0, 2.0, -0.5, 3.0], device=cuda))
    px.mx_product(conns, x, out=x)  # no destination is a source
    want = few[1].astype(np.float64) + 2.0 * few[3] - 0.5 * few[2]
    got = x[torch.tensor([n - 3, 1], device=cuda)].cpu().numpy()
    bound = 5 * _mx.U32 * (np.abs(few[1]) + 2 * np.abs(few[3]) + np.abs(few[2]))
    assert (np.abs(got[0] - want) <= bound).all() and np.array_equal(got[1], np.float32(3.0) * few[3])
    # quantised rows and their gradient
    ck = px.mx_quantize(x, "e4m3", keep_nonzero=True)
    codes, scales = _mx.quantize(few, "e4m3", True)
    np.testing.assert_array_equal(ck.codes[ids].cpu().numpy(), codes)
    np.testing.assert_array_equal(ck.scales[ids].cpu().numpy(), scales)
    a = _mx.values(codes, scales, "e4m3", batch)
    f, t = np.array([0, 3, 2, 1, 3]), np.array([3, 2, 3, 0, 0])
    bucket = {"from_id": torch.from_numpy(pick[f].astype(np.int32)).to(cuda),
              "to_id": torch.from_numpy(pick[t].astype(np.int32)).to(cuda),
              "dead": torch.zeros(5, dtype=torch.uint8, device=cuda)}
    out = px.mx_edge_grad(bucket, x, ck).cpu().numpy()
    prod = few[t].astype(np.float64) * a[f]
    assert (np.abs(out - prod.sum(1) / batch) <= (batch + 4) * _mx.U32 * np.abs(prod).sum(1) / batch).all()
    g = px.mx_unit_grad(x, ck, "tanh", out=x)[ids].cpu().numpy()
    up = few.astype(np.float64)
    assert (np.abs(g - up * (1 - a * a)) <= 4 * _mx.U32 * np.abs(up) * (1 + a * a)).all()
    back = px.mx_dequantize(ck)
    np.testing.assert_array_equal(back[ids].cpu().numpy(), a.astype(np.float32))
    del x, ck, back
    # few samples: the codes (a whole block a unit) pass 4 GiB long before the gradients do
    n = (1 << 27) + 64
    g = torch.zeros((n, 4), device=cuda)
    rows = px.MxRows.empty(n, 4, "e4m3", cuda, zero=True)
    ids = torch.tensor([n - 1, 3, n - 33, 64], device=cuda)
    px.mx_quantize(torch.from_numpy(few[:, :4].copy()).to(cuda), "e4m3", ids=ids, out=rows)
    g[ids] = torch.from_numpy(few[:, 4:8].copy()).to(cuda)
    a4 = _mx.values(*_mx.quantize(few[:, :4], "e4m3"), "e4m3", 4)
    bucket = {"from_id": ids.to(torch.int32), "to_id": ids.flip(0).to(torch.int32),
              "dead": torch.zeros(4, dtype=torch.uint8, device=cuda)}
    prod = few[::-1, 4:8].astype(np.float64) * a4
    out = px.mx_edge_grad(bucket, g, rows).cpu().numpy()
    assert (np.abs(out - prod.sum(1) / 4) <= 8 * _mx.U32 * np.abs(prod).sum(1) / 4).all()
    del g, rows
    # 8-bit rows past 4 GiB
    n = (1 << 22) + 4096
    rows = px.MxRows.empty(n, batch, "e4m3", cuda, zero=True)
    ids = torch.tensor([n - 1, n - 2, 0, 7], device=cuda)
    px.mx_quantize(torch.from_numpy(few).to(cuda), "e4m3", keep_nonzero=True, ids=ids, out=rows)
    np.testing.assert_array_equal(rows.codes[ids].cpu().numpy(), codes)
    conns = px.MxConns(torch.tensor([0], dtype=torch.int32, device=cuda), torch.tensor([0, 2], device=cuda),
                       torch.tensor([n - 1, n - 2], dtype=torch.int32, device=cuda), "f32",
                       weight=torch.tensor([1.5, -1.0], device=cuda))
    out = px.mx_product(conns, rows, out=torch.zeros((1, batch), device=cuda)).cpu().numpy()[0]
    assert (np.abs(out - (1.5 * a[0] - a[1])) <= 4 * _mx.U32 * (1.5 * np.abs(a[0]) + np.abs(a[1]))).all()


def test_product_skips_what_is_out_of_range(cuda):
    rng = np.random.default_rng(1)
    conns, off, src, w, units = _graph(rng, [10, 40, 3], 20, "e2m1", cuda)
    src = src.copy()
    src[[0, 12, 51]] = [-1, 20, 1 << 30]
    units = units.copy()
    units[1] = 99
    x = rng.standard_normal((20, 6)).astype(np.float32)
    bad = px.MxConns(torch.from_numpy(units).to(cuda), conns.offsets, torch.from_numpy(src).to(cuda), "e2m1",
                     block_offsets=conns.block_offsets, codes=conns.codes, scales=conns.scales)
    out = torch.full((8, 6), 3.0, device=cuda)
    px.mx_product(bad, torch.from_numpy(x).to(cuda), out=out)
    y, err = _mx.product(off, src, w, x.astype(np.float64), units, 8, "identity", 20)
    on = np.isin(np.arange(8), units)
    _within(out.cpu().numpy()[on], y[on], err[on])
    assert (out.cpu().numpy()[~on] == 3).all()
    # offsets past the arrays read nothing beyond them
    wild = px.MxConns(conns.units, torch.tensor([-7, 40, 1 << 40, 1 << 41], device=cuda), conns.src, "e2m1",
                      block_offsets=torch.tensor([-3, 1 << 20, 1 << 41, 1 << 50], device=cuda), codes=conns.codes,
                      scales=conns.scales)
    assert torch.isfinite(px.mx_product(wild, torch.from_numpy(x).to(cuda))).all()
    # new rows elsewhere are zero
    new = px.mx_product(conns, torch.from_numpy(x).to(cuda)).cpu().numpy()
    assert new.shape == (20, 6) and not new[~np.isin(np.arange(20), conns.units.cpu().numpy())].any()


def test_product_poisoned_rows_reach_only_their_edges(cuda):
    rng = np.random.default_rng(6)
    conns, off, src, w, units = _graph(rng, [4, 4, 4, 4], 16, "f32", cuda)
    x = rng.standard_normal((16, 64)).astype(np.float32)
    x[src[0], 33] = np.nan
    hit = np.array([(src[off[i]:off[i + 1]] == src[0]).any() for i in range(4)])
    for xd, first in ((torch.from_numpy(x).to(cuda), 33), (px.mx_quantize(torch.from_numpy(x).to(cuda), "e4m3"), 32)):
        out = px.mx_product(conns, xd).cpu().numpy()[units[units < 16]]
        bad = np.isnan(out)
        assert bad[hit[units < 16], 33].all() and not bad[:, :first].any() and not bad[~hit[units < 16]].any()


# ---------------------------------------------------------------------------
# the paths that use them
# ---------------------------------------------------------------------------
def _mlp_net(widths, density, rng, hidden="relu", opt=None, batch_loss=None, out="identity"):
    offsets = np.concatenate([[0], np.cumsum(widths)])
    frm, to = [], []
    for layer in range(len(widths) - 1):
        s, d = np.meshgrid(np.arange(offsets[layer], offsets[layer + 1]),
                           np.arange(offsets[layer + 1], offsets[layer + 2]), indexing="ij")
        keep = rng.random(s.shape) < density
        frm.append(s[keep]), to.append(d[keep])
    # a few edges that skip a level
    frm.append(np.arange(offsets[0], offsets[0] + 5)), to.append(np.arange(offsets[2], offsets[2] + 5))
    frm, to = np.concatenate(frm).astype(np.int32), np.concatenate(to).astype(np.int32)
    w = (rng.standard_normal(frm.size) * 0.3).astype(np.float32)

    class Net(px.Network):
        forward_pass = px.ForwardPass(hidden, output_activation=out)
        backward_pass = px.BackwardPass(hidden)
        loss = batch_loss or px.MSELoss()
        update_conn = opt or px.optim.sgd(0.05)
        batch_reduction = px.MeanFloatFirstRest()
        propagation = px.Propagation.TOPOLOGICAL

    n = int(offsets[-1])
    return Net, n, frm, to, w, list(range(widths[0])), list(range(int(offsets[-2]), n))


def _topological(level, frm, to, w, x, inputs, outputs, hidden, out_act):
    """Rows and error bounds of a layered forward in 64 bits, edges into
    deeper units only (slope of each activation at most 1)."""
    n = level.size
    y, err = np.zeros((n, x.shape[1])), np.zeros((n, x.shape[1]))
    y[inputs] = x
    is_out = np.isin(np.arange(n), outputs)
    for lv in range(1, int(level.max()) + 1):
        for u in np.nonzero(level == lv)[0]:
            e = to == u
            t = w[e, None] * y[frm[e]]
            s = np.abs(t).sum(0)
            y[u] = _mx.act(out_act if is_out[u] else hidden, t.sum(0))
            err[u] = ((e.sum() + 2) * _mx.U32 * s + (np.abs(w[e])[:, None] * err[frm[e]]).sum(0)) * 1.01 \
                + 8 * _mx.U32 * np.abs(y[u])
    return y, err


@pytest.mark.parametrize("fmt", mx.CHECKPOINT_FORMATS)
@pytest.mark.parametrize("hidden,opt_kind,loss", [("relu", "sgd", "mse"), ("tanh", "adam", "softmax"),
                                                  ("sigmoid", "momentum", "mse")])
@pytest.mark.parametrize("batch", [8, 36])
def test_checkpointed_step(cuda, fmt, hidden, opt_kind, loss, batch):
    """Two steps: the forward, the loss and the checkpoint's codes against the
    float32 step on the same state; the backward and the update against a
    restatement in 64 bits that reads the step's own checkpoint."""
    rng = np.random.default_rng(batch)
    opt = {"sgd": px.optim.sgd(0.05), "adam": px.optim.adam(0.01), "momentum": px.optim.momentum(0.05)}[opt_kind]
    net, n, frm, to, w, inputs, outputs = _mlp_net(
        [24, 40, 33, 10], 0.4, rng, hidden, opt, px.SoftmaxCrossEntropyLoss() if loss == "softmax" else px.MSELoss())
    built = [px.NetworkBuilder.from_edges(net, n, frm, to, weights=w, input_ids=inputs, output_ids=outputs,
                                          capacity_headroom=0.1, device=cuda) for _ in range(2)]
    (static, state), (_, ref_state) = built
    step = px.make_step(net, static, batch_size=batch, device=cuda, activation_checkpoint=fmt)
    ref = px.make_step(net, static, batch_size=batch, device=cuda)
    level = state.units["level"].cpu().numpy()
    is_out = np.isin(np.arange(n), outputs)
    for it in range(2):
        host = [{k: v.cpu().numpy().copy() for k, v in b.items()} for b in state.conns]
        for mine, theirs in zip(state.conns, ref_state.conns):  # the reference starts from this step's state
            for k in mine:
                theirs[k].copy_(mine[k])
        x = rng.standard_normal((batch, len(inputs))).astype(np.float32)
        t = rng.standard_normal((batch, len(outputs))).astype(np.float32)
        if loss == "softmax":
            t = np.eye(len(outputs), dtype=np.float32)[rng.integers(0, len(outputs), batch)]
        res = step(state, px.StepInputs(x, t))
        want = ref(ref_state, px.StepInputs(x, t))
        # both forwards sum the same float32 products in whatever order: the repository's bar for an activation
        np.testing.assert_allclose(float(res.loss), float(want.loss), rtol=1e-5, atol=1e-6)
        np.testing.assert_allclose(state.units["activation"].cpu().numpy(), ref_state.units["activation"].cpu().numpy(),
                                   rtol=1e-5, atol=1e-6)
        a32 = ref.act_b.cpu().numpy()
        a = px.mx_dequantize(step.checkpoint).cpu().numpy().astype(np.float64)
        assert (np.abs(a - a32) <= 2 * _mx.half_step(a32, np.abs(a32) * 1e-5 + 1e-6, fmt) + np.abs(a32) * 1e-5 + 1e-6
                ).all()  # one whole step: keep_nonzero may round up from next to 0
        np.testing.assert_array_equal(np.sign(a)[a32 != 0], np.sign(a32)[a32 != 0])
        # the backward from the checkpoint, and a bound that carries each row's error down
        seed = step.seed_b.cpu().numpy().astype(np.float64)
        grad, err = np.zeros((n, batch)), np.zeros((n, batch))
        prime = np.where(is_out[:, None], 1.0, _mx.act_prime(hidden, a)) if hidden != "relu" else \
            np.where(is_out[:, None], 1.0, (a > 0).astype(float))
        for lv in range(int(level.max()), 0, -1):
            for u in np.nonzero(level == lv)[0]:
                s, sa, se, cnt = seed[u].copy(), np.abs(seed[u]), np.zeros(batch), 0
                for b in host:
                    e = (b["from_id"] == u) & (b["dead"] == 0)
                    tw = b["weight"][e].astype(np.float64)[:, None]
                    s += (tw * grad[b["to_id"][e]]).sum(0)
                    sa += np.abs(tw * grad[b["to_id"][e]]).sum(0)
                    se += (np.abs(tw) * err[b["to_id"][e]]).sum(0)
                    cnt += int(e.sum())
                grad[u] = s * prime[u]
                slope = np.abs(prime[u]) + 4 * _mx.U32 * (1 + a[u] ** 2)
                err[u] = ((cnt + 4) * _mx.U32 * sa + se) * slope * 1.01 + 4 * _mx.U32 * np.abs(s) * (1 + a[u] ** 2)
        _within(step.grad_b.cpu().numpy(), grad, err)
        for b, h in zip(state.conns, host):
            live = h["dead"] == 0
            f, to_ = h["from_id"][live], h["to_id"][live]
            g = (grad[to_] * a[f]).sum(1) / batch
            eg = ((err[to_] * np.abs(a[f])).sum(1) + (batch + 4) * _mx.U32 * np.abs(grad[to_] * a[f]).sum(1)) / batch
            w0 = h["weight"][live].astype(np.float64)
            if opt_kind == "sgd":
                w1, slope = w0 - opt.lr * g, opt.lr
            elif opt_kind == "momentum":
                v = opt.b1 * h["opt/v"][live].astype(np.float64) + g
                w1, slope = w0 - opt.lr * v, opt.lr
            else:
                t_ = h["opt/t"][live] + 1.0
                m = opt.b1 * h["opt/m"][live] + (1 - opt.b1) * g
                v = opt.b2 * h["opt/v"][live] + (1 - opt.b2) * g * g
                mh, vh = m / (1 - opt.b1 ** t_), v / (1 - opt.b2 ** t_)
                w1 = w0 - opt.lr * mh / (np.sqrt(vh) + opt.eps)
                # d/dg of the direction: at most 2 / (sqrt(vh) + eps); the betas' float32 forms move it by 1e-5 of lr
                slope = 2 * opt.lr / (np.sqrt(vh) + opt.eps)
            got = b["weight"].cpu().numpy()[live]
            bound = np.minimum(slope * eg, 2 * opt.lr) * 1.01 + 4 * _mx.U32 * (np.abs(w0) + np.abs(w1)) + \
                opt.lr * (np.abs(g) * 4 * _mx.U32 if opt_kind != "adam" else 2e-5)
            assert (np.abs(got - w1) <= bound).all(), f"step {it}"
            np.testing.assert_array_equal(b["dead"].cpu().numpy(), h["dead"])


def test_checkpointed_step_holds_fewer_bytes_and_refuses_other_edges(cuda):
    rng = np.random.default_rng(0)
    net, n, frm, to, w, inputs, outputs = _mlp_net([64, 512, 512, 10], 0.05, rng)
    static, state = px.NetworkBuilder.from_edges(net, n, frm, to, weights=w, input_ids=inputs, output_ids=outputs,
                                                 device=cuda)
    step = px.make_step(net, static, batch_size=1024, device=cuda, activation_checkpoint="e4m3")
    plain = px.make_step(net, static, batch_size=1024, device=cuda)

    def held(fn):
        rows = {t.data_ptr(): t.numel() * t.element_size() for t in (fn.acc_b, fn.act_b, fn.grad_b, fn.seed_b)}
        ck = fn.checkpoint
        return sum(rows.values()) + (0 if ck is None else ck.codes.numel() + ck.scales.numel())

    assert held(plain) == 16 * n * 1024 and held(step) == (8 * 1024 + 33 * 32) * n
    x, t = rng.standard_normal((1024, 64)).astype(np.float32), rng.standard_normal((1024, 10)).astype(np.float32)
    step(state, px.StepInputs(x, t))
    # an edge that does not go deeper (an edge into an input): refused, nothing was run
    frm2, to2 = np.append(frm, 64).astype(np.int32), np.append(to, 3).astype(np.int32)
    static, state = px.NetworkBuilder.from_edges(net, n, frm2[frm2 < 64], to2[frm2 < 64], input_ids=inputs,
                                                 output_ids=outputs, device=cuda)
    state.conns[0]["to_id"][0] = 3
    bad = px.make_step(net, static, batch_size=1024, device=cuda, activation_checkpoint="e4m3")
    with pytest.raises(ValueError, match="deeper"):
        bad(state, px.StepInputs(x, t))


@pytest.mark.parametrize("weights", [*FMTS, "f32"])
@pytest.mark.parametrize("rows", ["f32", "e4m3", "e2m1"])
@pytest.mark.parametrize("batch", [1, 5, 64])
def test_infer(cuda, weights, rows, batch):
    rng = np.random.default_rng(batch)
    net, n, frm, to, w, inputs, outputs = _mlp_net([24, 40, 33, 10], 0.4, rng, "tanh")
    outputs = [*outputs, 30, 2]  # an output that also feeds others, and an input that is an output
    static, state = px.NetworkBuilder.from_edges(net, n, frm, to, weights=w, input_ids=inputs, output_ids=outputs,
                                                 capacity_headroom=0.2, device=cuda)
    infer = px.make_infer(net, static, state, weights=weights, rows=rows)
    x = rng.standard_normal((batch, len(inputs))).astype(np.float32)
    got = infer(x)
    assert tuple(got.shape) == (batch, len(outputs)) and got.dtype == torch.float32
    got = got.cpu().numpy().T
    level = state.units["level"].cpu().numpy()
    # the weights as held: blocks of 32 in-edges of a unit, in slot order
    hw = w.astype(np.float64)
    order = np.concatenate([b["from_id"].cpu().numpy()[b["dead"].cpu().numpy() == 0].astype(np.int64) * n +
                            b["to_id"].cpu().numpy()[b["dead"].cpu().numpy() == 0] for b in state.conns])
    where = {k: i for i, k in enumerate(frm.astype(np.int64) * n + to)}
    slots = np.array([where[k] for k in order])
    frm, to, hw = frm[slots], to[slots], hw[slots]
    if weights != "f32":
        for u in range(n):
            e = np.nonzero(to == u)[0]
            if len(e):
                q = _mx.quantize(hw[e][None].astype(np.float32), weights)
                hw[e] = _mx.values(*q, weights, len(e))[0]
    if rows == "f32":
        y, err = _topological(level, frm, to, hw, x.T.astype(np.float64), inputs, outputs, "tanh", "identity")
        _within(got, y[outputs], err[outputs] + np.where(np.isin(outputs, inputs), 0, 1e-30)[:, None])
        if weights == "f32":  # and the training step's forward
            step = px.make_step(net, static, batch_size=64, device=cuda)
            full = np.zeros((64, len(inputs)), np.float32)
            full[:batch] = x
            step(state, px.StepInputs(full, np.zeros((64, len(outputs)), np.float32)))
            np.testing.assert_allclose(got, step.act_b.cpu().numpy()[outputs][:, :batch], rtol=1e-5, atol=1e-6)
        return
    # quantised rows: a walk that quantises each level's rows; a value next to a border may go either way, so every
    # difference it can make is carried: half a step of every source in both walks
    def walk():
        y, err = np.zeros((n, batch)), np.zeros((n, batch))
        y[inputs] = _mx.values(*_mx.quantize(x.T, rows), rows, batch)
        exact = np.zeros((n, batch))
        exact[inputs] = x.T
        for lv in range(1, int(level.max()) + 1):
            for u in np.nonzero(level == lv)[0]:
                e = to == u
                tt = hw[e, None] * y[frm[e]]
                z = _mx.act("identity" if u in outputs else "tanh", tt.sum(0))
                er = ((e.sum() + 2) * _mx.U32 * np.abs(tt).sum(0) + (np.abs(hw[e])[:, None] * err[frm[e]]).sum(0)) * 1.01 \
                    + 8 * _mx.U32 * np.abs(z)
                exact[u], err[u] = z, er
                if u in frm:  # its rows: the device may stand one step beside where the error reaches a border
                    lo = _mx.values(*_mx.quantize((z - er)[None].astype(np.float32), rows), rows, batch)[0]
                    hi = _mx.values(*_mx.quantize((z + er)[None].astype(np.float32), rows), rows, batch)[0]
                    y[u] = _mx.values(*_mx.quantize(z[None].astype(np.float32), rows), rows, batch)[0]
                    flip = np.maximum(np.abs(lo - y[u]), np.abs(hi - y[u]))
                    out_err = er.copy()
                    err[u] = flip
                    exact_err[u] = out_err
                else:
                    exact_err[u] = er
        return exact

    exact_err = np.zeros((n, batch))
    exact = walk()
    _within(got, exact[outputs], exact_err[outputs] + 1e-30)


def test_infer_of_a_pruned_net(cuda):
    """Units left without in-edges (sigmoid of 0, not 0), sources without any
    (level 0, not an input), and outputs nothing reaches: as the training
    step's forward."""
    rng = np.random.default_rng(77)
    net, n, frm, to, w, inputs, outputs = _mlp_net([16, 30, 20, 6], 0.4, rng, "sigmoid")
    frm, to = np.append(frm, n).astype(np.int32), np.append(to, 50).astype(np.int32)  # a source that is no input
    w = np.append(w, np.float32(0.7))
    static, state = px.NetworkBuilder.from_edges(net, n + 2, frm, to, weights=w, input_ids=inputs,
                                                 output_ids=[*outputs, n + 1], device=cuda)
    for b in state.conns:
        kill = torch.from_numpy(rng.random(b["dead"].numel()) < 0.7).to(cuda) | (b["to_id"] == outputs[0])
        b["dead"][kill] = 1
    x = rng.standard_normal((8, len(inputs))).astype(np.float32)
    got = px.make_infer(net, static, state, weights="f32")(x).cpu().numpy().T
    step = px.make_step(net, static, batch_size=8, device=cuda)
    step(state, px.StepInputs(x, np.zeros((8, len(outputs) + 1), np.float32)))
    np.testing.assert_allclose(got, step.act_b.cpu().numpy()[[*outputs, n + 1]], rtol=1e-5, atol=1e-6)
    assert not got[0].any() and not got[-1].any()  # identity outputs of nothing


def test_captured_and_replayed(cuda):
    """Each operator captured once and replayed on new values in the same
    buffers, two graphs of the same inference sharing nothing."""
    rng = np.random.default_rng(3)
    net, n, frm, to, w, inputs, outputs = _mlp_net([24, 40, 33, 10], 0.4, rng)
    static, state = px.NetworkBuilder.from_edges(net, n, frm, to, weights=w, input_ids=inputs, output_ids=outputs,
                                                 device=cuda)
    infer = px.make_infer(net, static, state, weights="e2m1", rows="e4m3")
    bucket = state.conns[0]
    x = torch.zeros((32, 24), device=cuda)
    g = torch.randn((n, 32), device=cuda)
    act = torch.randn((n, 32), device=cuda)

    def run():
        ck = px.mx_quantize(act, "e4m3", keep_nonzero=True)
        return infer(x), px.mx_edge_grad(bucket, g, ck), px.mx_unit_grad(g, ck, "tanh"), px.mx_dequantize(ck)

    run()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = run()
        graphs.append((graph, outs))
    for _ in range(3):
        x.copy_(torch.randn_like(x)), g.copy_(torch.randn_like(g)), act.copy_(torch.randn_like(act))
        for graph, _ in graphs:
            graph.replay()
        want = run()
        for _, outs in graphs:
            for a, b in zip(outs, want):
                assert torch.equal(a, b)


def test_checkpointed_step_captured(cuda):
    """A captured step replays as the eager one: the same state after each."""
    rng = np.random.default_rng(31)
    net, n, frm, to, w, inputs, outputs = _mlp_net([24, 64, 48, 10], 0.3, rng)
    pair = [px.NetworkBuilder.from_edges(net, n, frm, to, weights=w, input_ids=inputs, output_ids=outputs, device=cuda)
            for _ in range(2)]
    steps = [px.make_step(net, static, batch_size=32, device=cuda, activation_checkpoint="e5m2") for static, _ in pair]
    x, t = torch.zeros((32, 24), device=cuda), torch.zeros((32, 10), device=cuda)
    run = lambda i: steps[i](pair[i][1], px.StepInputs(x, t))  # noqa: E731
    run(0), run(1)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = run(0)
    for _ in range(4):
        x.copy_(torch.randn_like(x)), t.copy_(torch.randn_like(t))
        graph.replay()
        want = run(1)
        # the two forwards and backwards add the same float32 products with atomics: the repository's bar
        torch.testing.assert_close(res.loss, want.loss, rtol=1e-5, atol=1e-6)
        for a, b in zip(pair[0][1].conns, pair[1][1].conns):
            # an activation next to a border of e5m2 may round either way: half a step (2^-3) of one sample's share
            torch.testing.assert_close(a["weight"], b["weight"], rtol=1e-3, atol=1e-4)


def test_two_streams_at_once(cuda):
    rng = np.random.default_rng(3)
    net, n, frm, to, w, inputs, outputs = _mlp_net([64, 400, 300, 10], 0.2, rng)
    static, state = px.NetworkBuilder.from_edges(net, n, frm, to, weights=w, input_ids=inputs, output_ids=outputs,
                                                 device=cuda)
    infer = px.make_infer(net, static, state, weights="e2m1", rows="e2m1")
    xs = [torch.randn((200, 64), device=cuda) for _ in range(2)]
    want = [infer(x).clone() for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(infer(xs[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, want[i]) for o in got[i])


def test_train_then_answer(cuda):
    """The operators together, as they are used: checkpointed training steps
    on a growing net, then answers from 4-bit weights on the grown arena."""
    rng = np.random.default_rng(12)
    net, n, frm, to, w, inputs, outputs = _mlp_net([24, 64, 48, 10], 0.3, rng)
    net.add_conn = None

    class Grown(px.Network):
        forward_pass = px.ForwardPass("relu", output_activation="identity")
        backward_pass = px.BackwardPass("relu")
        loss = px.MSELoss()
        update_conn = px.optim.sgd(0.02)
        batch_reduction = px.MeanFloatFirstRest()
        propagation = px.Propagation.TOPOLOGICAL
        prune_conn = px.MagnitudePrune(0.02)
        add_conn = px.ProposeAddConn(proposals_per_proposer=2, max_new_per_level=20, direction="deeper",
                                     max_level_gap=2, init=("hash_uniform", 0.1))

    static, state = px.NetworkBuilder.from_edges(Grown, n, frm, to, weights=w, input_ids=inputs, output_ids=outputs,
                                                 capacity_headroom=0.5, device=cuda)
    step = px.make_step(Grown, static, batch_size=64, device=cuda, activation_checkpoint="e4m3")
    before = px.live_conn_count(state)
    teacher = rng.standard_normal((24, 10)).astype(np.float32) * 0.2
    for _ in range(5):
        x = rng.standard_normal((64, 24)).astype(np.float32)
        res = step(state, px.StepInputs(x, x @ teacher))
        assert np.isfinite(float(res.loss))
    assert px.live_conn_count(state) != before
    x = rng.standard_normal((7, 24)).astype(np.float32)
    full = np.zeros((64, 24), np.float32)
    full[:7] = x
    exact = px.make_infer(Grown, static, state, weights="f32")(x).cpu().numpy()
    four = px.make_infer(Grown, static, state)(x).cpu().numpy()
    ref = px.make_step(Grown, static, batch_size=64, device=cuda)
    ref(state, px.StepInputs(full, np.zeros((64, 10), np.float32)))
    # the restated step's own forward on the same arena (its growth ran after it)
    np.testing.assert_allclose(exact, ref.act_b.cpu().numpy()[outputs][:, :7].T, rtol=1e-5, atol=1e-6)
    assert four.shape == exact.shape and np.isfinite(four).all()


def test_reads_the_struct_of_the_call(cuda):
    """A conns struct outlives the call only through its tensors."""
    rng = np.random.default_rng(1)
    conns, off, src, w, units = _graph(rng, [3, 4], 9, "f32", cuda)
    assert ctypes.sizeof(conns._c) == 80
    x = torch.ones((9, 2), device=cuda)
    a = px.mx_product(conns, x)
    b = px.mx_product(px.MxConns(conns.units, conns.offsets, conns.src, "f32", weight=conns.weight), x)
    assert torch.equal(a, b)


def _levels_net(**kw):
    class Net(px.Network):
        forward_pass = px.ForwardPass(kw.get("hidden", "identity"), output_activation="identity")
        backward_pass = px.BackwardPass(kw.get("hidden", "identity"))
        loss = px.MSELoss()
        update_conn = px.optim.sgd(0.5)
        batch_reduction = px.MeanFloatFirstRest()
        propagation = px.Propagation.TOPOLOGICAL

    return Net


def _built_from(net, n, edges, outputs, dev):
    frm, to, w = zip(*edges)
    return px.NetworkBuilder.from_edges(net, n, list(frm), list(to), weights=list(w), input_ids=(0, 1),
                                        output_ids=outputs, device=dev)


@pytest.mark.parametrize("fmt", mx.CHECKPOINT_FORMATS)
def test_checkpoint_keeps_nothing_of_another_state(cuda, fmt):
    """Two states of one static, a unit at level 1 in the first and at level 0
    (without in-edges) in the second: its activation is 0 there, and its
    out-edges' gradient with it."""
    net = _levels_net()
    first = [(0, 2, 1.0), (1, 3, 1.0), (2, 4, 2.0), (3, 4, 1.0)]
    second = [(1, 3, 1.0), (2, 4, 2.0), (3, 4, 1.0)]
    static, a = _built_from(net, 5, first, (4,), cuda)
    static_b, b = _built_from(net, 5, second, (4,), cuda)
    _, fresh = _built_from(net, 5, second, (4,), cuda)
    assert static == static_b
    x, t = np.full((8, 2), 3.0, np.float32), np.zeros((8, 1), np.float32)
    step = px.make_step(net, static, batch_size=8, device=cuda, activation_checkpoint=fmt)
    step(a, px.StepInputs(x, t))
    step(b, px.StepInputs(x, t))
    px.make_step(net, static, batch_size=8, device=cuda, activation_checkpoint=fmt)(fresh, px.StepInputs(x, t))
    for mine, want in zip(b.conns, fresh.conns):
        assert torch.equal(mine["weight"], want["weight"])
    still = (b.conns[0]["from_id"] == 2) & (b.conns[0]["dead"] == 0)
    assert b.conns[0]["weight"][still].tolist() == [2.0]
    assert not px.mx_dequantize(step.checkpoint)[2].any()


@pytest.mark.parametrize("rows", ["f32", "e4m3", "e2m1"])
@pytest.mark.parametrize("batched", [False, True])
def test_infer_of_units_that_no_level_applies(cuda, rows, batched):
    """A level-0 unit that is no input keeps the activation its state holds in
    the streaming step and reads 0 in the batched one; so does an output."""
    class Net(px.Network):
        forward_pass = px.ForwardPass("identity")
        propagation = px.Propagation.TOPOLOGICAL
        batch_reduction = px.MeanFloatFirstRest() if batched else None

    static, state = _built_from(Net, 6, [(0, 2, 2.0), (3, 2, 4.0), (2, 4, 1.0), (3, 4, -1.0)], (4, 5, 3), cuda)
    state.units["activation"][3] = 0.5
    state.units["activation"][5] = 0.25
    infer = px.make_infer(Net, static, state, weights="f32", rows=rows)
    for x in ([1.0, 2.0], [-3.0, 0.0]):
        got = infer(np.array([x] * (8 if batched else 1), np.float32)).cpu().numpy()
        if batched:
            step = px.make_step(Net, static, batch_size=8, device=cuda)
            step(state, px.StepInputs(np.array([x] * 8, np.float32)))
            want = step.act_b.cpu().numpy()[[4, 5, 3]].T
        else:
            px.make_step(Net, static, device=cuda)(state, px.StepInputs(np.array(x, np.float32)))
            want = state.units["activation"].cpu().numpy()[[4, 5, 3]][None]
        np.testing.assert_array_equal(got, want)  # few bits: every sum is exact


def test_checkpointed_step_knows_its_states(cuda):
    """Training on two states in turn, with growth and prune, looks at neither
    again (a capture could not); an edit in place is seen."""
    rng = np.random.default_rng(21)
    net, n, frm, to, w, inputs, outputs = _mlp_net([24, 64, 48, 10], 0.3, rng)

    class Grown(net):
        prune_conn = px.MagnitudePrune(0.02)
        add_conn = px.ProposeAddConn(proposals_per_proposer=2, max_new_per_level=20, direction="deeper",
                                     max_level_gap=2, init=("hash_uniform", 0.1))

    built = [px.NetworkBuilder.from_edges(Grown, n, frm, to, weights=w, input_ids=inputs, output_ids=outputs,
                                          capacity_headroom=0.5, device=cuda) for _ in range(2)]
    static, states = built[0][0], [s for _, s in built]
    step = px.make_step(Grown, static, batch_size=32, device=cuda, activation_checkpoint="e4m3")
    x, t = torch.randn((32, 24), device=cuda), torch.randn((32, 10), device=cuda)
    for _ in range(3):
        for s in states:
            step(s, px.StepInputs(x, t))
    known = dict(step._checked)
    for s in states:
        step(s, px.StepInputs(x, t))
    assert step._checked == known and len(known) == 2
    graph = torch.cuda.CUDAGraph()
    fixed = px.make_step(net, static, batch_size=32, device=cuda, activation_checkpoint="e4m3")
    fixed(states[0], px.StepInputs(x, t)), fixed(states[1], px.StepInputs(x, t))
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        fixed(states[0], px.StepInputs(x, t))  # not the state seen last
    graph.replay()
    torch.cuda.synchronize()
    states[0].units["level"][outputs[0]] = 1
    with pytest.raises(ValueError, match="deeper"):
        step(states[0], px.StepInputs(x, t))


@pytest.mark.parametrize("fmt", mx.CHECKPOINT_FORMATS)
def test_edge_grad_of_the_largest_gradients(cuda, fmt):
    """Gradients up to float32's largest against small activations, slot by
    slot and as one product: sums that float32 holds stay finite."""
    rng = np.random.default_rng(11)
    n, batch = 70, 256
    g = (rng.standard_normal((n, batch)) * np.exp2(rng.integers(-40, 90, (n, 1)))).astype(np.float32)
    big = np.finfo(np.float32).max
    g[::3, ::7] = big * rng.choice([1.0, -1.0, 1 - 2.0 ** -9, 1 - 2.0 ** -16], g[::3, ::7].shape)
    x = (rng.standard_normal((n, batch)) * 2.0 ** -12).astype(np.float32)
    x[:, 5:9] = 0.0
    ck = _rows(x, fmt, True, cuda)
    a = _mx.values(ck.codes.cpu().numpy(), ck.scales.cpu().numpy(), fmt, batch)
    for cap in (1000, 1 << 18):
        assert (mx.edge_grad_scratch_bytes(cap, batch, n) > 0) == (cap > 1000)
        f, t = rng.integers(0, n, cap).astype(np.int32), rng.integers(0, n, cap).astype(np.int32)
        dev = {"from_id": torch.from_numpy(f).to(cuda), "to_id": torch.from_numpy(t).to(cuda),
               "dead": torch.zeros(cap, dtype=torch.uint8, device=cuda)}
        pairs, size = g.astype(np.float64) @ a.T / batch, np.abs(g).astype(np.float64) @ np.abs(a).T / batch
        got = px.mx_edge_grad(dev, torch.from_numpy(g).to(cuda), ck).cpu().numpy()
        _within(got, pairs[t, f], size[t, f] * (batch + 4) * _mx.U32 * 1.01, f"{cap} slots")


@pytest.mark.parametrize("rows", FMTS)
@pytest.mark.parametrize("weights", ["e2m1", "f32"])
@pytest.mark.parametrize("degrees,batch", [("one", 7), ("one", 20), ("ragged", 33), ("ragged", 64), ("ragged", 100),
                                           ("long", 250), ("single", 20), ("single", 300)])
def test_product_of_large_rows_and_weights(cuda, rows, weights, degrees, batch):
    """Weights whose product with a block's scale passes float32's range: every
    sample whose own products stay in it is as in float32, a 0 among them."""
    rng = np.random.default_rng(batch)
    num_src = 12
    degrees = {**DEGREES, "single": [1] * 40}[degrees]
    conns, off, src, w, units = _graph(rng, degrees, num_src, "f32", cuda)
    w = (np.sign(w) * np.exp2(rng.integers(-20, 40, w.size)) * rng.choice([1.0, 1.5], w.size)).astype(np.float32)
    w[0] = 1.5 * 2.0 ** 39
    if weights == "f32":
        conns = px.MxConns(conns.units, conns.offsets, conns.src, "f32", weight=torch.from_numpy(w).to(cuda))
    else:
        deg = np.asarray(degrees)
        dst = torch.from_numpy(np.repeat(np.arange(deg.size), deg)).to(cuda)
        made = px.MxConns.from_edges(conns.src, dst, torch.from_numpy(w).to(cuda),
                                     torch.arange(deg.size, dtype=torch.int32, device=cuda), weights=weights)
        conns = px.MxConns(conns.units, made.offsets, made.src, weights, block_offsets=made.block_offsets,
                           codes=made.codes, scales=made.scales)
        v = _mx.values(made.codes.cpu().numpy(), made.scales.cpu().numpy()[:, None], weights, 32).reshape(-1)
        blk = made.block_offsets.cpu().numpy()
        w = np.concatenate([v[blk[i] * 32:blk[i] * 32 + deg[i]] for i in range(deg.size)])
    x = rng.standard_normal((num_src, batch)) * np.exp2(rng.integers(-30, 20, (num_src, batch)))
    x[:, ::5] = 0.0
    x[:, 3::11] *= 2.0 ** 100  # a few samples of a block, whose scale then is large
    x[src[0], 3] = 2.0 ** 120
    x = x.astype(np.float32)
    xd = _rows(x, rows, False, cuda)
    xv = _mx.values(xd.codes.cpu().numpy(), xd.scales.cpu().numpy(), rows, batch)
    total = len(units) + 4
    got = px.mx_product(conns, xd, out=torch.zeros((total, batch), device=cuda)).cpu().numpy()
    y, err = _mx.product(off, src, w, xv, units, total, "identity", num_src)
    top = np.zeros((total, batch))
    for i, u in enumerate(units):
        e = np.arange(off[i], off[i + 1])
        if e.size:
            top[u] = np.abs(w[e, None] * xv[src[e]]).sum(0)
    fits = top < 2.0 ** 126
    assert fits.any() and not fits[units].all()
    _within(got[fits], y[fits], err[fits])
    assert not np.isfinite(got[(top > 2.0 ** 129) & (np.abs(y) > 2.0 ** 128.5)]).any()


def test_relu_keeps_what_is_not_a_number(cuda):
    rng = np.random.default_rng(4)
    for many, batch in ((700, 40), (11000, 1), (11000, 8), (11000, 16), (3, 300)):
        conns, off, src, w, units = _graph(rng, [5] * many, 16, "f32", cuda)
        x = rng.standard_normal((16, batch)).astype(np.float32)
        x[src[0], batch // 2] = np.nan
        x[src[7], 0] = np.inf
        xf = torch.from_numpy(x).to(cuda)
        total = len(units) + 3
        for xd in (xf, *(px.mx_quantize(xf, fmt) for fmt in FMTS)):
            ident = px.mx_product(conns, xd, out=torch.zeros((total, batch), device=cuda))
            relu = px.mx_product(conns, xd, activation="relu", out=torch.zeros((total, batch), device=cuda))
            assert torch.isnan(ident).any()
            assert torch.equal(torch.isnan(relu), torch.isnan(ident))
            assert torch.equal(torch.nan_to_num(relu, 0.0), torch.clamp_min(torch.nan_to_num(ident, 0.0), 0.0))
            for fmt in FMTS:
                q = px.mx_product(conns, xd, activation="relu", out=px.MxRows.empty(total, batch, fmt, cuda, zero=True))
                bad = torch.nn.functional.pad(~torch.isfinite(relu), (0, -batch % 32)).view(total, -1, 32).any(2)
                assert torch.equal(q.scales == 255, bad)


@pytest.mark.parametrize("fmt", mx.CHECKPOINT_FORMATS)
def test_relu_apply_keeps_what_is_not_a_number(cuda, fmt):
    rows = torch.randn((20, 70), device=cuda)
    rows[3, 40], rows[7, 2] = float("nan"), float("inf")
    want = torch.relu(rows)
    ck = px.MxRows.empty(20, 70, fmt, cuda)
    px.mx_unit_apply(rows, ck, "relu")
    assert torch.equal(torch.isnan(rows), torch.isnan(want)) and torch.equal(torch.nan_to_num(rows), torch.nan_to_num(want))
    bad = torch.zeros((20, 3), dtype=torch.bool, device=cuda)
    bad[3, 1] = bad[7, 0] = True
    assert torch.equal(ck.scales == 255, bad)
    net, n, frm, to, w, inputs, outputs = _mlp_net([24, 40, 33, 10], 0.4, np.random.default_rng(1))
    static, state = px.NetworkBuilder.from_edges(net, n, frm, to, weights=w, input_ids=inputs, output_ids=outputs, device=cuda)
    x = np.random.default_rng(2).standard_normal((40, 24)).astype(np.float32)
    x[33, 5] = np.nan
    for r, first in (("f32", 33), ("e4m3", 32)):
        got = torch.isnan(px.make_infer(net, static, state, weights="f32", rows=r)(x))
        assert got[first:].any() and not got[:first].any() and (r != "f32" or not got[34:].any())


@pytest.mark.parametrize("n,cap,batch", [(64, 4096, 16384), (2, 5, 1 << 17), (16, 20000, 5001)])
def test_edge_grad_of_a_long_batch(cuda, n, cap, batch):
    rng = np.random.default_rng(batch)
    b, dev = _bucket(rng, n, cap, cuda)
    g = rng.standard_normal((n, batch)).astype(np.float32)
    ck = _rows(rng.standard_normal((n, batch)).astype(np.float32), "e4m3", True, cuda)
    a = _mx.values(ck.codes.cpu().numpy(), ck.scales.cpu().numpy(), "e4m3", batch)
    f, t = b["from_id"].astype(np.int64), b["to_id"].astype(np.int64)
    live = (b["dead"] == 0) & (f >= 0) & (f < n) & (t >= 0) & (t < n)
    f, t = np.where(live, f, 0), np.where(live, t, 0)
    pairs, size = g.astype(np.float64) @ a.T / batch, np.abs(g).astype(np.float64) @ np.abs(a).T / batch
    got = px.mx_edge_grad(dev, torch.from_numpy(g).to(cuda), ck).cpu().numpy()
    _within(got, np.where(live, pairs[t, f], 0.0), np.where(live, size[t, f] * (batch + 4) * _mx.U32 * 1.01, 0.0))


def test_checkpointed_step_of_a_small_net_with_many_slots(cuda):
    """The update as one product of all pairs, reached through the step: one
    SGD step from the step's own gradient rows and checkpoint, in 64 bits."""
    rng = np.random.default_rng(41)
    net, n, frm, to, w, inputs, outputs = _mlp_net([40, 50, 10], 0.5, rng, opt=px.optim.sgd(0.05))
    static, state = px.NetworkBuilder.from_edges(net, n, frm, to, weights=w, input_ids=inputs, output_ids=outputs,
                                                 capacity_align=1 << 16, device=cuda)
    assert all(mx.edge_grad_scratch_bytes(b["dead"].numel(), 1024, n) > 0 for b in state.conns)
    step = px.make_step(net, static, batch_size=1024, device=cuda, activation_checkpoint="e4m3")
    before = [{k: b[k].cpu().numpy() for k in ("from_id", "to_id", "dead", "weight")} for b in state.conns]
    step(state, px.StepInputs(rng.standard_normal((1024, 40)).astype(np.float32),
                              rng.standard_normal((1024, 10)).astype(np.float32)))
    g, a = step.grad_b.cpu().numpy(), px.mx_dequantize(step.checkpoint).cpu().numpy().astype(np.float64)
    for h, b in zip(before, state.conns):
        live, dw, err = _edge_reference(h, g, a, n)
        w0 = h["weight"].astype(np.float64)
        got = b["weight"].cpu().numpy()
        lr = float(np.float32(0.05))
        # the gradient's error, then a rounding of lr * dw and one of the difference
        bound = lr * err + 2 * _mx.U32 * (np.abs(w0) + lr * np.abs(dw)) * 1.01
        assert live.any() and (np.abs(got - (w0 - lr * dw))[live] <= bound[live]).all()
        np.testing.assert_array_equal(got[~live], h["weight"][~live])


def test_four_bit_answers_after_training(cuda):
    """A trained net's answers from 4-bit weights: those of its weights as
    held, off the float32 net's by no more than the weights' rounding carries
    forward, so that a class it leads by more than that stays the class."""
    rng = np.random.default_rng(51)
    net, n, frm, to, w, inputs, outputs = _mlp_net([16, 40, 30, 5], 0.5, rng, batch_loss=px.SoftmaxCrossEntropyLoss())
    static, state = px.NetworkBuilder.from_edges(net, n, frm, to, weights=w, input_ids=inputs, output_ids=outputs,
                                                 device=cuda)
    step = px.make_step(net, static, batch_size=64, device=cuda, activation_checkpoint="e4m3")
    centres = rng.standard_normal((5, 16)) * 2
    for _ in range(60):
        label = rng.integers(0, 5, 64)
        x = (centres[label] + rng.standard_normal((64, 16)) * 0.3).astype(np.float32)
        step(state, px.StepInputs(x, np.eye(5, dtype=np.float32)[label]))
    label = rng.integers(0, 5, 200)
    x = (centres[label] + rng.standard_normal((200, 16)) * 0.3).astype(np.float32)
    got = px.make_infer(net, static, state)(x).cpu().numpy().T
    host = [{k: b[k].cpu().numpy() for k in ("from_id", "to_id", "dead", "weight")} for b in state.conns]
    frm, to, w = (np.concatenate([b[k][b["dead"] == 0] for b in host]) for k in ("from_id", "to_id", "weight"))
    level, held = state.units["level"].cpu().numpy(), w.astype(np.float64)
    for u in range(n):
        e = np.nonzero(to == u)[0]
        if e.size:
            held[e] = _mx.values(*_mx.quantize(w[e][None], "e2m1"), "e2m1", e.size)[0]
    xt = x.T.astype(np.float64)
    y4, err = _topological(level, frm, to, held, xt, inputs, outputs, "relu", "identity")
    _within(got, y4[outputs], err[outputs] + 1e-30)
    y, _ = _topological(level, frm, to, w.astype(np.float64), xt, inputs, outputs, "relu", "identity")
    off = np.zeros_like(y)
    for lv in range(1, int(level.max()) + 1):  # |w4 x4 - w x| <= |w4 - w| |x| + |w4| |x4 - x|, ReLU's slope at most 1
        for u in np.nonzero(level == lv)[0]:
            e = to == u
            off[u] = (np.abs(held[e] - w[e])[:, None] * np.abs(y[frm[e]]) + np.abs(held[e])[:, None] * off[frm[e]]).sum(0)
    bound = off[outputs] * 1.01 + err[outputs] + 1e-30
    assert (np.abs(got - y[outputs]) <= bound).all()
    order = np.sort(y[outputs], axis=0)
    sure = order[-1] - order[-2] > 2 * bound.max(0)
    assert np.array_equal(got.argmax(0)[sure], y[outputs].argmax(0)[sure])
