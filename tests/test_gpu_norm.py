"""Norm, gate and residual between blocks (p8x_norm_residual) against the formula in 64 bits.

Tolerances: inputs are read exactly; mean and variance are f32 sums of up to C terms in a tree of at most 32 + 10 levels
(relative error < 42 2^-24 of the sum of absolute values), their root halves it, a handful of f32 operations follow: 4e-6
of the largest |x| of the row (a layer norm subtracts a mean, so errors are of the row's size), then one rounding."""
import numpy as np
import pytest

import p8x
from kvcase import BF16, F16, F32, from_bits, half_ulp, to_bits

pytestmark = pytest.mark.gpu
SIZE = {F32: 4, F16: 2, BF16: 2}


def norm64(v, kind, w, b, eps):
    if kind == p8x.NORM_NONE:
        return v
    if kind == p8x.NORM_LAYER:
        v = v - v.mean(1, keepdims=True)
    v = v / np.sqrt((v * v).mean(1, keepdims=True) + eps)
    return v * (1.0 if w is None else w) + (0.0 if b is None else b)


def run(n, C, y=F32, h=F32, x=F32, post=p8x.NORM_NONE, pre=p8x.NORM_RMS, gate=None, act=p8x.GATE_LINEAR, bias=False, alpha=0.7, pad=0, in_place=False,
        has_y=True, has_x=True, has_h=True, off=0, scale=1.0, weights=True, seed=0):
    """pad: elements between rows; off: elements by which every buffer starts later; gate: None, or (dtype, shared)"""
    rng = np.random.default_rng(seed + n + C)
    ld = C + pad
    eps = float(np.float32(1e-5))

    def buf(dtype, rows, values):
        a = np.zeros(rows * ld + off, np.float32)
        a[off:].reshape(rows, ld)[:, :C] = values
        bits = to_bits(a, dtype)
        return p8x.DeviceBuffer.from_numpy(bits), bits

    def vals(bits, dtype, rows):
        return from_bits(bits[off:].reshape(rows, ld)[:, :C].copy(), dtype)

    yd, yb = buf(y, n, scale * rng.standard_normal((n, C)) * np.exp(rng.standard_normal(C) * 0.5) + 0.3)
    hd, hb = buf(h, n, 2 * scale * rng.standard_normal((n, C)) + 1.0)
    w = [(1 + 0.2 * rng.standard_normal(C)).astype(np.float32) for _ in range(4)]
    wd = [p8x.DeviceBuffer.from_numpy(v) for v in w]
    rows = 0 if gate is None else 1 if gate[1] else n
    gd, gb = buf(gate[0], rows, rng.standard_normal((rows, C))) if gate else (None, None)
    hod = hd if in_place else buf(h, n, -5.0)[0]
    xd, _ = buf(x, n, -5.0)

    def at(b, dtype):
        return b.addr + off * SIZE[dtype]
    p8x.NormResidual(n, C, h=at(hd, h), y=at(yd, y) if has_y else None, h_out=at(hod, h) if has_h else None, x=at(xd, x) if has_x else None, y_dtype=y,
                     h_dtype=h, x_dtype=x, ldy=ld, ldh=ld, ldho=ld, ldx=ld, post=post, w_post=wd[0] if weights else None, b_post=wd[1] if bias else None, eps_post=eps, pre=pre,
                     w_pre=wd[2] if weights else None, b_pre=wd[3] if bias else None, eps_pre=eps, gate=at(gd, gate[0]) if gate else None,
                     gate_dtype=gate[0] if gate else F32, ld_gate=0 if gate and gate[1] else ld, gate_act=act, alpha=alpha).run()
    p8x.synchronize()
    hr = vals(hb, h, n)
    if has_y:
        g = vals(gb, gate[0], rows) if gate else 1.0
        if act == p8x.GATE_SIGMOID and gate:
            g = 1 / (1 + np.exp(-g))
        hr = hr + float(np.float32(alpha)) * g * norm64(vals(yb, y, n), post, w[0] if weights else None, w[1] if bias else None, eps)
    xr = norm64(hr, pre, w[2] if weights else None, w[3] if bias else None, eps)
    for on, d, dt, ref in ((has_h, hod, h, hr), (has_x, xd, x, xr)):
        if not on:
            continue
        bits = d.to_numpy(np.float32 if dt == F32 else np.uint16, (n * ld + off,))
        got = vals(bits, dt, n)
        tol = half_ulp(dt) * np.abs(ref) + 4e-6 * np.abs(ref).max(1, keepdims=True) + (2.0 ** -24 if dt == F16 else 0)
        assert (np.abs(got - ref) <= tol).all(), (np.abs(got - ref).max(), tol.min())
        rest = from_bits(bits[off:].reshape(n, ld)[:, C:].copy(), dt)
        assert (rest == 0).all() and (bits[:off] == 0).all()   # nothing between the rows is written


@pytest.mark.parametrize("C", [1, 2, 7, 63, 64, 65, 255, 1000, 2560, 4096, 5120, 9999, 17408, 32768])
@pytest.mark.parametrize("post,pre", [(p8x.NORM_NONE, p8x.NORM_RMS), (p8x.NORM_RMS, p8x.NORM_RMS), (p8x.NORM_LAYER, p8x.NORM_LAYER)])
def test_norm_widths(C, post, pre):
    run(3, C, post=post, pre=pre, bias=pre == p8x.NORM_LAYER)


@pytest.mark.parametrize("y", [F32, F16, BF16])
@pytest.mark.parametrize("h", [F32, F16, BF16])
@pytest.mark.parametrize("x", [F32, F16, BF16])
def test_norm_types(y, h, x):
    run(5, 520, y, h, x, post=p8x.NORM_RMS, gate=(y, False), act=p8x.GATE_SIGMOID)


@pytest.mark.parametrize("gate", [(F32, False), (F32, True), (BF16, False), (F16, True)])
@pytest.mark.parametrize("act", [p8x.GATE_LINEAR, p8x.GATE_SIGMOID])
def test_norm_gates(gate, act):
    run(4, 768, post=p8x.NORM_RMS, gate=gate, act=act)


@pytest.mark.parametrize("o", [dict(pad=1), dict(pad=4, off=4), dict(off=1), dict(pad=3, off=2, y=BF16, x=F16, h=BF16), dict(in_place=True), dict(has_y=False),
                               dict(has_x=False), dict(has_h=False), dict(pre=p8x.NORM_NONE, x=BF16), dict(weights=False), dict(alpha=0.0),
                               dict(alpha=-1.5, bias=True, post=p8x.NORM_LAYER), dict(pad=8, off=8, y=F16, h=F16, x=F16)])
def test_norm_layouts(o):
    run(6, 1024, **{"post": p8x.NORM_RMS, **o})
    run(2, 1026, **{"post": p8x.NORM_RMS, **o})


@pytest.mark.parametrize("n", [1, 2, 255, 257, 1500])
def test_norm_rows(n):
    run(n, 640, post=p8x.NORM_RMS, x=BF16, gate=(F32, True))


def test_norm_zero_rows_and_special_values():
    """a row of zeros gives zeros (eps), an infinity or NaN stays in its row"""
    n, C = 4, 320
    y = np.zeros((n, C), np.float32)
    h = np.zeros((n, C), np.float32)
    h[1:] = np.random.default_rng(0).standard_normal((3, C))
    h[2, 5], h[3, 7] = np.inf, np.nan
    yd, hd, xd = (p8x.DeviceBuffer.from_numpy(a) for a in (y, h, np.ones((n, C), np.float32)))
    p8x.NormResidual(n, C, h=hd, y=yd, x=xd, post=p8x.NORM_RMS).run()
    p8x.synchronize()
    x = xd.to_numpy(np.float32, (n, C))
    ref = h[1] / np.sqrt((h[1].astype(np.float64) ** 2).mean() + 1e-6)
    assert (x[0] == 0).all() and np.abs(x[1] - ref).max() < 4e-6 * np.abs(ref).max()
    assert np.isnan(x[2, 5]) and (np.delete(x[2], 5) == 0).all() and np.isnan(x[3]).all()


def test_norm_replays_in_a_graph():
    n, C = 3, 2048
    h = np.random.default_rng(1).standard_normal((n, C)).astype(np.float32)
    hd, yd, xd = (p8x.DeviceBuffer.from_numpy(a) for a in (h, h[::-1].copy(), np.zeros_like(h)))
    call = p8x.NormResidual(n, C, h=hd, y=yd, x=xd, post=p8x.NORM_RMS)
    call.run()
    p8x.synchronize()
    want = xd.to_numpy(np.uint32, (n, C)).copy()
    st = p8x.Stream()
    g = p8x.Graph(lambda s: call.run(s), st)
    for _ in range(3):
        xd.fill(0)
        p8x.synchronize()
        g.launch(st)
        st.sync()
        assert np.array_equal(want, xd.to_numpy(np.uint32, (n, C)))
    g.release()
    st.release()
