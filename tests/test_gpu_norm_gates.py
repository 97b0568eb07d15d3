"""Sigmoid gates of any size in p8x_norm_residual: infinities and values whose product with log2 e overflows give 0 or 1, a NaN
stays in its row. Tolerances as in test_gpu_norm (the sigmoid is one of its f32 operations)."""
import numpy as np
import pytest

import p8x
from kvcase import BF16, F16, F32, from_bits, to_bits
from test_gpu_norm import norm64

pytestmark = pytest.mark.gpu
EDGES = [0.0, -0.0, 1e-40, 87.0, -87.0, 88.8, -88.8, 100.0, -100.0, 126.5, -126.5, 149.0, -149.0, 65504.0, -65504.0, 2.35e38, -2.35e38, 2.37e38, -2.37e38, 3e38,
         -3e38, 3.4e38, -3.4e38, np.inf, -np.inf]


@pytest.mark.parametrize("gate", [F32, F16, BF16])
@pytest.mark.parametrize("C", [320, 321, 4096])
@pytest.mark.parametrize("shared", [False, True])
def test_sigmoid_gates_of_any_size(gate, C, shared):
    rng = np.random.default_rng(C)
    n = 4
    y, h = rng.standard_normal((n, C)).astype(np.float32), rng.standard_normal((n, C)).astype(np.float32)
    g = (3 * rng.standard_normal((1 if shared else n, C))).astype(np.float32)
    g[:, :len(EDGES)] = EDGES
    if not shared:
        g[3, C // 2] = np.nan
    bits = to_bits(g, gate)
    yd, hd, gd, od, xd = (p8x.DeviceBuffer.from_numpy(a) for a in (y, h, bits, np.zeros_like(h), np.zeros_like(h)))
    p8x.NormResidual(n, C, h=hd, y=yd, h_out=od, x=xd, post=p8x.NORM_RMS, gate=gd, gate_dtype=gate, ld_gate=0 if shared else C,
                     gate_act=p8x.GATE_SIGMOID, alpha=0.7).run()
    p8x.synchronize()
    with np.errstate(over="ignore"):
        s = 1 / (1 + np.exp(-from_bits(bits, gate)))
    hr = h + float(np.float32(0.7)) * s * norm64(y.astype(np.float64), p8x.NORM_RMS, None, None, float(np.float32(1e-6)))
    xr = norm64(hr, p8x.NORM_RMS, None, None, float(np.float32(1e-6)))
    for d, ref in ((od, hr), (xd, xr)):
        got = d.to_numpy(np.float32, (n, C)).astype(np.float64)
        assert np.array_equal(np.isnan(got), np.isnan(ref))
        clean = ~np.isnan(ref).any(1)
        got, ref = got[clean], ref[clean]
        assert (np.abs(got - ref) <= 2.0 ** -24 * np.abs(ref) + 4e-6 * np.abs(ref).max(1, keepdims=True)).all(), np.abs(got - ref).max()
