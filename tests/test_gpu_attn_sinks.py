"""Attention whose slots differ widely in weight: a few that take nearly all of it (sinks) with values of zero, and a long tail
whose weights, far below theirs, make up the result (p8x_attn_tree).

Tolerances. All values are positive, so errors are relative to the result: a weight's is that of its score (|score| < 40, an
error of a few 2^-24 of it: 1e-5) and of its rounding, 2^-17 of itself or 2^-19 of the largest of its 32 slots, which are mostly of one level here; the sums are
f32. That is the bound of test_gpu_attn, 2e-5 for f32 queries and 4e-5 for 16-bit ones, here of the result itself; then one
rounding to the type."""
import numpy as np
import pytest

import p8x
from kvcase import BF16, F16, F32, Case, from_bits, half_ulp, to_bits
from test_gpu_attn import run_attn

pytestmark = pytest.mark.gpu


def levels_case(level, value, toks, heads, kv, D, cache, q, seed, spread=0.0, page=64):
    """level [n]: how far a slot's score is above the drafted tokens' (spread: plus a normal of that size), value [n]: of what size
    its value is. A drafted token's value is that of the last slot."""
    n = len(level)
    c = Case([n], [toks], heads=heads, kv=kv, D=D, cache=cache, q=q, fused=False, seed=seed, page=page, mask="chain")
    rng = np.random.default_rng(seed)
    qv = 0.05 * rng.standard_normal((c.n, heads, D))
    qv[:, :, 0], qv[:, :, 1] = 8.0, 1.0
    c.qb = to_bits(qv.astype(np.float32), q)

    def rows(m, lv, val):
        k = 0.05 * rng.standard_normal((m, kv, D))
        k[:, :, 0] = (np.asarray(lv, np.float64) / (8.0 * c.scale))[:, None]
        k[:, :, 1] = spread * rng.standard_normal((m, kv)) / c.scale
        return to_bits(k.astype(np.float32), cache), to_bits((np.asarray(val)[:, None, None] * (1 + 0.25 * rng.random((m, kv, D)))).astype(np.float32), cache)
    k, v = rows(n, level, value)
    for j in range(n):
        c.row(c.kb, 0, j)[:], c.row(c.vb, 0, j)[:] = k[j], v[j]
    k, v = rows(c.n, np.full(c.n, level[-1]), np.full(c.n, value[-1]))
    c.knb, c.vnb = (to_bits(from_bits(b, cache).astype(np.float32), c.kt) for b in (k, v))
    return c


def check(c, workspace):
    out, lse = run_attn(c, workspace=workspace)
    ref, rl = c.attention()
    got = from_bits(out, c.qt)
    tol = (half_ulp(c.qt) + (2e-5 if c.qt == F32 else 4e-5)) * np.abs(ref) + (2.0 ** -25 if c.qt == F16 else 0)
    assert (np.abs(got - ref) <= tol).all(), (np.abs(got / ref - 1).max(), tol.max() / np.abs(ref).max())
    assert (np.abs(lse - rl) <= 1e-5 * (1 + np.abs(rl))).all()


# tokens, heads: one row tile, two, rows shared through LDS
ROWS = [(1, 4), (8, 4), (20, 4)]
TYPES = [(F16, F32), (F16, F16), (BF16, F32), (BF16, BF16)]


@pytest.mark.parametrize("cache,q", TYPES)
@pytest.mark.parametrize("toks,heads", ROWS)
@pytest.mark.parametrize("depth", [8, 15, 20, 26])
@pytest.mark.parametrize("workspace", [False, True])
def test_sinks(depth, toks, heads, cache, q, workspace):
    """256 sinks (a tile for each of a workgroup's waves), then the tail"""
    n = 4096
    level = np.full(n, -float(depth))
    level[:256] = 0.0
    value = np.where(level < 0, min(40000.0, np.exp(depth) / n), 0.0)
    check(levels_case(level, value, toks, heads, 1, 128, cache, q, depth), workspace)


@pytest.mark.parametrize("D", [64, 256])
@pytest.mark.parametrize("cache,q", TYPES)
@pytest.mark.parametrize("toks,heads", ROWS)
def test_sinks_head_dims(D, toks, heads, cache, q):
    level = np.full(3000, -16.0)
    level[:256] = 0.0
    check(levels_case(level, np.where(level < 0, 2000.0, 0.0), toks, heads, 1, D, cache, q, 1), False)


@pytest.mark.parametrize("cache,q", TYPES)
@pytest.mark.parametrize("toks,heads", ROWS)
@pytest.mark.parametrize("seed", [0, 1, 2])
def test_levels_up_and_down(seed, toks, heads, cache, q):
    """stretches of 32 to 512 slots at levels up to 15 apart, each as much of the result as it is long"""
    rng = np.random.default_rng(seed)
    level = np.concatenate([np.full(32 * int(rng.integers(1, 17)), rng.choice([0.0, -4.0, -7.0, -11.0, -15.0])) for _ in range(24)])
    check(levels_case(level, 0.01 * np.exp(-level), toks, heads, 1, 128, cache, q, seed), seed % 2 == 1)


@pytest.mark.parametrize("cache,q", TYPES)
@pytest.mark.parametrize("toks,heads", ROWS)
def test_sinks_over_a_spread_tail(toks, heads, cache, q):
    """a tail whose scores are spread by 1, as they are in earnest: the largest of a tile's 32 is some e^2 above their median, the
    sum 32 e^0.5 of it. Weights are held to 2^-19 of the tile's largest (2^-22 for f32 queries): e^1.5 2^-19 = 9e-6 of the sum"""
    level = np.full(6000, -18.0)
    level[:256] = 0.0
    check(levels_case(level, np.where(level < 0, 8000.0, 0.0), toks, heads, 1, 128, cache, q, 7, spread=1.0), False)


@pytest.mark.parametrize("cache,q", TYPES)
@pytest.mark.parametrize("toks,heads", ROWS)
def test_scores_falling_without_end(toks, heads, cache, q):
    """each tile some e^2 below the one before, far beyond what could matter: nothing overflows, the first tiles are the result"""
    n = 32 * 150
    level = -2.0 * (np.arange(n) // 32)
    c = levels_case(level, np.ones(n), toks, heads, 1, 128, cache, q, 9)
    check(c, False)
