"""Append of accepted tokens to the cache (p8x_kv_append) and eviction to a budget (p8x_kv_evict): every bit of the
cache, scores, positions and lengths against a plain implementation."""
import numpy as np
import pytest

import p8x
from kvcase import BF16, F16, F32, Case, from_bits, to_bits

pytestmark = pytest.mark.gpu


def append_ref(c, at, pos):
    k, v, pos, ends = c.kb.copy(), c.vb.copy(), pos.copy(), []
    for s in range(c.S):
        n = c.lens[s]
        acc = c.accepted(s)[:max(0, c.max_len - n)]
        for r, j in enumerate(acc):
            tok = c.first[s] + j
            pos[s, :, n + r] = at[tok]
            if not c.there(s, n + r):
                continue
            for pool, new in ((k, c.knb), (v, c.vnb)):
                c.row(pool, s, n + r)[:] = to_bits(from_bits(new[tok], c.kt).astype(np.float32), c.cache)
        ends.append(n + len(acc))
    return k, v, pos, np.array(ends, np.int32)


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("lens,toks,o", [
    ([0], [1], {}),
    ([15, 0, 33], [3, 64, 1], dict(page=16)),
    ([5, 100], [500, 3], dict(page=48, D=64, heads=6, kv=3, accept=None)),
    ([40, 60], [30, 10], dict(max_len=64)),
    ([7, 9], [0, 2], dict(D=256, layout="slot", table=False)),
])
@pytest.mark.parametrize("cache,q", [(F16, F32), (BF16, F32), (BF16, BF16)])
def test_append(lens, toks, o, cache, q, in_place):
    o = dict(o)
    every = "accept" in o
    o.pop("accept", None)
    c = Case(lens, toks, cache=cache, q=q, seed=sum(toks), mask="chain" if every else "tree", **o) if not every else Case(
        lens, toks, cache=cache, q=q, seed=sum(toks), mask="none", **o)
    if not every:
        c.accept = np.array([int(c.mask[c.first[s] + c.toks[s] - 1]) if c.toks[s] else 0 for s in range(c.S)], np.uint64)
    at = np.arange(100, 100 + c.n, dtype=np.int32)
    pos = np.full((c.S, c.kv, c.max_len), -7, np.int32)
    cache_, d = c.make_cache(), c.drafts(q=False)
    pd = c.dev(pos)
    ld = c.lend if in_place else c.dev(np.full(c.S, -1, np.int32))
    p8x.KvAppend(cache_, accept=None if c.accept is None else c.dev(c.accept), at=c.dev(at), pos=pd, len_out=ld, **d).run()
    p8x.synchronize()
    k, v, rp, ends = append_ref(c, at, pos)
    assert np.array_equal(c.kd.to_numpy(np.uint16, c.pool_shape), k)
    assert np.array_equal(c.vd.to_numpy(np.uint16, c.pool_shape), v)
    assert np.array_equal(pd.to_numpy(np.int32, pos.shape), rp)
    assert np.array_equal(ld.to_numpy(np.int32, (c.S,)), ends)


def test_append_rounds_like_the_cache_and_drops_pages_outside():
    c = Case([14, 3], [6, 2], cache=F16, q=F32, fused=False, seed=1)
    c.knb[0, 0, :6] = [65504.0, 65520.0, np.inf, -np.inf, np.nan, 2.0 ** -25]   # largest, overflow to inf, subnormal tie to 0
    c.pages[0, 1] = -1
    cache, d = c.make_cache(), c.drafts(q=False)
    ld = c.dev(np.zeros(2, np.int32))
    p8x.KvAppend(cache, len_out=ld, **d).run()
    p8x.synchronize()
    k, v, _, ends = append_ref(c, np.zeros(c.n, np.int32), np.zeros((2, c.kv, c.max_len), np.int32))
    got = from_bits(c.kd.to_numpy(np.uint16, c.pool_shape), F16)
    assert np.array_equal(got, from_bits(k, F16), equal_nan=True)
    assert np.array_equal(c.vd.to_numpy(np.uint16, c.pool_shape), v)
    assert np.array_equal(ld.to_numpy(np.int32, (2,)), ends)


# ---- evict
def evict_ref(c, budget, sinks, recent, score, pos, score_out, pos_out):
    k, v, so, po = c.kb.copy(), c.vb.copy(), score_out.copy(), None if pos is None else pos_out.copy()
    for s in range(c.S):
        n = c.lens[s]
        for h in range(c.kv):
            sc = score[s, h, :n]
            m = min(n, budget)
            so[s, h, :m] = sc[:m]
            if pos is not None:
                po[s, h, :m] = pos[s, h, :m]
            if n <= budget:
                continue
            p = None if pos is None else pos[s, h, :n].astype(np.int64)
            safe = np.zeros(n, bool) if p is None else (p < sinks) | ((p >= p.max() + 1 - recent) if recent else False)
            val = np.where(np.isnan(sc), -np.inf, sc).astype(np.float64)
            order = sorted(range(n), key=lambda j: (not safe[j], bool(np.isnan(sc[j])) and not safe[j], -val[j] if not safe[j] else 0.0, j))
            kept = np.zeros(n, bool)
            kept[order[:budget]] = True
            src, dst = np.flatnonzero(kept[budget:]) + budget, np.flatnonzero(~kept[:budget])
            assert len(src) == len(dst)
            for a, b in zip(src, dst):
                so[s, h, b] = sc[a]
                if pos is not None:
                    po[s, h, b] = pos[s, h, a]
                if c.there(s, a) and c.there(s, b):
                    for pool in (k, v):
                        c.row(pool, s, b)[h] = c.row(pool, s, a)[h]
    return k, v, so, po, np.minimum(c.lens, budget).astype(np.int32)


def run_evict(c, budget, sinks=0, recent=0, kind="skewed", with_pos=True, in_place=False, seed=0):
    rng = np.random.default_rng(seed)
    shape = (c.S, c.kv, c.max_len)
    score = np.exp(3 * rng.standard_normal(shape)).astype(np.float32)
    if kind == "ties":
        score = rng.integers(0, 3, shape).astype(np.float32)
    elif kind == "equal":
        score[:] = 0.25
    elif kind == "odd":   # both zeros, negative, infinite, NaN
        score = rng.choice(np.array([0.0, -0.0, -1.5, 2.0, np.inf, -np.inf, np.nan, 1e-42], np.float32), shape)
    pos = None
    if with_pos:
        pos = np.stack([[rng.permutation(3 * c.max_len)[:c.max_len] for _ in range(c.kv)] for _ in range(c.S)]).astype(np.int32)
    cache = c.make_cache()
    sd, pd = c.dev(score), c.dev(pos) if with_pos else None
    blank_s, blank_p = np.full(shape, -9.0, np.float32), np.full(shape, -9, np.int32)
    so = sd if in_place else c.dev(blank_s)
    po = None if pos is None else pd if in_place else c.dev(blank_p)
    lo = c.lend if in_place else c.dev(np.full(c.S, -1, np.int32))
    call = p8x.KvEvict(cache, budget, score=sd, len_out=lo, score_out=so, pos=pd, pos_out=po, n_sink=sinks, n_recent=recent)
    call.run()
    p8x.synchronize()
    k, v, rs, rp, rl = evict_ref(c, budget, sinks, recent, score, pos, score if in_place else blank_s, pos if in_place else blank_p)
    assert np.array_equal(lo.to_numpy(np.int32, (c.S,)), rl)
    assert np.array_equal(so.to_numpy(np.uint32, shape), rs.view(np.uint32))
    if with_pos:
        assert np.array_equal(po.to_numpy(np.int32, shape), rp)
    assert np.array_equal(c.kd.to_numpy(np.uint16, c.pool_shape), k)
    assert np.array_equal(c.vd.to_numpy(np.uint16, c.pool_shape), v)


@pytest.mark.parametrize("lens,budget,sinks,recent,o", [
    ([1], 1, 0, 1, {}),
    ([2], 1, 0, 0, {}),
    ([17, 0, 16], 16, 4, 4, dict(page=16)),
    ([100, 64, 65], 64, 4, 8, dict(page=48)),
    ([700, 1500], 333, 0, 100, dict(page=32, kv=3, heads=3, layout="slot")),
    ([1100], 1025, 3, 0, dict(D=64, kv=1, heads=1)),
    ([2050, 2049], 2048, 0, 2048, dict(D=64, kv=1, heads=1, page=64)),
    ([130], 500, 4, 4, dict(D=256)),
])
@pytest.mark.parametrize("kind", ["skewed", "ties", "equal", "odd"])
def test_evict(lens, budget, sinks, recent, o, kind):
    run_evict(Case(lens, [0] * len(lens), fused=False, seed=budget, **o), budget, sinks, recent, kind)


def test_evict_long():
    """more slots than a workgroup holds at a time"""
    run_evict(Case([40007], [0], fused=False, heads=1, kv=1, D=64, page=64, seed=2), 20011, 4, 1000, "skewed")
    run_evict(Case([70001], [0], fused=False, heads=1, kv=1, D=64, page=64, seed=3), 333, 0, 0, "ties", with_pos=False)


@pytest.mark.parametrize("kind", ["skewed", "ties", "equal", "odd"])
@pytest.mark.parametrize("lens,budget,recent", [([4097, 5000], 4096, 64), ([20011, 31], 77, 9), ([32700, 9000], 16001, 0)])
def test_evict_of_thousands(lens, budget, recent, kind):
    """rows whose keys a workgroup holds in shared memory, many groups of 64 a wave"""
    run_evict(Case(lens, [0, 0], fused=False, heads=1, kv=1, D=64, page=64, seed=8), budget, 3, recent, kind)


def test_evict_in_place_without_positions_and_pages_outside():
    run_evict(Case([300, 200], [0, 0], fused=False, seed=4), 128, 4, 16, "skewed", in_place=True)
    run_evict(Case([300, 90], [0, 0], fused=False, seed=5, table=False, layout="slot", cache=BF16), 100, with_pos=False)
    c = Case([300], [0], fused=False, seed=6)
    c.pages[0, 1], c.pages[0, 15] = -1, c.n_pages
    run_evict(c, 100, 2, 2)


def test_evict_and_append_replay_in_a_graph():
    """captured once, replayed with other work between; each replay starts from the same cache"""
    c = Case([200, 150], [4, 2], seed=7, cache=F16, q=F32)
    cache, d = c.make_cache(), c.drafts(q=False)
    score = np.random.default_rng(3).random((2, c.kv, c.max_len)).astype(np.float32)
    sd, so, lo, lo2 = c.dev(score), c.dev(np.zeros_like(score)), c.dev(np.zeros(2, np.int32)), c.dev(np.zeros(2, np.int32))
    ev, ap = p8x.KvEvict(cache, 100, score=sd, score_out=so, len_out=lo), p8x.KvAppend(cache, len_out=lo2, **d)

    def both(st):
        ev.run(st)
        ap.run(st)

    def results():
        p8x.synchronize()
        return [c.kd.to_numpy(np.uint16, c.pool_shape).copy(), c.vd.to_numpy(np.uint16, c.pool_shape).copy(), so.to_numpy(np.uint32, score.shape).copy(),
                lo.to_numpy(np.int32, (2,)).copy(), lo2.to_numpy(np.int32, (2,)).copy()]

    def reset():
        for b, a in ((c.kd, c.kb), (c.vd, c.vb)):
            p8x.hip_check(p8x.hip().hipMemcpy(b.ptr, a.ctypes.data, a.nbytes, p8x.H2D), "copy")
        so.fill(0); lo.fill(0); lo2.fill(0)
        p8x.synchronize()
    both(None)
    want = results()
    st = p8x.Stream()
    g = p8x.Graph(both, st)
    for _ in range(3):
        reset()
        g.launch(st)
        st.sync()
        assert all(np.array_equal(a, b) for a, b in zip(want, results()))
        reset()
        both(None)
        assert all(np.array_equal(a, b) for a, b in zip(want, results()))
    g.release()
    st.release()
