"""Attention of drafted tokens over the cache (p8x_attn_tree) and the accumulated attention weight (p8x_kv_score)
against the formula in 64 bits.

Tolerances. Scores: products of 16-bit (or f32) operands summed in f32 over head_dim terms of size |q||k|: an error of a few
2^-24 times sqrt(head_dim) |q| |k| scale, below 4e-6 for the inputs here (|scores| < 12), which is a relative error of the
weight; the exponential and its argument add 2^-22. The weights are kept to 16 bits or more: 2^-17 of a weight, of either
sign. Their sum over the slots times |v| <= max|v|: out is within 2e-5 max|v| of the formula for f32 queries (whose
weights are kept to f32), 4e-5 max|v| for 16-bit ones, and then rounded to its type."""
import numpy as np
import pytest

import p8x
from kvcase import BF16, F16, F32, Case, from_bits, half_ulp

pytestmark = pytest.mark.gpu


def run_attn(c, mask=True, workspace=True, lse=True):
    cache, d = c.make_cache(), c.drafts(mask=mask)
    npdt = np.float32 if c.qt == F32 else np.uint16
    out = c.dev(np.full((c.n, c.H, c.D), 0x7E7E if npdt == np.uint16 else 7.0, npdt))
    ls = c.dev(np.full((c.n, c.H), 7.0, np.float32)) if lse else None
    kw = {} if workspace else dict(workspace=0, workspace_bytes=0)
    call = p8x.AttnTree(cache, out, lse=ls, **kw, **d)
    call.run()
    p8x.synchronize()
    first = out.to_numpy(npdt, (c.n, c.H, c.D)).copy()
    fl = ls.to_numpy(np.float32, (c.n, c.H)).copy() if lse else None
    call.run()   # the workspace is left as it was found
    p8x.synchronize()
    assert first.tobytes() == out.to_numpy(npdt, (c.n, c.H, c.D)).tobytes()
    if lse:
        assert np.array_equal(fl.view(np.uint32), ls.to_numpy(np.uint32, (c.n, c.H)))
    return first, fl


def check_attn(c, out, lse, mask=True):
    used = int(c.first[-1])
    ref, rl = c.attention(mask)
    got = from_bits(out, c.qt)
    vmax = np.nanmax(np.abs([from_bits(b[np.isfinite(from_bits(b, t))], t).max(initial=0) for b, t in ((c.vb, c.cache), (c.vnb, c.kt))] + [1.0]))
    tol = half_ulp(c.qt) * np.abs(ref) + (2e-5 if c.qt == F32 else 4e-5) * vmax
    bad = ~(np.abs(got - ref) <= tol)[:used]
    assert not bad.any(), (np.argwhere(bad)[:4], np.nanmax(np.abs(got - ref)[:used]), tol.min())
    if lse is not None:
        a, b = lse[:used].astype(np.float64), rl[:used]
        with np.errstate(invalid="ignore"):   # -inf - -inf
            same = (a == b) | (np.abs(a - b) <= 1e-5 * (1 + np.abs(b)))
        assert same.all(), np.argwhere(~same)[:4]
    # rows of no sequence stay as they were
    assert (out[used:] == (7.0 if c.qt == F32 else 0x7E7E)).all()


SHAPES = [
    # lens, toks, options
    ([1], [1], {}),
    ([0], [1], {}),
    ([15, 16, 17], [1, 2, 3], {}),
    ([31, 32, 33, 0, 1], [5, 1, 8, 2, 1], dict(heads=6, kv=2)),
    ([100, 3, 257], [7, 64, 17], dict(heads=5, kv=1, page=48)),
    ([511, 64], [33, 64], dict(heads=8, kv=2, page=32)),
    ([1000], [1], dict(heads=8, kv=1)),
    ([5003], [2], dict(heads=4, kv=1, page=64)),
    ([700], [64], dict(heads=8, kv=1, page=256)),
    ([130, 40], [3, 9], dict(heads=3, kv=3)),
]


@pytest.mark.parametrize("cache,q", [(F16, F32), (BF16, F32), (F16, F16), (BF16, BF16)])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_attn_shapes(shape, cache, q):
    lens, toks, o = SHAPES[shape]
    c = Case(lens, toks, cache=cache, q=q, seed=shape, layout=("head", "slot")[shape % 2], **o)
    check_attn(c, *run_attn(c))


@pytest.mark.parametrize("D", [64, 256])
@pytest.mark.parametrize("cache,q", [(F16, F16), (BF16, F32)])
@pytest.mark.parametrize("shape", [2, 3, 4, 5, 7])
def test_attn_head_dims(D, cache, q, shape):
    lens, toks, o = SHAPES[shape]
    c = Case(lens, toks, cache=cache, q=q, D=D, seed=40 + shape, **o)
    check_attn(c, *run_attn(c))


@pytest.mark.parametrize("mask", ["chain", "none", "any"])
@pytest.mark.parametrize("lens,toks", [([0, 20, 0], [3, 64, 64]), ([2000], [10])])
def test_attn_masks(mask, lens, toks):
    """masks that leave a row empty (no slots, no bits): zeros and lse -inf"""
    c = Case(lens, toks, cache=BF16, q=BF16, mask=mask, seed=3)
    check_attn(c, *run_attn(c))


def test_attn_null_mask_is_causal():
    c = Case([37, 5], [9, 64], seed=5, mask="none")
    check_attn(c, *run_attn(c, mask=False), mask=False)


def test_attn_without_workspace_or_lse():
    c = Case([3000, 20], [4, 2], seed=6, heads=8, kv=2)
    a, _ = run_attn(c, workspace=False, lse=False)
    check_attn(c, a, None)


@pytest.mark.parametrize("table,extra", [(False, 0), (False, 5), (True, 3)])
def test_attn_contiguous_cache_and_rows_of_no_sequence(table, extra):
    c = Case([77, 300], [3, 2], seed=7, table=table, extra=extra, layout="slot", page=16)
    check_attn(c, *run_attn(c))


def test_attn_separate_types_of_drafts():
    """16-bit queries with f32 drafts (rounded as the cache stores them), and f32 queries with 16-bit drafts"""
    for q, kv in ((F16, F32), (F32, F16)):
        c = Case([50, 130], [6, 11], seed=8, q=q, kv_in=kv, fused=False, cache=F16)
        check_attn(c, *run_attn(c))


@pytest.mark.parametrize("q", [F32, F16])
def test_attn_pages_outside_the_pool_hold_no_slots(q):
    c = Case([200, 90], [3, 2], seed=9, q=q)
    c.pages[0, 2], c.pages[0, 12], c.pages[1, 0] = -1, c.n_pages, 1 << 30
    check_attn(c, *run_attn(c))


@pytest.mark.parametrize("cache,q", [(F16, F32), (BF16, BF16)])
@pytest.mark.parametrize("what", [np.inf, -np.inf, np.nan])
def test_attn_what_a_mask_hides_does_not_reach(cache, q, what):
    """a drafted token with infinite or NaN keys and values: its own branch and no other sees them"""
    c = Case([40], [12], seed=10, cache=cache, q=q, fused=False, heads=4, kv=2)
    c.knb[5, 0, 3] = c.vnb[5, 0, 7] = c.vnb[5, 1, 100] = to = np.float32(what) if c.kt == F32 else np.uint16({np.inf: 0x7C00, -np.inf: 0xFC00}.get(what, 0x7E00) if c.kt == F16 else {np.inf: 0x7F80, -np.inf: 0xFF80}.get(what, 0x7FC0))
    del to
    hit = np.array([int(m) >> 5 & 1 for m in c.mask], bool)
    assert hit.any() and not hit.all()
    out, lse = run_attn(c)
    clean = Case([40], [12], seed=10, cache=cache, q=q, fused=False, heads=4, kv=2)
    o2, l2 = run_attn(clean)
    assert np.array_equal(out[~hit], o2[~hit]) and np.array_equal(lse[~hit], l2[~hit])
    check_attn(clean, np.where(hit[:, None, None], o2, out), np.where(hit[:, None], l2, lse))
    f = from_bits(out, c.qt)
    assert not np.isfinite(f[hit][:, 2:, 100]).any()   # kv head 1: finite keys, one value that is not
    assert np.isfinite(f[hit][:, 2:, :100]).all() and np.isfinite(f[hit][:, 2:, 101:]).all()


def test_attn_large_scores():
    """scores far beyond the exponential's range: the largest takes all"""
    c = Case([64], [4], seed=11, heads=4, kv=2, fused=False, q=F32, cache=BF16)
    c.qb *= 300.0
    out, lse = run_attn(c)
    ref, rl = c.attention()
    # weights differ by exp of a score's error here: |score| < 4000 at 2^-22
    assert np.abs(from_bits(out, F32) - ref).max() < 8e-3 and np.abs(lse - rl).max() < 4e-3


def test_attn_tiny_and_huge_queries_keep_f32_accuracy():
    """f32 queries beyond the range of 16-bit parts: scale carries the rest"""
    for f in (2.0 ** 40, 2.0 ** -40):
        c = Case([90], [3], seed=12, fused=False, q=F32, cache=F16)
        c.qb *= np.float32(f)
        c.scale = float(np.float32(c.scale / f))
        check_attn(c, *run_attn(c))


def test_attn_large_offsets():
    """a pool whose second page lies past 2^32 bytes and 2^31 elements"""
    D, kv, page, n = 64, 1, 64, 100
    stride = (1 << 31) + 4096
    c = Case([n], [2], seed=13, D=D, kv=kv, heads=2, page=page, max_len=128, cache=F16, q=F32)
    c.pages[:] = [[1, 0]]
    rng = np.random.default_rng(1)
    for pool in (c.kb, c.vb):
        pool[:2] = rng.standard_normal(pool[:2].shape).astype(np.float16).view(np.uint16)
    ref = Case.attention(c)
    big = [p8x.DeviceBuffer(2 * (stride + page * D)) for _ in range(2)]
    for b, pool in zip(big, (c.kb, c.vb)):
        for p in range(2):
            a = np.ascontiguousarray(pool[p])
            p8x.hip_check(p8x.hip().hipMemcpy(b.addr + 2 * stride * p, a.ctypes.data, a.nbytes, p8x.H2D), "copy")
    lend, pages = c.dev(np.array([n], np.int32)), c.dev(c.pages)
    cache = p8x.KvCache(F16, 1, kv, D, big[0], big[1], page_stride=stride, head_stride=page * D, slot_stride=D, page_size=page, n_pages=2, len=lend,
                        max_len=128, pages=pages, ld_pages=2)
    out, lse = p8x.DeviceBuffer(4 * 2 * 2 * D), p8x.DeviceBuffer(4 * 4)
    d = c.drafts()
    p8x.AttnTree(cache, out, lse=lse, **d).run()
    sc, so = c.dev(np.zeros((1, 1, 128), np.float32)), c.dev(np.zeros((1, 1, 128), np.float32))
    p8x.KvScore(cache, lse, sc, so, decay=1.0, **d).run()
    p8x.synchronize()
    assert np.abs(out.to_numpy(np.float32, (2, 2, D)) - ref[0]).max() < 1e-4
    s64 = c.score(lse.to_numpy(np.float32, (2, 2)), np.zeros((1, 1, 128)), np.zeros((1, 1, 128)), 1.0)
    assert np.abs(so.to_numpy(np.float32, (1, 1, 128)) - s64).max() < 1e-5
    for b in big:
        b.free()


@pytest.mark.parametrize("op", ["attn", "score"])
def test_graph_replays_equal_eager(op):
    c = Case([900, 40], [5, 3], seed=14, heads=8, kv=2, q=BF16, cache=BF16)
    cache, d = c.make_cache(), c.drafts()
    out, lse = c.dev(np.zeros((c.n, c.H, c.D), np.uint16)), c.dev(np.zeros((c.n, c.H), np.float32))
    attn = p8x.AttnTree(cache, out, lse=lse, **d)
    attn.run()
    sc, so = c.dev(np.ones((c.S, c.kv, c.max_len), np.float32)), c.dev(np.zeros((c.S, c.kv, c.max_len), np.float32))
    call, res, shape, dt = (attn, out, (c.n, c.H, c.D), np.uint16) if op == "attn" else (p8x.KvScore(cache, lse, sc, so, decay=0.5, **d), so, (c.S, c.kv, c.max_len), np.uint32)
    call.run()
    p8x.synchronize()
    want = res.to_numpy(dt, shape).copy()
    st = p8x.Stream()
    g = p8x.Graph(lambda s: call.run(s), st)
    for _ in range(4):
        res.fill(0)
        p8x.synchronize()
        g.launch(st)
        st.sync()
        assert np.array_equal(want, res.to_numpy(dt, shape))
        call.run()
        p8x.synchronize()
    g.release()
    st.release()


# ---- scores. A weight's relative error is that of its score (above): 2e-5 of the sum, plus f32 rounding of the sum.
@pytest.mark.parametrize("cache,q", [(F16, F32), (BF16, F32), (F16, F16), (BF16, BF16)])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_score_shapes(shape, cache, q):
    lens, toks, o = SHAPES[shape]
    c = Case(lens, toks, cache=cache, q=q, seed=60 + shape, layout=("slot", "head")[shape % 2], **o)
    for accept in (None, "path", "zero"):
        run_score(c, accept)


@pytest.mark.parametrize("D", [64, 256])
@pytest.mark.parametrize("cache,q", [(F16, F16), (BF16, F32)])
@pytest.mark.parametrize("shape", [3, 4, 8])
def test_score_head_dims(D, cache, q, shape):
    lens, toks, o = SHAPES[shape]
    run_score(Case(lens, toks, cache=cache, q=q, D=D, seed=80 + shape, **o), "path")


def run_score(c, accept, in_place=False, decay=0.75):
    rng = np.random.default_rng(2)
    c.accept = None if accept is None else np.zeros(c.S, np.uint64) if accept == "zero" else np.array(
        [int(c.mask[c.first[s] + c.toks[s] - 1]) | 0xF000000000000000 for s in range(c.S)], np.uint64)   # bits past the tokens are ignored
    _, rl = c.attention()
    lse = np.where(np.isfinite(rl), rl, 0).astype(np.float32)
    old = rng.random((c.S, c.kv, c.max_len)).astype(np.float32)
    cache, d = c.make_cache(), c.drafts()
    sd, ld = c.dev(old), c.dev(lse)
    od = sd if in_place else c.dev(np.full(old.shape, -3.0, np.float32))
    acc = None if c.accept is None else c.dev(c.accept)
    p8x.KvScore(cache, ld, sd, od, accept=acc, decay=decay, **d).run()
    p8x.synchronize()
    got = od.to_numpy(np.float32, old.shape).astype(np.float64)
    ref = c.score(lse, old, old if in_place else np.full(old.shape, -3.0), decay)
    assert (np.abs(got - ref) <= 2e-5 * np.abs(ref) + 1e-7).all(), np.abs(got - ref).max()


def test_score_in_place_pages_outside_and_full_cache():
    run_score(Case([300, 20], [4, 3], seed=20), "path", in_place=True)
    c = Case([200, 90], [3, 2], seed=21)
    c.pages[0, 2], c.pages[1, 0] = -1, c.n_pages
    run_score(c, None)
    run_score(Case([60, 62], [8, 9], max_len=64, seed=22), None)   # drafts past max_len have no slot


def test_score_without_tokens_decays():
    c = Case([33, 5], [0, 0], seed=23, fused=False)
    old = np.random.default_rng(0).random((2, c.kv, c.max_len)).astype(np.float32)
    cache = c.make_cache()
    sd = c.dev(old)
    p8x.KvScore(cache, c.dev(np.zeros(1, np.float32)), sd, decay=0.5, n_tokens=0, max_tokens=0, first=c.dev(c.first)).run()
    p8x.synchronize()
    want = old.copy()
    for s in range(2):
        want[s, :, :c.lens[s]] *= np.float32(0.5)
    assert np.array_equal(sd.to_numpy(np.float32, old.shape), want)
