"""Attention of drafted tokens where a sequence has many rows (tokens times heads of a group), so that a workgroup's waves
share keys and values through LDS; and where there are many sequences. Tolerances as in test_gpu_attn."""
import numpy as np
import pytest

import p8x
from kvcase import BF16, F16, F32, Case, from_bits
from test_gpu_attn import check_attn, run_attn, run_score

pytestmark = pytest.mark.gpu

# lens, toks, heads, kv: 34 .. 2048 rows, one row tile and several, one workgroup a segment and several, lengths around the
# tiles of 32 and the stages of 64 slots, none
ROWS = [
    ([0, 1, 31], [17, 20, 33], 4, 2),
    ([95, 64, 65, 129], [31, 32, 33, 13], 10, 2),
    ([4000, 10], [64, 7], 8, 2),
    ([77], [64], 32, 1),
    ([0, 33], [64, 64], 16, 2),
    ([9001], [40], 3, 1),
]


@pytest.mark.parametrize("cache,q", [(F16, F32), (BF16, F32), (F16, F16), (BF16, BF16)])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("shape", range(len(ROWS)))
def test_many_rows(shape, D, cache, q):
    lens, toks, heads, kv = ROWS[shape]
    c = Case(lens, toks, heads=heads, kv=kv, D=D, cache=cache, q=q, seed=100 + shape, page=(16, 64)[shape % 2], layout=("slot", "head")[shape % 2])
    check_attn(c, *run_attn(c))


@pytest.mark.parametrize("mask", ["none", "any", "chain"])
def test_many_rows_masks(mask):
    c = Case([0, 50, 700], [64, 64, 40], heads=8, kv=2, cache=F16, q=F32, mask=mask, seed=110)
    check_attn(c, *run_attn(c))


@pytest.mark.parametrize("q", [F32, F16])
def test_many_rows_pages_outside_the_pool(q):
    c = Case([200, 90, 64], [40, 33, 17], heads=8, kv=2, q=q, seed=111)
    c.pages[0, 2], c.pages[0, 12], c.pages[1, 0], c.pages[2, :4] = -1, c.n_pages, 1 << 30, -5   # the last sequence's all
    check_attn(c, *run_attn(c))


@pytest.mark.parametrize("cache,q", [(F16, F32), (BF16, BF16)])
@pytest.mark.parametrize("what", [np.inf, -np.inf, np.nan])
def test_many_rows_what_a_mask_hides_does_not_reach(cache, q, what):
    def case():
        return Case([40, 2000], [40, 40], seed=112, cache=cache, q=q, fused=False, heads=4, kv=2)
    c = case()
    bits = {F16: {np.inf: 0x7C00, -np.inf: 0xFC00}, BF16: {np.inf: 0x7F80, -np.inf: 0xFF80}}
    to = np.float32(what) if c.kt == F32 else np.uint16(bits[c.kt].get(what, 0x7FC0 if c.kt == BF16 else 0x7E00))
    hit = np.zeros(c.n, bool)
    for s, j in ((0, 5), (1, 35)):
        c.knb[c.first[s] + j, 0, 3] = c.vnb[c.first[s] + j, 0, 7] = c.vnb[c.first[s] + j, 1, 100] = to
        for i in range(40):
            hit[c.first[s] + i] = int(c.mask[c.first[s] + i]) >> j & 1
    assert hit.any() and not hit.all()
    clean = case()
    (out, lse), (o2, l2) = run_attn(c), run_attn(clean)
    assert np.array_equal(out[~hit], o2[~hit]) and np.array_equal(lse[~hit], l2[~hit])
    check_attn(clean, np.where(hit[:, None, None], o2, out), np.where(hit[:, None], l2, lse))
    f = from_bits(out, c.qt)
    assert not np.isfinite(f[hit][:, 2:, 100]).any() and np.isfinite(f[hit][:, 2:, :100]).all()


@pytest.mark.parametrize("toks", [2, 40])
@pytest.mark.parametrize("cache,q", [(F16, F16), (BF16, F32)])
def test_negative_and_zero_scale(cache, q, toks):
    for scale in (-0.125, 0.0):
        c = Case([130, 9], [toks, 1], cache=cache, q=q, seed=113)
        c.scale = scale
        check_attn(c, *run_attn(c))
        run_score(c, "path")


def test_many_sequences():
    """more sequences than a wave has lanes, some of them empty of slots or tokens"""
    lens = [(37 * s) % 101 for s in range(150)]
    toks = [s % 4 if s != 80 else 45 for s in range(150)]
    c = Case(lens, toks, heads=4, kv=2, D=64, seed=114)
    check_attn(c, *run_attn(c))
    run_score(c, "path")


def test_sequences_beyond_the_work_of_one_wave_of_workgroups():
    """1200 segments without a split, and with several row tiles"""
    c = Case([5 + s % 60 for s in range(300)], [1] * 300, heads=4, kv=4, D=64, seed=115)
    check_attn(c, *run_attn(c))
    c = Case([33 + s for s in range(20)], [64] * 20, heads=16, kv=2, D=64, seed=116, q=F16)
    check_attn(c, *run_attn(c))


def test_large_offsets():
    """a pool whose second page lies past 2^32 bytes and 2^31 elements: rows shared through LDS, then append and eviction"""
    D, page, n, toks, budget = 64, 64, 100, 40, 90
    stride = (1 << 31) + 4096
    c = Case([n], [toks], seed=118, D=D, kv=1, heads=2, page=page, max_len=192, cache=F16, q=F32)
    c.pages = np.array([[1, 0, 2]], np.int32)
    rng = np.random.default_rng(1)
    for pool in (c.kb, c.vb):
        pool[:3] = rng.standard_normal(pool[:3].shape).astype(np.float16).view(np.uint16)
    ref, rl = c.attention()
    big = [p8x.DeviceBuffer(2 * (2 * stride + page * D)) for _ in range(2)]
    for b, pool in zip(big, (c.kb, c.vb)):
        for p in range(3):
            a = np.ascontiguousarray(pool[p])
            p8x.hip_check(p8x.hip().hipMemcpy(b.addr + 2 * stride * p, a.ctypes.data, a.nbytes, p8x.H2D), "copy")
    lend = c.dev(np.array([n], np.int32))
    cache = p8x.KvCache(F16, 1, 1, D, big[0], big[1], page_stride=stride, head_stride=page * D, slot_stride=D, page_size=page, n_pages=3, len=lend,
                        max_len=192, pages=c.dev(c.pages), ld_pages=3)
    out, lse, d = c.dev(np.zeros((toks, 2, D), np.float32)), c.dev(np.zeros((toks, 2), np.float32)), c.drafts()
    p8x.AttnTree(cache, out, lse=lse, **d).run()
    p8x.KvAppend(cache, len_out=lend, **d).run()
    score = rng.random((1, 1, 192)).astype(np.float32)
    sd = c.dev(score)
    p8x.KvEvict(cache, budget, score=sd, len_out=lend).run()
    p8x.synchronize()
    assert np.abs(out.to_numpy(np.float32, ref.shape) - ref).max() < 1e-4 and np.abs(lse.to_numpy(np.float32, rl.shape) - rl).max() < 1e-4
    assert lend.to_numpy(np.int32, (1,))[0] == budget
    kept = np.zeros(n + toks, bool)
    kept[np.argsort(-score[0, 0, :n + toks], kind="stable")[:budget]] = True
    at = np.arange(budget)
    at[np.flatnonzero(~kept[:budget])] = np.flatnonzero(kept[budget:]) + budget
    for b, pool, new in zip(big, (c.kb, c.vb), (c.knb, c.vnb)):
        rows = np.concatenate([[c.row(pool, 0, j)[0] for j in range(n)], np.ascontiguousarray(new[:, 0]).astype(np.float16).view(np.uint16)])[at]
        for j in range(budget):
            p, o = c.place(0, j)
            got = np.zeros(D, np.uint16)
            p8x.hip_check(p8x.hip().hipMemcpy(got.ctypes.data, b.addr + 2 * (stride * p + o * D), got.nbytes, p8x.D2H), "copy")
            assert np.array_equal(got, rows[j]), j
        b.free()


def test_one_workspace_for_calls_of_any_shape():
    """in turn: few segments with many records, many with few, rows shared through LDS, more segments than counters"""
    cases = [Case([6000], [3], heads=4, kv=1, D=128, seed=120), Case([150 + s for s in range(60)], [2] * 60, heads=4, kv=2, D=64, seed=121),
             Case([3000, 64], [40, 40], heads=4, kv=2, seed=122), Case([5 + s % 90 for s in range(1100)], [1] * 1100, heads=4, kv=4, D=64, seed=123)]
    calls, most = [], 0
    for c in cases:
        cache, d, out = c.make_cache(), c.drafts(), c.dev(np.zeros((c.n, c.H, c.D), np.float32))
        own = p8x.AttnTree(cache, out, **d)
        most = max(most, own._args[-1])
        own.run()
        p8x.synchronize()
        calls.append((c, cache, d, out, out.to_numpy(np.float32, (c.n, c.H, c.D)).copy()))
    ws = p8x.DeviceBuffer(most)
    ws.fill(0)
    for size in (most, most // 5):
        for i in (0, 1, 2, 0, 3, 1, 0, 2, 1):
            c, cache, d, out, want = calls[i]
            out.fill(0x7F)
            p8x.AttnTree(cache, out, workspace=ws, workspace_bytes=size, **d).run()
            p8x.synchronize()
            got = out.to_numpy(np.float32, want.shape)
            # (another split in a smaller workspace: sums in another order)
            assert np.abs(got - want).max() <= (0 if size == most else 1e-5), (i, size)
    for c, _, _, _, want in calls[:3]:
        check_attn(c, want, None)


def test_calls_on_a_stream_of_their_own():
    """every call ordered by the stream that it is given, with uploads on that stream just before"""
    c = Case([300, 64], [5, 40], heads=4, kv=2, seed=117, cache=BF16, q=BF16)
    cache, d = c.make_cache(), c.drafts()
    out, lse = c.dev(np.zeros((c.n, c.H, c.D), np.uint16)), c.dev(np.zeros((c.n, c.H), np.float32))
    sc = c.dev(np.ones((c.S, c.kv, c.max_len), np.float32))
    st = p8x.Stream()
    p8x.AttnTree(cache, out, lse=lse, **d).run(st)
    p8x.KvScore(cache, lse, sc, decay=0.5, **d).run(st)
    st.sync()
    check_attn(c, out.to_numpy(np.uint16, (c.n, c.H, c.D)), lse.to_numpy(np.float32, (c.n, c.H)))
    ref = c.score(lse.to_numpy(np.float32, (c.n, c.H)), np.ones((c.S, c.kv, c.max_len)), np.ones((c.S, c.kv, c.max_len)), 0.5)
    assert (np.abs(sc.to_numpy(np.float32, ref.shape) - ref) <= 2e-5 * np.abs(ref) + 1e-7).all()
    st.release()
