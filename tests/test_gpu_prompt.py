"""Causal attention of new tokens over the cache that holds them (p8x_attn_prompt) against the formula in 64 bits, within the
bounds that promptcase derives."""
import numpy as np
import pytest

import p8x
from kvcase import BF16, F16, F32, from_bits, to_bits
from promptcase import Prompt

pytestmark = pytest.mark.gpu
TYPES = [(F16, F16), (BF16, BF16), (F16, F32), (BF16, F32)]

SHAPES = [
    # slots, new tokens, options
    ([1], [1], {}),
    ([5, 1, 0, 70], [5, 1, 0, 3], dict(heads=6, kv=2)),
    ([63, 64, 65], [63, 64, 65], dict(heads=5, kv=1, page=48)),
    ([200, 129], [100, 1], dict(heads=3, kv=3, page=32)),
    ([31, 33, 2], [32, 40, 9], dict(heads=4, kv=2)),            # fewer slots than tokens: the first see nothing
    ([700], [130], dict(heads=8, kv=2, page=256)),
    ([1030, 20, 400], [1, 20, 260], dict(heads=7, kv=1)),
    ([300], [300], dict(heads=2, kv=2, page=16)),
    ([5000], [3], dict(heads=4, kv=1, page=64)),
]


@pytest.mark.parametrize("cache,q", TYPES)
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_shapes(shape, cache, q):
    lens, toks, o = SHAPES[shape]
    c = Prompt(lens, toks, cache=cache, q=q, seed=shape, layout=("head", "slot")[shape % 2], **o)
    c.check(*c.run())


@pytest.mark.parametrize("D", [64, 256])
@pytest.mark.parametrize("cache,q", TYPES)
@pytest.mark.parametrize("shape", [1, 2, 3, 4, 6, 8])
def test_head_dims(D, cache, q, shape):
    lens, toks, o = SHAPES[shape]
    c = Prompt(lens, toks, cache=cache, q=q, D=D, seed=20 + shape, layout=("slot", "head")[shape % 2], **o)
    c.check(*c.run())


@pytest.mark.parametrize("cache,q,out", [(F16, F16, BF16), (BF16, BF16, F16), (F16, F32, BF16), (BF16, F32, F16), (F16, F32, F16)])
def test_types_of_the_result(cache, q, out):
    c = Prompt([90, 40], [33, 40], cache=cache, q=q, out=out, seed=30)
    c.check(*c.run())


@pytest.mark.parametrize("q", [F32, F16])
def test_without_lse_or_workspace_and_with_little(q):
    c = Prompt([3000, 90], [5, 70], cache=F16, q=q, heads=4, kv=1, seed=31)
    full, lse = c.run()
    c.check(full, lse)
    c.check(*c.run(workspace=0))
    c.check(*c.run(workspace=p8x.DeviceBuffer(64)))
    some = p8x.DeviceBuffer(1 << 20)
    some.fill(0xFF)   # any contents
    a = c.run(workspace=some)
    c.check(*a)
    b = c.run(workspace=some)
    assert a[0].tobytes() == b[0].tobytes() and a[1].tobytes() == b[1].tobytes()
    assert c.run(lse=False)[0].tobytes() == full.tobytes()


@pytest.mark.parametrize("table,extra", [(False, 0), (False, 5), (True, 3)])
def test_contiguous_cache_and_rows_of_no_sequence(table, extra):
    c = Prompt([100, 257], [77, 30], table=table, extra=extra, seed=32, cache=BF16, q=BF16)
    c.check(*c.run())


def test_tokens_past_max_tokens_are_left():
    """max_tokens below a sequence's tokens: the further ones are none of the call's, as in the append"""
    c = Prompt([50, 20], [20, 6], cache=F16, q=F16, seed=33)
    ref = Prompt([50, 20], [20, 6], cache=F16, q=F16, seed=33)
    c.tk = 12
    ref.toks[0] = 12
    ref.first = c.first
    out, lse = c.run()
    want, wl, tol, ltol = ref.causal()
    rows = list(range(12)) + list(range(20, 26))
    assert (np.abs(from_bits(out, F16) - want)[rows] <= tol[rows]).all() and (np.abs(lse - wl)[rows] <= ltol[rows]).all()
    assert (out[12:20] == 0x7E7E).all() and (lse[12:20] == 7.0).all()


def test_rows_out_of_order_are_no_sequence():
    c = Prompt([30, 30, 30], [4, 4, 4], cache=F16, q=F16, seed=34)
    c.first = np.array([0, 4, 2, 90], np.int32)   # the second's end before its start, the third's behind the rows
    out, lse = c.run()
    want, wl, tol, ltol = Prompt([30, 30, 30], [4, 0, 0], cache=F16, q=F16, seed=34, extra=8).causal()
    assert (out[4:] == 0x7E7E).all() and (lse[4:] == 7.0).all() and np.isfinite(from_bits(out[:4], F16)).all()


@pytest.mark.parametrize("cache,q", TYPES)
def test_pages_outside_the_pool_hold_no_slots(cache, q):
    c = Prompt([300, 130, 70], [60, 130, 70], cache=cache, q=q, page=16, seed=35)
    c.pages[0, 2], c.pages[0, 12], c.pages[1, 0], c.pages[2, :5] = -1, c.n_pages, 1 << 30, -5   # the last sequence's all
    c.check(*c.run())


@pytest.mark.parametrize("D,cache,q", [(128, F16, F16), (128, BF16, F32), (64, BF16, BF16), (256, F16, F32)])
@pytest.mark.parametrize("what", [np.inf, -np.inf, np.nan])
def test_what_a_token_does_not_see_does_not_reach_it(D, cache, q, what):
    """keys and values of later tokens, of slots past the length and of pages that are not there"""
    c = Prompt([150, 40], [100, 40], cache=cache, q=q, D=D, page=16, seed=36)
    clean = c.causal()
    bad = to_bits(np.float32(what), cache)
    late = {0: (90, 91, 133, 149), 1: (17, 39)}
    for s, js in late.items():
        for j in js:
            c.row(c.kb, s, j)[:, ::3] = bad
            c.row(c.vb, s, j)[:, 1::2] = bad
    out, lse = c.run()
    got = from_bits(out, c.out_t)
    for s, js in late.items():
        n, nt, a = c.lens[s], c.toks[s], c.first[s]
        blind = max(0, js[0] - (n - nt))   # tokens before the first that sees one
        assert (np.abs(got - clean[0]) <= clean[2])[a:a + blind].all()
        assert (np.abs(lse - clean[1]) <= clean[3])[a:a + blind].all()
        assert not np.isfinite(got[a + blind:a + nt, :, 1::2]).any()


@pytest.mark.parametrize("what", [np.inf, -np.inf, np.nan])
@pytest.mark.parametrize("cache,q", [(F16, F16), (BF16, F32)])
def test_odd_values_alone(cache, q, what):
    """a later token whose key is ordinary and whose values are not: those that see it get them in the elements that have them"""
    c = Prompt([97], [97], cache=cache, q=q, seed=37)
    clean = c.causal()
    for j in (40, 95):
        c.row(c.vb, 0, j)[:, 5] = to_bits(np.float32(what), cache)
    got = from_bits(c.run()[0], c.out_t)
    ok = np.abs(got - clean[0]) <= clean[2]
    assert ok[:40].all() and ok[:, :, :5].all() and ok[:, :, 6:].all()
    assert not np.isfinite(got[40:, :, 5]).any()


@pytest.mark.parametrize("cache,q", TYPES)
def test_negative_and_zero_scale(cache, q):
    for scale in (-0.1, 0.0):
        c = Prompt([90, 33], [50, 33], cache=cache, q=q, seed=38)
        c.scale = float(np.float32(scale))
        c.check(*c.run())


@pytest.mark.parametrize("cache,q", TYPES)
def test_large_scores(cache, q):
    """scores far beyond the exponential's range, of either sign"""
    c = Prompt([200], [100], cache=cache, q=q, seed=39)
    c.qb = to_bits(from_bits(c.qb, q).astype(np.float32) * 40, q)
    c.check(*c.run())


@pytest.mark.parametrize("cache,q", TYPES)
@pytest.mark.parametrize("depth", [8, 15, 26, 60])
def test_sinks(cache, q, depth):
    """a first slot that takes nearly all of the weight and has next to no values: the rest decides the result"""
    c = Prompt([400, 120], [90, 120], cache=cache, q=q, heads=2, kv=1, seed=40)
    rng = np.random.default_rng(1)
    for s in range(2):
        a = c.first[s]
        u = np.zeros(c.D, np.float32)
        u[0] = 8.0
        k = rng.standard_normal((c.lens[s], c.D)).astype(np.float32) * 0.3
        k[:, 0] = 0
        k[0] = 0
        k[0, 0] = depth / 8.0 / c.scale
        for j in range(c.lens[s]):
            c.row(c.kb, s, j)[:] = to_bits(k[j], cache)
        c.row(c.vb, s, 0)[:] = 0
        q1 = rng.standard_normal((c.toks[s], c.H, c.D)).astype(np.float32)
        q1[:, :, 0] = 8.0
        c.qb[a:a + c.toks[s]] = to_bits(q1, q)
    out, lse = c.run()
    ref, rl, tol, ltol = c.causal()
    # relative to what the rest makes: the weights' bounds apply to it, the sums' to all
    f32 = q == F32
    uw = {(F16, False): 2.0 ** -11, (BF16, False): 2.0 ** -8, (F16, True): 2.0 ** -22, (BF16, True): 2.0 ** -24}[cache, f32]
    floor = 0.0 if cache == BF16 else 2.0 ** -22 if f32 else 2.0 ** -17
    got, big = from_bits(out, c.out_t), np.abs(ref).max(axis=2, keepdims=True)
    # the first 64 slots hold the sink: there a weight is held to floor of the sink's; behind them to floor of their own tile's
    rest = np.exp(-float(depth)) * 4.0 * 400
    for s in range(2):
        for i in range(1, c.toks[s]):
            tok, end = c.first[s] + i, c.lens[s] - c.toks[s] + i + 1
            near = floor * min(end, 64) * 4.0
            far = rest * (uw + floor * 64 + 2.0 ** -12 * (c.D + 8) * 2.0 ** -12 * 64 + 2.0 ** -18)
            half = {F16: 2.0 ** -11, BF16: 2.0 ** -8, F32: 2.0 ** -24}[c.out_t] * np.abs(ref[tok]) + (2.0 ** -25 if c.out_t == F16 else 0)
            assert (np.abs(got[tok] - ref[tok]) <= near + far + half * 1.01).all(), (s, i, np.abs(got[tok] - ref[tok]).max(), near, far)
    assert (np.abs(lse - rl) <= ltol + 64 * floor).all()


def test_tail_behind_the_sink_keeps_its_bits():
    """fp16: slots behind the sink's 64, e^-20 below it, are held to the type's step of themselves"""
    for depth in (15, 20, 30):
        c = Prompt([512], [40], cache=F16, q=F16, heads=2, kv=1, seed=41)
        for j in range(512):
            c.row(c.kb, 0, j)[:] = 0
        k0 = np.zeros(c.D, np.float32)
        k0[0] = depth / 8.0 / c.scale
        c.row(c.kb, 0, 0)[:] = to_bits(k0, F16)
        for j in range(64):   # the sink and the rest of its tile: no values
            c.row(c.vb, 0, j)[:] = 0
        q = from_bits(c.qb, F16).astype(np.float32)
        q[:, :, 0] = 8.0
        c.qb = to_bits(q, F16)
        out, _ = c.run()
        ref = c.causal()[0]
        big = np.abs(ref).max()
        # all behind the sink have the same weight, rounded to 2^-11 of itself; sums of 448 terms; subnormal results of fp16
        tol = (2.0 ** -11 + 512 * 2.0 ** -23 + 2.0 ** -16) * 448 * np.exp(-float(depth)) * 4.5 + 2.0 ** -11 * np.abs(ref) + 2.0 ** -25
        assert (np.abs(from_bits(out, F16) - ref) <= tol).all(), (depth, np.abs(from_bits(out, F16) - ref).max(), big)


def test_scores_falling_and_rising():
    """each tile far below, or above, the one before: nothing overflows, the largest are the result"""
    for cache, q in TYPES:
        for sign in (-1, 1):
            c = Prompt([1000], [9], cache=cache, q=q, heads=2, kv=1, seed=42)
            for j in range(1000):
                k = from_bits(c.row(c.kb, 0, j), cache).astype(np.float32) * 0.1
                k[:, 0] = sign * (j // 64) * 2.0 / c.scale
                c.row(c.kb, 0, j)[:] = to_bits(k, cache)
            qq = from_bits(c.qb, q).astype(np.float32)
            qq[:, :, 0] = 8.0
            c.qb = to_bits(qq, q)
            c.check(*c.run())


def test_many_sequences():
    rng = np.random.default_rng(5)
    toks = rng.integers(0, 12, 90).tolist()
    lens = [t + int(x) for t, x in zip(toks, rng.integers(0, 60, 90))]
    toks[7], lens[7] = 150, 300
    c = Prompt(lens, toks, cache=BF16, q=BF16, heads=4, kv=2, seed=43)
    c.check(*c.run())


def test_strides_of_queries_and_results():
    """queries inside wider rows with heads apart, results likewise; what lies between stays"""
    c = Prompt([120, 30], [60, 11], cache=BF16, q=BF16, heads=4, kv=2, seed=44)
    hs, ld = c.D + 16, 4 * (c.D + 16) + 40
    wide = np.full((c.n, ld), 0x7FC0, np.uint16)
    for h in range(4):
        wide[:, h * hs:h * hs + c.D] = c.qb[:, h]
    od = c.dev(np.full((c.n, ld), 0x1234, np.uint16))
    ls = c.dev(np.zeros((c.n, 4), np.float32))
    p8x.AttnPrompt(c.make_cache(), od, out_dtype=BF16, lse=ls, ld_out=ld, head_stride_out=hs, n_tokens=c.n, max_tokens=c.tk, first=c.dev(c.first), n_heads=4,
                   q=c.dev(wide), q_dtype=BF16, ld_q=ld, head_stride_q=hs, scale=c.scale).run()
    p8x.synchronize()
    got = od.to_numpy(np.uint16, (c.n, ld))
    mine = np.zeros(ld, bool)
    for h in range(4):
        mine[h * hs:h * hs + c.D] = True
    assert (got[:, ~mine] == 0x1234).all()
    c.check(np.stack([got[:, h * hs:h * hs + c.D] for h in range(4)], 1), ls.to_numpy(np.float32, (c.n, 4)))


def test_large_offsets():
    """a pool of more than 2^32 elements: sequences and their slots far apart"""
    c = Prompt([70, 40], [30, 40], cache=F16, q=F16, heads=2, kv=1, table=False, max_len=96, seed=45)
    stride = (1 << 31) + 4096
    pools = []
    for host in (c.kb, c.vb):
        b = p8x.DeviceBuffer(2 * (2 * stride + 96 * c.D))
        for s in range(2):
            rows = np.ascontiguousarray(host[s, 0])
            p8x.hip_check(p8x.hip().hipMemcpy(b.addr + 2 * (s + 1) * stride, rows.ctypes.data, rows.nbytes, p8x.H2D), "copy")
        pools.append(b)
    # sequence s in page s + 1 of a pool whose pages are 2^31 elements apart
    table = np.array([[1], [2]], np.int32)
    cache = p8x.KvCache(F16, 2, 1, c.D, pools[0], pools[1], page_stride=stride, head_stride=c.D, slot_stride=c.D, page_size=96, n_pages=3,
                        len=c.dev(np.asarray(c.lens, np.int32)), max_len=96, pages=c.dev(table), ld_pages=1)
    out, ls = c.dev(np.zeros((c.n, 2, c.D), np.uint16)), c.dev(np.zeros((c.n, 2), np.float32))
    p8x.AttnPrompt(cache, out, out_dtype=F16, lse=ls, n_tokens=c.n, max_tokens=c.tk, first=c.dev(c.first), n_heads=2, q=c.dev(c.qb), q_dtype=F16,
                   scale=c.scale).run()
    p8x.synchronize()
    c.check(out.to_numpy(np.uint16, (c.n, 2, c.D)), ls.to_numpy(np.float32, (c.n, 2)))
    for b in pools:
        b.free()


@pytest.mark.parametrize("lens,toks", [([900, 50], [3, 50]), ([600], [300])])
def test_graph_replays_equal_eager(lens, toks):
    c = Prompt(lens, toks, cache=BF16, q=BF16, heads=4, kv=2, seed=46)
    call = c.make()
    st = p8x.Stream()
    out, lse = c.run(stream=st, call=call)
    c.check(out, lse)
    g = p8x.Graph(lambda s: call.run(s), st)
    for _ in range(3):
        c.od.fill(0xFF)
        p8x.synchronize()
        g.launch(st)
        st.sync()
        a = c.results()
        assert a[0].tobytes() == out.tobytes() and a[1].tobytes() == lse.tobytes()
        c.run(call=call)
    g.release()


def test_two_streams_with_a_workspace_each():
    cs = [Prompt([2000 + 100 * i], [4], cache=F16, q=F16, heads=4, kv=1, seed=47 + i) for i in range(2)]
    calls, sts = [c.make() for c in cs], [p8x.Stream(), p8x.Stream()]
    want = [c.run(call=k) for c, k in zip(cs, calls)]
    for _ in range(5):
        for k, st in zip(calls, sts):
            k.run(st)
        for st in sts:
            st.sync()
        for c, w in zip(cs, want):
            got = c.results()
            assert got[0].tobytes() == w[0].tobytes() and got[1].tobytes() == w[1].tobytes()
