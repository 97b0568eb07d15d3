"""Rotary positions (p8x_rope) and the append with the rotation on the way (p8x_kv_append_rope) against the formula in 64 bits.

Tolerance. Angles are exact to 2^-32 of a turn (1.5e-9); sine and cosine and the two products and their sum add a few 2^-24
each, the norm (a sum of at most 256 squares, in 8 terms and 5 sums of two, a root and two products) less than 2^-20 of an
element: below 2^-20 amplitude (|a| + |b|) together, a and b being the pair after the norm. Then half a step of the type."""
import numpy as np
import pytest

import p8x
from kvcase import BF16, F16, F32, Case, from_bits, half_ulp, to_bits

pytestmark = pytest.mark.gpu


def reference(x, pos, freq, layout, n_rot, amp, w=None, eps=1e-6):
    """(rotated heads, bound before the rounding) of x [n][heads][D] in 64 bits"""
    x = np.asarray(x, np.float64)
    if w is not None:
        x = x / np.sqrt((x ** 2).mean(-1, keepdims=True) + eps) * w
    y, size = x.copy(), np.abs(x)
    for i in range(n_rot // 2):
        a, b = (i, i + n_rot // 2) if layout == p8x.ROPE_HALF else (2 * i, 2 * i + 1)
        t = np.array([2 * np.pi * (((int(p) * int(freq[i])) % (1 << 64)) / 2.0 ** 64) for p in pos])[:, None]
        va, vb = x[..., a], x[..., b]
        y[..., a], y[..., b] = amp * (va * np.cos(t) - vb * np.sin(t)), amp * (vb * np.cos(t) + va * np.sin(t))
        size[..., a] = size[..., b] = amp * (np.abs(va) + np.abs(vb))
    return y, 2.0 ** -20 * size


def close(bits, dtype, ref, bound):
    got = from_bits(bits, dtype)
    tol = bound + half_ulp(dtype) * (np.abs(ref) + bound) + {F32: 1e-37, F16: 2.0 ** -25, BF16: 1e-37}[dtype]
    assert (np.abs(got - ref) <= tol).all(), (np.abs(got - ref) / tol).max()


def blank(n, heads, D, dtype):
    return np.full((n, heads, D), 3, np.float32 if dtype == F32 else np.uint16)


def read(buf, n, heads, D, dtype):
    return buf.to_numpy(np.float32 if dtype == F32 else np.uint16, (n, heads, D))


POSITIONS = [0, 1, 7, 1001, 131071, 1000003, 2 ** 31 - 1, -1, -5000, -2 ** 31]


@pytest.mark.parametrize("D,n_rot", [(8, 8), (64, 64), (64, 24), (80, 32), (96, 96), (128, 128), (128, 64), (128, 8), (128, 0), (176, 80), (256, 256), (256, 104)])
@pytest.mark.parametrize("layout", [p8x.ROPE_HALF, p8x.ROPE_PAIRS])
def test_widths_and_parts(D, n_rot, layout):
    rng = np.random.default_rng(D + n_rot)
    n, H, kv = len(POSITIONS), 5, 3
    freq, amp = p8x.rope_frequencies(n_rot, 500000.0)
    q, k = rng.standard_normal((n, H, D)).astype(np.float32), rng.standard_normal((n, kv, D)).astype(np.float32)
    dev = p8x.DeviceBuffer.from_numpy
    fd, pos = dev(freq), np.array(POSITIONS, np.int32)
    rot = p8x.Rotation(n_rot, fd, layout, amp)
    qo, ko = dev(blank(n, H, D, F32)), dev(blank(n, kv, D, BF16))
    p8x.Rope(rot, n, D, dev(pos), n_heads=H, q=dev(q), q_out=qo, n_kv=kv, k=dev(k), k_out=ko, k_out_dtype=BF16).run()
    p8x.synchronize()
    close(read(qo, n, H, D, F32), F32, *reference(q, pos, freq, layout, n_rot, amp))
    close(read(ko, n, kv, D, BF16), BF16, *reference(k, pos, freq, layout, n_rot, amp))


@pytest.mark.parametrize("t_in", [F32, F16, BF16])
@pytest.mark.parametrize("t_out", [F32, F16, BF16])
@pytest.mark.parametrize("norm", [None, "q", "k", "both"])
def test_types_and_norms(t_in, t_out, norm):
    rng = np.random.default_rng(7)
    n, H, kv, D, n_rot = 13, 4, 2, 128, 96
    freq, amp = p8x.rope_frequencies(n_rot, 10000.0, p8x.ROPE_YARN, factor=8.0, original=4096)
    assert amp > 1.2
    bits = [to_bits(rng.standard_normal((n, h, D)) * 3, t_in) for h in (H, kv)]
    w = [(1 + 0.3 * rng.standard_normal(D)).astype(np.float32) if norm in (name, "both") else None for name in ("q", "k")]
    pos = rng.integers(0, 200000, n).astype(np.int32)
    dev = p8x.DeviceBuffer.from_numpy
    wd = [None if a is None else dev(a) for a in w]
    rot = p8x.Rotation(n_rot, dev(freq), p8x.ROPE_HALF, amp, w_q=wd[0], w_k=wd[1], eps=1e-5)
    qo, ko = dev(blank(n, H, D, t_out)), dev(blank(n, kv, D, t_out))
    p8x.Rope(rot, n, D, dev(pos), n_heads=H, q=dev(bits[0]), q_dtype=t_in, q_out=qo, q_out_dtype=t_out, n_kv=kv, k=dev(bits[1]), k_dtype=t_in, k_out=ko,
             k_out_dtype=t_out).run()
    p8x.synchronize()
    for buf, b, a, h in ((qo, bits[0], w[0], H), (ko, bits[1], w[1], kv)):
        close(read(buf, n, h, D, t_out), t_out, *reference(from_bits(b, t_in), pos, freq, p8x.ROPE_HALF, n_rot, amp, a, 1e-5))


@pytest.mark.parametrize("layout", [p8x.ROPE_HALF, p8x.ROPE_PAIRS])
@pytest.mark.parametrize("n,H,kv,D", [(1, 32, 8, 128), (3, 1, 1, 64), (700, 40, 8, 128), (64, 7, 1, 256), (2000, 3, 3, 80)])
def test_in_place_inside_a_row_of_products(n, H, kv, D, layout):
    """queries and keys in one buffer with the values, which stay; the same bits as to other rows"""
    rng = np.random.default_rng(n)
    ld = (H + 2 * kv) * D + 8
    x = rng.standard_normal((n, ld)).astype(np.float32)
    n_rot = D // 16 * 8
    freq, amp = p8x.rope_frequencies(n_rot, 10000.0)
    dev = p8x.DeviceBuffer.from_numpy
    pos = dev(rng.integers(0, 9000, n).astype(np.int32))
    rot = p8x.Rotation(n_rot, dev(freq), layout, amp)
    b = dev(x)
    p8x.Rope(rot, n, D, pos, n_heads=H, q=b, ld_q=ld, n_kv=kv, k=b.addr + 4 * H * D, ld_k=ld).run()
    qo, ko = dev(blank(n, H, D, F32)), dev(blank(n, kv, D, F32))
    src = dev(x)
    p8x.Rope(rot, n, D, pos, n_heads=H, q=src, ld_q=ld, q_out=qo, n_kv=kv, k=src.addr + 4 * H * D, ld_k=ld, k_out=ko).run()
    p8x.synchronize()
    got = b.to_numpy(np.float32, (n, ld))
    q, k = got[:, :H * D].reshape(n, H, D), got[:, H * D:(H + kv) * D].reshape(n, kv, D)
    assert q.tobytes() == read(qo, n, H, D, F32).tobytes() and k.tobytes() == read(ko, n, kv, D, F32).tobytes()
    assert np.array_equal(got[:, (H + kv) * D:], x[:, (H + kv) * D:])
    p = pos.to_numpy(np.int32, (n,))[:40]
    close(q[:40], F32, *reference(x[:40, :H * D].reshape(-1, H, D), p, freq, layout, n_rot, amp))


def test_queries_or_keys_alone_and_of_different_widths():
    rng = np.random.default_rng(9)
    n, H, kv, D = 21, 6, 2, 128
    q, k = to_bits(rng.standard_normal((n, H, D)), F16), rng.standard_normal((n, kv, D)).astype(np.float32)
    freq, amp = p8x.rope_frequencies(D)
    dev = p8x.DeviceBuffer.from_numpy
    pos = np.arange(n, dtype=np.int32)
    rot, pd = p8x.Rotation(D, dev(freq)), dev(pos)
    both, one = [dev(blank(n, H, D, F32)), dev(blank(n, kv, D, F16))], [dev(blank(n, H, D, F32)), dev(blank(n, kv, D, F16))]
    kw_q, kw_k = dict(n_heads=H, q=dev(q), q_dtype=F16), dict(n_kv=kv, k=dev(k), k_out_dtype=F16)
    p8x.Rope(rot, n, D, pd, q_out=both[0], k_out=both[1], **kw_q, **kw_k).run()
    p8x.Rope(rot, n, D, pd, q_out=one[0], **kw_q).run()
    p8x.Rope(rot, n, D, pd, k_out=one[1], **kw_k).run()
    p8x.synchronize()
    for a, b, h, t in ((both[0], one[0], H, F32), (both[1], one[1], kv, F16)):
        assert read(a, n, h, D, t).tobytes() == read(b, n, h, D, t).tobytes()
    close(read(both[0], n, H, D, F32), F32, *reference(from_bits(q, F16), pos, freq, p8x.ROPE_HALF, D, 1.0))


# ---- append
def append(c, rot, at=True, pos=True, in_place=False, q=True, q_out=None):
    """runs it on the case; returns (q out, K pool, V pool, pos, len)"""
    cache, d = c.make_cache(), c.drafts(q=False, mask=False)
    od = c.dev(blank(c.n, c.H, c.D, c.cache))
    size = 4 if c.qt == F32 else 2
    src = c.dev(c.buf) if c.buf is not None else c.dev(c.qb)
    pd = c.dev(np.full((c.S, c.kv, c.max_len), -9, np.int32)) if pos else None
    out_len = c.lend if in_place else c.dev(np.zeros(c.S, np.int32))
    kw = dict(n_heads=c.H, q=src, q_dtype=c.qt, q_out=od, q_out_dtype=c.cache, ld_q=c.ld if c.buf is not None else None) if q else {}
    p8x.KvAppendRope(cache, rot, at=c.dev(c.at) if at else None, pos=pd, len_out=out_len, **kw, **d).run()
    p8x.synchronize()
    return (read(od, c.n, c.H, c.D, c.cache), c.kd.to_numpy(np.uint16, c.pool_shape), c.vd.to_numpy(np.uint16, c.pool_shape),
            pd.to_numpy(np.int32, (c.S, c.kv, c.max_len)) if pos else None, out_len.to_numpy(np.int32, (c.S,)))


def check_append(c, rot, layout, freq, n_rot, amp, w_q=None, w_k=None, **o):
    at = o.get("at", True)
    q, k, v, pos, ln = append(c, rot, **o)
    where = np.zeros(c.n, np.int64)
    used = np.zeros(c.n, bool)
    want_pos = np.full((c.S, c.kv, c.max_len), -9)
    kb, vb = c.kb.copy(), c.vb.copy()
    for s in range(c.S):
        for i in range(min(c.toks[s], c.tk)):
            tok = c.first[s] + i
            used[tok] = True
            where[tok] = c.at[tok] if at else c.lens[s] + i
    ref, bound = reference(from_bits(c.knb, c.kt), where, freq, layout, n_rot, amp, w_k)
    for s in range(c.S):
        got = min(c.toks[s], c.tk, c.max_len - c.lens[s])
        assert ln[s] == c.lens[s] + got
        for i in range(got):
            tok, slot = c.first[s] + i, c.lens[s] + i
            want_pos[s, :, slot] = where[tok]
            if c.there(s, slot):
                close(c.row(k, s, slot), c.cache, ref[tok], bound[tok])
                assert np.array_equal(c.row(v, s, slot), to_bits(from_bits(c.vnb[tok], c.kt).astype(np.float32), c.cache))
                c.row(kb, s, slot)[:] = c.row(k, s, slot)
                c.row(vb, s, slot)[:] = c.row(v, s, slot)
    assert np.array_equal(k, kb) and np.array_equal(v, vb)   # nothing else changed
    if pos is not None:
        assert np.array_equal(pos, want_pos)
    if o.get("q", True):
        ref, bound = reference(from_bits(c.qb, c.qt), where, freq, layout, n_rot, amp, w_q)
        close(q[used], c.cache, ref[used], bound[used])
        assert (q[~used] == 3).all()


CASES = [
    ([0], [1], {}),
    ([5, 0, 70, 16], [3, 1, 0, 40], dict(heads=6, kv=2)),
    ([100], [333], dict(heads=5, kv=1, page=48)),
    ([60, 62, 64, 3], [9, 2, 7, 5], dict(max_len=64, heads=3, kv=3)),    # tokens past max_len
    ([7, 9], [4, 2], dict(table=False, extra=3)),
]


@pytest.mark.parametrize("cache,q", [(F16, F32), (BF16, F32), (BF16, BF16), (F16, F16)])
@pytest.mark.parametrize("shape", range(len(CASES)))
@pytest.mark.parametrize("in_place", [False, True])
def test_append(shape, cache, q, in_place):
    lens, toks, o = CASES[shape]
    c = Case(lens, toks, cache=cache, q=q, seed=shape, layout=("head", "slot")[shape % 2], **o)
    rng = np.random.default_rng(shape)
    c.at = rng.integers(0, 100000, c.n).astype(np.int32)
    layout, n_rot = (p8x.ROPE_HALF, 128) if shape % 2 else (p8x.ROPE_PAIRS, 64)
    freq, amp = p8x.rope_frequencies(n_rot, 500000.0, p8x.ROPE_BANDS, factor=8.0, original=8192, low=1, high=4)
    w = [(1 + 0.2 * rng.standard_normal(c.D)).astype(np.float32) for _ in range(2)] if shape % 3 else [None, None]
    rot = p8x.Rotation(n_rot, c.dev(freq), layout, amp, w_q=None if w[0] is None else c.dev(w[0]), w_k=None if w[1] is None else c.dev(w[1]))
    check_append(c, rot, layout, freq, n_rot, amp, *w, in_place=in_place)
    check_append(Case(lens, toks, cache=cache, q=q, seed=shape, layout=("head", "slot")[shape % 2], **o), rot, layout, freq, n_rot, amp, *w, at=False, pos=False,
                 q=False)


@pytest.mark.parametrize("D", [64, 256])
def test_append_head_dims_pages_outside_and_max_tokens(D):
    c = Case([40, 10], [30, 8], cache=BF16, q=F32, D=D, seed=4, page=16)
    c.at = np.arange(c.n, dtype=np.int32) * 1000
    c.pages[0, 3], c.pages[1, 0] = -1, c.n_pages
    c.tk = 20   # further tokens are none of the call's
    freq, amp = p8x.rope_frequencies(D, 10000.0, p8x.ROPE_LINEAR, factor=2.0)
    check_append(c, p8x.Rotation(D, c.dev(freq)), p8x.ROPE_HALF, freq, D, amp)


@pytest.mark.parametrize("q,kv_in", [(F32, F16), (F16, F32)])
def test_append_queries_of_another_width(q, kv_in):
    c = Case([20, 0], [9, 5], cache=F16, q=q, kv_in=kv_in, fused=False, seed=5)
    c.at = np.arange(c.n, dtype=np.int32)
    freq, amp = p8x.rope_frequencies(128)
    check_append(c, p8x.Rotation(128, c.dev(freq)), p8x.ROPE_HALF, freq, 128, amp)


def test_append_is_rope_then_append():
    """the bits of p8x_rope to the cache's type, and of p8x_kv_append's values"""
    c = Case([33, 7], [50, 11], cache=BF16, q=F32, seed=6, heads=8, kv=2)
    c.at = (np.arange(c.n) * 37).astype(np.int32)
    freq, amp = p8x.rope_frequencies(128)
    rot = p8x.Rotation(128, c.dev(freq), p8x.ROPE_HALF, amp)
    q, k, v, pos, _ = append(c, rot)
    b = c.dev(c.buf)
    p8x.Rope(rot, c.n, 128, c.dev(c.at), n_heads=c.H, q=b, ld_q=c.ld, n_kv=c.kv, k=b.addr + 4 * c.at_k, ld_k=c.ld).run()
    cache = c.make_cache()
    p8x.KvAppend(cache, len_out=c.dev(np.zeros(2, np.int32)), n_tokens=c.n, max_tokens=c.tk, first=c.dev(c.first), k=b.addr + 4 * c.at_k, v=b.addr + 4 * c.at_v,
                 ld_kv=c.ld).run()
    p8x.synchronize()
    assert np.array_equal(k, c.kd.to_numpy(np.uint16, c.pool_shape)) and np.array_equal(v, c.vd.to_numpy(np.uint16, c.pool_shape))
    rows = b.to_numpy(np.float32, (c.n, c.ld))[:, :c.H * 128].reshape(c.n, c.H, 128)
    assert np.array_equal(q, to_bits(rows, BF16))


def test_graph_replays_equal_eager():
    c = Case([10, 3], [60, 4], cache=F16, q=F32, seed=8)
    c.at = np.arange(c.n, dtype=np.int32)
    freq, amp = p8x.rope_frequencies(128)
    rot, cache, d = p8x.Rotation(128, c.dev(freq)), c.make_cache(), c.drafts(q=False, mask=False)
    od, ln = c.dev(blank(c.n, c.H, c.D, F16)), c.dev(np.zeros(2, np.int32))
    calls = [p8x.KvAppendRope(cache, rot, at=c.dev(c.at), len_out=ln, n_heads=c.H, q=c.dev(c.buf), ld_q=c.ld, q_out=od, q_out_dtype=F16, **d)]
    x = c.dev(c.buf)
    dst = c.dev(blank(c.n, c.H, c.D, F32))
    calls.append(p8x.Rope(rot, c.n, 128, c.dev(c.at), n_heads=c.H, q=x, ld_q=c.ld, q_out=dst))
    st = p8x.Stream()

    def results():
        return [b.to_numpy(np.uint8, (b.nbytes,)).tobytes() for b in (od, ln, dst, c.kd, c.vd)]
    for call in calls:
        call.run(st)
    st.sync()
    want = results()
    g = p8x.Graph(lambda s: [call.run(s) for call in calls], st)
    for _ in range(3):
        for b in (od, ln, dst):
            b.fill(0xFF)
        p8x.synchronize()
        g.launch(st)
        st.sync()
        assert results() == want
        for call in calls:
            call.run()
        p8x.synchronize()
    g.release()
