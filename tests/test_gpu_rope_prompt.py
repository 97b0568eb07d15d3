"""The calls of a rotary model together: a prompt at once gives what its tokens give one after another, and trees of drafted
tokens what their paths do."""
import numpy as np
import pytest

import p8x
from kvcase import BF16, F16, F32, from_bits, half_ulp
from p8x import tree_decode as td
from test_gpu_rope import reference
from test_gpu_tree_decode import SMALL, close

pytestmark = pytest.mark.gpu


class Layer:
    """q, k, v of one layer with random Pingala-8 weights, and a paged cache of one sequence"""

    def __init__(self, dtype, hidden=512, heads=8, kv=2, D=128, max_len=400, page=32, seed=0):
        rng = np.random.default_rng(seed)
        self.dtype, self.heads, self.kv, self.D, self.max_len = dtype, heads, kv, D, max_len
        slots = [p8x.synth_random(int(rng.integers(1, 1 << 31)), r * D, hidden) for r in (heads, kv, kv)]
        p8x.share_input(slots, [(heads * D, hidden), (kv * D, hidden), (kv * D, hidden)])
        self.w = [p8x.Tensor(s, r * D, hidden) for s, r in zip(slots, (heads, kv, kv))]
        self.ld = (heads + 2 * kv) * D
        dev = p8x.DeviceBuffer
        freq, amp = p8x.rope_frequencies(D, 10000.0, p8x.ROPE_YARN, factor=4.0, original=64)
        norm = [(1 + 0.2 * rng.standard_normal(D)).astype(np.float32) for _ in range(2)]
        self.rot = p8x.Rotation(D, dev.from_numpy(freq), amplitude=amp, w_q=dev.from_numpy(norm[0]), w_k=dev.from_numpy(norm[1]))
        pages = -(-max_len // page)
        self.table = dev.from_numpy(rng.permutation(pages + 2)[:pages].astype(np.int32))
        size = 2 * (pages + 2) * page * kv * D
        self.k, self.v, self.len = dev(size), dev(size), dev.from_numpy(np.zeros(1, np.int32))
        self.cache = p8x.KvCache(dtype, 1, kv, D, self.k, self.v, page_stride=page * kv * D, head_stride=page * D, slot_stride=D, page_size=page,
                                 n_pages=pages + 2, len=self.len, max_len=max_len, pages=self.table, ld_pages=pages)
        self.pos = dev.from_numpy(np.full((kv, max_len), -1, np.int32))

    def rows(self, x):
        """the products of x's rows: one buffer"""
        n = len(x)
        xd, out, cols = p8x.DeviceBuffer.from_numpy(x), p8x.DeviceBuffer(4 * n * self.ld), [0, self.heads * self.D, (self.heads + self.kv) * self.D]
        for w, c in zip(self.w, cols):
            w.mul_mat_dev(xd, p8x.F32, n, out.addr + 4 * c, ldy=self.ld)
        p8x.synchronize()
        return out, [out.addr + 4 * c for c in cols]

    def prompt(self, out, at, n, a, b, out_t=F32, q_t=F32):
        """tokens a .. b - 1 of the products, appended at once and attended for: (result bits, lse)"""
        dev, keep = p8x.DeviceBuffer, []
        size = 4 if q_t == F32 else 2
        q, o, lse = dev(size * (b - a) * self.heads * self.D), dev((4 if out_t == F32 else 2) * (b - a) * self.heads * self.D), dev(4 * (b - a) * self.heads)
        first = dev.from_numpy(np.array([0, b - a], np.int32))
        step = 4 * a * self.ld
        p8x.KvAppendRope(self.cache, self.rot, pos=self.pos, len_out=self.len, n_tokens=b - a, max_tokens=b - a, first=first, k=at[1] + step, v=at[2] + step,
                         ld_kv=self.ld, n_heads=self.heads, q=at[0] + step, ld_q=self.ld, q_out=q, q_out_dtype=q_t).run()
        p8x.AttnPrompt(self.cache, o, out_dtype=out_t, lse=lse, n_tokens=b - a, max_tokens=b - a, first=first, n_heads=self.heads, q=q, q_dtype=q_t,
                       scale=self.D ** -0.5).run()
        p8x.synchronize()
        return (o.to_numpy(np.float32 if out_t == F32 else np.uint16, (b - a, self.heads, self.D)).copy(),
                lse.to_numpy(np.float32, (b - a, self.heads)).copy())

    def token(self, out, at, i):
        """token i alone, as a tree of one: (result, lse)"""
        dev, step = p8x.DeviceBuffer, 4 * i * self.ld
        o, lse, pos = dev(4 * self.heads * self.D), dev(4 * self.heads), dev.from_numpy(np.array([i], np.int32))
        d = dict(n_tokens=1, max_tokens=1, first=dev.from_numpy(np.array([0, 1], np.int32)), k=at[1] + step, v=at[2] + step, ld_kv=self.ld)
        p8x.Rope(self.rot, 1, self.D, pos, n_heads=self.heads, q=at[0] + step, ld_q=self.ld, n_kv=self.kv, k=at[1] + step, ld_k=self.ld).run()
        p8x.AttnTree(self.cache, o, lse=lse, n_heads=self.heads, q=at[0] + step, ld_q=self.ld, scale=self.D ** -0.5, **d).run()
        p8x.KvAppend(self.cache, at=pos, pos=self.pos, len_out=self.len, **d).run()
        p8x.synchronize()
        return o.to_numpy(np.float32, (self.heads, self.D)).copy(), lse.to_numpy(np.float32, (self.heads,)).copy()


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_prompt_equals_its_tokens(dtype):
    """f32 queries: both ways hold weights to 2^-17 of themselves or better and sum in f32: within 2^-15 of max|v| of each other"""
    x = np.random.default_rng(1).standard_normal((230, 512)).astype(np.float32)
    L = Layer(dtype)
    out, at = L.rows(x)
    parts = [L.prompt(out, at, 230, a, b) for a, b in ((0, 150), (150, 151), (151, 230))]   # in chunks
    got, lse = np.concatenate([p[0] for p in parts]), np.concatenate([p[1] for p in parts])
    assert L.len.to_numpy(np.int32, (1,))[0] == 230
    k, v = L.k.to_numpy(np.uint8, (L.k.nbytes,)).copy(), L.v.to_numpy(np.uint8, (L.v.nbytes,)).copy()
    pos = L.pos.to_numpy(np.int32, (2, 400)).copy()
    M = Layer(dtype)
    out, at = M.rows(x)
    vmax = np.abs(out.to_numpy(np.float32, (230, M.ld))[:, (M.heads + M.kv) * M.D:]).max()
    for i in range(230):
        o, z = M.token(out, at, i)
        assert np.abs(got[i] - o).max() <= 2.0 ** -15 * vmax, i
        assert np.abs(lse[i] - z).max() <= 1e-5 * (1 + np.abs(z).max()), i
    # the same caches, bit for bit: slots in use only
    used = L.cache.max_len
    assert M.len.to_numpy(np.int32, (1,))[0] == 230 and np.array_equal(pos, M.pos.to_numpy(np.int32, (2, used)))
    page, D, kv = 32, 128, 2
    table = L.table.to_numpy(np.int32, (-(-used // page),))
    for mine, other in ((k, M.k), (v, M.v)):
        a = mine.view(np.uint16).reshape(-1, kv, page, D)
        b = other.to_numpy(np.uint16, a.shape)
        for j in range(230):
            assert np.array_equal(a[table[j // page], :, j % page], b[table[j // page], :, j % page]), j


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_prompt_in_16_bits_is_near_the_one_in_f32(dtype):
    """queries rounded to the cache's type (2^-11 or 2^-8 of each score's terms, twice as a weight), weights and results too"""
    x = np.random.default_rng(2).standard_normal((100, 512)).astype(np.float32)
    L, M = Layer(dtype), Layer(dtype)
    out, at = L.rows(x)
    full, _ = L.prompt(out, at, 100, 0, 100)
    some, _ = M.prompt(out, at, 100, 0, 100, out_t=dtype, q_t=dtype)
    u = half_ulp(dtype)
    vmax = np.abs(out.to_numpy(np.float32, (100, L.ld))[:, (L.heads + L.kv) * L.D:]).max()
    # |q . k| scale: heads normed to sqrt(D), weights of norms below 2, amplitude 1.14 squared: at most 4 * 1.3 * sqrt(128) = 59
    assert np.abs(from_bits(some, dtype) - full).max() <= (2 * 59 * u + 3 * u) * vmax


def test_rotary_tree_equals_each_of_its_paths():
    m = td.Model(**SMALL, rope_base=10000.0)
    plain = td.Model(**SMALL)
    prompt = np.random.default_rng(0).integers(0, 256, 21).tolist()
    tokens, parents = [5, 9, 200, 9, 77, 1, 3], [-1, 0, 0, 1, 2, 4, 0]
    d = td.Decoder(m, 128)
    d.prompt(prompt)
    tree = d.forward(tokens, parents)
    p = td.Decoder(plain, 128)
    p.prompt(prompt)
    p.forward(tokens, parents)
    # the first layer's products are the same: here rotated by each token's place behind the prompt
    rows = [x.layers[0]["qkv"].to_numpy(np.float32, (8, x.ld))[:7] for x in (d, p)]
    freq, amp = p8x.rope_frequencies(128, 10000.0)
    for a, b in ((0, m.heads), (m.heads, m.heads + m.kv)):
        got, x = (r[:, a * 128:b * 128].reshape(7, b - a, 128) for r in rows)
        ref, bound = reference(x, d.depth, freq, p8x.ROPE_HALF, 128, amp)
        assert (np.abs(got - ref) <= bound + 2.0 ** -24 * np.abs(ref)).all()
    assert np.array_equal(rows[0][:, (m.heads + m.kv) * 128:], rows[1][:, (m.heads + m.kv) * 128:])   # values as they were
    for leaf in (3, 5, 6):
        path = [leaf]
        while parents[path[0]] >= 0:
            path.insert(0, parents[path[0]])
        one = td.Decoder(m, 128)
        one.prompt(prompt)
        for i in path:
            close(tree[i], one.forward([tokens[i]], [-1])[0])
            one.keep([0])
