"""p8x_attn_prompt where the rows are many: eight waves a workgroup, whole segments, ragged sequences, several row tiles."""
import numpy as np
import pytest

from kvcase import BF16, F16, F32, from_bits, to_bits
from promptcase import Prompt

pytestmark = pytest.mark.gpu

MANY = [
    # slots, new tokens, options: at least a row tile of 256 for each of the 256 compute units
    ([300], [300], dict(heads=256, kv=32, page=48)),
    ([700, 90, 513], [200, 90, 257], dict(heads=128, kv=64, page=16)),
    ([257] * 9, [65, 0, 257, 1, 256, 100, 128, 33, 64], dict(heads=80, kv=16, page=32)),
    ([1100], [1030], dict(heads=64, kv=64, page=64)),
]


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("cache", [F16, BF16])
@pytest.mark.parametrize("shape", range(len(MANY)))
def test_many_rows(shape, cache, D):
    lens, toks, o = MANY[shape]
    c = Prompt(lens, toks, cache=cache, q=cache, D=D, seed=100 + shape, layout=("head", "slot")[shape % 2], **o)
    out, lse = c.run()
    c.check(out, lse)
    again = c.run()
    assert out.tobytes() == again[0].tobytes() and lse.tobytes() == again[1].tobytes()


@pytest.mark.parametrize("cache", [F16, BF16])
def test_many_rows_f32(cache):
    lens, toks, o = MANY[0]
    c = Prompt(lens, toks, cache=cache, q=F32, seed=110, **o)
    c.check(*c.run())


def test_pages_outside_the_pool():
    c = Prompt([400, 333], [250, 333], cache=BF16, q=BF16, heads=256, kv=32, page=16, seed=111)
    c.pages[0, 1], c.pages[0, 20], c.pages[1, :3] = -1, c.n_pages, -7
    c.check(*c.run())


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("what", [np.inf, -np.inf, np.nan])
def test_odd_values_of_later_tokens(what, D):
    c = Prompt([420], [300], cache=F16, q=F16, D=D, heads=256, kv=32, page=64, seed=112)
    clean = c.causal()
    for j in (125, 200, 419):
        c.row(c.vb, 0, j)[:, 5] = to_bits(np.float32(what), F16)
    got = from_bits(c.run()[0], F16)
    ok = np.abs(got - clean[0]) <= clean[2]
    assert ok[:5].all() and ok[:, :, :5].all() and ok[:, :, 6:].all()
    assert not np.isfinite(got[5:, :, 5]).any()


def test_odd_keys_of_later_tokens():
    c = Prompt([300], [300], cache=BF16, q=BF16, heads=256, kv=32, page=64, seed=113)
    clean = c.causal()
    c.row(c.kb, 0, 130)[:] = to_bits(np.float32(np.nan), BF16)
    got = from_bits(c.run()[0], BF16)
    assert (np.abs(got - clean[0]) <= clean[2])[:130].all() and not np.isfinite(got[130:]).any()


@pytest.mark.parametrize("depth", [10, 30])
@pytest.mark.parametrize("cache", [F16, BF16])
def test_sink(cache, depth):
    """a first slot that takes nearly all, without values: the others, of the same weight, decide the result"""
    c = Prompt([300], [260], cache=cache, q=cache, heads=256, kv=32, page=64, seed=114)
    for j in range(300):
        c.row(c.kb, 0, j)[:] = 0
    c.row(c.kb, 0, 0)[:, 0] = to_bits(np.float32(depth / 8.0 / c.scale), cache)
    for j in range(64):   # the sink and the rest of its tile
        c.row(c.vb, 0, j)[:] = 0
    q = from_bits(c.qb, cache).astype(np.float32)
    q[:, :, 0] = 8.0
    c.qb = to_bits(q, cache)
    got, ref = from_bits(c.run()[0], cache), c.causal()[0]
    u = {F16: 2.0 ** -11, BF16: 2.0 ** -8}[cache]
    # weights of e^-depth / (1 + 299 e^-depth), held to u of themselves behind the sink's tile; sums of at most 300 terms
    tol = (u + 400 * 2.0 ** -23 + 2.0 ** -15) * 236 * np.exp(-float(depth)) * 5.0 + u * np.abs(ref) + (2.0 ** -25 if cache == F16 else 0)
    assert (np.abs(got - ref) <= tol).all()


def test_sequences_that_overlap():
    # `first` goes up and down: every other sequence has the same token, which makes more segments than any workspace is meant for
    S = 81
    c = Prompt([900] * S, [1] + [0] * (S - 1), cache=F16, q=F16, heads=32, kv=8, page=64, seed=130)
    c.pages[:] = c.pages[0]
    want = c.causal()
    c.first = np.array([i % 2 for i in range(S + 1)], np.int32)
    out, lse = c.run()
    # a workgroup writes the whole of a row or nothing of it
    assert (np.abs(from_bits(out[:1], F16) - want[0][:1]) <= want[2][:1]).all()
    assert (np.abs(lse[:1] - want[1][:1]) <= want[3][:1]).all()


@pytest.mark.parametrize("cache,q", [(F16, F16), (BF16, F32)])
@pytest.mark.parametrize("toks", [1, 5, 32])
@pytest.mark.parametrize("n", [32, 33, 64, 65, 96, 97, 129, 544, 545, 897, 1500])
def test_halves_and_parts_end_anywhere(n, toks, cache, q):
    # 128 rows: two halves of the slots, each of none, one or more tiles, whole or in parts
    c = Prompt([n], [min(n, toks)], cache=cache, q=q, heads=16, kv=4, page=32, seed=140 + n)
    c.check(*c.run())


@pytest.mark.parametrize("n", [70, 700])
@pytest.mark.parametrize("what", [np.inf, np.nan])
def test_odd_values_and_missing_pages_in_the_second_half(what, n):
    c = Prompt([n, n - 3], [30, 1], cache=BF16, q=BF16, heads=16, kv=4, page=16, seed=150)
    c.pages[0, (n - 40) // 16] = -1
    clean = c.causal()
    for j in (n - 1, n - 9):   # the last tokens', hidden from those before
        c.row(c.vb, 0, j)[:, 3] = to_bits(np.float32(what), BF16)
    got = from_bits(c.run()[0], BF16)
    ok = np.abs(got - clean[0]) <= clean[2]
    assert ok[:30 - 9].all() and ok[:31, :, :3].all() and ok[:31, :, 4:].all() and ok[30].all()
    assert not np.isfinite(got[30 - 9:30, :, 3]).any()
