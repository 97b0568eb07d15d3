"""p8x_attn_prompt where segments are split over workgroups and joined: infinities and NaN that a token sees reach it as they do
without a split."""
import ctypes

import numpy as np
import pytest

import p8x
from kvcase import BF16, F16, F32, from_bits, to_bits
from promptcase import Prompt

pytestmark = pytest.mark.gpu
TYPES = [(F16, F16), (BF16, BF16), (F16, F32), (BF16, F32)]
# slots, new tokens, options: long contexts of few rows, so that each segment has several parts
SPLIT = [
    ([5000], [1], dict(heads=4, kv=1, page=64)),
    ([3000], [70], dict(heads=4, kv=1, page=32)),
    ([2600, 0, 4000], [2, 0, 3], dict(heads=4, kv=2, page=64)),
]


def make(shape, cache, q, seed):
    lens, toks, opt = SPLIT[shape]
    return Prompt(lens, toks, cache=cache, q=q, seed=seed, **opt)


def both(c):
    """results split over workgroups, and whole (without a workspace)"""
    cache = c.make_cache()
    d = p8x._drafts(cache, n_tokens=c.n, max_tokens=c.tk, first=c.dev(c.first), n_heads=c.H, q=c.dev(c.qb), q_dtype=c.qt, scale=c.scale)
    assert p8x.lib().p8x_attn_prompt_workspace(ctypes.byref(cache.c), ctypes.byref(d)) > 0
    return c.run(), c.run(workspace=0)


def same(c, split, whole):
    """the same places that are not finite, and the same lse there"""
    a, b = from_bits(split[0], c.out_t), from_bits(whole[0], c.out_t)
    assert np.array_equal(np.isfinite(a), np.isfinite(b))
    assert np.array_equal(np.isnan(split[1]), np.isnan(whole[1])) and np.array_equal(np.isneginf(split[1]), np.isneginf(whole[1]))


@pytest.mark.parametrize("cache,q", TYPES)
@pytest.mark.parametrize("shape", range(len(SPLIT)))
def test_query_of_nan(shape, cache, q):
    c = make(shape, cache, q, 160 + shape)
    clean = c.causal()
    tok, head = c.n - 1, 2
    c.qb[tok, head, 7:8] = to_bits(np.float32(np.nan), q)
    results = both(c)
    other = np.ones((c.n, c.H), bool)
    other[tok, head] = False
    for out, lse in results:
        got = from_bits(out, c.out_t)
        assert np.isnan(got[tok, head]).all() and np.isnan(lse[tok, head])
        assert (np.abs(got - clean[0]) <= clean[2])[other].all() and (np.abs(lse - clean[1]) <= clean[3])[other].all()
    same(c, *results)


@pytest.mark.parametrize("cache,q", TYPES)
@pytest.mark.parametrize("at", ["first", "middle", "all"])
@pytest.mark.parametrize("shape", range(len(SPLIT)))
def test_keys_of_nan_over_whole_parts(shape, at, cache, q):
    """a long range of slots whose keys are NaN: more than a part holds (at most a quarter of the slots here)"""
    c = make(shape, cache, q, 165 + shape)
    clean = c.causal()
    n = c.lens[-1]
    for j in range(*{"first": (0, n // 2 + 1), "middle": (n // 4, 3 * n // 4 + 1), "all": (0, n)}[at]):
        c.row(c.kb, c.S - 1, j)[:, 11] = to_bits(np.float32(np.nan), cache)
    results = both(c)
    a = int(c.first[-2])
    for out, lse in results:
        got = from_bits(out, c.out_t)
        assert np.isnan(got[a:c.n]).all() and np.isnan(lse[a:c.n]).all()
        assert (np.abs(got - clean[0]) <= clean[2])[:a].all() and (np.abs(lse - clean[1]) <= clean[3])[:a].all()
    same(c, *results)


@pytest.mark.parametrize("cache,q", TYPES)
@pytest.mark.parametrize("shape", [0, 1])
def test_keys_of_nan_up_to_any_tile(shape, cache, q):
    """wherever the first parts end: some of these ranges are whole parts and nothing of the next"""
    lens, toks, opt = SPLIT[shape]
    c = make(shape, cache, q, 169)
    call = c.make()
    nan = np.full(c.D, to_bits(np.float32(np.nan), cache), np.uint16)
    for end in range(32, lens[0] - toks[0], 32):
        for j in range(end - 32, end):
            p, o = c.place(0, j)
            at = 2 * c.D * (p * c.page + o)   # one key/value head
            p8x.hip_check(p8x.hip().hipMemcpy(c.kd.addr + at, nan.ctypes.data, nan.nbytes, p8x.H2D), "copy")
        out, lse = c.run(call=call)
        assert np.isnan(from_bits(out, c.out_t)).all() and np.isnan(lse).all(), end


@pytest.mark.parametrize("cache", [F16, BF16])
@pytest.mark.parametrize("at", ["first", "middle", "all"])
def test_infinite_keys_over_whole_parts(at, cache):
    """16-bit queries: scores of inf in the rows of one sign are NaN, scores of -inf in those of the other weigh nothing"""
    c = make(1, cache, cache, 170)
    qq = from_bits(c.qb, cache)
    qq[:, 0::2, 5], qq[:, 1::2, 5] = 1.0, -1.0
    c.qb = to_bits(qq, cache)
    n = c.lens[0]
    span = {"first": (0, n // 2 + 1), "middle": (n // 4, 3 * n // 4 + 1), "all": (0, n)}[at]
    # what the heads of the other sign see of the range: nothing
    hidden = make(1, cache, cache, 170)
    hidden.qb = c.qb
    for j in range(*span):
        c.row(c.kb, 0, j)[:, 5] = to_bits(np.float32(np.inf), cache)
    here = hidden.there
    hidden.there = lambda s, j: here(s, j) and not span[0] <= j < span[1]
    ref, rl, tol, ltol = hidden.causal()
    results = both(c)
    for out, lse in results:
        got = from_bits(out, c.out_t)
        assert np.isnan(got[:, 0::2]).all() and np.isnan(lse[:, 0::2]).all()
        if at == "all":
            assert (got[:, 1::2] == 0).all() and np.isneginf(lse[:, 1::2]).all()
        else:
            assert (np.abs(got - ref) <= tol)[:, 1::2].all() and (np.abs(lse - rl) <= ltol)[:, 1::2].all()
    same(c, *results)


@pytest.mark.parametrize("cache", [F16, BF16])
@pytest.mark.parametrize("shape", range(len(SPLIT)))
def test_infinite_values_beside_scores_of_minus_infinity(shape, cache):
    """a weight of 0 of an infinite value is NaN, also where all weights are 0; lse stays -inf"""
    c = make(shape, cache, cache, 175)
    qq = from_bits(c.qb, cache)
    qq[:, :, 5] = -1.0
    c.qb = to_bits(qq, cache)
    for s in range(c.S):
        for j in range(c.lens[s]):
            c.row(c.kb, s, j)[:, 5] = to_bits(np.float32(np.inf), cache)
        if c.lens[s]:
            c.row(c.vb, s, 700)[:, 9] = to_bits(np.float32(np.inf), cache)
    results = both(c)
    for out, lse in results:
        got = from_bits(out, c.out_t)
        assert np.isnan(got[:, :, 9]).all() and (np.delete(got, 9, 2) == 0).all() and np.isneginf(lse).all()
    same(c, *results)
