"""How far below a row's largest weight others keep their bits (p8x_attn_prompt): to 2^-64 of the sum of the row's weights on an fp16
cache, 2^-110 on a bf16 one, in whole segments, halves and joined parts."""
import numpy as np
import pytest

from kvcase import BF16, F16, F32, from_bits, half_ulp, to_bits
from promptcase import Prompt

pytestmark = pytest.mark.gpu

SHAPES = [
    # slots, new tokens: halves; parts of them; workgroups of 256 rows
    ([640], [20], dict(heads=2, kv=1)),
    ([3000], [3], dict(heads=2, kv=1, page=32)),
    ([2300], [150], dict(heads=2, kv=1, page=64, max_len=2304)),
]


def case(shape, cache, q, out, scores, valued):
    """scores: log2 of each slot's weight, the same for all rows; valued: the slots that have values"""
    lens, toks, o = SHAPES[shape]
    c = Prompt(lens, toks, cache=cache, q=q, out=out, seed=180 + shape, **o)
    c.scale = 1.0
    qq = np.zeros((c.n, c.H, c.D), np.float32)
    qq[:, :, 0] = 1.0
    qq[:, :, 1:] = np.random.default_rng(1).standard_normal((c.n, c.H, c.D - 1))   # of elements that no key has
    c.qb = to_bits(qq, q)
    for j in range(lens[0]):
        k = np.zeros(c.D, np.float32)
        k[0] = scores[j] * np.log(2.0)
        c.row(c.kb, 0, j)[:] = to_bits(k, cache)
        if j not in valued:
            c.row(c.vb, 0, j)[:] = 0
    return c


def check(c, valued):
    """Each weight w, of a sum of 1: half a step (two in a row for scores, sums as in promptcase), on fp16 2^-17 or 2^-22 of the largest of its
    64 slots, and the limit."""
    out, lse = c.run()
    got = from_bits(out, c.out_t)
    ref, rl, _, ltol = c.causal()
    n, nt = c.lens[0], c.toks[0]
    f32 = c.qt == F32
    uw = {(F16, False): 2.0 ** -11, (BF16, False): 2.0 ** -8, (F16, True): 2.0 ** -22, (BF16, True): 2.0 ** -24}[c.cache, f32]
    floor = 0.0 if c.cache == BF16 else 2.0 ** -22 if f32 else 2.0 ** -17
    limit = 2.0 ** -64 if c.cache == F16 else 2.0 ** -110
    k = np.array([from_bits(c.row(c.kb, 0, j)[0, :1], c.cache)[0] for j in range(n)])
    v = np.abs(np.array([from_bits(c.row(c.vb, 0, j)[0], c.cache) for j in range(n)]))
    big = np.abs(k).max()
    es = (c.D + 8) * 2.0 ** -24 * big + 2.0 ** -21 * big + 2.0 ** -22 * big + 2.0 ** -21
    for i in range(nt):
        see = n - nt + i + 1
        w = np.exp(k[:see] - rl[i, 0])
        # the largest of the 64 slots on either side holds that of any tile of at most 64 with the slot in it
        near = np.array([w[max(0, j - 63):j + 64].max() if j in valued else 0.0 for j in range(see)])
        err = ((w * (uw + 2 * es + 2 * (see + 64) * 2.0 ** -24) + floor * near + limit)[:, None] * v[:see]).sum(0) * 1.01
        tol = err + half_ulp(c.out_t) * (np.abs(ref[i]) + err)
        assert (np.abs(got[i] - ref[i]) <= tol).all(), (i, np.abs(got[i] - ref[i]).max(), tol.max(), np.abs(ref[i]).max())
    assert (np.abs(lse - rl) <= ltol).all()
    return got, err


@pytest.mark.parametrize("cache,q,out,depth", [(F16, F32, F32, 30), (F16, F32, F32, 50), (F16, F32, F32, 57), (F16, F32, BF16, 57), (F16, F16, BF16, 57),
                                               (BF16, F32, F32, 57), (BF16, F32, F32, 100), (BF16, BF16, BF16, 100)])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_tail_far_below_a_first_slot(shape, cache, q, out, depth):
    """a first slot without values that takes all but 2^-depth: what is returned is the tail's"""
    n = SHAPES[shape][0][0]
    scores = np.zeros(n)
    scores[0] = depth
    valued = set(range(n // 2, n // 2 + 8))
    got, err = check(case(shape, cache, q, out, scores, valued), valued)
    assert np.abs(got).max() > 8 * np.abs(err).max()   # more than the bounds


@pytest.mark.parametrize("cache,q,out,up", [(F16, F32, F32, 20), (F16, F32, F32, 55), (F16, F16, BF16, 55), (BF16, F32, F32, 55), (BF16, BF16, BF16, 100)])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_slot_below_one_that_follows_a_long_tail(shape, cache, q, out, up):
    """first a slot, then a tail 2^-100 below it, then a slot 2^up above without values: what is returned is the first slot's"""
    n, nt = SHAPES[shape][0][0], SHAPES[shape][1][0]
    scores = np.full(n, -100.0)
    scores[0], scores[n - nt - 70] = 0, up
    valued = {0}
    got, err = check(case(shape, cache, q, out, scores, valued), valued)
    assert np.abs(got).max() > 8 * np.abs(err).max()
