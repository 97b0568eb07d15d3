"""Batches of many sequences and sequences that are none: p8x_attn_prompt where segments of more than 64 sequences are split over
workgroups, and `first` out of order, in full against the formula."""
import ctypes

import numpy as np
import pytest

import p8x
from kvcase import BF16, F16, F32, from_bits
from promptcase import Prompt

pytestmark = pytest.mark.gpu


# 128 compute units' worth of segments at most, so that they are split; 150 of up to 64 rows take two rounds of workgroups
@pytest.mark.parametrize("S,most,heads", [(70, 40, 4), (100, 6, 4), (150, 3, 8)])
@pytest.mark.parametrize("cache,q", [(F16, F16), (BF16, F32)])
def test_split_segments_of_many_sequences(S, most, heads, cache, q):
    rng = np.random.default_rng(S)
    toks = rng.integers(0, most + 1, S)
    lens = toks + rng.integers(0, 300, S)
    for s, n in ((1, 2600), (S // 2, 1), (63, 1900), (64, 3100), (S - 1, 1500)):
        lens[s], toks[s] = n, max(1, min(toks[s], n))
    toks[0] = toks[65] = 0
    c = Prompt(lens.tolist(), toks.tolist(), cache=cache, q=q, heads=heads, kv=1, page=64, seed=190 + S)
    cd = c.make_cache()
    d = p8x._drafts(cd, n_tokens=c.n, max_tokens=c.tk, first=c.dev(c.first), n_heads=c.H, q=c.dev(c.qb), q_dtype=c.qt, scale=c.scale)
    assert p8x.lib().p8x_attn_prompt_workspace(ctypes.byref(cd.c), ctypes.byref(d)) > 0   # may be split
    c.check(*c.run())


@pytest.mark.parametrize("cache,q", [(F16, F16), (BF16, BF16), (F16, F32)])
def test_rows_out_of_order_leave_the_others_right(cache, q):
    c = Prompt([30, 40, 50, 300], [4, 5, 6, 7], cache=cache, q=q, seed=195)
    want, wl, tol, ltol = c.causal()
    c.first = np.array([0, 4, 2, 90, 97], np.int32)   # the second's end before its start, the third's and the last's behind the rows
    out, lse = c.run()
    assert (np.abs(from_bits(out, c.out_t) - want) <= tol)[:4].all() and (np.abs(lse - wl) <= ltol)[:4].all()
    assert (out[4:] == (7.0 if c.out_t == F32 else 0x7E7E)).all() and (lse[4:] == 7.0).all()
