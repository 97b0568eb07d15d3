"""Eviction of rows whose keys stay in registers, at the lengths where the number of keys a lane changes, of sequences far shorter than
their rows, and of protected slots that are more than the budget: every bit, as in test_gpu_kv."""
import numpy as np
import pytest

import p8x
from kvcase import Case
from test_gpu_kv import evict_ref, run_evict

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["skewed", "ties", "equal", "odd"])
@pytest.mark.parametrize("max_len", [63, 64, 128, 129, 2047, 2048, 2049, 4096, 4097, 8191, 8192, 8193])
def test_rows_around_the_forms_limits(max_len, kind):
    lens = [max_len, max_len // 2 + 1, 1]
    run_evict(Case(lens, [0] * 3, fused=False, heads=1, kv=1, D=64, page=64, max_len=max_len, seed=max_len), max(1, max_len // 3), 2 if max_len > 6 else 0,
              max_len // 16, kind)


@pytest.mark.parametrize("max_len", [200, 3000, 8000])
def test_short_sequences_in_long_rows(max_len):
    """waves without slots, budgets just above and below the slots in use"""
    for budget in (1, 63, 64, 65, 99):
        run_evict(Case([100, 64, 65, 0, 2], [0] * 5, fused=False, kv=2, D=64, page=32, max_len=max_len, seed=budget), budget, 0, min(budget, 7), "ties")


@pytest.mark.parametrize("n", [40, 1500, 5000, 9000])
def test_more_protected_slots_than_stay(n):
    """positions need not be different: of too many protected slots the lowest stay"""
    rng = np.random.default_rng(n)
    c = Case([n, n // 2], [0, 0], fused=False, heads=2, kv=2, D=64, page=64, seed=n)
    shape, budget = (2, 2, c.max_len), n // 4
    score = rng.random(shape).astype(np.float32)
    pos = np.where(rng.random(shape) < 0.6, 1, rng.integers(10, 50, shape)).astype(np.int32)   # some 0.6 below n_sink
    cache = c.make_cache()
    sd, pd, so, po, lo = (c.dev(a) for a in (score, pos, np.zeros_like(score), np.zeros_like(pos), np.zeros(2, np.int32)))
    p8x.KvEvict(cache, budget, score=sd, len_out=lo, score_out=so, pos=pd, pos_out=po, n_sink=2, n_recent=1).run()
    p8x.synchronize()
    k, v, rs, rp, rl = evict_ref(c, budget, 2, 1, score, pos, np.zeros_like(score), np.zeros_like(pos))
    assert np.array_equal(lo.to_numpy(np.int32, (2,)), rl) and np.array_equal(so.to_numpy(np.float32, shape), rs)
    assert np.array_equal(po.to_numpy(np.int32, shape), rp)
    assert np.array_equal(c.kd.to_numpy(np.uint16, c.pool_shape), k) and np.array_equal(c.vd.to_numpy(np.uint16, c.pool_shape), v)
