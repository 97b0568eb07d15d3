"""Attention where what lies below the sinks of test_gpu_attn_sinks is a few slots only, so that most of their tile is not there:
the cache's last slots, drafted tokens, half tiles without a page. Tolerances as there."""
import numpy as np
import pytest

from test_gpu_attn_sinks import ROWS, TYPES, check, levels_case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cache,q", TYPES)
@pytest.mark.parametrize("toks,heads", ROWS)
@pytest.mark.parametrize("few", [1, 3, 17, 33])
def test_last_slots_and_drafts(few, toks, heads, cache, q):
    """with and without values of the drafted tokens"""
    level = np.concatenate([np.zeros(256), np.full(few, -15.0)])
    c = levels_case(level, np.where(level < 0, 20000.0, 0.0), toks, heads, 1, 128, cache, q, few)
    check(c, False)
    c.knb[:] = 0   # level 0
    c.vnb[:] = 0
    check(c, False)


@pytest.mark.parametrize("cache,q", TYPES)
@pytest.mark.parametrize("toks,heads", ROWS)
def test_half_tiles(toks, heads, cache, q):
    level = np.concatenate([np.zeros(256), np.full(512, -15.0)])
    c = levels_case(level, np.where(level < 0, 20000.0, 0.0), toks, heads, 1, 128, cache, q, 5, page=16)
    c.pages[0, 17::2] = -1
    check(c, False)
