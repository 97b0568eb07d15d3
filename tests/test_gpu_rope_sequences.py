"""p8x_kv_append_rope over very many sequences, one of them long."""
import numpy as np
import pytest

import p8x
from kvcase import F16, from_bits, half_ulp, to_bits
from test_gpu_rope import reference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("S,long", [(300, 5000), (65535, 200000)])
def test_a_long_prompt_among_single_tokens(S, long):
    """every sequence one token but for one; all but that one and the last without a page"""
    D, at = 64, S // 3
    page = (long + 15) // 16 * 16
    toks = np.ones(S, np.int64)
    toks[at] = long
    first = np.concatenate([[0], np.cumsum(toks)]).astype(np.int32)
    n = int(first[-1])
    rng = np.random.default_rng(S)
    k, v = (to_bits(rng.standard_normal((n, D)), F16) for _ in range(2))
    dev = p8x.DeviceBuffer.from_numpy
    table = np.full((S, 1), -1, np.int32)
    table[at], table[-1] = 1, 0
    lens = rng.integers(0, 9, S).astype(np.int32)
    lens[at] = 0
    kd, vd = (dev(np.zeros((2, page, D), np.uint16)) for _ in range(2))
    ln, new = dev(lens), dev(np.full(S, -1, np.int32))
    cache = p8x.KvCache(F16, S, 1, D, kd, vd, page_stride=page * D, head_stride=D, slot_stride=D, page_size=page, n_pages=2, len=ln, max_len=page,
                        pages=dev(table), ld_pages=1)
    freq, amp = p8x.rope_frequencies(D, 10000.0)
    rot = p8x.Rotation(D, dev(freq), amplitude=amp)
    p8x.KvAppendRope(cache, rot, len_out=new, n_tokens=n, max_tokens=long, first=dev(first), k=dev(k), v=dev(v), kv_dtype=F16).run()
    p8x.synchronize()
    assert np.array_equal(new.to_numpy(np.int32, (S,)), lens + toks)
    gk, gv = (b.to_numpy(np.uint16, (2, page, D)) for b in (kd, vd))
    a = first[at]
    assert np.array_equal(gv[1, :long], v[a:a + long]) and not gv[1, long:].any() and not gk[1, long:].any()
    assert np.array_equal(gv[0, lens[-1]], v[-1]) and np.count_nonzero(gv[0].any(1)) == 1 and np.count_nonzero(gk[0].any(1)) == 1
    # all of them as p8x_rope has them, some against the formula
    turned = dev(np.zeros((long, D), np.uint16))
    p8x.Rope(rot, long, D, dev(np.arange(long, dtype=np.int32)), n_heads=1, q=dev(k[a:a + long]), q_dtype=F16, q_out=turned, q_out_dtype=F16).run()
    p8x.synchronize()
    assert np.array_equal(gk[1, :long], turned.to_numpy(np.uint16, (long, D)))
    some = np.unique(np.concatenate([np.arange(500), np.arange(0, long, 97), [long - 1]]))
    for rows, slots, got in ((k[a + some], some, gk[1, some]), (k[-1:], lens[-1:], gk[0, lens[-1]:lens[-1] + 1])):
        ref, bound = reference(from_bits(rows, F16)[:, None], slots, freq, p8x.ROPE_HALF, D, amp)
        assert (np.abs(from_bits(got, F16) - ref[:, 0]) <= bound[:, 0] + half_ulp(F16) * (np.abs(ref[:, 0]) + bound[:, 0]) + 2.0 ** -25).all()
