"""Frequencies of rotary positions, and the argument checks of the calls of a prompt: all of them on the host."""
import numpy as np
import pytest

import p8x
from test_kv_refusals import A, BAD_CACHE, cache, drafts, refused

EVERY = dict(kind=p8x.ROPE_YARN, factor=4.0, original=4096, low=1.0, high=32.0)


def turns(freq):
    return np.array([int(f) for f in freq], dtype=object)


@pytest.mark.parametrize("n_rot,base", [(128, 500000.0), (64, 10000.0), (96, 1e6), (8, 2.0), (2, 10000.0)])
@pytest.mark.parametrize("kind", [p8x.ROPE_PLAIN, p8x.ROPE_LINEAR, p8x.ROPE_BANDS, p8x.ROPE_YARN])
def test_frequencies(n_rot, base, kind):
    """the definition in 80-bit numbers; powers, products and quotients in 64 bits are off by some 2^-53 each"""
    factor, original, low, high = 8.0, 8192.0, 1.0, 4.0
    factors = np.linspace(1.0, 3.0, n_rot // 2)
    freq, amp = p8x.rope_frequencies(n_rot, base, kind, factor=factor, original=original, low=low, high=high, factors=factors)
    ld = np.longdouble
    tau = ld(2) * np.arccos(ld(-1))
    for i in range(n_rot // 2):
        th = ld(base) ** (-2 * ld(i) / n_rot) / ld(factors[i])
        if kind == p8x.ROPE_LINEAR:
            th /= factor
        elif kind == p8x.ROPE_BANDS:
            wave = tau / th
            if wave > original / low:
                th /= factor
            elif wave >= original / high:
                a = (original / wave - low) / (high - low)
                th = (1 - a) * th / factor + a * th
        elif kind == p8x.ROPE_YARN:
            def pair(b):
                return n_rot * np.log(original / (b * tau)) / (2 * np.log(ld(base)))
            lo, hi = max(np.floor(pair(high)), 0), min(np.ceil(pair(low)), n_rot - 1)
            a = min(ld(1), max(ld(0), (i - lo) / max(hi - lo, ld(0.001))))
            th = a * th / factor + (1 - a) * th
        want = th / tau
        assert abs(ld(int(freq[i])) / ld(2) ** 64 - want % 1) <= want * ld(2) ** -49 + ld(2) ** -64
    assert amp == (np.float32(0.1 * np.log(8.0) + 1) if kind == p8x.ROPE_YARN else 1.0)


def test_frequencies_of_nothing_and_of_factors_below_one():
    assert len(p8x.rope_frequencies(0)[0]) == 0
    assert p8x.rope_frequencies(64, **{**EVERY, "factor": 0.5})[1] == 1.0
    fast = p8x.rope_frequencies(8, 10000.0, p8x.ROPE_LINEAR, factor=0.01)[0]   # 15.9 turns a position: whole ones do nothing
    assert abs(int(fast[0]) / 2.0 ** 64 - (100 / (2 * np.pi)) % 1) < 1e-13


@pytest.mark.parametrize("bad", [dict(kind=4), dict(kind=-1), dict(base=0.0), dict(base=-2.0), dict(base=float("inf")), dict(base=1.0), dict(factor=0.0),
                                 dict(factor=float("nan")), dict(original=0.0), dict(low=0.0), dict(low=33.0), dict(high=float("inf")),
                                 dict(factors=np.zeros(32)), dict(factors=np.ones(31))], ids=str)
def test_bad_scalings(bad):
    with pytest.raises(p8x.P8xError) as e:
        p8x.rope_frequencies(64, **{**EVERY, **bad})
    assert "p8x_rope_frequencies" in str(e.value)


def test_bad_frequency_counts():
    for n in (-2, 7):
        with pytest.raises(p8x.P8xError):
            p8x.rope_frequencies(n)


def rotation(**o):
    return p8x.Rotation(**{**dict(n_rot=64, freq=A, layout=p8x.ROPE_HALF), **o})


def rope(r=None, **o):
    return p8x.Rope(r or rotation(), **{**dict(n=3, head_dim=128, pos=A, n_heads=4, q=A, n_kv=2, k=A, ld_k=1024), **o})


def append(c=None, d=None, r=None, **o):
    return p8x.KvAppendRope(c or cache(), r or rotation(), **{**dict(n_heads=4, q=A, q_out=A, q_out_dtype=p8x.F16, ld_q_out=512), **o}, **(d or tokens()))


def tokens(**o):
    return {k: v for k, v in drafts(**o).items() if k not in ("n_heads", "q", "scale")}


BAD_ROTATION = [dict(layout=2), dict(layout=-1), dict(n_rot=-8), dict(n_rot=136), dict(n_rot=12), dict(freq=None), dict(freq=A + 8), dict(w_q=A + 4), dict(w_k=A + 8),
                dict(amplitude=float("nan")), dict(amplitude=float("inf"))]


@pytest.mark.parametrize("bad", BAD_ROTATION, ids=str)
def test_bad_rotations(bad):
    refused(rope(rotation(**bad)))
    refused(append(r=rotation(**bad)))


@pytest.mark.parametrize("bad", [dict(n=-1), dict(head_dim=0), dict(head_dim=100), dict(head_dim=264), dict(pos=None), dict(n_heads=-1), dict(q=None), dict(q=A + 8),
                                 dict(q_dtype=3), dict(k_out_dtype=7, k_out=A), dict(ld_q=514), dict(ld_q=64), dict(head_stride_q=64), dict(head_stride_q=130),
                                 dict(q_out=A + 4), dict(q_out=A, q_out_dtype=p8x.F16), dict(q_out=A, ld_q_out=1024), dict(k_out=A, ld_k=1024, ld_k_out=516),
                                 dict(n_heads=0, n_kv=0), dict(n_heads=70000, ld_q=70000 * 128)], ids=str)
def test_bad_ropes(bad):
    refused(rope(**bad))


def test_no_tokens_need_no_positions():
    rope(n=0, pos=None).run()


@pytest.mark.parametrize("bad", BAD_CACHE, ids=str)
def test_bad_caches(bad):
    refused(append(cache(**bad)))
    refused(prompt(cache(**bad)))


@pytest.mark.parametrize("bad", [dict(n_tokens=-1), dict(max_tokens=-1), dict(first=None), dict(k=None), dict(v=None), dict(kv_dtype=p8x.BF16), dict(k=A + 4),
                                 dict(ld_kv=130), dict(head_stride_kv=64)], ids=str)
def test_bad_tokens(bad):
    refused(append(d=tokens(**bad)))


def test_bad_append_queries():
    for bad in (dict(q_out=A + 8), dict(ld_q_out=514), dict(q_dtype=9)):
        refused(append(**bad))


def prompt(c=None, **o):
    d = dict(n_tokens=4, max_tokens=3, first=A, n_heads=4, q=A, scale=0.1, out=A, workspace=A, workspace_bytes=64)
    d.update(o)
    return p8x.AttnPrompt(c or cache(), **d)


@pytest.mark.parametrize("bad", [dict(n_tokens=-1), dict(max_tokens=-1), dict(first=None), dict(n_heads=3), dict(n_heads=0), dict(q=None), dict(q=A + 8),
                                 dict(q_dtype=p8x.BF16), dict(ld_q=514), dict(head_stride_q=130), dict(scale=float("nan")), dict(mask=A), dict(out=None),
                                 dict(out=A + 8), dict(out_dtype=3), dict(ld_out=514), dict(head_stride_out=64), dict(workspace=A + 4),
                                 dict(q_dtype=p8x.F16, out_dtype=p8x.F32), dict(n_heads=70000, ld_q=128 * 70000, ld_out=128 * 70000)], ids=str)
def test_bad_prompts(bad):
    refused(prompt(**bad))


def test_bad_workspace():
    with pytest.raises(p8x.P8xError):
        prompt(workspace=A, workspace_bytes=None)
    assert p8x.lib().p8x_attn_prompt_workspace(None, None) == 0


def test_no_tokens_is_no_work():
    prompt(n_tokens=0, q=None, out=None).run()
    prompt(max_tokens=0, q=None, out=None).run()


def test_more_tokens_than_are_counted():
    refused(append(d=tokens(max_tokens=(1 << 30) + 1)))
    refused(prompt(max_tokens=(1 << 30) + 1))
    refused(prompt(n_tokens=1 << 29))
