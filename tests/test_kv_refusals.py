"""Argument checks of the calls between the linears: all of them on the host, before any GPU work."""
import ctypes

import pytest

import p8x

A = 0x1000   # an address that is never read


def cache(**o):
    a = dict(dtype=p8x.F16, n_seq=2, n_kv=2, head_dim=128, k=A, v=A, page_stride=4096, head_stride=2048, slot_stride=128, page_size=16, n_pages=8,
             len=A, max_len=64, pages=A, ld_pages=4)
    return p8x.KvCache(**{**a, **o})


def drafts(**o):
    a = dict(n_tokens=4, max_tokens=3, first=A, k=A, v=A, n_heads=4, q=A, scale=0.1)
    return {**a, **o}


BAD_CACHE = [dict(dtype=p8x.F32), dict(n_seq=0), dict(n_kv=0), dict(max_len=0), dict(head_dim=96), dict(head_dim=0), dict(k=None), dict(v=None), dict(len=None),
             dict(k=A + 8), dict(v=A + 2), dict(page_stride=4100), dict(slot_stride=64), dict(slot_stride=132), dict(head_stride=64), dict(page_size=24),
             dict(page_size=0), dict(n_pages=0), dict(ld_pages=3), dict(n_seq=70000), dict(max_len=(1 << 30) + 1),
             dict(pages=None, ld_pages=0, page_size=63), dict(pages=None, ld_pages=0, page_size=64, n_pages=1)]
BAD_DRAFTS = [dict(n_tokens=-1), dict(max_tokens=-1), dict(first=None), dict(k=None), dict(v=None), dict(kv_dtype=p8x.BF16), dict(k=A + 4),
              dict(ld_kv=130), dict(ld_kv=64), dict(head_stride_kv=64), dict(head_stride_kv=130)]
BAD_QUERIES = [dict(max_tokens=65), dict(q=None), dict(n_heads=3), dict(n_heads=0), dict(q_dtype=p8x.BF16), dict(q=A + 8), dict(ld_q=514), dict(head_stride_q=130),
               dict(scale=float("nan")), dict(scale=float("inf")), dict(q_dtype=p8x.F16, ld_q=516)]


def attn(c, d, **o):
    return p8x.AttnTree(c, **{**dict(out=A, workspace=A, workspace_bytes=64), **o}, **d)


def score(c, d, **o):
    return p8x.KvScore(c, **{**dict(lse=A, score=A, score_out=A), **o}, **d)


def append(c, d, **o):
    return p8x.KvAppend(c, **o, **d)


def evict(c, **o):
    return p8x.KvEvict(c, **{**dict(budget=16, score=A, len_out=A, pos=A, n_sink=2, n_recent=3, workspace=A, workspace_bytes=1 << 20), **o})


def refused(call):
    with pytest.raises(p8x.P8xError) as e:
        call.run()
    assert call._name in str(e.value)


@pytest.mark.parametrize("bad", BAD_CACHE, ids=str)
def test_bad_caches(bad):
    for make in (attn, score, append):
        refused(make(cache(**bad), drafts()))
    refused(evict(cache(**bad)))


@pytest.mark.parametrize("bad", BAD_DRAFTS, ids=str)
def test_bad_drafts(bad):
    for make in (attn, score, append):
        if not (make is score and bad == dict(v=None)):   # scores read no values
            refused(make(cache(), drafts(**bad)))


@pytest.mark.parametrize("bad", BAD_QUERIES, ids=str)
def test_bad_queries(bad):
    refused(attn(cache(), drafts(**bad)))
    refused(score(cache(), drafts(**bad)))


@pytest.mark.parametrize("bad", [dict(out=None), dict(out=A + 8), dict(ld_out=514), dict(head_stride_out=64), dict(workspace=A + 4)], ids=str)
def test_bad_attn(bad):
    refused(attn(cache(), drafts(), **bad))


def test_bad_score_append():
    for bad in (dict(lse=None), dict(score=None, score_out=A), dict(decay=float("nan"))):
        refused(score(cache(), drafts(), **bad))
    refused(append(cache(), drafts(max_tokens=65), accept=A))   # the accepted set has 64 bits


@pytest.mark.parametrize("bad", [dict(budget=0), dict(n_sink=-1), dict(n_recent=-1), dict(n_sink=10, n_recent=7), dict(score=None, score_out=A), dict(len_out=None),
                                 dict(pos=None), dict(workspace_bytes=100), dict(workspace=A + 4), dict(n_sink=(1 << 31) - 1, n_recent=16)], ids=str)
def test_bad_evict(bad):
    refused(evict(cache(), **bad))


@pytest.mark.parametrize("bad", [dict(n=-1), dict(C=0), dict(C=p8x.MAX_DRAFT * 512 + 1), dict(h=None), dict(x=None, h_out=None), dict(h_dtype=3), dict(y_dtype=9),
                                 dict(x_dtype=-1), dict(gate=A, gate_dtype=7), dict(post=3), dict(pre=-1), dict(gate=A, gate_act=2), dict(ldh=31), dict(ldy=31), dict(ldx=31),
                                 dict(ldho=31), dict(gate=A, ld_gate=31), dict(h=A + 2), dict(x=A + 1, x_dtype=p8x.F16), dict(w_pre=A + 2)], ids=str)
def test_bad_norm(bad):
    a = dict(n=2, C=32, h=A, y=A, h_out=A, x=A)
    refused(p8x.NormResidual(**{**a, **bad}))


def test_null_structs():
    L = p8x.lib()
    c, d = cache().c, p8x._drafts(cache(), **drafts())
    assert L.p8x_norm_residual(None, None) == p8x.P8X_ERR_ARG
    assert L.p8x_attn_tree(None, ctypes.byref(d), A, 512, 0, None, None, 0, None) == p8x.P8X_ERR_ARG
    assert L.p8x_attn_tree(ctypes.byref(c), None, A, 512, 0, None, None, 0, None) == p8x.P8X_ERR_ARG
    assert L.p8x_kv_evict(ctypes.byref(c), None, None) == p8x.P8X_ERR_ARG
    assert L.p8x_attn_workspace(None, None) == 0 and L.p8x_kv_evict_workspace(None, 4) == 0


def test_nothing_to_do_is_no_error():
    p8x.NormResidual(0, 32, h=A, x=A).run()
    attn(cache(), drafts(n_tokens=0, max_tokens=0)).run()


def test_slot_strides_beyond_offsets_within_a_page():
    """attention and scores keep a slot's offset in its half page in 32 bits"""
    big = dict(slot_stride=1 << 26, head_stride=128, page_stride=1 << 31)
    for make in (attn, score):
        with pytest.raises(p8x.P8xError) as e:
            make(cache(**big), drafts()).run()
        assert e.value.code == p8x.P8X_ERR_UNSUPPORTED if hasattr(e.value, "code") else "2^26" in str(e.value)
