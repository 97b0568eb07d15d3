"""Workspaces that a caller gives to the attention and the eviction: a buffer's own size is taken where none is said, an address alone
has none and is refused. CPU only (nothing runs)."""
import ctypes

import pytest

import p8x
from test_kv_refusals import A, cache, drafts


class Buffer(p8x.DeviceBuffer):
    """a buffer of some size that is never touched"""

    def __init__(self, nbytes):
        self.nbytes, self.ptr = nbytes, ctypes.c_void_p(A)

    def free(self):
        pass


def attn(**o):
    return p8x.AttnTree(cache(), A, **o, **drafts())._args[-1]


def evict(**o):
    return p8x.KvEvict(cache(), 16, A, A, pos=A, **o)._args[-1]._obj.workspace_bytes


@pytest.mark.parametrize("make", [attn, evict])
def test_size_of_a_workspace(make):
    assert make(workspace=Buffer(4096)) == 4096
    assert make(workspace=Buffer(4096), workspace_bytes=1024) == 1024   # part of it
    assert make(workspace=A, workspace_bytes=1024) == 1024
    with pytest.raises(p8x.P8xError, match="workspace_bytes"):
        make(workspace=A)
    with pytest.raises(p8x.P8xError, match="workspace_bytes"):
        make(workspace=Buffer(4096), workspace_bytes=4097)


def test_attention_without_a_workspace():
    assert attn(workspace=0, workspace_bytes=0) == 0 and attn(workspace=0) == 0
