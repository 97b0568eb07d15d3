"""The ordering check of the K-chunk fix-up (test_asm_ordering) on the attention's unit, whose workgroups publish records of
a segment's parts the same way. CPU only (hipcc cross-compiles)."""
import os
import subprocess

import pytest

from test_asm_ordering import CSRC, HIPCC, hipflags, unordered_publications


@pytest.mark.skipif(not os.path.exists(HIPCC), reason="hipcc not installed")
def test_attn_records_complete_before_arrival(tmp_path):
    out = str(tmp_path / "attn.s")
    subprocess.run([HIPCC] + hipflags() + ["--cuda-device-only", "-S", os.path.join(CSRC, "p8x_attn.hip"), "-o", out], check=True,
                   stderr=subprocess.DEVNULL, timeout=600)
    n, bad = unordered_publications(open(out).read().splitlines())
    assert n > 0 and bad == 0, f"{bad} of {n} atomic adds follow an sc1 store without s_waitcnt vmcnt(0)"
