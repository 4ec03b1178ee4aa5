"""Calls that paged_attention_decode's C entry has to refuse, before any CUDA call (the pointers here are
never dereferenced; one that is not refused would end in a launch error on a machine without a GPU)."""

import ctypes

import pytest
import torch

from gdn_b200 import _lib

MB = 1 << 20
L3 = ctypes.c_int64 * 3

pytestmark = pytest.mark.skipif(torch.cuda.is_available(), reason="its addresses are made up")


def attend(gdn_lib, **over):
    """B 2, 8 / 2 heads of 128: q and output 4096 bytes each, lse 64, k and v 1024, each cache 81920."""
    a = dict(q=1 * MB, kc=2 * MB, vc=3 * MB, tables=4 * MB, lens=5 * MB, k=6 * MB, v=7 * MB, scale=0.0, window=0,
             sinks=0, out=8 * MB, lse=9 * MB, ws=10 * MB, ws_bytes=1 << 40, dtype=0, B=2, HQ=8, HKV=2, D=128,
             pages=10, page=16, width=4, stride=4, ks=L3(4096, 256, 128), vs=L3(4096, 256, 128), bad=None,
             stream=None)
    a.update(over)
    return gdn_lib.gdn_paged_attention_decode(*a.values())


@pytest.mark.parametrize("over", [
    # CTAs write rows of the output while others, ahead of them, still read new rows
    dict(out=6 * MB), dict(out=7 * MB), dict(out=6 * MB + 1008), dict(out=7 * MB - 4080),
    dict(k=8 * MB + 4080), dict(v=8 * MB - 1008),
    dict(lse=6 * MB), dict(lse=7 * MB + 1020), dict(lse=1 * MB + 4092), dict(lse=8 * MB - 60),
    dict(lse=2 * MB + 81916), dict(lse=3 * MB), dict(lse=4 * MB + 28), dict(lse=5 * MB + 4),
    dict(out=4 * MB + 16), dict(out=5 * MB - 4080),
])
def test_outputs_may_not_overlap_inputs(gdn_lib, over):
    assert attend(gdn_lib, **over) == _lib.GDN_ERR_ALIAS


@pytest.mark.parametrize("over", [
    dict(), dict(out=6 * MB + 1024), dict(out=7 * MB - 4096), dict(lse=8 * MB + 4096), dict(lse=1 * MB + 4096),
    dict(lse=None), dict(k=None, v=None, out=6 * MB),
])
def test_neighbours_are_no_overlap(gdn_lib, over):
    assert attend(gdn_lib, **over) == _lib.GDN_ERR_LAUNCH      # as far as a machine without a GPU goes
