"""The plan of a paged_attention_decode call, as seen in its workspace, which only cut rows need; and the
sizes at which the serving operators' C entries stop."""

import ctypes

import pytest

from gdn_b200 import _lib

# CTAs that are resident at a time: 148 SMs, two CTAs each for heads of 64 and 128, one for 256
PLACES = {64: 296, 128: 296, 256: 148}
BLOCK = {64: 128, 128: 64, 256: 64}         # tokens a CTA takes at a time


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("waves", [1, 2, 3])
@pytest.mark.parametrize("HKV", [1, 2, 4])
def test_a_long_row_is_cut_whatever_the_number_of_rows(gdn_lib, D, waves, HKV):
    """The lengths are not known on the host: as many rows as CTAs do not share the work evenly when one
    of them is long."""
    ws = gdn_lib.gdn_paged_attention_workspace_bytes
    for short in (0, 1, 8):                  # at and just below a multiple of the places
        B = (waves * PLACES[D] - short) // HKV
        for n in (26 * BLOCK[D], 8192, 32768, 131072):
            assert ws(B, 8 * HKV, HKV, D, n) > 0, (B, HKV, n)


@pytest.mark.parametrize("D", [64, 128, 256])
def test_short_rows_stay_whole(gdn_lib, D):
    ws = gdn_lib.gdn_paged_attention_workspace_bytes
    for B in (1, 100, 148, 296, 592, 5000, 30000):
        assert ws(B, 8, 1, D, BLOCK[D]) == 0                   # one block each: nothing to share
    assert ws(PLACES[D], 8, 1, D, 16 * BLOCK[D]) == 0
    assert ws(1, 8, 1, D, 2 * BLOCK[D]) == 0


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("B,HQ,HKV", [(1, 8, 2), (3, 48, 2), (500, 8, 8), (37, 64, 8), (148, 16, 2), (148, 8, 1),
                                      (296, 24, 2), (65535, 1, 1)])
def test_workspaces_grow_with_the_tokens(gdn_lib, D, B, HQ, HKV):
    """So a workspace for more tokens, as for the whole table, is enough for fewer, as of a window."""
    sizes = [gdn_lib.gdn_paged_attention_workspace_bytes(B, HQ, HKV, D, n)
             for n in (0, 1, 64, 100, 300, 600, 1000, 1600, 1700, 3300, 5000, 100000, 2**31 - 2048)]
    assert all(a <= b for a, b in zip(sizes, sizes[1:])) and sizes[0] == 0 and sizes[-1] > 0


MB = 1 << 20
L3 = ctypes.c_int64 * 3


def attend(gdn_lib, **over):
    """No pointer is dereferenced: the entry refuses each of these calls before it comes to the GPU."""
    a = dict(q=1 * MB, kc=2 * MB, vc=3 * MB, tables=4 * MB, lens=5 * MB, k=6 * MB, v=7 * MB, scale=0.0, window=0,
             sinks=0, out=8 * MB, lse=9 * MB, ws=10 * MB, ws_bytes=0, dtype=0, B=2, HQ=8, HKV=2, D=128,
             pages=10, page=16, width=4, stride=4, ks=L3(4096, 256, 128), vs=L3(4096, 256, 128), bad=None,
             stream=None)
    a.update(over)
    return gdn_lib.gdn_paged_attention_decode(*a.values())


@pytest.mark.parametrize("window,sinks,tokens", [(0, 0, 16000), (3000, 0, 3000), (3000, 100, 3100), (15999, 0, 15999),
                                                 (15000, 5000, 16000), (2**30 - 1, 2**30 - 1, 16000)])
def test_a_call_asks_for_what_it_can_see(gdn_lib, window, sinks, tokens):
    """One byte less than the size for its tokens is refused: those of the table of 1000 pages of 16, or the
    window and the first tokens where that is less."""
    size = gdn_lib.gdn_paged_attention_workspace_bytes(2, 8, 2, 128, tokens)
    assert size > 0
    assert attend(gdn_lib, width=1000, stride=1000, window=window, sinks=sinks,
                  ws_bytes=size - 1) == _lib.GDN_ERR_SHAPE


@pytest.mark.parametrize("over", [dict(B=65536), dict(B=65535, HQ=130, HKV=130)])
def test_documented_limits_of_attention(gdn_lib, over):
    assert attend(gdn_lib, **over) == _lib.GDN_ERR_SHAPE


@pytest.mark.parametrize("B,K,V", [(1, 1, 2**26 + 1), (2**25, 1, 10), (2**19, 64, 10)])
def test_documented_limits_of_selection(gdn_lib, B, K, V):
    assert gdn_lib.gdn_beam_select(MB, 0, V * K, V, 2 * MB, None, 0, B, K, V, 1, 3 * MB, 4 * MB, 5 * MB, 6 * MB,
                                   1 << 50, None) == _lib.GDN_ERR_SHAPE
