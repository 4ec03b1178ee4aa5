"""Where paged_attention_decode leaves rows whole: seen in the workspace, which only cut rows need."""

import pytest

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
