"""paged_attention_decode with one long row among as many short ones as fill the GPU.

Tolerances: those of test_paged_attention_gpu, whose inputs these are.
"""

import pytest
import torch

import gdn_b200
from test_paged_attention_gpu import check, expect, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D,B,HQ,HKV", [(128, 148, 4, 2), (128, 74, 8, 4), (256, 148, 2, 1), (64, 148, 4, 2),
                                        (128, 296, 4, 2)])
@pytest.mark.parametrize("longest", [1500, 1700, 5000])     # on both sides of where rows are cut
def test_one_long_row(D, B, HQ, HKV, longest):
    lens = [1 + i % 40 for i in range(B)]
    lens[B // 3], lens[B // 2] = longest, 0
    x = make(lens, HQ, HKV, D, 16, seed=B + D)
    want = expect(x)
    first = gdn_b200.paged_attention_decode(**x)
    check(x, first, want)
    again = gdn_b200.paged_attention_decode(**x)
    assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])
