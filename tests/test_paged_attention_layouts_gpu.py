"""paged_attention_decode where keys and values lie in different layouts.

Two caches may agree in some of their strides (page, token, head) and differ in others.  The
buffers here are large enough for either cache's offsets.  Tolerances: those of
test_paged_attention_gpu, whose inputs these are.
"""

import pytest
import torch

import gdn_b200
from gdn_b200 import serving
from test_paged_attention_gpu import check, expect, make

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16


def wide_rows(cache):
    """Rows of D in places of 2 D: strides (2 HKV D ps, 2 HKV D, 2 D)."""
    P, ps, HKV, D = cache.shape
    buf = torch.zeros((P, ps, HKV, 2 * D), dtype=cache.dtype, device="cuda")
    buf[..., :D] = cache
    return buf[..., :D]


def spare_heads(cache):
    """Rows side by side, as many heads unused behind them: strides (2 HKV D ps, 2 HKV D, D)."""
    P, ps, HKV, D = cache.shape
    buf = torch.zeros((P, ps, 2 * HKV, D), dtype=cache.dtype, device="cuda")
    buf[:, :, :HKV] = cache
    return buf[:, :, :HKV]


def head_major(cache):
    """Pages of [HKV, 2 ps, D], half of them unused: strides (2 HKV D ps, D, 2 ps D)."""
    P, ps, HKV, D = cache.shape
    buf = torch.zeros((P, HKV, 2 * ps, D), dtype=cache.dtype, device="cuda")
    buf[:, :, :ps] = cache.transpose(1, 2)
    return buf[:, :, :ps].transpose(1, 2)


def plain(cache):
    return cache


LAYOUTS = [(wide_rows, spare_heads), (spare_heads, wide_rows), (head_major, spare_heads),
           (wide_rows, head_major), (plain, wide_rows)]


@pytest.mark.parametrize("extension", [True, False])
@pytest.mark.parametrize("keys,values", LAYOUTS)
@pytest.mark.parametrize("ps", [1, 16])
@pytest.mark.parametrize("lens", [[200, 1, 0, 77], [2600, 70]])       # whole rows, cut rows
def test_keys_and_values_in_different_layouts(monkeypatch, lens, ps, keys, values, extension):
    if not extension:
        monkeypatch.setattr(serving, "_calls", serving._Nothing)
    for D, HQ, HKV, dtype in ((64, 8, 2, BF16), (128, 12, 3, FP16), (256, 6, 2, BF16)):
        x = make(lens, HQ, HKV, D, ps, dtype, seed=D + ps)
        want = expect(x)
        y = dict(x, k_cache=keys(x["k_cache"]), v_cache=values(x["v_cache"]))
        check(y, gdn_b200.paged_attention_decode(**y), want)


def test_one_head_of_any_stride():
    x = make([300, 40], 8, 1, 128, 16)
    want = expect(x)
    y = dict(x, k_cache=wide_rows(x["k_cache"]), v_cache=spare_heads(x["v_cache"]))
    check(y, gdn_b200.paged_attention_decode(**y), want)
