"""paged_attention_decode with many small weights beside large ones: none is lost.

In fp16 a weight is multiplied as 2^15 exp(x - m), so that the largest is 2^15 and one is
subnormal, with an absolute rounding of 2^-25, only below 2^-14: relative to the largest
weight of its warp, which is at most the row's, at most 2^-40 a token.  With u, A, e and n as
in test_paged_attention_gpu, and nothing left of that test's n 2^-25 max |v|:
    |o - exact|   <= u |o| + (u + 4 e + 2^-20 + 2 n 2^-24) A (1 + u) + n 2^-40 max|v| [fp16]
    |lse - exact| <= 2 e + 2^-20 + n 2^-24 + 2^-22 |lse|
An output that is subnormal in fp16 is rounded by at most 2^-25.  The 15 of the factor goes into
the exponent's second term, whose rounding e covers: |m| + 15 <= 2 M or both are below 16,
where 2^-24 16 < 2^-20.
"""

import pytest
import torch

import gdn_b200
from test_paged_attention_gpu import expect, make

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16


def check(x, got, want):
    out, lse, absv, mag, _, vc, _ = want
    o, l = got
    D, dt = x["q"].shape[-1], x["q"].dtype
    u = torch.finfo(dt).eps / 2
    n = int(x["seq_lens"].max().clamp(min=1))
    e = ((D + 4) * 2.0**-24 * mag)[..., None]
    tol = u * out.abs() + (u + 4 * e + 2.0**-20 + 2 * n * 2.0**-24) * absv * (1 + u)
    if dt == FP16:
        tol = tol + n * 2.0**-40 * float(vc.double().abs().max()) + 2.0**-25
    err = (o[:, 0].cpu().double() - out).abs()
    assert bool((err <= tol).all()), (float((err - tol).max()), float(err.max()))
    inf = torch.isinf(lse)
    assert torch.equal(torch.isinf(l.cpu()), inf)
    ltol = 2 * e[..., 0] + 2.0**-20 + n * 2.0**-24 + 2.0**-22 * lse.abs()
    assert bool(((l.cpu().double() - lse).abs() <= ltol)[~inf].all())


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("D,HQ,HKV", [(64, 8, 2), (64, 24, 1), (128, 16, 1), (256, 4, 2)])
@pytest.mark.parametrize("lens,window", [([300, 31, 2, 1, 0], 0), ([3000, 90], 0), ([3000, 90], 700)])
@pytest.mark.parametrize("drop", [9.0, 18.0, 24.0])
def test_weights_far_below_the_largest_are_counted(dtype, D, HQ, HKV, lens, window, drop):
    """Each 16th token's score is `drop` above the others', whose values carry the output:
    15 e^-drop of 30000, 2^-26 a weight at 18."""
    x = make(lens, HQ, HKV, D, 16, dtype, seed=D)
    x["q"].zero_()
    x["q"][..., 0] = 1.0
    for c in (x["k_cache"], x["k"]):
        c.zero_()
    x["k_cache"][:, 0, :, 0] = drop                # pages of 16: the first token of each
    x["v_cache"].fill_(30000.0)
    x["v_cache"][:, 0] = 0.0
    x["v"].fill_(30000.0)
    want = expect(x, window, 0, 1.0)
    check(x, gdn_b200.paged_attention_decode(**x, window=window, scale=1.0), want)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("spread", [0.3, 3.0])
def test_random_scores(dtype, D, spread):
    x = make([2000, 70, 1, 0, 333], 8, 2, D, 16, dtype, seed=3)
    x["q"] *= spread
    want = expect(x, 0, 0, None)
    check(x, gdn_b200.paged_attention_decode(**x), want)


@pytest.mark.parametrize("value", [60000.0, -65504.0])
def test_values_at_the_types_end(value):
    x = make([5000, 40], 8, 2, 128, 16, FP16, seed=4)
    for c in (x["v_cache"], x["v"]):
        c.fill_(value)
    want = expect(x)
    got = gdn_b200.paged_attention_decode(**x)
    assert bool(torch.isfinite(got[0]).all())
    check(x, got, want)
