"""beam_select's log-sum-exp: rows of large finite logits, long rows, rows that rise.

Tolerance, in units of 2^-24 of the score's absolute error.  A term's exponent x log2 e - c is less than 8
and, below, at most |x - m| log2 e + 1/2 in size.  It is rounded once, by half a step, so by at most
max(4, |x - m| log2 e + 1/2) units, times ln 2; log2 e itself is off by 0.22 relative; and the
weighted mean of |x - m| is at most ln V: 1.22 ln V + 3.2 < 25.3 for V <= 2^26.  The exponential 4; a
chain of at most 32 additions and the two that join four chains 34; everything behind is in 64 bits, scaled by
powers of two, but a slice's sum, stored in 32 (1), and the logarithm of the fraction (2).  Together
less than 67 units, 4e-6.
From |m| = 2^23 on c, and the limit above which a thread takes another, are rounded by up to half a step
of |m| log2 e each: the exponent is up to |m| 2^-23 log2 e larger, of which the rounding takes 2^-24, times
ln 2.  From 2^29 on different logits are 64 or more apart: only the largest counts.
"""

import math

import pytest
import torch

import gdn_b200
from oracle import serving_ref

pytestmark = pytest.mark.gpu
TOL = 4e-6


def check_scores(x, s, n, got):
    """The scores of what was chosen, against 64 bits."""
    toks, pars, news = (t.cpu() for t in got)
    rows = x.cpu().double()
    lse = torch.logsumexp(rows, -1)
    for b in range(x.shape[0]):
        for r in range(n):
            i, t = int(pars[b, r]), int(toks[b, r])
            want = float(s[b, i].double()) + (float(rows[b, i, t]) - float(lse[b, i]))
            more = min(float(rows[b, i].abs().max()), 2.0**29) * 2.0**-23 * 2.0**-24
            assert abs(float(news[b, r]) - want) <= TOL + more + abs(want) * 2.0**-24, (b, r, float(news[b, r]), want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("top", [3e7, 5e8, 1e9, 1e10, 1.7e13, 1e20, 9e29, 1e31, 3e38])
@pytest.mark.parametrize("sign", [1, -1])
def test_large_finite_logits(dtype, top, sign):
    """Rows whose largest logit is huge, or whose every logit is hugely negative."""
    x = torch.full((1, 3, 4000), -top if sign < 0 else 0.0)
    x[0, 0, [7, 3999]] = sign * top
    x[0, 1, 2000] = sign * top * (0.5 if sign < 0 else 1.0)
    x[0, 2, 5:9] = 1.0                                  # an ordinary row
    x[0, 2, 9:] = -top
    x, s = x.to(dtype).cuda(), torch.tensor([[-1.0, -2.0, -3.0]]).cuda()
    got = gdn_b200.beam_select(x, s, num_selected=6)
    cands = serving_ref.beam_candidates(x, s)[0]
    check_scores(x, s, 6, got)
    for r in range(6):
        assert (int(got[1][0, r]), int(got[0][0, r])) == cands[r][1:], (r, cands[:6])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("drop", [0.125, 1.0, 2.3, 7.0])
@pytest.mark.parametrize("V", [151936, 2**20 + 3])
def test_long_slices_of_equal_terms(dtype, drop, V):
    """So many rows that each is one slice: equal terms round the same way at every addition."""
    row = torch.full((V,), -drop)
    row[:2048:4] = 0.0                                  # the first vector of every thread holds one
    x = row.to(dtype).cuda().expand(224, 8, V)
    s = -torch.arange(8.0).expand(224, 8).contiguous().cuda()
    toks, pars, news = gdn_b200.beam_select(x, s, num_selected=8)
    want = s[0].double().cpu() - torch.logsumexp(row.to(dtype).double(), 0)
    assert bool((pars == 0).all()) and bool((toks == torch.arange(0, 32, 4, device="cuda")).all())
    err = (news.cpu().double() - want[0]).abs().max()
    assert float(err) <= TOL + abs(float(want[0])) * 2.0**-24, float(err)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("B", [1, 224])
def test_rising_rows(dtype, B):
    """The running maximum grows all along the row: the sums are scaled at every step."""
    V = 300007
    row = torch.linspace(-30.0, 0.0, V).to(dtype)
    x = row.cuda().expand(B, 8, V)
    s = torch.zeros(B, 8).cuda()
    toks, pars, news = gdn_b200.beam_select(x, s, num_selected=3)
    first = int((row == row.max()).nonzero()[0])
    want = float(row.double().max() - torch.logsumexp(row.double(), 0))
    assert int(toks[0, 0]) == first and int(pars[0, 0]) == 0
    assert float((news[:, 0].cpu().double() - want).abs().max()) <= TOL + abs(want) * 2.0**-24


@pytest.mark.parametrize("sign", [1, -1])
def test_slices_on_both_sides_of_the_largest_exact_size(sign):
    """2^29 in one slice, the next larger or smaller logits in the others."""
    x = torch.full((1, 1, 40000), sign * 2.0**29)
    x[..., 20000:] += -64.0 if sign > 0 else -128.0
    x, s = x.cuda(), torch.zeros(1, 1).cuda()
    check_scores(x, s, 2, gdn_b200.beam_select(x, s, num_selected=2))


def test_equal_rows_tie_in_long_slices():
    x = (torch.randn(1, 1, 151937, generator=torch.Generator().manual_seed(3)) * 2.5)
    x = x.to(torch.bfloat16).cuda().expand(300, 8, 151937).clone()     # rows begin anywhere
    toks, pars, news = gdn_b200.beam_select(x, torch.zeros(300, 8, device="cuda"))
    assert bool((news == news[0]).all()) and bool((toks == toks[0]).all())
    assert pars[0].tolist() == list(range(8)) and len(set(toks[0].tolist())) == 1
    assert math.isfinite(float(news[0, 0]))
