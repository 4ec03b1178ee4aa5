"""beam_select on rows of large finite logits.

Tolerance: that of test_beam_select_gpu, whose c is m log2 e as rounded.  From |m| = 2^23 on that is off
by up to |m| 2^-23, 32 at most, of which a term's exponent carries 2^-24 more.  From 2^29 on different
logits are 64 or more apart: only the largest counts.
"""

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
