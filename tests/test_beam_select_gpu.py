"""beam_select on the GPU against its definition in 64 bits.

Tolerance.  A score is cum + (x - lse) in 64 bits, rounded once to fp32 (2^-24 relative).
lse's error is the softmax-weighted mean of its terms' relative errors.  A term's exponent
x log2 e - c is rounded once and its factor once: at most 1.5 |x - m| 2^-24 in the exponent to
e, whose weighted mean is at most 1.5 ln V 2^-24 < 20 2^-24; the exponential is off by 2^-22; a
chain of k positive fp32 additions by k 2^-24, here k <= 40 (a thread's at most 16 vectors in
four chains, then the warp's lanes), 64 bits beyond, and 2^-24 for a slice's sum.  Together
(20 + 4 + 40 + 1) 2^-24 < 4e-6.  Two candidates of different beams whose scores are nearer
than twice that may come in either order; all others must come exactly.
"""

import math

import pytest
import torch

import gdn_b200
from oracle import serving_ref

pytestmark = pytest.mark.gpu
TOL = 4e-6


def check(logits, scores, n, finished=None, eos=0):
    toks, pars, news = gdn_b200.beam_select(logits, scores, num_selected=n, finished=finished,
                                            eos_token=eos)
    every = serving_ref.beam_candidates(logits, scores, finished, eos)
    for b, cands in enumerate(every):
        got = list(zip(news[b].tolist(), pars[b].tolist(), toks[b].tolist()))
        exact = {(i, t): s for s, i, t in cands}
        k = min(n, len(cands))
        assert len({(i, t) for _, i, t in got[:k]}) == k
        for r in range(k):
            s, i, t = got[r]
            assert (i, t) in exact, (b, r, got[r], cands[:k + 1])
            tol = TOL + abs(exact[i, t]) * 2.0**-24
            assert abs(s - exact[i, t]) <= tol, (b, r, s, exact[i, t])
            assert abs(cands[r][0] - exact[i, t]) <= 2 * TOL, (b, r, got[r], cands[r])
            if (i, t) != cands[r][1:]:
                # another one only where different beams are too near to tell
                assert i != cands[r][1]
        # within a beam the order is exact: logit, then token
        for i in set(p for _, p, _ in got[:k]):
            mine = [t for _, p, t in got[:k] if p == i]
            assert mine == [t for _, p, t in cands if p == i][:len(mine)]
        assert got[k:] == [(-math.inf, -1, -1)] * (n - k)
    return toks, pars, news


def make(B, K, V, dtype, seed=0, spread=2.5):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(B, K, V, generator=g) * spread).to(dtype).cuda()
    s = (-8 - 4 * torch.rand(B, K, generator=g)).cuda()
    return x, s


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("B,K,V,n", [(1, 1, 1, 1), (1, 1, 2, 3), (2, 3, 7, 8), (3, 4, 1000, 4),
                                     (1, 5, 4097, 10), (2, 8, 32001, 16), (1, 32, 5003, 64),
                                     (1, 64, 333, 33), (70, 2, 130, 2), (1, 2, 200000, 5)])
def test_sizes_and_types(dtype, B, K, V, n):
    x, s = make(B, K, V, dtype, seed=V)
    check(x, s, n)


def test_ties_go_to_the_lower_beam_and_token():
    x = torch.zeros(2, 4, 5000, dtype=torch.bfloat16, device="cuda")
    s = torch.zeros(2, 4, device="cuda")
    t, p, _ = gdn_b200.beam_select(x, s, num_selected=40)
    assert t.tolist() == [list(range(40))] * 2 and p.tolist() == [[0] * 40] * 2
    x[:, :, 777] = 1.0                               # then one token per beam, then the rest
    t, p, _ = gdn_b200.beam_select(x, s, num_selected=6)
    assert t.tolist() == [[777] * 4 + [0, 1]] * 2 and p.tolist() == [[0, 1, 2, 3, 0, 0]] * 2
    x = torch.zeros(1, 1, 100, device="cuda")
    x[0, 0, 50:] = -0.0                              # -0 and +0 are equal
    t, _, _ = gdn_b200.beam_select(x, torch.zeros(1, 1, device="cuda"), num_selected=60)
    assert t[0].tolist() == list(range(60))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("V", [777, 5003, 40000, 151937])
def test_equal_rows_tie_wherever_they_lie(dtype, V):
    """Equal beams have equal scores, bit for bit, whatever their alignment and their place in
    the batch: the lower beam comes first for each token."""
    g = torch.Generator().manual_seed(V)
    x = (torch.randn(1, 1, V, generator=g) * 3).to(dtype).expand(5, 7, V).contiguous().cuda()
    s = torch.full((5, 7), -2.5, device="cuda")
    t, p, v = gdn_b200.beam_select(x, s, num_selected=21)
    row = x[0, 0].float().cpu()
    top = row.sort(descending=True, stable=True).indices[:30].tolist()
    # equal scores: the lower beam, within a beam the lower token (16-bit logits repeat)
    want = sorted(((-float(row[k]), i, k) for i in range(7) for k in top))[:21]
    assert t.tolist() == [[k for _, _, k in want]] * 5
    assert p.tolist() == [[i for _, i, _ in want]] * 5
    for r in v.tolist():
        assert len(set(r)) == len(set(x for x, _, _ in want))


@pytest.mark.parametrize("spread", [2.0, 30.0])
@pytest.mark.parametrize("B,K,V,n", [(8, 32, 50257, 32), (2, 64, 40000, 64)])
def test_a_few_beams_far_ahead(B, K, V, n, spread):
    """The first candidates of few slices reach the result, so that they bound it loosely."""
    x, s = make(B, K, V, torch.float32, seed=int(spread))
    f = torch.rand(B, K, generator=torch.Generator().manual_seed(n)) < 0.2
    check(x, s * spread, n, f.cuda(), eos=2)


def test_many_requests_of_few_tokens():
    x, s = make(600, 8, 130, torch.float32, seed=3)
    f = torch.rand(600, 8, generator=torch.Generator().manual_seed(1)) < 0.4
    s[5] = -math.inf
    check(x, s, 5, f.cuda(), eos=7)
    x, s = make(300, 3, 2500, torch.bfloat16, seed=4)
    f = torch.rand(300, 3, generator=torch.Generator().manual_seed(2)) < 0.5
    check(x, s, 6, f.cuda(), eos=7)


@pytest.mark.parametrize("order", ["ascending", "descending", "blocks", "hot", "hot ties",
                                   "hot and one above"])
def test_sorted_logits(order):
    V = 60000
    row = torch.linspace(-20, 20, V)
    if order == "descending":
        row = row.flip(0)
    if order == "blocks":                            # the best ones all side by side
        row = torch.cat([torch.full((30000,), -5.0), torch.linspace(5, 6, 64),
                         torch.full((V - 30064,), -4.0)])
    if order.startswith("hot"):                      # large ones where a sample may miss them
        row = torch.full((V,), -5.0)
        row[3000:33000] = 5.0 if "ties" in order else torch.linspace(5, 6, 30000)
        if "above" in order:
            row[3000:33000] = 5.0
            row[20000:20100] = 7.0
    x = row.repeat(2, 2, 1).to(torch.float32).cuda()
    check(x, torch.tensor([[-1.0, -1.5], [0.0, -30.0]]).cuda(), 64)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("n", [1, 16, 17, 64])
def test_hot_regions_of_every_type(dtype, n):
    g = torch.Generator().manual_seed(n)
    x = torch.randn(1, 2, 150001, generator=g)
    x[0, 0, 9000:40000] += 8.0
    x[0, 1, -3000:] += 6.0
    check(x.to(dtype).cuda(), torch.tensor([[-1.0, -0.5]]).cuda(), n)


def test_tokens_masked_with_the_lowest_value():
    """A grammar's mask: a few tokens left, all others at the type's lowest value."""
    for dtype in (torch.bfloat16, torch.float16, torch.float32):
        x, s = make(3, 4, 50000, dtype, seed=8)
        keep = torch.zeros(50000, dtype=torch.bool)
        keep[torch.tensor([5, 17, 49999, 30000, 30001])] = True
        x[:, :, ~keep] = torch.finfo(dtype).min
        check(x, s, 4)
        check(x, s, 32)                              # some masked ones have to be taken


def test_coarse_bf16_logits_with_many_ties():
    x, s = make(3, 4, 20011, torch.float32, seed=5)
    x = (x * 2).round().div(2).to(torch.bfloat16)
    check(x, s, 50)


def test_masked_dead_and_broken_rows():
    x, s = make(6, 4, 999, torch.float32, seed=9)
    x[0, :, 5:] = -math.inf                          # 5 tokens a beam left
    x[1, 1] = -math.inf                              # a beam without tokens
    x[2, 0, 17] = math.nan                           # a broken beam
    x[3, 2, 3] = math.inf
    s[4, 1:] = -math.inf                             # the first step: one live beam
    s[5] = -math.inf                                 # nothing at all
    check(x, s, 24)
    t, p, v = gdn_b200.beam_select(x, s, num_selected=24)
    assert (p[1] != 1).all() and (p[2] != 0).all() and (p[3] != 2).all()
    assert (t[5] == -1).all() and torch.isinf(v[5]).all()
    assert (t[0, 20:] == -1).all() and (t[0, :20] >= 0).all()


def test_lowest_finite_logits_are_chosen_last():
    x = torch.full((1, 2, 300), torch.finfo(torch.float32).min, device="cuda")
    x[0, 0, 7] = 0.0
    x[0, 1] = -math.inf
    x[0, 1, 9] = -3.0
    check(x, torch.tensor([[-1.0, -2.0]]).cuda(), 8)
    y = torch.full((1, 1, 300), torch.finfo(torch.bfloat16).min, dtype=torch.bfloat16, device="cuda")
    check(y, torch.zeros(1, 1, device="cuda"), 8)


def test_finished_beams():
    x, s = make(4, 5, 4000, torch.bfloat16, seed=2)
    f = torch.zeros(4, 5, dtype=torch.bool)
    f[0, 2] = f[1, 0] = f[1, 4] = f[2] = True
    s[2, 3] = -math.inf
    s[1, 0] = math.nan
    x[2] = math.nan                                  # a finished beam's logits are not looked at
    t, p, v = check(x, s, 10, f.cuda(), eos=3999)
    assert (t[2, :4] == 3999).all() and (t[2, 4:] == -1).all()


def test_strided_and_unaligned_logits():
    x, s = make(3, 4, 1003, torch.bfloat16, seed=4)
    big = torch.full((3, 9, 1031), 50.0, dtype=torch.bfloat16, device="cuda")
    big[:, 1:9:2, 13:13 + 1003] = x
    view = big[:, 1:9:2, 13:13 + 1003]
    a = check(x, s, 8)
    b = check(view, s, 8)
    assert all(torch.equal(u, w) for u, w in zip(a, b))
    one = x[:, :1].expand(3, 4, 1003)                # one row for all beams
    check(one, s, 8)


def test_graph_streams_empty_and_repeat():
    x, s = make(5, 4, 30000, torch.bfloat16, seed=6)
    eager = gdn_b200.beam_select(x, s, num_selected=8)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs = []
    with torch.cuda.stream(side):
        for _ in range(2):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                got = gdn_b200.beam_select(x, s, num_selected=8)
            graphs.append((g, got))
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(3):
        with torch.cuda.stream(s1):
            graphs[0][0].replay()
        with torch.cuda.stream(s2):
            graphs[1][0].replay()
    torch.cuda.synchronize()
    for _, got in graphs:
        assert all(torch.equal(u, w) for u, w in zip(eager, got))
    t, p, v = gdn_b200.beam_select(x[:0], s[:0])
    assert t.shape == p.shape == v.shape == (0, 4)
