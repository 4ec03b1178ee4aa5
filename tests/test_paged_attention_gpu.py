"""paged_attention_decode on the GPU against its definition in 64 bits.

Tolerances.  Let u = torch.finfo(dtype).eps / 2 be a rounding to the tensors' type, A the
softmax's mean of |v|, n the visible tokens, and e = (D + 4) 2^-24 M the error of one score
in fp32 with M the largest scale * sum |q||k| (products of two 16-bit values are exact in
fp32; D additions, the scale, the subtraction of the maximum, base 2).  Each p carries a
relative error of 2 e (its own and the maximum's) + 2^-21 (the exponential), and one rounding
u to the type it is multiplied in (subnormal in fp16: at most 2^-25 absolutely, n 2^-25 A'
with A' the plain mean of |v|, bounded by max |v|); sums of n terms in fp32 add n 2^-24; the
result is rounded once, u |o|.  So
    |o - exact|   <= u |o| + (u + 4 e + 2^-20 + 2 n 2^-24) A (1 + u) + n 2^-25 max|v| [fp16]
    |lse - exact| <= 2 e + 2^-20 + n 2^-24 + 2^-22 |lse|
The sum of n terms never loses more than that, whatever its order.
"""

import math

import pytest
import torch

import gdn_b200
from oracle import serving_ref

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16


def make(lens, HQ, HKV, D, ps, dtype=BF16, width=None, seed=0, spare=3):
    g = torch.Generator().manual_seed(seed)
    B = len(lens)
    used = [-(-max(0, n) // ps) for n in lens]
    width = max(used + [1]) if width is None else width
    pages = sum(used) + spare
    order = torch.randperm(pages, generator=g)
    tables = torch.full((B, width), -1, dtype=torch.int32)
    at = 0
    for b, u in enumerate(used):
        u = min(u, width)
        tables[b, :u] = order[at:at + u].int()
        at += u
    r = lambda *s: torch.randn(*s, generator=g).to(dtype).cuda()  # noqa: E731
    return dict(q=r(B, 1, HQ, D), k_cache=r(pages, ps, HKV, D), v_cache=r(pages, ps, HKV, D),
                block_tables=tables.cuda(), seq_lens=torch.tensor(lens, dtype=torch.int32).cuda(),
                k=r(B, 1, HKV, D), v=r(B, 1, HKV, D))


def expect(x, window=0, num_sinks=0, scale=None):
    return serving_ref.attention(x["q"], x["k_cache"], x["v_cache"], x["block_tables"],
                                 x["seq_lens"], x.get("k"), x.get("v"), scale, window, num_sinks)


def check(x, got, want):
    out, lse, absv, mag, kc, vc, _ = want
    o, l = got
    D, dt = x["q"].shape[-1], x["q"].dtype
    u = torch.finfo(dt).eps / 2
    n = int(x["seq_lens"].max().clamp(min=1))
    e = ((D + 4) * 2.0**-24 * mag)[..., None]
    tol = u * out.abs() + (u + 4 * e + 2.0**-20 + 2 * n * 2.0**-24) * absv * (1 + u)
    if dt == FP16:
        tol = tol + n * 2.0**-25 * float(torch.nan_to_num(vc.double()).abs().max())
    err = (o[:, 0].cpu().double() - out).abs()
    assert bool((err <= tol).all()), float((err - tol).max())
    inf = torch.isinf(lse)
    assert torch.equal(torch.isinf(l.cpu()), inf)
    ltol = 2 * e[..., 0] + 2.0**-20 + n * 2.0**-24 + 2.0**-22 * lse.abs()
    assert bool(((l.cpu().double() - lse).abs() <= ltol)[~inf].all())
    assert torch.equal(x["k_cache"].cpu().view(torch.int16), kc.view(torch.int16))
    assert torch.equal(x["v_cache"].cpu().view(torch.int16), vc.view(torch.int16))


def run(x, **kw):
    return gdn_b200.paged_attention_decode(**x, **kw)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("HQ,HKV", [(1, 1), (8, 1), (12, 4), (14, 2), (40, 2), (16, 16)])
def test_heads_and_types(dtype, D, HQ, HKV):
    x = make([1, 2, 17, 63, 64, 65, 200, 0], HQ, HKV, D, 16, dtype, seed=D + HQ)
    want = expect(x)
    check(x, run(x), want)


@pytest.mark.parametrize("ps", [1, 3, 8, 16, 24, 64, 100, 300])
def test_page_sizes_and_lengths(ps):
    x = make([0, 1, 15, 16, 31, 33, 127, 129, 255, 257, 300], 8, 2, 128, ps, seed=ps)
    want = expect(x)
    check(x, run(x), want)


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 5), (16, 0), (64, 4), (100, 17), (5000, 3)])
def test_window_and_sinks(window, sinks):
    x = make([1, 5, 6, 16, 40, 68, 69, 117, 118, 1000], 8, 2, 64, 16, seed=window)
    want = expect(x, window, sinks)
    check(x, run(x, window=window, num_sinks=sinks), want)


@pytest.mark.parametrize("lens", [[5000], [4097, 1, 4096], [700] * 40, [1] * 300,
                                  [520] * 150 + [0, 1, 63, 64, 65, 2000],     # cut rows by share
                                  [500] * 300, [64] * 200 + [3000],
                                  [0] * 140 + [900, 0, 40]])
def test_long_split_and_many_rows(lens):
    x = make(lens, 8, 2, 128, 16, seed=len(lens))
    want = expect(x)
    check(x, run(x), want)


@pytest.mark.parametrize("D,HQ,HKV", [(64, 24, 1), (256, 12, 1), (256, 8, 2), (64, 4, 4), (128, 40, 1)])
@pytest.mark.parametrize("lens", [[3001, 64, 0, 1025], [130] * 9 + [2500]])
def test_cut_rows_of_other_shapes(D, HQ, HKV, lens):
    x = make(lens, HQ, HKV, D, 16, seed=HQ)
    want = expect(x)
    check(x, run(x), want)
    x = make(lens, HQ, HKV, D, 8, FP16, seed=HQ + 1)
    want = expect(x, 1500, 9)
    check(x, run(x, window=1500, num_sinks=9), want)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("HQ,HKV", [(17, 1), (25, 1), (32, 1), (48, 1), (66, 2), (64, 1)])
@pytest.mark.parametrize("lens", [[200, 3, 0, 33], [2600]])
def test_many_heads_to_a_key_value_head(D, HQ, HKV, lens):
    x = make(lens, HQ, HKV, D, 16, seed=HQ)
    want = expect(x, 70, 3)
    check(x, run(x, window=70, num_sinks=3), want)
    x = make(lens, HQ, HKV, D, 16, FP16, seed=HQ + D)
    want = expect(x)
    check(x, run(x), want)


def test_without_new_rows_reads_the_cache_only():
    x = make([1, 20, 333], 8, 2, 128, 16)
    del x["k"], x["v"]
    want = expect(x)
    check(x, run(x), want)


@pytest.mark.parametrize("scale", [0.0, 0.3, -0.1])
def test_scale(scale):
    x = make([50, 3], 4, 4, 64, 8)
    want = expect(x, scale=scale)
    check(x, run(x, scale=scale), want)


def test_table_entries_out_of_range_hide_their_tokens():
    x = make([100, 100, 64, 20, 33], 8, 2, 128, 16)
    P = x["k_cache"].shape[0]
    x["block_tables"][0, 2] = -1
    x["block_tables"][1, 0] = P
    x["block_tables"][1, 6] = P + 7                # the new token's page: seen, not stored
    x["block_tables"][2, :] = 2**31 - 1
    x["block_tables"][3, 1] = -5
    x["block_tables"][4, :] = -1
    want = expect(x)
    bad = torch.zeros(1, dtype=torch.int32, device="cuda")
    check(x, run(x, bad_index_count=bad), want)
    assert int(bad) == want[-1] == 2 + 4
    del x["k"], x["v"]                              # now rows 4 and 2 see nothing
    want = expect(x)
    assert math.isinf(want[1][4, 0]) and math.isinf(want[1][2, 0])
    bad.zero_()
    check(x, run(x, bad_index_count=bad), want)
    assert int(bad) == want[-1]


@pytest.mark.parametrize("sinks,window", [(0, 20), (3, 20), (17, 20), (3, 500)])
def test_bad_pages_are_counted_once_with_a_window(sinks, window):
    x = make([100, 30, 90], 8, 2, 64, 16)
    x["block_tables"][:, ::2] = 1000
    want = expect(x, window, sinks)
    bad = torch.zeros(1, dtype=torch.int32, device="cuda")
    check(x, run(x, window=window, num_sinks=sinks, bad_index_count=bad), want)
    assert int(bad) == want[-1]


@pytest.mark.parametrize("HQ,HKV", [(12, 1), (40, 2)])
@pytest.mark.parametrize("lens", [[100, 30, 90], [1500], [5] * 200])
def test_bad_pages_with_two_warps_to_a_tile(HQ, HKV, lens):
    x = make(lens, HQ, HKV, 256, 16)
    x["block_tables"][:, 1::3] = 99999
    want = expect(x)
    bad = torch.zeros(1, dtype=torch.int32, device="cuda")
    check(x, run(x, bad_index_count=bad), want)
    assert int(bad) == want[-1]


def test_lengths_beyond_the_table_and_negative():
    x = make([40, -3, 10], 8, 2, 128, 16, width=3)
    x["seq_lens"][0] = 49
    want = expect(x)
    bad = torch.zeros(1, dtype=torch.int32, device="cuda")
    check(x, run(x, bad_index_count=bad), want)
    assert int(bad) == want[-1] == 1


def test_garbage_behind_the_last_token_is_harmless():
    x = make([1, 18, 70], 8, 2, 128, 16)
    for b, n in enumerate([1, 18, 70]):
        page = int(x["block_tables"][b, (n - 1) // 16])
        for c in (x["k_cache"], x["v_cache"]):
            c[page, (n - 1) % 16:] = float("nan")     # the new token's place too
    want = expect(x)
    got = run(x)
    assert bool(torch.isfinite(got[0].float()).all())
    check(x, got, want)


def test_infinities_in_values_and_large_scores():
    x = make([30, 30], 4, 2, 64, 16)
    x["q"] *= 30                                     # one token takes nearly all the weight
    page = int(x["block_tables"][1, 0])
    x["v_cache"][page, 3, 0, 5] = float("inf")
    got = run(x)
    o = got[0][:, 0].cpu().float()
    # the infinity reaches dim 5 of the heads that read kv head 0 of row 1: inf or nan
    # (weight 0 times inf) there, finite values everywhere else
    assert not bool(torch.isfinite(o[1, :2, 5]).any())
    o[1, :2, 5] = 0
    assert bool(torch.isfinite(o).all())


def test_equal_scores_and_scores_of_minus_infinity():
    x = make([64], 2, 1, 64, 16)
    x["q"].zero_()
    want = expect(x)
    check(x, run(x), want)
    x["q"].fill_(1.0)
    x["k_cache"].zero_()
    page = int(x["block_tables"][0, 1])
    x["k_cache"][page, 2, 0, 0] = float("-inf")      # one token with score -inf: weight 0
    x["k"].zero_()
    o, lse = run(x)
    assert bool(torch.isfinite(o.float()).all())
    assert abs(float(lse[0, 0]) - math.log(63)) < 1e-5


def test_strided_caches_and_tables():
    B, HQ, HKV, D, ps = 3, 8, 2, 128, 16
    lens = [33, 1, 90]
    x = make(lens, HQ, HKV, D, ps)
    want = expect(x)
    base = run({k: v.clone() for k, v in x.items()})
    P = x["k_cache"].shape[0]
    both = torch.empty((P, 2, HKV, ps, D + 8), dtype=BF16, device="cuda")   # head-major, padded
    both[:, 0, :, :, :D] = x["k_cache"].transpose(1, 2)
    both[:, 1, :, :, :D] = x["v_cache"].transpose(1, 2)
    wide = torch.full((B, x["block_tables"].shape[1] + 5), 7, dtype=torch.int32, device="cuda")
    wide[:, :x["block_tables"].shape[1]] = x["block_tables"]
    y = dict(x, k_cache=both[:, 0, :, :, :D].transpose(1, 2),
             v_cache=both[:, 1, :, :, :D].transpose(1, 2),
             block_tables=wide[:, :x["block_tables"].shape[1]])
    got = run(y)
    check(y, got, want)
    assert torch.equal(got[0], base[0]) and torch.equal(got[1], base[1])


def test_shared_pages_and_empty_batch():
    x = make([48, 40, 47], 8, 2, 64, 16)
    x["block_tables"][1, :2] = x["block_tables"][0, :2]
    x["block_tables"][2, :2] = x["block_tables"][0, :2]
    want = expect(x)
    check(x, run(x), want)
    e = {k: (v[:0] if k not in ("k_cache", "v_cache") else v) for k, v in x.items()}
    o, lse = run(e)
    assert o.shape == (0, 1, 8, 64) and lse.shape == (0, 8)


def test_offsets_beyond_32_bits():
    """A cache of more than 2^31 elements: the last pages lie behind 4 GB."""
    D, HKV, ps = 128, 2, 16
    P = 2**31 // (ps * HKV * D) + 64                 # 4.3 GB each
    kc = torch.zeros((P, ps, HKV, D), dtype=BF16, device="cuda")
    vc = torch.zeros((P, ps, HKV, D), dtype=BF16, device="cuda")
    small = make([40, 40], 4, HKV, D, ps)
    pages = torch.tensor([[P - 1, 5, P - 7], [P - 3, P - 4, 0]], dtype=torch.int32)
    want = expect(small)
    for b in range(2):
        for j in range(3):
            s = int(small["block_tables"][b, j])
            kc[pages[b, j]] = small["k_cache"][s]
            vc[pages[b, j]] = small["v_cache"][s]
    y = dict(small, k_cache=kc, v_cache=vc, block_tables=pages.cuda())
    got = run(y)
    base = run(small)
    assert torch.equal(got[0], base[0]) and torch.equal(got[1], base[1])
    check(small, base, want)
    for b in range(2):
        last = int(pages[b, 2])
        assert torch.equal(kc[last, 7], small["k"][b, 0]) and torch.equal(vc[last, 7], small["v"][b, 0])


def test_captured_replayed_and_other_streams():
    x = make([300, 77, 0, 1], 16, 2, 256, 16)
    want = expect(x)
    eager = run({k: v.clone() for k, v in x.items()})
    graphs = []
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run({k: v.clone() for k, v in x.items()})
        for _ in range(2):
            gph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(gph, stream=side):
                got = run(x)
            graphs.append((gph, got))
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(3):                               # both at once: they share no workspace
        with torch.cuda.stream(s1):
            graphs[0][0].replay()
        with torch.cuda.stream(s2):
            graphs[1][0].replay()
    torch.cuda.synchronize()
    for _, got in graphs:
        assert torch.equal(got[0], eager[0]) and torch.equal(got[1], eager[1])
    check(x, graphs[0][1], want)
    # lengths are read on the device: a replay follows them
    x["seq_lens"].copy_(torch.tensor([299, 5, 4, 0], dtype=torch.int32))
    want = expect(x)
    graphs[0][0].replay()
    torch.cuda.synchronize()
    check(x, graphs[0][1], want)


def test_repeats_bit_for_bit():
    x = make([3000, 100, 2049], 16, 2, 128, 16)
    first = run(x)
    for _ in range(5):
        again = run(x)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])
