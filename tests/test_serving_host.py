"""Refusals of the serving operators, on the CPU: the Python entries check before any library
call, the C entries before any CUDA call (their pointers here are never dereferenced)."""

import ctypes

import pytest
import torch

import gdn_b200
from gdn_b200 import _lib, serving

P = 1 << 20
BF16, I32 = torch.bfloat16, torch.int32
L3 = ctypes.c_int64 * 3


def attend(gdn_lib, **over):
    a = dict(q=P, kc=P, vc=P, tables=P, lens=P, k=P, v=P, scale=0.0, window=0, sinks=0, out=2 * P,
             lse=P, ws=P, ws_bytes=1 << 40, dtype=0, B=2, HQ=8, HKV=2, D=128, pages=10, page=16,
             width=4, stride=4, ks=L3(4096, 256, 128), vs=L3(4096, 256, 128), bad=None, stream=None)
    a.update(over)
    return gdn_lib.gdn_paged_attention_decode(*a.values())


@pytest.mark.parametrize("over,code", [
    (dict(D=96), _lib.GDN_ERR_SHAPE), (dict(HQ=7), _lib.GDN_ERR_SHAPE),
    (dict(HKV=0), _lib.GDN_ERR_SHAPE), (dict(B=-1), _lib.GDN_ERR_SHAPE),
    (dict(pages=0), _lib.GDN_ERR_SHAPE), (dict(page=0), _lib.GDN_ERR_SHAPE),
    (dict(width=1 << 28), _lib.GDN_ERR_SHAPE), (dict(dtype=2), _lib.GDN_ERR_ARG),
    (dict(dtype=-1), _lib.GDN_ERR_ARG), (dict(window=-1), _lib.GDN_ERR_ARG),
    (dict(sinks=-1), _lib.GDN_ERR_ARG), (dict(scale=float("nan")), _lib.GDN_ERR_ARG),
    (dict(q=None), _lib.GDN_ERR_NULL), (dict(kc=None), _lib.GDN_ERR_NULL),
    (dict(tables=None), _lib.GDN_ERR_NULL), (dict(lens=None), _lib.GDN_ERR_NULL),
    (dict(k=None), _lib.GDN_ERR_NULL), (dict(out=None), _lib.GDN_ERR_NULL),
    (dict(ks=None), _lib.GDN_ERR_NULL), (dict(q=P + 8), _lib.GDN_ERR_ALIGN),
    (dict(v=P + 2), _lib.GDN_ERR_ALIGN), (dict(lens=P + 2), _lib.GDN_ERR_ALIGN),
    (dict(ks=L3(4096, 260, 128)), _lib.GDN_ERR_ALIGN), (dict(stride=-1), _lib.GDN_ERR_SHAPE),
    (dict(), _lib.GDN_ERR_ALIAS),          # keys and values stored into the same cache
    (dict(out=P), _lib.GDN_ERR_ALIAS), (dict(out=P + 4096), _lib.GDN_ERR_ALIAS),
    (dict(width=40, ws=None, vc=4 * P), _lib.GDN_ERR_NULL),
    (dict(width=40, ws=P + 8, vc=4 * P), _lib.GDN_ERR_ALIGN),
    (dict(width=40, ws_bytes=64, vc=4 * P), _lib.GDN_ERR_SHAPE),
])
def test_attention_c_entry_refuses(gdn_lib, over, code):
    assert attend(gdn_lib, **over) == code


def test_attention_c_entry_does_nothing_for_an_empty_batch(gdn_lib):
    assert attend(gdn_lib, B=0, q=None, out=None) == _lib.GDN_OK


def test_attention_workspace_covers_what_the_call_asks_for(gdn_lib):
    """A windowed call needs the workspace of its window; every size of the table is enough."""
    ws = gdn_lib.gdn_paged_attention_workspace_bytes
    assert ws(1, 8, 2, 128, 64) == 0 and ws(0, 8, 2, 128, 4096) == 0 and ws(1, 7, 2, 128, 4096) == 0
    for D in (64, 128, 256):
        for B, HQ, HKV in ((1, 8, 2), (3, 48, 2), (500, 8, 8)):
            sizes = [ws(B, HQ, HKV, D, n) for n in (1, 100, 600, 1000, 5000, 100000)]
            assert all(a <= b for a, b in zip(sizes[-3:], sizes[-2:])) and sizes[-1] > 0


def select(gdn_lib, **over):
    a = dict(logits=P, dtype=0, sb=4000, sk=1000, scores=P, finished=None, eos=0, B=2, K=4, V=1000,
             n=4, tokens=P, parents=P, out=P, ws=P, ws_bytes=1 << 40, stream=None)
    a.update(over)
    return gdn_lib.gdn_beam_select(*a.values())


@pytest.mark.parametrize("over,code", [
    (dict(B=-1), _lib.GDN_ERR_SHAPE), (dict(K=0), _lib.GDN_ERR_SHAPE), (dict(V=0), _lib.GDN_ERR_SHAPE),
    (dict(n=0), _lib.GDN_ERR_SHAPE), (dict(n=65), _lib.GDN_ERR_LIMIT), (dict(K=65), _lib.GDN_ERR_LIMIT),
    (dict(dtype=3), _lib.GDN_ERR_ARG), (dict(sk=-1), _lib.GDN_ERR_ARG),
    (dict(finished=P, eos=1000), _lib.GDN_ERR_ARG), (dict(finished=P, eos=-1), _lib.GDN_ERR_ARG),
    (dict(logits=None), _lib.GDN_ERR_NULL), (dict(ws=None), _lib.GDN_ERR_NULL),
    (dict(logits=P + 1), _lib.GDN_ERR_ALIGN), (dict(dtype=2, logits=P + 2), _lib.GDN_ERR_ALIGN),
    (dict(ws=P + 8), _lib.GDN_ERR_ALIGN), (dict(ws_bytes=8), _lib.GDN_ERR_SHAPE),
])
def test_selection_c_entry_refuses(gdn_lib, over, code):
    assert select(gdn_lib, **over) == code


def pools(*spec):
    n = len(spec)
    return ((ctypes.c_void_p * n)(*[s[0] for s in spec]), (ctypes.c_int64 * n)(*[s[1] for s in spec]),
            (ctypes.c_int64 * n)(*[s[2] for s in spec]), n)


def test_page_c_entries_refuse(gdn_lib):
    one = pools((P, 64, 64))
    f = gdn_lib.gdn_copy_pages
    assert f(*one, 0, P, P, 1, None, None) == _lib.GDN_ERR_SHAPE
    assert f(*one, 2**30 + 1, P, P, 1, None, None) == _lib.GDN_ERR_SHAPE
    assert f(*one, 4, P, P, -1, None, None) == _lib.GDN_ERR_SHAPE
    assert f(*one, 4, P, P, 4097, None, None) == _lib.GDN_ERR_LIMIT
    assert f(*pools(*[(P + (i << 30), 64, 64) for i in range(33)]), 4, P, P, 1, None, None) == _lib.GDN_ERR_LIMIT
    assert f(*one, 4, None, P, 1, None, None) == _lib.GDN_ERR_NULL
    assert f(*one, 4, P + 2, P, 1, None, None) == _lib.GDN_ERR_ALIGN
    assert f(*one, 4, P, P, 1, P + 1, None) == _lib.GDN_ERR_ALIGN
    assert f(*pools((None, 64, 64)), 4, P, P, 1, None, None) == _lib.GDN_ERR_NULL
    assert f(*pools((P, 0, 64)), 4, P, P, 1, None, None) == _lib.GDN_ERR_SHAPE
    assert f(*pools((P, 64, 63)), 4, P, P, 1, None, None) == _lib.GDN_ERR_ALIAS
    # the same pool twice, a pool inside another one, halves that overlap by a byte
    assert f(*pools((P, 64, 64), (P, 64, 64)), 4, P, P, 1, None, None) == _lib.GDN_ERR_ALIAS
    assert f(*pools((P, 64, 64), (P + 128, 16, 32)), 4, P, P, 1, None, None) == _lib.GDN_ERR_ALIAS
    assert f(*pools((P, 33, 64), (P + 32, 32, 64)), 4, P, P, 1, None, None) == _lib.GDN_ERR_ALIAS
    assert f(*one, 4, P, P, 0, None, None) == _lib.GDN_OK
    # interleaved halves are fine (nothing to copy: no launch)
    assert f(*pools((P, 32, 64), (P + 32, 32, 64)), 4, P, P, 0, None, None) == _lib.GDN_OK

    f = gdn_lib.gdn_alloc_pages
    assert f(P, 0, P, 1, P, P, 4, None) == _lib.GDN_ERR_SHAPE
    assert f(P, 4, P, 2, P, P, 4, None) == _lib.GDN_ERR_SHAPE
    assert f(None, 4, P, 1, P, P, 4, None) == _lib.GDN_ERR_NULL
    assert f(P, 4, P, 1, P + 2, P, 4, None) == _lib.GDN_ERR_ALIGN
    f = gdn_lib.gdn_free_pages
    assert f(P, 0, P, 1, None, None) == _lib.GDN_ERR_SHAPE
    assert f(P, 4, None, 1, None, None) == _lib.GDN_ERR_NULL
    assert f(P, 4, P + 1, 1, None, None) == _lib.GDN_ERR_ALIGN

    def fork(**over):
        a = dict(tables=P, stride=4, lens=P, parents=P, ref=P, nt=2 * P, nl=2 * P, rows_in=2,
                 rows_out=2, width=4, pages=8, ps=16)
        a.update({k: v for k, v in over.items() if k in a})
        tail = dict(ws=P, ws_bytes=24, bad=None, stream=None)
        tail.update({k: v for k, v in over.items() if k in tail})
        return gdn_lib.gdn_fork_pages(*a.values(), *one, *tail.values())

    for over, code in [(dict(ps=0), _lib.GDN_ERR_SHAPE), (dict(rows_in=-1), _lib.GDN_ERR_SHAPE),
                       (dict(width=1 << 28), _lib.GDN_ERR_SHAPE), (dict(ws_bytes=23), _lib.GDN_ERR_SHAPE),
                       (dict(pages=0), _lib.GDN_ERR_SHAPE), (dict(ref=None), _lib.GDN_ERR_NULL),
                       (dict(parents=None), _lib.GDN_ERR_NULL), (dict(nt=P), _lib.GDN_ERR_ALIAS),
                       (dict(nl=P), _lib.GDN_ERR_ALIAS), (dict(lens=P + 1), _lib.GDN_ERR_ALIGN),
                       (dict(rows_in=0, rows_out=0), _lib.GDN_OK)]:
        assert fork(**over) == code, over

    f = gdn_lib.gdn_compact_pages
    assert f(P, 0, P, 1, P, P, *one, P, 1 << 20, None) == _lib.GDN_ERR_SHAPE
    assert f(P, 8, P, -1, P, P, *one, P, 1 << 20, None) == _lib.GDN_ERR_SHAPE
    assert f(P, 8, P, 1, P, P, *one, P, 8, None) == _lib.GDN_ERR_SHAPE
    assert f(P, 8, None, 1, P, P, *one, P, 1 << 20, None) == _lib.GDN_ERR_NULL
    assert f(P, 8, P, 1, P + 2, P, *one, P, 1 << 20, None) == _lib.GDN_ERR_ALIGN


def test_python_attention_refuses():
    q = torch.zeros(2, 1, 8, 128, dtype=BF16)
    kc = torch.zeros(5, 16, 2, 128, dtype=BF16)
    t, n = torch.zeros(2, 3, dtype=I32), torch.zeros(2, dtype=I32)
    f = gdn_b200.paged_attention_decode
    with pytest.raises(ValueError, match="CUDA tensor"):
        f(q, kc, kc, t, n)
    with pytest.raises(ValueError, match="4-D"):
        f(q[:, 0], kc, kc, t, n)
    with pytest.raises(TypeError, match="bfloat16 or float16"):
        f(q.float(), kc, kc, t, n)
    with pytest.raises(ValueError, match="head_dim"):
        f(q[..., :96], kc, kc, t, n)


def test_cache_layout_rules():
    check = lambda c: serving._check_cache(c, "k_cache", BF16, 2, 128, c.device)  # noqa: E731
    with pytest.raises(ValueError, match="expected"):
        check(torch.zeros(5, 16, 2, 128, dtype=BF16))
    with pytest.raises(TypeError):
        check(torch.zeros(5, 16, 2, 128))
    with pytest.raises(ValueError, match="4-D"):
        check(torch.zeros(5, 32, 128, dtype=BF16))


def test_python_selection_and_pages_refuse():
    with pytest.raises(ValueError, match="CUDA tensor"):
        gdn_b200.beam_select(torch.zeros(1, 2, 9), torch.zeros(1, 2))
    with pytest.raises(TypeError, match="logits"):
        gdn_b200.beam_select(torch.zeros(1, 2, 9, dtype=torch.float64), torch.zeros(1, 2))
    with pytest.raises(ValueError, match="3-D"):
        gdn_b200.beam_select(torch.zeros(2, 9), torch.zeros(1, 2))
    i = torch.zeros(1, dtype=I32)
    with pytest.raises(ValueError, match="CUDA tensor"):
        gdn_b200.copy_pages(torch.zeros(4, 4), i, i)
    with pytest.raises(ValueError, match="num_pages"):
        gdn_b200.copy_pages(torch.zeros(4), i, i)
    with pytest.raises(ValueError, match="32 pools"):
        gdn_b200.copy_pages([torch.zeros(4, 4)] * 33, i, i)
    for f in (lambda r: gdn_b200.alloc_pages(r, torch.ones(1, dtype=torch.bool)),
              lambda r: gdn_b200.free_pages(r, i), gdn_b200.compact_pages,
              lambda r: gdn_b200.fork_pages(i[None], i, i, r, 16)):
        with pytest.raises(ValueError, match="CUDA tensor"):
            f(torch.zeros(4, dtype=I32))
        with pytest.raises(TypeError, match="refcounts"):
            f(torch.zeros(4))
        with pytest.raises(ValueError, match="1-D"):
            f(torch.zeros(4, 4, dtype=I32))
