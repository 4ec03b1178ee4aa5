"""The serving operators' two ways into the library, the CPython extension and ctypes: the same
answers, and the same refusals, which the extension leaves to Python."""

import pytest
import torch

import gdn_b200
from gdn_b200 import _lib, build, serving

I32, BF16 = torch.int32, torch.bfloat16


def test_extension_declines_what_python_refuses(gdn_lib):
    build.build_torch()
    calls = _lib.torch_calls()
    z = torch.zeros(2, 2)
    i = torch.zeros(2, dtype=I32)
    assert calls.attend(*[z] * 5, None, None, None, 0, 0, None, None) is None
    assert calls.attend(None, *[z] * 4, None, None, None, 0, 0, None, None) is None
    assert calls.attend(z) is None
    assert calls.select(torch.zeros(1, 2, 9), torch.zeros(1, 2), None, None, 0) is None
    assert calls.select(torch.zeros(1, 2, 9), torch.zeros(1, 2), "many", None, 0) is None
    assert calls.copy(z, i, i, None) is None and calls.copy([], i, i, None) is None
    assert calls.copy(3, i, i, None) is None
    assert calls.alloc(i, i) is None and calls.release(i, i, None) is None
    assert calls.fork(i[None], i, i, i, 16, (), None) is None
    assert calls.fork(i[None], i, i, i, 2**40, (), None) is None
    assert calls.compact(i, None, ()) is None


def both(monkeypatch, call):
    """The call's results through the extension, and through ctypes alone."""
    made = []
    calls = serving._torch_calls()
    assert calls is not serving._Nothing, "the extension is not built"

    class Spy:
        def __getattr__(self, name):
            def f(*args):
                made.append(getattr(calls, name)(*args))
                return made[-1]
            return f

    monkeypatch.setattr(serving, "_calls", Spy())
    a = call()
    assert made and made[0] is not None, "the extension declined"
    monkeypatch.setattr(serving, "_calls", serving._Nothing)
    b = call()
    monkeypatch.undo()
    return a, b


def same(a, b):
    if isinstance(a, torch.Tensor):
        return torch.equal(a, b) and a.dtype == b.dtype
    return len(a) == len(b) and all(same(x, y) for x, y in zip(a, b))


def cuda(x):
    return torch.tensor(x, dtype=I32, device="cuda")


@pytest.mark.gpu
@pytest.mark.parametrize("window,new,given", [(0, True, True), (100, False, False), (5, True, False)])
def test_attention_both_ways(monkeypatch, window, new, given):
    g = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=g).to(BF16).cuda()  # noqa: E731
    q, kv, k, v = r(2, 1, 8, 128), r(60, 2, 16, 2, 128), r(2, 1, 2, 128), r(2, 1, 2, 128)
    tables, lens = torch.randperm(60, generator=g).int().view(2, 30).cuda(), cuda([470, 33])
    bad = torch.zeros(1, dtype=I32, device="cuda")
    tables[1, 0] = 60

    def call():
        out = torch.full_like(q, 7.0) if given else None
        o, lse = gdn_b200.paged_attention_decode(
            q, kv[:, 0], kv[:, 1], tables, lens, k=k if new else None, v=v if new else None,
            scale=0.1, window=window, num_sinks=3, output=out, bad_index_count=bad)
        assert out is None or o.data_ptr() == out.data_ptr()
        return o, lse, kv.clone(), bad.clone()

    a, b = both(monkeypatch, call)
    assert same(a[:3], b[:3]) and int(b[3]) == 2 * int(a[3]) == 2
    with pytest.raises(ValueError, match="kv heads"):
        gdn_b200.paged_attention_decode(q[:, :, :3].contiguous(), kv[:, 0], kv[:, 1], tables, lens)
    with pytest.raises(TypeError, match="v_cache"):
        gdn_b200.paged_attention_decode(q, kv[:, 0], kv[:, 1].half(), tables, lens)
    with pytest.raises(_lib.GdnError, match="overlap"):
        gdn_b200.paged_attention_decode(q, kv[:, 0], kv[:, 1], tables, lens, output=q)


@pytest.mark.gpu
def test_selection_both_ways(monkeypatch):
    g = torch.Generator().manual_seed(1)
    x = torch.randn(3, 4, 999, generator=g).cuda()
    s, f = -torch.rand(3, 4, generator=g).cuda(), (torch.rand(3, 4, generator=g) < 0.3).cuda()
    for kw in ({}, dict(num_selected=9), dict(finished=f, eos_token=5)):
        a, b = both(monkeypatch, lambda: gdn_b200.beam_select(x, s, **kw))
        assert same(a, b)
    with pytest.raises(ValueError, match="64"):
        gdn_b200.beam_select(x, s, num_selected=65)
    with pytest.raises(ValueError, match="eos_token"):
        gdn_b200.beam_select(x, s, finished=f, eos_token=999)
    with pytest.raises(ValueError, match="shape"):
        gdn_b200.beam_select(x, s[:, :3])


@pytest.mark.gpu
def test_pages_both_ways(monkeypatch):
    g = torch.Generator().manual_seed(2)
    start = torch.randn(12, 3, 40, generator=g).cuda()
    refs0 = cuda([1, 0, 2, 1, 0, 0, 1, 1, 0, 3, 0, 0])
    tables, lens = cuda([[0, 2], [3, 6], [7, 9]]), cuda([9, 12, 16])

    def copy():
        pool = start.clone()
        gdn_b200.copy_pages([pool, pool.new_zeros(12, 2)], cuda([0, 1, 12]), cuda([1, 0, 3]))
        return pool

    def fork():
        pool, refs = start.clone(), refs0.clone()
        t, n = gdn_b200.fork_pages(tables, lens, cuda([0, 0, 2, 1, 1]), refs, 8, pools=(pool,))
        return t, n, refs, pool

    def compact():
        pool, refs, t = start.clone(), refs0.clone(), tables.clone()
        remap, live = gdn_b200.compact_pages(refs, t, pools=pool)
        return remap, live, refs, t, pool

    def turnover():
        refs, bad = refs0.clone(), cuda([0])
        gdn_b200.free_pages(refs, tables, bad_index_count=bad)
        return gdn_b200.alloc_pages(refs, torch.tensor([True, False, True]).cuda()), refs, bad

    for call in (copy, fork, compact, turnover):
        a, b = both(monkeypatch, call)
        assert same(a, b), call
    # what the extension declines and ctypes makes: int64 indices, pages with a pitch
    pool = start.clone()
    gdn_b200.copy_pages(pool[:, :2], cuda([0, 1]).long(), cuda([1, 0]))
    assert torch.equal(pool[0, :2], start[1, :2]) and torch.equal(pool[0, 2], start[0, 2])
    with pytest.raises(ValueError, match="4096"):
        gdn_b200.copy_pages(pool, torch.zeros(4097, dtype=I32, device="cuda"),
                            torch.zeros(4097, dtype=I32, device="cuda"))
    with pytest.raises(_lib.GdnError, match="overlap"):
        gdn_b200.copy_pages([pool, pool], cuda([0]), cuda([1]))
