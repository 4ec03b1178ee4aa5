"""The page operators on the GPU: bytes and whole numbers, compared exactly."""

import pytest
import torch

import gdn_b200
from oracle import serving_ref

pytestmark = pytest.mark.gpu
I32 = torch.int32


def rand_pool(shape, dtype, g):
    if dtype.is_floating_point:
        return torch.randn(shape, generator=g).to(dtype).cuda()
    return torch.randint(-100, 100, shape, generator=g).to(dtype).cuda()


def ints(v):
    return torch.tensor(v, dtype=I32).cuda()


def counter():
    return torch.zeros(1, dtype=I32, device="cuda")


@pytest.mark.parametrize("shape,dtype", [((12, 8, 128, 16), torch.float32), ((12, 7), torch.bfloat16),
                                         ((12, 1), torch.uint8), ((12, 3, 5), torch.float16),
                                         ((12, 1000, 4), torch.int32), ((12, 33), torch.int64),
                                         ((12, 20000), torch.float32)])
def test_copy_is_simultaneous(shape, dtype):
    g = torch.Generator().manual_seed(shape[-1])
    for src, dst in [([0, 1, 2, 3], [1, 2, 3, 0]),            # a cycle
                     ([5, 5, 5], [5, 6, 7]),                  # one parent, one of them itself
                     ([3, 4], [4, 3]), ([9], [2]), ([], []),
                     ([1, 2, 8], [7, 7, 7]),                  # the last pair wins
                     ([1, 2, 7], [7, 7, 7]),
                     ([-1, 2, 11, 0], [3, -1, 0, 11])]:
        pool = rand_pool(shape, dtype, g)
        want, _ = serving_ref.copy(pool, torch.tensor(src), torch.tensor(dst))
        gdn_b200.copy_pages(pool, ints(src), ints(dst))
        assert torch.equal(pool.cpu(), want), (src, dst)


@pytest.mark.parametrize("n,slots,elems", [(300, 512, 700), (1024, 1030, 128), (4096, 5000, 40),
                                           (2000, 2000, 12), (33, 33, 16384)])
def test_copy_many(n, slots, elems):
    g = torch.Generator().manual_seed(n)
    pool = rand_pool((slots, elems), torch.float32, g)
    src = torch.randint(-1, slots + 1, (n,), generator=g)
    dst = torch.randint(-1, slots + 1, (n,), generator=g)     # with repeats
    want, bad = serving_ref.copy(pool, src, dst)
    c = counter()
    gdn_b200.copy_pages(pool, src.int().cuda(), dst.cuda(), bad_index_count=c)
    assert torch.equal(pool.cpu(), want)
    assert int(c) == bad


def test_copy_several_pools_strided_and_wide_indices():
    g = torch.Generator().manual_seed(1)
    kv = rand_pool((9, 2, 16, 2, 64), torch.bfloat16, g)
    conv = rand_pool((9, 3, 77), torch.bfloat16, g)
    padded = rand_pool((9, 50), torch.float32, g)
    pools = [kv[:, 0], kv[:, 1], conv, padded[:, :37]]
    src = torch.tensor([0, 1, 8, 2**33, 4, -2**40], dtype=torch.int64).cuda()
    dst = torch.tensor([1, 0, 3, 5, 2**32 + 2, 6], dtype=torch.int64).cuda()
    c = counter()
    want = [serving_ref.copy(p, src.cpu(), dst.cpu())[0] for p in pools]
    rest = padded[:, 37:].cpu().clone()
    gdn_b200.copy_pages(pools, src, dst, bad_index_count=c)
    for p, w in zip(pools, want):
        assert torch.equal(p.cpu(), w)
    assert torch.equal(padded[:, 37:].cpu(), rest) and int(c) == 2


def test_copy_beyond_32_bit_offsets():
    P, elems = 70, 16 * 1024 * 1024                  # 64 MB a page, 4.7 GB
    pool = torch.zeros((P, elems), dtype=torch.float32, device="cuda")
    pool[P - 1] = torch.arange(elems, device="cuda").float()
    pool[3] = 7.0
    gdn_b200.copy_pages(pool, ints([P - 1, 3]), ints([3, P - 2]))
    assert torch.equal(pool[3], pool[P - 1]) and bool((pool[P - 2] == 7.0).all())


@pytest.mark.parametrize("P,n,seed", [(1, 1, 0), (5, 9, 1), (1000, 300, 2), (70000, 5000, 3),
                                      (1025, 1024, 4), (4096, 1, 5)])
def test_alloc_and_free(P, n, seed):
    g = torch.Generator().manual_seed(seed)
    ref = torch.randint(0, 3, (P,), generator=g, dtype=I32)
    need = torch.rand(n, generator=g) < 0.7
    want_ref, want = serving_ref.alloc(ref, need)
    r = ref.cuda()
    pages = gdn_b200.alloc_pages(r, need.cuda())
    assert torch.equal(pages.cpu(), want) and torch.equal(r.cpu(), want_ref)
    out = torch.randint(-2, P + 2, (n, 3), generator=g, dtype=I32)
    want_ref, bad = serving_ref.free(want_ref, out)
    c = counter()
    gdn_b200.free_pages(r, out.cuda(), bad_index_count=c)
    assert torch.equal(r.cpu(), want_ref) and int(c) == bad


def test_alloc_when_nothing_is_free_or_needed():
    r = torch.ones(50, dtype=I32, device="cuda")
    assert gdn_b200.alloc_pages(r, torch.ones(3, dtype=torch.bool, device="cuda")).tolist() == [-1] * 3
    r.zero_()
    assert gdn_b200.alloc_pages(r, torch.zeros(3, dtype=torch.bool, device="cuda")).tolist() == [-1] * 3
    assert int(r.sum()) == 0
    assert gdn_b200.alloc_pages(r, torch.zeros(0, dtype=torch.bool, device="cuda")).numel() == 0
    gdn_b200.free_pages(r, torch.zeros(0, dtype=I32, device="cuda"))


def tables_for(lens, ps, width, g, extra):
    """Rows with pages of their own, one of them also sharing another's first page."""
    used = [-(-max(0, n) // ps) for n in lens]
    P = sum(used) + extra
    order = torch.randperm(P, generator=g).int()
    t = torch.full((len(lens), width), -1, dtype=I32)
    ref = torch.zeros(P, dtype=I32)
    at = 0
    for r, u in enumerate(used):
        t[r, :u] = order[at:at + u]
        at += u
        ref[t[r, :u].long()] += 1
    return t, ref


@pytest.mark.parametrize("lens,parents,ps,extra", [
    ([5, 16, 33], [0, 0, 1, 1, 2, 2, 2], 16, 8),
    ([5, 16, 33], [2], 16, 0),
    ([1], [0] * 12, 4, 30),
    ([20, 7, 40, 0], [3, -1, 2, 9, 0, 2, 0], 8, 5),
    ([20, 7, 40], [0, 0, 0, 1, 1, 2, 2], 8, 2),           # too few pages for the copies
    ([20, 7, 40], [], 8, 1),
    ([64] * 40, [i // 2 for i in range(40)], 16, 3),
    ([63] * 300, [i // 3 * 2 for i in range(310)], 16, 400),
])
def test_fork(lens, parents, ps, extra):
    g = torch.Generator().manual_seed(len(parents))
    t, ref = tables_for(lens, ps, max(-(-max(lens) // ps), 1) + 2, g, extra)
    P = ref.numel()
    pools = [rand_pool((P, ps, 2, 8), torch.bfloat16, g), rand_pool((P, ps, 3), torch.float32, g)]
    want = serving_ref.fork(t, torch.tensor(lens), torch.tensor(parents), ref, ps, pools)
    r, c = ref.cuda(), counter()
    nt, nl = gdn_b200.fork_pages(t.cuda(), ints(lens), ints(parents), r, ps, pools=pools,
                                 bad_index_count=c)
    assert torch.equal(nt.cpu(), want[0]) and torch.equal(nl.cpu(), want[1])
    assert torch.equal(r.cpu(), want[2]) and int(c) == want[4]
    for p, w in zip(pools, want[3]):
        assert torch.equal(p.cpu(), w)


def test_fork_with_shared_pages_and_bad_entries():
    g = torch.Generator().manual_seed(3)
    t, ref = tables_for([40, 40, 25], 8, 6, g, 6)
    t[1, :3] = t[0, :3]                               # a shared prefix
    ref.zero_()
    for v in t.flatten().tolist():
        if v >= 0:
            ref[v] += 1
    t[2, 1], t[2, 3] = -1, 10_000                     # bad entries, the partial page's too
    pool = rand_pool((ref.numel(), 8), torch.float32, g)
    lens, parents = [40, 37, 25], [1, 1, 2, 2, 1]
    want = serving_ref.fork(t, torch.tensor(lens), torch.tensor(parents), ref, 8, [pool])
    r, c = ref.cuda(), counter()
    nt, nl = gdn_b200.fork_pages(t.cuda(), ints(lens), torch.tensor(parents).cuda(), r, 8, pools=pool,
                                 bad_index_count=c)
    assert torch.equal(nt.cpu(), want[0]) and torch.equal(nl.cpu(), want[1])
    assert torch.equal(r.cpu(), want[2]) and torch.equal(pool.cpu(), want[3][0])
    assert int(c) == want[4]


def test_fork_without_pools_and_empty():
    t, ref = tables_for([9, 9], 4, 3, torch.Generator().manual_seed(0), 4)
    r = ref.cuda()
    nt, nl = gdn_b200.fork_pages(t.cuda(), ints([9, 9]), ints([1, 1]), r, 4)
    want = serving_ref.fork(t, torch.tensor([9, 9]), torch.tensor([1, 1]), ref, 4)
    assert torch.equal(nt.cpu(), want[0]) and torch.equal(r.cpu(), want[2])
    e = torch.empty((0, 3), dtype=I32, device="cuda")
    nt, nl = gdn_b200.fork_pages(e, ints([]), ints([]), r, 4)
    assert nt.shape == (0, 3) and nl.shape == (0,) and torch.equal(r.cpu(), want[2])


@pytest.mark.parametrize("P,live", [(1, 0.0), (1, 1.0), (7, 0.5), (64, 0.0), (64, 1.0), (1000, 0.3),
                                    (5003, 0.9), (3000, 0.05), (70001, 0.5)])
def test_compact(P, live):
    g = torch.Generator().manual_seed(P)
    ref = torch.randint(1, 4, (P,), generator=g, dtype=I32) * (torch.rand(P, generator=g) < live).int()
    t = torch.randint(-3, P + 3, (13, 5), generator=g, dtype=I32)
    pools = [rand_pool((P, 36), torch.bfloat16, g), rand_pool((P, 3), torch.uint8, g)]
    want = serving_ref.compact(ref, t, pools)
    r, tt = ref.cuda(), t.cuda()
    remap, n = gdn_b200.compact_pages(r, tt, pools=pools)
    assert torch.equal(remap.cpu(), want[0]) and int(n) == want[1]
    assert torch.equal(r.cpu(), want[2]) and torch.equal(tt.cpu(), want[3])
    for p, w in zip(pools, want[4]):
        assert torch.equal(p[:want[1]].cpu(), w[:want[1]])
        assert torch.equal(p.cpu(), w)


@pytest.mark.parametrize("P", [5, 4096, 16385, 40003])
def test_counts_that_do_not_begin_on_16_bytes(P):
    g = torch.Generator().manual_seed(P)
    ref = torch.randint(-1, 3, (P,), generator=g, dtype=I32)
    for off in (1, 2, 3):
        r = torch.full((P + 8,), 7, dtype=I32, device="cuda")
        r[off:off + P] = ref.cuda()
        want = serving_ref.compact(ref, None, [])
        remap, n = gdn_b200.compact_pages(r[off:off + P])
        assert torch.equal(remap.cpu(), want[0]) and int(n) == want[1]
        assert torch.equal(r[off:off + P].cpu(), want[2])
        assert r[:off].eq(7).all() and r[off + P:].eq(7).all()
        r[off:off + P] = ref.cuda()
        free = (ref <= 0).nonzero()[:, 0].tolist()
        need = torch.ones(len(free) + 3, dtype=torch.bool, device="cuda")
        pages = gdn_b200.alloc_pages(r[off:off + P], need)
        assert pages.tolist() == free + [-1] * 3
        assert r[off:off + P].gt(0).all() and r[:off].eq(7).all() and r[off + P:].eq(7).all()


def test_compact_without_tables_or_pools():
    r = ints([0, 2, 0, 1])
    remap, n = gdn_b200.compact_pages(r)
    assert remap.tolist() == [-1, 1, -1, 0] and int(n) == 2 and r.tolist() == [1, 2, 0, 0]


def test_in_graphs():
    g = torch.Generator().manual_seed(8)
    pool = rand_pool((20, 1000), torch.float32, g)
    start, src, dst = pool.clone(), ints([0, 1, 2]), ints([1, 2, 0])
    t, ref = tables_for([9, 12, 30], 8, 5, g, 10)
    t, ref, lens, par = t.cuda(), ref.cuda(), ints([9, 12, 30]), ints([0, 0, 2])
    ref0 = ref.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            gdn_b200.copy_pages(pool, src, dst)
            ref.copy_(ref0)
            nt, nl = gdn_b200.fork_pages(t, lens, par, ref, 8)
            remap, live = gdn_b200.compact_pages(ref, nt)
    torch.cuda.synchronize()
    want = serving_ref.fork(t, lens.cpu(), par.cpu(), ref0, 8)
    want_c = serving_ref.compact(want[2], want[0])
    for k in range(1, 4):
        graph.replay()
        torch.cuda.synchronize()
        idx = [(i - k) % 3 for i in range(3)]
        assert torch.equal(pool[:3], start[idx]) and torch.equal(pool[3:], start[3:])
        assert torch.equal(nt.cpu(), want_c[3]) and torch.equal(ref.cpu(), want_c[2])
        assert torch.equal(remap.cpu(), want_c[0]) and int(live) == want_c[1]
