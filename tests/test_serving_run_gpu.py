"""A beam search over a small stack of one GDN layer and one attention layer, with both caches
kept by the serving operators: prompts, forks into beams, steps, compaction, the end.

The layers' q, k, v and gates depend on the tokens alone, so each surviving beam's recurrent
state and cached rows must equal, bit for bit, those of its token history fed through the
same decode step without any fork or copy; the logits depend on both layers' outputs.
"""

import pytest
import torch

import gdn_b200

pytestmark = pytest.mark.gpu

R, K, V, PS, D = 3, 4, 500, 8, 64          # requests, beams, vocabulary, page size, attention dim
H, HV, HQ, HKV = 4, 8, 8, 2
I32 = torch.int32


class Stack:
    def __init__(self, seed):
        g = torch.Generator().manual_seed(seed)
        r = lambda *s: torch.randn(*s, generator=g).to(torch.bfloat16).cuda()  # noqa: E731
        self.gq, self.gk, self.gv = r(V, H, 128), r(V, H, 128), r(V, HV, 128)
        self.a, self.b = r(V, HV), r(V, HV)
        self.A_log = torch.rand(HV, generator=g).cuda()
        self.dt = torch.randn(HV, generator=g).cuda()
        self.q, self.k, self.v = r(V, HQ, D), r(V, HKV, D), r(V, HKV, D)
        self.out = (torch.randn(HV * 128 + HQ * D, V, generator=g) * 0.15).cuda()

    def gdn(self, tokens, pool, slots):
        t = tokens.long()
        o, _ = gdn_b200.gated_delta_rule_decode_pretranspose(
            self.gq[t][:, None], self.gk[t][:, None], self.gv[t][:, None], None, self.A_log,
            self.a[t][:, None], self.dt, self.b[t][:, None], initial_state=pool,
            initial_state_indices=slots)
        return o

    def step(self, tokens, pool, slots, caches, tables, lens):
        t = tokens.long()
        g = self.gdn(tokens, pool, slots)
        o, _ = gdn_b200.paged_attention_decode(
            self.q[t][:, None], *caches, tables, lens, k=self.k[t][:, None], v=self.v[t][:, None])
        x = torch.cat([g.flatten(1), o.flatten(1)], 1).float()
        return (x @ self.out).to(torch.bfloat16)


def grow(tables, lens, refcounts):
    """One more token per row: a page where the last one is full."""
    need = lens % PS == 0
    pages = gdn_b200.alloc_pages(refcounts, need)
    at = (lens // PS).long()[:, None]
    tables.scatter_(1, at, torch.where(need[:, None], pages[:, None], tables.gather(1, at)))
    lens += 1


@pytest.mark.parametrize("seed", [0, 1])
def test_beam_search_over_both_caches(seed):
    s = Stack(seed)
    g = torch.Generator().manual_seed(100 + seed)
    prompts = [torch.randint(0, V, (n,), generator=g).tolist() for n in (13, 8, 21)]
    pages, width, steps = 150, 12, 30
    caches = [torch.full((pages, PS, HKV, D), float("nan"), dtype=torch.bfloat16, device="cuda")
              for _ in range(2)]
    pool = torch.zeros((R * K, HV, 128, 128), device="cuda")
    refcounts = torch.zeros(pages, dtype=I32, device="cuda")
    tables = torch.full((R, width), -1, dtype=I32, device="cuda")
    lens = torch.zeros(R, dtype=I32, device="cuda")
    slots = torch.arange(0, R * K, K, dtype=I32, device="cuda")
    # prompts token by token; shorter ones wait as padding rows (length 0, slot -1)
    logits = [None] * R
    for i in range(max(map(len, prompts))):
        on = [r for r in range(R) if i < len(prompts[r])]
        rows = torch.tensor(on, device="cuda")
        t, n = tables[rows], lens[rows]
        grow(t, n, refcounts)
        tables[rows], lens[rows] = t, n
        tokens = torch.tensor([prompts[r][i] if r in on else 0 for r in range(R)], device="cuda")
        active = torch.zeros(R, dtype=torch.bool, device="cuda")
        active[rows] = True
        x = s.step(tokens, pool, torch.where(active, slots, -1), caches, tables,
                   torch.where(active, lens, 0))
        for r in on:
            logits[r] = x[r]
    # K beams per request from one row each
    first = torch.stack(logits)[:, None]
    tokens, _, scores = gdn_b200.beam_select(first, torch.zeros(R, 1, device="cuda"), num_selected=K)
    parents = torch.arange(R, device="cuda").repeat_interleave(K)
    tables, lens = gdn_b200.fork_pages(tables, lens, parents, refcounts, PS, pools=caches)
    all_slots = torch.arange(R * K, dtype=I32, device="cuda")
    gdn_b200.copy_pages(pool, slots.repeat_interleave(K), all_slots)
    history = [prompts[r] + [int(tokens[r, j])] for r in range(R) for j in range(K)]
    base = torch.arange(0, R * K, K, device="cuda")[:, None]
    for i in range(steps):
        grow(tables, lens, refcounts)
        x = s.step(tokens.flatten(), pool, all_slots, caches, tables, lens)
        tokens, par, scores = gdn_b200.beam_select(x.view(R, K, V), scores)
        parents = (base + par).flatten()
        tables, lens = gdn_b200.fork_pages(tables, lens, parents, refcounts, PS, pools=caches)
        gdn_b200.copy_pages(pool, parents, all_slots)
        history = [history[p] + [t] for p, t in zip(parents.tolist(), tokens.flatten().tolist())]
        if i % 10 == 9:
            remap, live = gdn_b200.compact_pages(refcounts, tables, pools=caches)
            assert int(live) == int((refcounts > 0).sum())
            assert int(tables.max()) < int(live)
    # every reference is a table entry and the other way round
    held = tables[tables >= 0].long()
    assert torch.equal(torch.bincount(held, minlength=pages).int(), refcounts)
    assert (scores[:, :-1] >= scores[:, 1:]).all()
    # the beams' caches are those of their histories (the last token is not fed yet)
    assert len(set(map(tuple, history))) == R * K
    fed = [h[:-1] for h in history]
    assert lens.tolist() == [len(h) for h in fed]
    alone = torch.zeros((R * K, HV, 128, 128), device="cuda")
    for i in range(max(map(len, fed))):
        t = torch.tensor([h[i] if i < len(h) else 0 for h in fed], device="cuda")
        on = torch.tensor([i < len(h) for h in fed], device="cuda")
        s.gdn(t, alone, torch.where(on, all_slots, -1))
    assert torch.equal(pool, alone)
    for row, h in enumerate(fed):
        t = torch.tensor(h, device="cuda")
        pg = tables[row, :-(-len(h) // PS)].long()
        for cache, src in zip(caches, (s.k, s.v)):
            assert torch.equal(cache[pg].flatten(0, 1)[:len(h)], src[t])
    gdn_b200.free_pages(refcounts, tables)
    assert int(refcounts.abs().sum()) == 0
