"""Plain definitions of the serving operators, in 64 bits and Python loops, on the CPU.

``attention`` / ``beam`` return 64-bit values; the page operators return what their pools,
tables and reference counts become.  Written from the definitions in include/gdn_b200.h.
"""

from __future__ import annotations

import math

import torch


def attention(q, k_cache, v_cache, tables, lens, k=None, v=None, scale=None, window=0, sinks=0):
    """(output [B,HQ,D], lse [B,HQ], mean |v| under the softmax [B,HQ,D], largest
    scale * sum |q||k| [B,HQ], k_cache, v_cache after the call, bad count)."""
    q, kc, vc = q.cpu().double(), k_cache.cpu().clone(), v_cache.cpu().clone()
    tables, lens = tables.cpu(), lens.cpu()
    B, _, HQ, D = q.shape
    P, ps, HKV, _ = kc.shape
    width = tables.shape[1]
    if scale is None or scale == 0:                     # 0 stands for it too, as in the GDN entries
        scale = 1.0 / math.sqrt(D)
    out = torch.zeros(B, HQ, D, dtype=torch.float64)
    absv = torch.zeros(B, HQ, D, dtype=torch.float64)
    lse = torch.full((B, HQ), -math.inf, dtype=torch.float64)
    mag = torch.zeros(B, HQ, dtype=torch.float64)
    bad = 0
    seen_rows = []
    for b in range(B):
        n = max(0, int(lens[b]))
        fits = n <= width * ps
        bad += not fits
        n = min(n, width * ps)
        new = k is not None and n > 0 and fits
        toks = range(n)
        if window and n > sinks + window:
            toks = list(range(sinks)) + list(range(n - window, n))
        rows, counted = [], set()
        for t in toks:
            page = int(tables[b, t // ps])
            if page >= P and t // ps not in counted:
                counted.add(t // ps)
                bad += 1
            ok = 0 <= page < P
            if new and t == n - 1:
                if ok:
                    kc[page, t % ps] = k[b, 0].cpu()
                    vc[page, t % ps] = v[b, 0].cpu()
                rows.append(None)
            elif ok:
                rows.append((page, t % ps))
        seen_rows.append(rows)
    for b, rows in enumerate(seen_rows):
        if not rows:
            continue
        at = torch.tensor([r if r is not None else (0, 0) for r in rows])
        K, V = kc[at[:, 0], at[:, 1]].double(), vc[at[:, 0], at[:, 1]].double()
        if rows[-1] is None:
            K[-1], V[-1] = k[b, 0].cpu().double(), v[b, 0].cpu().double()
        for h in range(HQ):
            g = h // (HQ // HKV)
            x = scale * (K[:, g] @ q[b, 0, h])
            lse[b, h] = torch.logsumexp(x, 0)
            w = torch.softmax(x, 0)
            out[b, h] = w @ V[:, g]
            absv[b, h] = w @ V[:, g].abs()
            mag[b, h] = abs(scale) * (K[:, g].abs() @ q[b, 0, h].abs()).max()
    return out, lse, absv, mag, kc, vc, bad


def beam_candidates(logits, scores, finished=None, eos=0):
    """Per request the list of (score, beam, token) of all candidates, best first."""
    x, cum = logits.cpu().double(), scores.cpu().double()
    B, K, V = x.shape
    every = []
    for b in range(B):
        cands = []
        for i in range(K):
            if finished is not None and bool(finished[b, i]):
                if math.isfinite(cum[b, i]):
                    cands.append((float(cum[b, i]), i, eos))
                continue
            row = x[b, i]
            if row.isnan().any() or not math.isfinite(row.max()) or not math.isfinite(cum[b, i]):
                continue
            s = cum[b, i] + (row - torch.logsumexp(row, 0))
            order = torch.sort(row, descending=True, stable=True).indices
            cands += [(float(s[t]), i, int(t)) for t in order[:64].tolist()
                      if math.isfinite(s[t])]
        cands.sort(key=lambda c: -c[0])                 # stable: beam, then logit, then token
        every.append(cands)
    return every


def copy(pool, src, dst):
    """pool after the simultaneous copy, and the bad count."""
    pool = pool.cpu()
    out, P, bad = pool.clone(), pool.shape[0], 0
    for s, d in zip(src.tolist(), dst.tolist()):
        if s < 0 or d < 0:
            continue
        if s >= P or d >= P:
            bad += 1
            continue
        out[d] = pool[s]
    return out, bad


def alloc(refcounts, need):
    ref = refcounts.tolist()
    free = [p for p, c in enumerate(ref) if c <= 0]
    pages = []
    for want in need.tolist():
        page = free.pop(0) if want and free else -1
        if page >= 0:
            ref[page] = 1
        pages.append(page)
    return torch.tensor(ref, dtype=torch.int32), torch.tensor(pages, dtype=torch.int32)


def free(refcounts, pages):
    ref, bad = refcounts.tolist(), 0
    for p in pages.flatten().tolist():
        if p < 0:
            continue
        if p >= len(ref) or ref[p] <= 0:
            bad += 1
        else:
            ref[p] -= 1
    return torch.tensor(ref, dtype=torch.int32), bad


def fork(tables, lens, parents, refcounts, ps, pools=()):
    """(new tables, new lens, refcounts, pools after, bad count)."""
    tables, lens, ref = tables.cpu(), lens.tolist(), refcounts.tolist()
    pools = [p.cpu().clone() for p in pools]
    rows, width = tables.shape
    P, bad = len(ref), 0
    children = [sum(1 for q in parents.tolist() if q == r) for r in range(rows)]
    n_of = [min(max(0, n), width * ps) for n in lens]
    for r in range(rows):
        for j in range(-(-n_of[r] // ps)):
            page = int(tables[r, j])
            if 0 <= page < P:
                full = j < n_of[r] // ps
                ref[page] += children[r] - 1 if full else min(children[r], 1) - 1
    out = torch.full((len(parents), width), -1, dtype=torch.int32)
    new_lens, seen = [], set()
    for i, q in enumerate(parents.tolist()):
        if not 0 <= q < rows:
            bad += q >= rows
            new_lens.append(0)
            continue
        used = -(-n_of[q] // ps)
        out[i, :used] = tables[q, :used]
        new_lens.append(n_of[q])
        if q in seen and n_of[q] % ps and 0 <= int(tables[q, used - 1]) < P:
            page = next((p for p, c in enumerate(ref) if c <= 0), -1)
            out[i, used - 1] = page
            if page < 0:
                bad += 1
            else:
                ref[page] = 1
                for pool in pools:
                    pool[page] = pool[int(tables[q, used - 1])]
        seen.add(q)
    return (out, torch.tensor(new_lens, dtype=torch.int32), torch.tensor(ref, dtype=torch.int32),
            pools, bad)


def compact(refcounts, tables=None, pools=()):
    """(remap, live count, refcounts, tables, pools after)."""
    ref = refcounts.tolist()
    live = [p for p, c in enumerate(ref) if c > 0]
    L = len(live)
    holes = [p for p in range(L) if ref[p] <= 0]
    movers = [p for p in live if p >= L]
    remap = [p if c > 0 else -1 for p, c in enumerate(ref)]
    pools = [p.cpu().clone() for p in pools]
    for s, d in zip(movers, holes):
        remap[s] = d
        ref[d], ref[s] = ref[s], 0
        for pool in pools:
            pool[d] = pool[s]
    if tables is not None:
        tables = tables.cpu().clone()
        flat = tables.view(-1)
        for i, t in enumerate(flat.tolist()):
            if 0 <= t < len(ref):
                flat[i] = remap[t]
    return (torch.tensor(remap, dtype=torch.int32), L, torch.tensor(ref, dtype=torch.int32),
            tables, pools)
