"""The serving operators next to the GDN decode step, as measured cases.

Three operators that a server runs around each decode step:

* ``attend`` - softmax attention of one new token over a paged key-value cache, the other
  token mixer of a stack that alternates GDN and attention layers.  The new token's key and
  value are appended to the cache in the same call.
* ``beam``   - beam search's selection over beams and vocabulary.
* ``copy`` / ``fork`` / ``compact`` / ``turnover`` - the pages of a cache (slots of the pooled
  recurrent state, pages of the key-value cache): copying them as one simultaneous
  assignment, forking sequences, closing the holes of a pool, freeing and allocating.

``own`` False computes each operator in elementary torch operations; True calls gdn_b200.
"""

import math
import os
import sys

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _gdn():
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                       "flashinfer-competition-codebase_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import gdn_b200

    return gdn_b200


# --------------------------------------------------------------------------- the cases


def _attend(name, batch, heads, kv_heads, dim, page, longest, dtype="bf16", window=0, sinks=0,
            shortest=0.5):
    return {"op": "attend", "name": name, "batch": batch, "heads": heads, "kv_heads": kv_heads,
            "dim": dim, "page": page, "longest": longest, "dtype": dtype, "window": window,
            "sinks": sinks, "shortest": shortest}


def _beam(name, batch, beams, vocab, selected, dtype="bf16", finished=0.0, first=False):
    return {"op": "beam", "name": name, "batch": batch, "beams": beams, "vocab": vocab,
            "selected": selected, "dtype": dtype, "finished": finished, "first": first}


def listed():
    return [
        # one user, short context, the attention layer of one rank of a 4-way head split: latency
        _attend("attend one short", 1, 4, 1, 128, 16, 100),
        # a full serving batch of ragged contexts, grouped heads
        _attend("attend batch ragged", 64, 32, 8, 128, 16, 8191),
        # one user with a very long document, few key-value heads of 256
        _attend("attend one long", 1, 16, 2, 256, 64, 131072, shortest=1.0),
        # sliding-window layers with first tokens kept visible, fp16, small heads, odd pages
        _attend("attend window fp16", 128, 14, 2, 64, 24, 20001, "fp16", 1024, 4),
        # one request of 4 beams with a small vocabulary: latency
        _beam("beam one request", 1, 4, 32000, 4),
        # a full batch of 8 beams, 2 candidates kept per beam, a large vocabulary
        _beam("beam full batch", 64, 8, 151936, 16, finished=0.1),
        # wide beams over fp32 logits of an odd vocabulary
        _beam("beam wide fp32", 8, 32, 50257, 32, "fp32", finished=0.25),
        # reordering the recurrent states of one request's beams (8 v-heads, fp32)
        {"op": "copy", "name": "copy one request", "slots": 16, "pairs": 4, "elems": 8 * 128 * 128,
         "dtype": "fp32", "pools": 1},
        # reordering 64 requests x 4 beams in the decode benchmark's pool layout (32 v-heads)
        {"op": "copy", "name": "copy full batch", "slots": 320, "pairs": 256,
         "elems": 32 * 128 * 128, "dtype": "fp32", "pools": 1},
        # beam reorder of a paged cache: tables, reference counts, copies of the partial pages
        {"op": "fork", "name": "fork full batch", "batch": 64, "beams": 8, "page": 16,
         "kv_heads": 8, "dim": 128, "longest": 4000},
        # closing the holes of a key-value pool after many requests have left
        {"op": "compact", "name": "compact half full", "pages": 8191, "page": 16, "kv_heads": 8,
         "dim": 128, "live": 0.5, "rows": 64},
        # requests that leave give up their pages, new ones take theirs
        {"op": "turnover", "name": "turnover", "pages": 65536, "leaving": 4000, "coming": 1000},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attend", "attend", "attend", "beam", "beam", "copy", "fork", "compact",
                     "turnover"])
    if op == "attend":
        dim = rng.choice([64, 128, 256])
        kv_heads = rng.choice([1, 2, 3, 4, 8])
        group = rng.choice([1, 2, 4, 5, 7, 8, 12, 16, 24])
        batch = _log(rng, 1, 160)
        # at most the largest listed case's values (64 x 6144 x 8 x 128) in the cache
        most = min(131072, 390_000_000 // (batch * kv_heads * dim))
        longest = _log(rng, 1, max(1, most))
        window = rng.choice([0, 0, _log(rng, 1, 4096)])
        sinks = rng.choice([0, 1, 4, 17]) if window else 0
        page = rng.choice([1, 8, 16, 16, 32, 64, 100, 256])
        c = _attend("", batch, kv_heads * group, kv_heads, dim, page, longest,
                    rng.choice(["bf16", "bf16", "fp16"]), window, sinks, rng.uniform(0.0, 1.0))
    elif op == "beam":
        beams = rng.choice([1, 2, 3, 4, 5, 8, 12, 16, 32])
        vocab = _log(rng, 128, 200000)
        batch = max(1, min(_log(rng, 1, 128), 77_000_000 // (vocab * beams)))
        selected = rng.choice([beams, min(64, 2 * beams), min(64, 2 * beams + 1)])
        c = _beam("", batch, beams, vocab, selected, rng.choice(["bf16", "fp16", "fp32"]),
                  rng.choice([0.0, 0.0, 0.3]), rng.random() < 0.2)
        if c["dtype"] == "fp32":
            c["batch"] = max(1, batch // 2)
    elif op == "copy":
        dtype = rng.choice(["fp32", "bf16"])
        elems = rng.choice([8, 16, 32]) * rng.choice([128 * 128, 128 * 3, 1001])
        pools = rng.choice([1, 1, 2, 5])
        most = 130_000_000 // (elems * pools)
        pairs = min(_log(rng, 1, 1024), max(1, most))
        c = {"op": op, "slots": pairs + rng.randint(0, pairs + 4), "pairs": pairs, "elems": elems,
             "dtype": dtype, "pools": pools}
    elif op == "fork":
        c = {"op": op, "batch": _log(rng, 1, 64), "beams": rng.choice([1, 2, 4, 5, 8]),
             "page": rng.choice([8, 16, 32, 64]), "kv_heads": rng.choice([1, 2, 8]),
             "dim": rng.choice([64, 128, 256]), "longest": _log(rng, 1, 4000)}
    elif op == "compact":
        c = {"op": op, "pages": _log(rng, 16, 8191), "page": rng.choice([16, 32]),
             "kv_heads": rng.choice([1, 2, 8]), "dim": rng.choice([64, 128]),
             "live": rng.uniform(0.1, 0.9), "rows": _log(rng, 1, 128)}
    else:
        pages = _log(rng, 64, 65536)
        c = {"op": op, "pages": pages, "leaving": rng.randint(1, max(1, pages // 8)),
             "coming": rng.randint(1, max(1, pages // 8))}
    c.pop("name", None)
    return c


# --------------------------------------------------------------------------- inputs


def _lengths(case):
    """Ragged lengths of the batch in some order: evenly spread between the shortest share and
    the longest; of a batch of 16 or more one row is padding (length 0)."""
    n, longest = case["batch"], case["longest"]
    low = max(1, int(case.get("shortest", 0.25) * longest))
    lens = [longest - (longest - low) * i // max(1, n - 1) for i in range(n)]
    if n >= 16:
        lens[n // 2] = 0
    return lens


def _shuffled(values, gen):
    return [values[i] for i in torch.randperm(len(values), generator=gen).tolist()]


def _visible(case, n):
    return min(n, case["sinks"] + case["window"]) if case["window"] else n


def _prepare_attend(case, gen, cuda):
    dt = _DTYPES[case["dtype"]]
    B, HQ, HKV, D, ps = (case[k] for k in ("batch", "heads", "kv_heads", "dim", "page"))
    lens = _shuffled(_lengths(case), gen)
    width = max(1, -(-case["longest"] // ps))
    used = [-(-n // ps) for n in lens]
    spare = sum(used)                                   # a page that padding rows point at
    order = torch.randperm(spare, generator=gen) if spare else torch.zeros(0, dtype=torch.int64)
    tables = torch.full((B, width), spare, dtype=torch.int32)
    at = 0
    for b, u in enumerate(used):
        tables[b, :u] = order[at:at + u].to(torch.int32)
        at += u
    cache = [torch.empty((spare + 1, ps, HKV, D), dtype=dt, device="cuda").normal_(generator=cuda)
             for _ in range(2)]
    new = [torch.empty((B, 1, HKV, D), dtype=dt, device="cuda").normal_(generator=cuda)
           for _ in range(2)]
    q = torch.empty((B, 1, HQ, D), dtype=dt, device="cuda").normal_(generator=cuda) * 1.5
    return {"q": q, "k_cache": cache[0], "v_cache": cache[1], "tables": tables.cuda(),
            "lens": torch.tensor(lens, dtype=torch.int32).cuda(), "k": new[0], "v": new[1]}


def _prepare_beam(case, gen, cuda):
    B, K, V = case["batch"], case["beams"], case["vocab"]
    logits = torch.empty((B, K, V), dtype=_DTYPES[case["dtype"]], device="cuda")
    logits.normal_(0.0, 2.5, generator=cuda)
    scores = -8.0 - 4.0 * torch.rand((B, K), generator=gen)
    scores = scores.sort(dim=1, descending=True).values
    if case["first"]:                                   # the first step: one live beam
        scores[:, 0], scores[:, 1:] = 0.0, -math.inf
    finished = torch.rand((B, K), generator=gen) < case["finished"]
    return {"logits": logits, "scores": scores.cuda(),
            "finished": finished.cuda() if case["finished"] else None, "eos": V - 1}


def _prepare_copy(case, gen, cuda):
    slots, n = case["slots"], case["pairs"]
    dst = torch.randperm(slots, generator=gen)[:n]
    src = dst[torch.randint(0, n, (n,), generator=gen)]  # parents among the beams themselves
    pools = [torch.empty((slots, case["elems"]), dtype=_DTYPES[case["dtype"]],
                         device="cuda").normal_(generator=cuda) for _ in range(case["pools"])]
    return {"pools": pools, "src": src.to(torch.int32).cuda(), "dst": dst.to(torch.int32).cuda()}


def _prepare_fork(case, gen, cuda):
    B, K, ps = case["batch"], case["beams"], case["page"]
    lens = _shuffled(_lengths(case), gen)
    width = max(1, -(-case["longest"] // ps))
    full = [n // ps for n in lens]
    total = sum(f + K for f in full)                     # shared full pages, one partial per beam
    pages = total + B * K + 1                            # free pages for the copies, one spare
    order = torch.randperm(pages - 1, generator=gen).to(torch.int32)
    tables = torch.full((B * K, width), -1, dtype=torch.int32)
    refcounts = torch.zeros(pages, dtype=torch.int32)
    refcounts[pages - 1] = 1
    at = 0
    for b, n in enumerate(lens):
        f = full[b]
        tables[b * K:(b + 1) * K, :f] = order[at:at + f]
        refcounts[order[at:at + f].long()] = K
        at += f
        if n % ps:
            tables[b * K:(b + 1) * K, f] = order[at:at + K]
            refcounts[order[at:at + K].long()] = 1
            at += K
    parents = torch.cat([b * K + torch.randint(0, K, (K,), generator=gen) for b in range(B)])
    shape = (pages, ps, case["kv_heads"], case["dim"])
    pools = [torch.empty(shape, dtype=torch.bfloat16, device="cuda").normal_(generator=cuda)
             for _ in range(2)]
    return {"tables": tables.cuda(), "refcounts": refcounts.cuda(), "pools": pools,
            "lens": torch.tensor(lens, dtype=torch.int32).repeat_interleave(K).cuda(),
            "parents": parents.to(torch.int32).cuda(), "page": ps}


def _prepare_compact(case, gen, cuda):
    P, rows = case["pages"], case["rows"]
    live = torch.randperm(P, generator=gen)[:max(1, int(P * case["live"]))]
    refcounts = torch.zeros(P, dtype=torch.int32)
    refcounts[live] = torch.randint(1, 4, (live.numel(),), generator=gen, dtype=torch.int32)
    width = -(-live.numel() // rows)
    tables = torch.full((rows * width,), -1, dtype=torch.int32)
    tables[:live.numel()] = live.to(torch.int32)
    shape = (P, case["page"], case["kv_heads"], case["dim"])
    pools = [torch.empty(shape, dtype=torch.bfloat16, device="cuda").normal_(generator=cuda)
             for _ in range(2)]
    return {"refcounts": refcounts.cuda(), "tables": tables.view(rows, width).cuda(),
            "pools": pools}


def _prepare_turnover(case, gen, cuda):
    P = case["pages"]
    refcounts = torch.randint(0, 3, (P,), generator=gen, dtype=torch.int32)
    held = refcounts.nonzero().flatten()
    leaving = held[torch.randperm(held.numel(), generator=gen)[:case["leaving"]]]
    need = torch.rand(case["coming"], generator=gen) < 0.75
    return {"refcounts": refcounts.cuda(), "leaving": leaving.to(torch.int32).cuda(),
            "need": need.cuda()}


_PREPARE = {"attend": _prepare_attend, "beam": _prepare_beam, "copy": _prepare_copy,
            "fork": _prepare_fork, "compact": _prepare_compact, "turnover": _prepare_turnover}


def prepare(case, seed):
    gen = torch.Generator().manual_seed(seed)
    cuda = torch.Generator(device="cuda").manual_seed(seed)
    state = _PREPARE[case["op"]](case, gen, cuda)
    state["case"] = dict(case)
    return state


# --------------------------------------------------------------------------- plain forms


def _plain_attend(s):
    case, ps = s["case"], s["case"]["page"]
    q, lens, tables = s["q"], s["lens"].long(), s["tables"].long()
    B, HQ, HKV, D = q.shape[0], case["heads"], case["kv_heads"], case["dim"]
    # append the new token (padding rows keep what their spare page holds)
    last = (lens - 1).clamp(min=0)
    page = tables.gather(1, (last // ps)[:, None])[:, 0]
    there = (lens > 0)[:, None, None]
    for cache, new in ((s["k_cache"], s["k"]), (s["v_cache"], s["v"])):
        cache[page, last % ps] = torch.where(there, new[:, 0], cache[page, last % ps])
    # the visible tokens: all, or the sinks and the window
    most = _visible(case, case["longest"])
    seen = lens if not case["window"] else lens.clamp(max=case["sinks"] + case["window"])
    i = torch.arange(most, device=q.device)[None]
    token = torch.where(i < case["sinks"], i, i + (lens - seen)[:, None]) if case["window"] else i
    valid = i < seen[:, None]
    token = torch.where(valid, token, 0)
    page = tables.gather(1, token // ps)
    keys = s["k_cache"][page, token % ps].float().permute(0, 2, 3, 1)
    qf = q[:, 0].float().reshape(B, HKV, HQ // HKV, D)
    x = torch.matmul(qf, keys) * (1.0 / math.sqrt(D))
    del keys
    x = x.masked_fill(~valid[:, None, None], -math.inf)
    m = x.amax(-1, keepdim=True).clamp(min=-3e38)
    p = torch.exp(x - m)
    total = p.sum(-1, keepdim=True, dtype=torch.float64)
    values = s["v_cache"][page, token % ps].float().permute(0, 2, 1, 3)
    o = torch.matmul(p, values) / total.clamp(min=1e-300).float()
    lse = (m.double() + torch.log(total)).float()
    o = torch.where((lens > 0)[:, None, None, None], o, 0.0)
    lse = torch.where((lens > 0)[:, None, None, None], lse, -math.inf)
    return {"output": o.reshape(B, 1, HQ, D).to(q.dtype), "lse": lse.reshape(B, HQ),
            "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _plain_beam(s):
    case, n = s["case"], s["case"]["selected"]
    B, K, V = s["logits"].shape
    x = s["logits"].float() + 0.0
    m = x.amax(-1, keepdim=True)
    # 64 bits for the sum and the scores: candidates of different beams are compared
    lse = m[..., 0].double() + torch.log(torch.exp(x - m).sum(-1, dtype=torch.float64))
    # one beam's candidates by logit, equal ones by token: (logit's ordered bits, ~token)
    bits = x.view(torch.int32)
    bits = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long()
    key = bits * 2**32 + (2**32 - 1 - torch.arange(V, device=x.device))
    token = 2**32 - 1 - (key.topk(min(n, V), dim=-1).values & 0xFFFFFFFF)
    score = s["scores"].double()[..., None] + (x.gather(-1, token).double() - lse[..., None])
    if s["finished"] is not None:                       # a finished beam stands for itself
        done = s["finished"][..., None]
        one = torch.where(torch.arange(token.shape[-1], device=x.device) == 0,
                          s["scores"].double()[..., None], -math.inf)
        score = torch.where(done, one, score)
        token = torch.where(done, s["eos"], token)
    score = torch.where(torch.isfinite(score), score, -math.inf).reshape(B, -1)
    token = token.reshape(B, -1)
    width = K * min(n, V)
    if width < n:
        pad = torch.zeros((B, n - width), device=x.device)
        score = torch.cat([score, pad.double() - math.inf], 1)
        token = torch.cat([token, pad.long()], 1)
    best, at = torch.sort(score, dim=-1, descending=True, stable=True)
    best, at = best[:, :n], at[:, :n]
    none = torch.isinf(best)
    parents = torch.where(none, -1, at // min(n, V)).int()
    tokens = torch.where(none, -1, token.gather(1, at)).int()
    return {"tokens": tokens, "parents": parents, "scores": best.float()}


def _plain_copy(s):
    src, dst = s["src"].long(), s["dst"].long()
    for pool in s["pools"]:
        pool[dst] = pool[src]
    return list(s["pools"])


def _first_free(refcounts):
    """Indices of the pages, the free ones first, each kind ascending."""
    return torch.argsort((refcounts > 0).int(), stable=True)


def _plain_fork(s):
    tables, lens, ps = s["tables"].long(), s["lens"].long(), s["page"]
    parents, refcounts = s["parents"].long(), s["refcounts"].clone()
    rows, width = tables.shape
    P, dev = refcounts.numel(), tables.device
    children = torch.zeros(rows, dtype=torch.int32, device=dev)
    children.index_add_(0, parents, torch.ones_like(parents, dtype=torch.int32))
    column = torch.arange(width, device=dev)
    full, part = (lens // ps)[:, None], ((lens % ps) > 0)[:, None]
    delta = torch.where(column < full, children[:, None] - 1, 0)
    at_part = (column == full) & part
    delta = torch.where(at_part, children[:, None].clamp(max=1) - 1, delta)
    held = (column < full) | at_part
    refcounts.index_add_(0, torch.where(held, tables, 0).flatten(), delta.flatten().int())
    # children after the first take a copy of the partial page
    i = torch.arange(parents.numel(), device=dev)
    first = torch.full((rows,), parents.numel(), device=dev)
    first = first.scatter_reduce(0, parents, i, "amin")
    wants = (first[parents] != i) & ((lens[parents] % ps) > 0)
    fresh = _first_free(refcounts)[(wants.cumsum(0) - 1).clamp(min=0)]
    dst = torch.where(wants, fresh, P - 1)               # P - 1: the spare page
    refcounts[dst] = 1
    new = torch.where((column < full) | at_part, tables, -1)[parents]
    here = (lens[parents] // ps)[:, None] == column
    src = torch.where(wants, torch.where(here, new, 0).sum(1), P - 1)
    new = torch.where(here & wants[:, None], fresh[:, None], new)
    for pool in s["pools"]:
        pool[dst] = pool[src]
    return {"tables": new.int(), "lens": lens[parents].int(), "refcounts": refcounts,
            "pools": s["pools"]}


def _plain_compact(s):
    refcounts = s["refcounts"]
    P = refcounts.numel()
    live = refcounts > 0
    page = torch.arange(P, device=refcounts.device)
    count = live.sum(dtype=torch.int32)
    src = (live & (page >= count)).nonzero()[:, 0]
    dst = (~live & (page < count)).nonzero()[:, 0]
    for pool in s["pools"]:
        pool[dst] = pool[src]
    remap = torch.where(live, page, -1).int()
    remap[src] = dst.int()
    counts = torch.where(page < count, refcounts, 0)
    counts[dst] = refcounts[src]
    tables = s["tables"]
    tables = torch.where(tables >= 0, remap[tables.clamp(min=0).long()], tables)
    return {"remap": remap, "live": count[None], "refcounts": counts, "tables": tables,
            "pools": s["pools"]}


def _plain_turnover(s):
    refcounts = s["refcounts"].clone()
    leaving = s["leaving"].long()
    refcounts.index_add_(0, leaving, torch.full_like(s["leaving"], -1))
    refcounts.clamp_(min=0)
    need = s["need"]
    rank = (need.cumsum(0) - 1).clamp(min=0)
    order = _first_free(refcounts)
    free = (refcounts <= 0).sum()
    got = need & (rank < free)
    pages = torch.where(got, order[rank.clamp(max=order.numel() - 1)], -1).int()
    taken = torch.cat([refcounts, refcounts[:1]])        # one more place for those without need
    taken[torch.where(got, pages.long(), refcounts.numel())] = 1
    return {"refcounts": taken[:-1], "pages": pages}


_PLAIN = {"attend": _plain_attend, "beam": _plain_beam, "copy": _plain_copy, "fork": _plain_fork,
          "compact": _plain_compact, "turnover": _plain_turnover}


# --------------------------------------------------------------------------- the framework


def _own_attend(s):
    case = s["case"]
    output, lse = _gdn().paged_attention_decode(
        s["q"], s["k_cache"], s["v_cache"], s["tables"], s["lens"], k=s["k"], v=s["v"],
        window=case["window"], num_sinks=case["sinks"])
    return {"output": output, "lse": lse, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _own_beam(s):
    tokens, parents, scores = _gdn().beam_select(
        s["logits"], s["scores"], num_selected=s["case"]["selected"], finished=s["finished"],
        eos_token=s["eos"])
    return {"tokens": tokens, "parents": parents, "scores": scores}


def _own_copy(s):
    _gdn().copy_pages(s["pools"], s["src"], s["dst"])
    return list(s["pools"])


def _own_fork(s):
    refcounts = s["refcounts"].clone()
    tables, lens = _gdn().fork_pages(s["tables"], s["lens"], s["parents"], refcounts, s["page"],
                                     pools=s["pools"])
    return {"tables": tables, "lens": lens, "refcounts": refcounts, "pools": s["pools"]}


def _own_compact(s):
    refcounts, tables = s["refcounts"].clone(), s["tables"].clone()
    remap, live = _gdn().compact_pages(refcounts, tables, pools=s["pools"])
    return {"remap": remap, "live": live, "refcounts": refcounts, "tables": tables,
            "pools": s["pools"]}


def _own_turnover(s):
    refcounts = s["refcounts"].clone()
    _gdn().free_pages(refcounts, s["leaving"])
    pages = _gdn().alloc_pages(refcounts, s["need"])
    return {"refcounts": refcounts, "pages": pages}


_OWN = {"attend": _own_attend, "beam": _own_beam, "copy": _own_copy, "fork": _own_fork,
        "compact": _own_compact, "turnover": _own_turnover}


def run(state):
    return (_OWN if own else _PLAIN)[state["case"]["op"]](state)


# --------------------------------------------------------------------------- work, 64 bits


def work(case):
    op = case["op"]
    if op == "attend":
        lens = _lengths(case)
        seen = sum(_visible(case, n) for n in lens)
        B, HQ, HKV, D = (case[k] for k in ("batch", "heads", "kv_heads", "dim"))
        pages = sum(-(-_visible(case, n) // case["page"]) for n in lens)
        # the visible cache rows, the new rows in and out, q, output, lse, tables and lengths
        return {"bytes": 4 * seen * HKV * D + 8 * B * HKV * D + 4 * B * HQ * D + 4 * B * HQ
                + 4 * pages + 4 * B, "flops": 4 * seen * HQ * D}
    if op == "beam":
        rows = case["batch"] * case["beams"]
        # a finished beam's logits need not be read
        read = rows * (1.0 - case["finished"]) if not case["first"] else case["batch"]
        size = 4 if case["dtype"] == "fp32" else 2
        return {"bytes": read * case["vocab"] * size + 5 * rows
                + 12 * case["batch"] * case["selected"], "flops": 4 * read * case["vocab"]}
    if op == "copy":
        n, size = case["pairs"], 4 if case["dtype"] == "fp32" else 2
        each = case["elems"] * size * case["pools"]
        sources = n * (1.0 - (1.0 - 1.0 / n) ** n)       # distinct sources, each read once
        moved = n - 1.0                                  # one of n is its own source on average
        return {"bytes": (min(sources, moved) + moved) * each + 8 * n if n > 1 else 8 * n,
                "flops": 0}
    if op == "fork":
        B, K, ps = case["batch"], case["beams"], case["page"]
        lens = _lengths(case)
        each = 2 * 2 * ps * case["kv_heads"] * case["dim"]
        entries = K * sum(-(-n // ps) for n in lens)
        parents = K * (1.0 - (1.0 - 1.0 / K) ** K)       # distinct parents of K children
        part = sum(1 for n in lens if n % ps)
        width = max(1, -(-case["longest"] // ps))
        more = K - parents                               # children after the first: copies
        return {"bytes": part * more * 2 * each + 4 * entries + 4 * B * K * width
                + 8 * (sum(n // ps for n in lens) + K * part) + 16 * B * K, "flops": 0}
    if op == "compact":
        P, live = case["pages"], max(1, int(case["pages"] * case["live"]))
        each = 2 * 2 * case["page"] * case["kv_heads"] * case["dim"]
        moved = live * (1.0 - live / P)                  # live pages behind the first `live`
        return {"bytes": 2 * moved * each + 12 * P + 8 * live, "flops": 0}
    # the reference counts are read and the changed ones written, once
    return {"bytes": 4 * case["pages"] + 8 * case["leaving"] + 9 * case["coming"], "flops": 0}


def _exact_attend(case, s):
    q, lens = s["q"][:, 0].double(), s["lens"].tolist()
    B, HQ, HKV, D, ps = q.shape[0], case["heads"], case["kv_heads"], case["dim"], case["page"]
    out = torch.zeros((B, 1, HQ, D), dtype=torch.float64, device=q.device)
    lse = torch.full((B, HQ), -math.inf, dtype=torch.float64, device=q.device)
    for b, n in enumerate(lens):
        if n == 0:
            continue
        pages = s["tables"][b, :-(-n // ps)].long()
        where = torch.ones(n, dtype=torch.bool, device=q.device)
        if case["window"]:
            where[case["sinks"]:max(case["sinks"], n - case["window"])] = False
        for h in range(HKV):
            keys, values = ((c[pages, :, h].reshape(-1, D)[:n]).double()
                            for c in (s["k_cache"], s["v_cache"]))
            keys[n - 1], values[n - 1] = s["k"][b, 0, h].double(), s["v"][b, 0, h].double()
            keys, values = keys[where], values[where]
            heads = slice(h * HQ // HKV, (h + 1) * HQ // HKV)
            x = (keys @ q[b, heads].T) / math.sqrt(D)    # [tokens, heads of the group]
            lse[b, heads] = torch.logsumexp(x, 0)
            out[b, 0, heads] = torch.softmax(x, 0).T @ values
    return {"output": out, "lse": lse, "k_cache": None, "v_cache": None}


def _exact_beam(case, s):
    n, eos = case["selected"], s["eos"]
    rows = []
    for b in range(case["batch"]):
        logp = torch.log_softmax(s["logits"][b].double(), -1) + s["scores"][b].double()[:, None]
        if s["finished"] is not None:
            done = s["finished"][b]
            logp[done] = -math.inf
            logp[done, eos] = s["scores"][b].double()[done]
        flat = logp.flatten()
        best = flat.topk(min(n, flat.numel())).values
        best = torch.cat([best, best.new_full((n - best.numel(),), -math.inf)])
        rows.append(torch.where(torch.isfinite(best), best, -math.inf))
    return {"tokens": None, "parents": None, "scores": torch.stack(rows)}


def exact(case, seed):
    if case["op"] not in ("attend", "beam"):
        return None                                      # bytes and whole numbers only
    s = prepare(case, seed)
    return _exact_attend(case, s) if case["op"] == "attend" else _exact_beam(case, s)
