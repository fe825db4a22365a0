"""Performance cases of decoding that branches over a paged cache: trees of drafted tokens that one
pass checks, and beams.  Each operator in its plain form (elementary torch operations) and through the
framework's own entry points.

Kinds of case:
  tree     paged_tree_attention: the drafted tokens of each sequence against its paged keys and against
           those of its own drafted tokens that it descends from.
  accept   accept_drafts: the longest path of each tree that the model's own choices confirm.
  compact  compact_paged_kv: keys and values of the confirmed tokens moved to where they belong, in all
           layers.
  beam     beam_select: the best continuations of each search, over its beams and the vocabulary.
  fork     fork_pages, copy_pages: page table rows reordered by the beams that continue, pages shared,
           freed, handed out, and copied where rows part.
"""
from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

DEV = "cuda:0"
NODES = 64  # of a tree at most


# ------------------------------------------------------------------ cases
def listed():
    mix = {"q_heads": 32, "kv_heads": 8, "head_dim": 128}   # the benchmark model's attention
    return [
        # One conversation, a chain of four drafted tokens behind the last one: latency.
        {"name": "tree_1x900_chain", "kind": "tree", "seqs": 1, "longest": 900, "nodes": 5, "ragged": 0, "pad": 0,
         "chain": True, "page": 16, **mix},
        # A batch of very different lengths and trees, rows of padding among them.
        {"name": "tree_24_ragged", "kind": "tree", "seqs": 24, "longest": 9001, "nodes": 40, "ragged": 5, "pad": 3,
         "chain": False, "page": 16, **mix},
        # Long contexts, small trees: the bandwidth of the device.
        {"name": "tree_16x32768", "kind": "tree", "seqs": 16, "longest": 32768, "nodes": 16, "ragged": 0, "pad": 0,
         "chain": False, "page": 64, **mix},
        # The largest trees: as much arithmetic as memory.
        {"name": "tree_8x16384_wide", "kind": "tree", "seqs": 8, "longest": 16384, "nodes": 64, "ragged": 0, "pad": 0,
         "chain": False, "page": 64, **mix},
        # A few conversations, and a full server.
        {"name": "accept_4", "kind": "accept", "seqs": 4, "nodes": 12, "ragged": 1, "chain": False},
        {"name": "accept_256", "kind": "accept", "seqs": 256, "nodes": 64, "ragged": 2, "chain": False},
        # One conversation's confirmed tokens in a few layers.
        {"name": "compact_1", "kind": "compact", "seqs": 1, "longest": 900, "nodes": 8, "deepest": 4, "layers": 4,
         "page": 16, "ragged": 1, **mix},
        # A full server's, in all layers of the benchmark model.
        {"name": "compact_64", "kind": "compact", "seqs": 64, "longest": 9001, "nodes": 64, "deepest": 9, "layers": 32,
         "page": 16, "ragged": 2, **mix},
        # One search: latency.
        {"name": "beam_1x4", "kind": "beam", "searches": 1, "beams": 4, "k": 8, "vocab": 32000, "dtype": "bf16"},
        # Many of them, a large vocabulary.
        {"name": "beam_64x4", "kind": "beam", "searches": 64, "beams": 4, "k": 8, "vocab": 131072, "dtype": "bf16"},
        # Two searches of a few hundred tokens, small caches.
        {"name": "fork_2x4", "kind": "fork", "searches": 2, "beams": 4, "longest": 333, "layers": 2, "page": 16,
         "ragged": 3, **mix},
        # Many of them.
        {"name": "fork_64x4", "kind": "fork", "searches": 64, "beams": 4, "longest": 1500, "layers": 4, "page": 64,
         "ragged": 4, **mix},
    ]


HEADS = ((32, 8, 128), (32, 8, 128), (8, 2, 64), (16, 16, 64), (32, 4, 128), (24, 8, 128), (16, 1, 128), (8, 4, 256),
         (40, 2, 128), (12, 4, 64))
PAGES = (8, 16, 16, 32, 64, 128)


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("tree", "tree", "accept", "compact", "beam", "beam", "fork"))
    nq, nkv, hd = rng.choice(HEADS)
    heads = {"q_heads": nq, "kv_heads": nkv, "head_dim": hd}
    page, ragged = rng.choice(PAGES), rng.randint(1, 999)
    if kind == "tree":
        seqs, nodes = _log(rng, 1, 64), _log(rng, 1, NODES)
        # No more memory and arithmetic than the largest listed cases have.
        most = min((1 << 31) // (seqs * nkv * hd * 4), int(1.3e11) // (4 * nq * hd * seqs * nodes))
        longest = _log(rng, 1, max(2, min(32768, most) - nodes))
        return {"kind": kind, "seqs": seqs, "longest": longest, "nodes": nodes, "ragged": rng.choice((0, ragged)),
                "pad": rng.randint(0, seqs // 4), "chain": rng.random() < 0.3, "page": page, **heads}
    if kind == "accept":
        return {"kind": kind, "seqs": _log(rng, 1, 256), "nodes": _log(rng, 1, NODES), "ragged": ragged,
                "chain": rng.random() < 0.3}
    if kind == "compact":
        seqs, nodes = _log(rng, 1, 64), _log(rng, 2, NODES)
        layers = max(1, min(_log(rng, 1, 32), (1 << 29) // (seqs * nkv * hd * (nodes + 2 * page))))
        return {"kind": kind, "seqs": seqs, "longest": _log(rng, 1, 9001), "nodes": nodes,
                "deepest": rng.randint(2, max(2, min(nodes, 9))), "layers": layers, "page": page, "ragged": ragged,
                **heads}
    beams = _log(rng, 1, 16)
    if kind == "beam":
        vocab = _log(rng, 300, 131072)
        return {"kind": kind, "searches": _log(rng, 1, 256 // beams), "beams": beams,
                "k": rng.choice((beams, 2 * beams)), "vocab": vocab,
                "dtype": rng.choice(("bf16", "fp32")) if vocab <= 65536 else "bf16"}
    beams = max(2, beams)
    searches = _log(rng, 1, 256 // beams)
    longest = _log(rng, 1, 1500)
    held = searches * (beams + 1) * (longest // 2 + page) * nkv * hd
    return {"kind": kind, "searches": searches, "beams": beams, "longest": longest,
            "layers": max(1, min(rng.randint(1, 4), (1 << 28) // held)), "page": page, "ragged": ragged, **heads}


def _lens(n, longest, ragged):
    """Keys of each sequence: all the longest, or spread below it."""
    if not ragged:
        return [longest] * n
    r = random.Random(ragged)
    lens = [1 + int((longest - 1) * r.random() ** 2) for _ in range(n)]
    lens[r.randrange(n)] = longest
    return lens


def _counts(n, nodes, ragged, pad=0):
    """Tokens of each tree: all the most, or spread below it; rows of padding have none."""
    r = random.Random(ragged + 17)
    counts = [r.randint(1, nodes) if ragged else nodes for _ in range(n)]
    counts[r.randrange(n)] = nodes
    return [0 if i >= n - pad else c for i, c in enumerate(counts)]


def _kept(case):
    """How many drafted tokens of each sequence are confirmed (the first always is)."""
    r = random.Random(case["ragged"] + 29)
    return [min(c, r.randint(1, case["deepest"])) for c in _counts(case["seqs"], case["nodes"], case["ragged"])]


def _fork_plan(case):
    """(keys of each beam, full pages that the beams of a search share, rows that continue)."""
    r = random.Random(case["ragged"])
    lens, shared, parents = [], [], []
    for s in range(case["searches"]):
        n = 1 + int((case["longest"] - 1) * r.random()) if s else case["longest"]
        lens.append(n)
        shared.append(r.randint(0, n // case["page"]))
        parents += [s * case["beams"] + min(r.randrange(case["beams"]), r.randrange(case["beams"]))
                    for _ in range(case["beams"])]
    return lens, shared, parents


# ------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(shape, g, std=1.0):
    return (torch.randn(shape, generator=g, device=DEV) * std).to(torch.bfloat16)


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _i64(values):
    """Bit patterns of 64 bits as int64."""
    return torch.tensor([v - (1 << 64) if v >> 63 else v for v in values], dtype=torch.int64, device=DEV)


def _tree(rng, n):
    """(parent, mask of the node and its ancestors) of each node; the first is the root."""
    parent, mask = [-1], [1]
    for i in range(1, n):
        p = rng.randrange(max(0, i - 8), i)  # a few branches at a time
        parent.append(p)
        mask.append(mask[p] | 1 << i)
    return parent, mask


def _pages_for(lens, page, first=None):
    """A shuffled pool's table for sequences of `lens` keys (entries below `first` are not there)."""
    return [(i, p) for i, n in enumerate(lens) for p in range(first[i] if first else 0, (n + page - 1) // page)]


def _table(need, rows, width, rng, spare):
    ids = list(range(len(need) + spare))
    rng.shuffle(ids)
    table = torch.full((rows, max(1, width)), -1, dtype=torch.int32)
    for (i, p), page in zip(need, ids):
        table[i, p] = page
    return table.to(DEV), max(1, len(ids))


def prepare(case, seed):
    g = _gen(seed)
    rng = random.Random(seed)
    kind = case["kind"]
    if kind == "beam":
        return _prepare_beam(case, g, rng)
    if kind == "accept":
        return _prepare_accept(case, rng)
    nq, nkv, hd, P = case["q_heads"], case["kv_heads"], case["head_dim"], case["page"]
    st = {"kind": kind, "nq": nq, "nkv": nkv, "hd": hd, "scaling": float(hd ** -0.5), "page": P}
    if kind == "fork":
        return _prepare_fork(case, g, rng, st)
    n = case["seqs"]
    lens = _lens(n, case["longest"], case["ragged"])
    if kind == "compact":
        # The pool holds the pages that the drafted tokens lie in; earlier ones are not read here.
        counts, kept = _counts(n, case["nodes"], case["ragged"]), _kept(case)
        ends = [a + b for a, b in zip(lens, counts)]
        need = _pages_for(ends, P, [v // P for v in lens])
        table, pages = _table(need, n, (max(ends) + P - 1) // P, rng, 3)
        paths = [sum(1 << i for i in [0] + rng.sample(range(1, c), m - 1)) for c, m in zip(counts, kept)]
        shape = (case["layers"], pages, nkv, P, hd)
        st.update(table=table, lens=_i32(lens), paths=_i64(paths), k_cache=_randn(shape, g), v_cache=_randn(shape, g))
        return st
    counts = _counts(n, case["nodes"], case["ragged"], case["pad"])
    lens = [0 if c == 0 else v for v, c in zip(lens, counts)]
    ends = [a + b for a, b in zip(lens, counts)]
    table, pages = _table(_pages_for(ends, P), n, (max(ends) + P - 1) // P, rng, 3)
    cuts = [0]
    for c in counts:
        cuts.append(cuts[-1] + c)
    trees = [[(2 << i) - 1 for i in range(c)] if case["chain"] else _tree(rng, c)[1][:c] for c in counts]
    # Keys that some queries like better than others: scores with a spread of a few units.
    st.update(q=_randn((cuts[-1], nq, hd), g, 1.5), k_cache=_randn((pages, nkv, P, hd), g),
              v_cache=_randn((pages, nkv, P, hd), g), table=table, lens=_i32(lens), cu=_i32(cuts),
              masks=None if case["chain"] else _i64([m for t in trees for m in t]),
              host_lens=lens, host_cuts=cuts, workspace=None)
    if own:
        from moeinfra_amd import ops

        st["workspace"] = ops.paged_tree_attention_workspace(n, nq, nkv, hd, DEV)
    return st


def _prepare_accept(case, rng):
    counts = _counts(case["seqs"], case["nodes"], case["ragged"])
    cuts, masks, drafts, targets = [0], [], [], []
    for c in counts:
        parent, mask = ([i - 1 for i in range(c)], [(2 << i) - 1 for i in range(c)]) if case["chain"] else _tree(rng, c)
        draft = [rng.randrange(32000) for _ in range(c)]
        # What the model chooses after each node: one of its drafted children three times of four.
        target = [rng.randrange(32000) for _ in range(c)]
        for i in range(c - 1, 0, -1):
            if rng.random() < 0.75:
                target[parent[i]] = draft[i]
        cuts.append(cuts[-1] + c)
        masks += mask
        drafts += draft
        targets += target
    token = lambda v: torch.tensor(v, dtype=torch.int64, device=DEV)
    return {"kind": "accept", "drafts": token(drafts), "targets": token(targets), "cu": _i32(cuts),
            "masks": None if case["chain"] else _i64(masks)}


def _prepare_beam(case, g, rng):
    S, W, V = case["searches"], case["beams"], case["vocab"]
    # A model's logits: a broad bulk and a few tokens far above it.
    x = torch.randn((S * W, V), generator=g, device=DEV) * 2.0
    peaks = torch.randn((S * W, V), generator=g, device=DEV) > 3.2
    x += torch.where(peaks, torch.rand((S * W, V), generator=g, device=DEV) * 9.0, 0.0)
    # Some searches may say only part of the vocabulary (a grammar's mask).
    masked = (torch.rand((S, 1, 1), generator=g, device=DEV) < 0.25).expand(S, W, 1).reshape(S * W, 1)
    gone = torch.rand((S * W, V), generator=g, device=DEV) < 0.9
    x = torch.where(masked & gone, -math.inf, x)
    scores = -20.0 * torch.rand((S, W), generator=g, device=DEV)
    # Every third search is at its first step: one beam only.
    first = torch.tensor([rng.random() < 0.33 for _ in range(S)], device=DEV)
    scores[:, 1:] = torch.where(first[:, None], -math.inf, scores[:, 1:])
    st = {"kind": "beam", "logits": x.to(torch.bfloat16 if case["dtype"] == "bf16" else torch.float32),
          "scores": scores, "k": case["k"], "workspace": None}
    if own:
        from moeinfra_amd import ops

        st["workspace"] = ops.beam_select_workspace(S, W, case["k"], DEV)
    return st


def _prepare_fork(case, g, rng, st):
    P, W = case["page"], case["beams"]
    lens, shared, parents = _fork_plan(case)
    rows = len(parents)
    width = case["longest"] // P + 2
    need = sum(s + W * ((n + P - 1) // P - s) for n, s in zip(lens, shared))
    ids = list(range(need + 2 * rows + 3))
    pages = len(ids)
    rng.shuffle(ids)
    table = np.full((rows, width), -1, dtype=np.int32)
    refs = np.zeros(pages, dtype=np.int32)
    at = 0
    for s, (n, both) in enumerate(zip(lens, shared)):
        held = (n + P - 1) // P
        table[s * W:(s + 1) * W, :both] = ids[at:at + both]
        at += both
        for b in range(s * W, (s + 1) * W):
            table[b, both:held] = ids[at:at + held - both]
            at += held - both
    np.add.at(refs, table[table >= 0], 1)
    shape = (case["layers"], pages, st["nkv"], P, st["hd"])
    st.update(table=torch.from_numpy(table).to(DEV), refs=torch.from_numpy(refs).to(DEV),
              lens=_i32([n for n in lens for _ in range(W)]), parents=_i32(parents), workspace=None,
              k_cache=_randn(shape, g), v_cache=_randn(shape, g))
    if own:
        from moeinfra_amd import ops

        st["workspace"] = ops.fork_pages_workspace(pages, DEV)
    return st


# ------------------------------------------------------------------ one pass
def run(st):
    kind = st["kind"]
    if not own:
        return {"tree": _plain_tree, "accept": _plain_accept, "compact": _plain_compact, "beam": _plain_beam,
                "fork": _plain_fork}[kind](st)
    from moeinfra_amd import ops

    if kind == "tree":
        return ops.paged_tree_attention(st["q"], st["k_cache"], st["v_cache"], st["table"], st["lens"], st["cu"],
                                        masks=st["masks"], scaling=st["scaling"], workspace=st["workspace"])
    if kind == "accept":
        paths, counts, tokens = ops.accept_drafts(st["targets"], st["drafts"], st["cu"], masks=st["masks"])
        return {"paths": paths, "counts": counts, "tokens": tokens}
    if kind == "compact":
        ops.compact_paged_kv(st["k_cache"], st["v_cache"], st["table"], st["lens"], st["paths"])
        return {"k_cache": st["k_cache"], "v_cache": st["v_cache"]}
    if kind == "beam":
        scores, rows, tokens = ops.beam_select(st["logits"], st["scores"], k=st["k"], workspace=st["workspace"])
        return {"scores": scores, "rows": rows, "tokens": tokens}
    # The rows go on as the next step finds them.
    st["table"], st["lens"], copies, missing = ops.fork_pages(st["table"], st["lens"], st["parents"], st["refs"],
                                                              st["page"], workspace=st["workspace"])
    ops.copy_pages(st["k_cache"], st["v_cache"], copies)
    return _forked(st, copies, missing)


def _forked(st, copies, missing):
    return {"table": st["table"], "lens": st["lens"], "refs": st["refs"], "copies": copies, "missing": missing,
            "k_cache": st["k_cache"], "v_cache": st["v_cache"]}


def _bits(words):
    """[n, 64] truth values of [n] words."""
    return ((words[:, None] >> torch.arange(NODES, device=DEV)) & 1).bool()


def _plain_tree(st):
    nq, nkv, hd, P = st["nq"], st["nkv"], st["hd"], st["page"]
    out = torch.empty_like(st["q"])
    for i, (lo, hi) in enumerate(zip(st["host_cuts"], st["host_cuts"][1:])):
        if lo == hi:
            continue
        m, n = hi - lo, st["host_lens"][i]
        pages = st["table"][i, :(n + m + P - 1) // P].long()
        k = st["k_cache"][pages].transpose(0, 1).reshape(nkv, -1, hd)[:, :n + m].float()
        v = st["v_cache"][pages].transpose(0, 1).reshape(nkv, -1, hd)[:, :n + m].float()
        q = st["q"][lo:hi].float().view(m, nkv, nq // nkv, hd).permute(1, 2, 0, 3).reshape(nkv, -1, hd)
        s = torch.matmul(q, k.transpose(1, 2)).view(nkv, nq // nkv, m, n + m) * st["scaling"]
        if st["masks"] is None:
            seen = torch.arange(m, device=DEV)[None, :] <= torch.arange(m, device=DEV)[:, None]
        else:
            seen = _bits(st["masks"][lo:hi])[:, :m]
        s[..., n:] = torch.where(seen, s[..., n:], -math.inf)
        e = torch.exp(s - s.amax(dim=-1, keepdim=True))
        o = torch.matmul(e.view(nkv, -1, n + m), v).view(nkv, nq // nkv, m, hd) / e.sum(dim=-1, keepdim=True)
        out[lo:hi] = o.permute(2, 0, 1, 3).reshape(m, nq, hd).to(torch.bfloat16)
    return out


def _plain_accept(st):
    cu = st["cu"].long()
    B, T = cu.numel() - 1, st["drafts"].numel()
    node = torch.arange(NODES, device=DEV)
    n = (cu[1:] - cu[:-1])[:, None]
    there = node[None, :] < n
    row = torch.where(there, cu[:-1, None] + node, 0).clamp(max=T - 1)
    if st["masks"] is None:
        parent = (node - 1).expand(B, NODES)
    else:
        up = _bits(st["masks"][row.reshape(-1)]).view(B, NODES, NODES) & (node[None, :] < node[:, None])
        parent = torch.where(up, node, -1).amax(dim=2)
    parent = torch.where(there, parent, -1)
    match = st["drafts"][row] == st["targets"][row].gather(1, parent.clamp(min=0))
    good = there & (node == 0)
    depth = torch.zeros((B, NODES), dtype=torch.int64, device=DEV) + good
    path = torch.where(good, torch.ones_like(depth) << node, 0)
    for i in range(1, NODES):  # (parents come before their children)
        p = parent[:, i:i + 1].clamp(min=0)
        good[:, i] = there[:, i] & (parent[:, i] >= 0) & match[:, i] & good.gather(1, p)[:, 0]
        depth[:, i] = torch.where(good[:, i], depth.gather(1, p)[:, 0] + 1, 0)
        path[:, i] = torch.where(good[:, i], path.gather(1, p)[:, 0] | torch.ones_like(n[:, 0]) << i, 0)
    best = torch.where(depth == depth.amax(dim=1, keepdim=True), node, NODES).amin(dim=1, keepdim=True)
    some = n[:, 0] > 0
    return {"paths": path.gather(1, best)[:, 0], "counts": depth.gather(1, best)[:, 0].to(torch.int32),
            "tokens": torch.where(some, st["targets"][row].gather(1, best)[:, 0], -1)}


def _plain_compact(st):
    P, table, lens = st["page"], st["table"], st["lens"].long()
    on = _bits(st["paths"])
    seq, bit = torch.nonzero(on, as_tuple=True)
    rank = torch.cumsum(on, dim=1)[seq, bit] - 1
    src, dst = lens[seq] + bit, lens[seq] + rank
    ps, pd = table[seq, src // P].long(), table[seq, dst // P].long()
    for cache in (st["k_cache"], st["v_cache"]):
        cache[:, pd, :, dst % P] = cache[:, ps, :, src % P]
    return {"k_cache": st["k_cache"], "v_cache": st["v_cache"]}


def _plain_beam(st):
    S, W = st["scores"].shape
    # In 64 bits: what is chosen hangs on the differences of sums over the vocabulary.
    x = st["logits"].double()
    x = torch.where(x.isnan(), -math.inf, x)
    m = x.amax(dim=1, keepdim=True)
    d = x - torch.where(m == -math.inf, 0.0, m)
    lse = torch.log(torch.exp(d).sum(dim=1, keepdim=True))
    total = (st["scores"].double().view(S * W, 1) + (d - torch.where(m == -math.inf, 0.0, lse))).view(S, -1)
    total = torch.where(total.isnan(), -math.inf, total)
    best, at = torch.sort(total, dim=1, descending=True, stable=True)       # ties: lowest index first
    best, at = best[:, :st["k"]], at[:, :st["k"]]
    V = st["logits"].shape[1]
    row = at // V + torch.arange(S, device=DEV)[:, None] * W
    none = best == -math.inf
    return {"scores": best.float(), "rows": torch.where(none, -1, row).to(torch.int32),
            "tokens": torch.where(none, -1, at % V)}


def _plain_fork(st):
    table, lens, refs, P = st["table"].long(), st["lens"].long(), st["refs"], st["page"]
    n, width = table.shape
    parents = st["parents"].long()
    real = (parents >= 0) & (parents < n)
    parents = parents.clamp(0, n - 1)
    new_lens = torch.where(real, lens[parents], 0)
    entry = torch.arange(width, device=DEV)[None, :]
    keep_to = (new_lens[:, None] + 1 + P - 1) // P                          # entries of a row from now on
    new = torch.where(real[:, None] & (entry < keep_to), table[parents], -1)
    pages = refs.numel()
    count = lambda t: torch.bincount(t[t >= 0].reshape(-1), minlength=pages)
    held = refs + count(new) - count(table)
    # Places that the next token is written to, row by row.
    first = (new_lens // P)[:, None]
    writes = real[:, None] & (entry >= first) & (entry < keep_to)
    rows, cols = torch.nonzero(writes, as_tuple=True)
    page = new[rows, cols]
    order = torch.arange(rows.numel(), device=DEV)
    writers = count(page)
    lowest = torch.full((pages,), rows.numel(), device=DEV).scatter_reduce_(0, page[page >= 0], order[page >= 0], "amin")
    safe = page.clamp(min=0)
    stays = (page >= 0) & (held[safe] == writers[safe]) & (lowest[safe] == order)
    wants = ~stays
    rank = torch.cumsum(wants, dim=0) - 1
    free = torch.nonzero(held <= 0)[:, 0]
    given = torch.full_like(page, -1)
    has = wants & (rank < free.numel())
    given[has] = free[rank[has]]
    held -= count(torch.where(wants, page, -1))
    held[given[has]] = 1
    new[rows, cols] = torch.where(wants, given, page)
    copies = torch.tensor([-1, -1, 0], device=DEV).repeat(parents.numel(), 1)
    part = has & (page >= 0) & (cols == new_lens[rows] // P) & (new_lens[rows] % P > 0)
    copies[rows[part]] = torch.stack((page, given, new_lens[rows] % P), dim=1)[part]
    missing = (wants & ~has).sum().reshape(1)
    refs.copy_(held)
    row = torch.arange(P, device=DEV)
    for src, dst, used in copies[copies[:, 1] >= 0].tolist():
        for cache in (st["k_cache"], st["v_cache"]):
            cache[:, dst, :, :used] = cache[:, src, :, :used]
    st["table"], st["lens"] = new.to(torch.int32), new_lens.to(torch.int32)
    return _forked(st, copies.to(torch.int32), missing.to(torch.int32))


# ------------------------------------------------------------------ work
def work(case):
    kind = case["kind"]
    if kind == "beam":
        rows, size = case["searches"] * case["beams"], 2 if case["dtype"] == "bf16" else 4
        # One difference, one scale, one exponential, one sum and one comparison per value.
        return {"bytes": rows * (case["vocab"] * size + 4) + case["searches"] * case["k"] * 16,
                "flops": 5 * rows * case["vocab"]}
    if kind == "accept":
        T = sum(_counts(case["seqs"], case["nodes"], case["ragged"]))
        return {"bytes": T * (16 if case["chain"] else 24) + 24 * case["seqs"], "flops": T}
    nq, nkv, hd, P = case["q_heads"], case["kv_heads"], case["head_dim"], case["page"]
    if kind == "compact":
        # The first confirmed token is in its place already; keys and values, read and written.
        moved = sum(m - 1 for m in _kept(case))
        return {"bytes": moved * case["layers"] * nkv * hd * 8 + 12 * case["seqs"], "flops": 0}
    if kind == "fork":
        lens, shared, parents = _fork_plan(case)
        W = case["beams"]
        parts = sum(max(0, parents.count(r) - 1) * (lens[r // W] % P) for r in range(len(parents)))
        entries = sum((lens[r // W] + P) // P for r in range(len(parents)))
        return {"bytes": parts * case["layers"] * nkv * hd * 8 + 12 * entries + 24 * len(parents), "flops": 0}
    counts = _counts(case["seqs"], case["nodes"], case["ragged"], case["pad"])
    lens = [0 if c == 0 else v for v, c in zip(_lens(case["seqs"], case["longest"], case["ragged"]), counts)]
    return {"bytes": sum(a + b for a, b in zip(lens, counts)) * nkv * hd * 4 + sum(counts) * nq * hd * 4,
            "flops": 4 * nq * hd * sum(c * (n + 1) for n, c in zip(lens, counts))}


# ------------------------------------------------------------------ the definition in 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    return {"tree": _exact_tree, "accept": _exact_accept, "compact": _exact_compact, "beam": _exact_beam,
            "fork": _exact_fork}[case["kind"]](st)


def _words(t):
    return [v & ((1 << 64) - 1) for v in t.cpu().tolist()]


def _exact_tree(st):
    nq, nkv, hd, P = st["nq"], st["nkv"], st["hd"], st["page"]
    out = torch.zeros(st["q"].shape, dtype=torch.double, device=DEV)
    words = None if st["masks"] is None else _words(st["masks"])
    for i, (lo, hi) in enumerate(zip(st["host_cuts"], st["host_cuts"][1:])):
        n, m = st["host_lens"][i], hi - lo
        if m == 0:
            continue
        j = torch.arange(n + m, device=DEV)
        page = st["table"][i].long()[j // P]
        hidden = torch.zeros((m, n + m), dtype=torch.bool)
        for a in range(m):
            word = (2 << a) - 1 if words is None else words[lo + a]
            for b in range(m):
                hidden[a, n + b] = not word >> b & 1
        hidden = hidden.to(DEV)
        for h in range(nkv):
            k, v = st["k_cache"][page, h, j % P].double(), st["v_cache"][page, h, j % P].double()
            for head in range(h * (nq // nkv), (h + 1) * (nq // nkv)):
                s = (st["q"][lo:hi, head].double() @ k.t() * st["scaling"]).masked_fill(hidden, -math.inf)
                out[lo:hi, head] = torch.softmax(s, dim=-1) @ v
    return out


def _exact_accept(st):
    cuts, drafts, targets = (st[n].cpu().tolist() for n in ("cu", "drafts", "targets"))
    words = None if st["masks"] is None else _words(st["masks"])
    paths, counts, tokens = [], [], []
    for lo, hi in zip(cuts, cuts[1:]):
        chains = {}
        for i in range(hi - lo):
            if i == 0:
                chains[0] = [0]
                continue
            above = [j for j in range(i) if ((2 << i) - 1 if words is None else words[lo + i]) >> j & 1]
            if above and above[-1] in chains and targets[lo + above[-1]] == drafts[lo + i]:
                chains[i] = chains[above[-1]] + [i]
        chain = max(chains.values(), key=len, default=[])  # (the first of the longest)
        paths.append(sum(1 << i for i in chain))
        counts.append(len(chain))
        tokens.append(targets[lo + chain[-1]] if chain else -1)
    return {"paths": _i64(paths), "counts": _i32(counts), "tokens": torch.tensor(tokens, device=DEV)}


def _exact_compact(st):
    P, table, lens = st["page"], st["table"].cpu(), st["lens"].cpu().tolist()
    out = {}
    for name in ("k_cache", "v_cache"):
        cache = st[name].double()
        for i, word in enumerate(_words(st["paths"])):
            bits = [b for b in range(NODES) if word >> b & 1]
            rows = [(int(table[i, (lens[i] + b) // P]), (lens[i] + b) % P) for b in bits]
            held = [cache[:, p, :, r].clone() for p, r in rows]
            for j, row in enumerate(held):
                cache[:, int(table[i, (lens[i] + j) // P]), :, (lens[i] + j) % P] = row
        out[name] = cache
    return out


def _exact_beam(st):
    S, W = st["scores"].shape
    k, V = st["k"], st["logits"].shape[1]
    scores, rows, tokens = [], [], []
    base = st["scores"].double().cpu().numpy()
    for s in range(S):
        x = st["logits"][s * W:(s + 1) * W].double().cpu().numpy()
        found = []
        for w in range(W):
            top = x[w].max()
            if top == -np.inf or base[s, w] == -np.inf:
                continue
            log_p = x[w] - top - np.log(np.exp(x[w] - top).sum())
            near = np.argpartition(-log_p, min(4 * k, V - 1))
            floor = log_p[near[min(4 * k, V - 1)]]  # (all that could be among the best, with their equals)
            found += [(-(base[s, w] + log_p[i]), w * V + int(i)) for i in np.nonzero(log_p >= floor)[0]
                      if log_p[i] > -np.inf]
        found = sorted(found)[:k]
        found += [(np.inf, None)] * (k - len(found))
        scores.append([-v for v, _ in found])
        rows.append([-1 if i is None else s * W + i // V for _, i in found])
        tokens.append([-1 if i is None else i % V for _, i in found])
    return {"scores": torch.tensor(scores, dtype=torch.double, device=DEV), "rows": _i32(rows),
            "tokens": torch.tensor(tokens, dtype=torch.int64, device=DEV)}


def _exact_fork(st):
    P, refs = st["page"], st["refs"].cpu().tolist()
    old, lens, parents = st["table"].cpu().tolist(), st["lens"].cpu().tolist(), st["parents"].cpu().tolist()
    width = len(old[0])
    new, new_lens = [], []
    for p in parents:
        n = lens[p] if 0 <= p < len(old) else 0
        row = old[p][:(n + P) // P] if 0 <= p < len(old) else []
        new.append(row + [-1] * (width - len(row)))
        new_lens.append(n)
    for rows, by in ((new, 1), (old, -1)):
        for row in rows:
            for p in row:
                if p >= 0:
                    refs[p] += by
    wants = [(i, n // P) for i, n in enumerate(new_lens) if 0 <= parents[i] < len(old) and n // P < width]
    by_page = {}
    for w in wants:
        by_page.setdefault(new[w[0]][w[1]], []).append(w)
    free = iter([p for p, r in enumerate(refs) if r <= 0])
    copies, missing, total = [[-1, -1, 0] for _ in parents], 0, dict(enumerate(refs))
    for i, e in wants:
        p = new[i][e]
        if p >= 0 and total[p] == len(by_page[p]) and by_page[p][0] == (i, e):
            continue
        fresh = next(free, -1)
        if p >= 0:
            refs[p] -= 1
        if fresh >= 0:
            refs[fresh] = 1
            if p >= 0 and new_lens[i] % P:
                copies[i] = [p, fresh, new_lens[i] % P]
        else:
            missing += 1
        new[i][e] = fresh
    out = {"table": _i32(new), "lens": _i32(new_lens), "refs": _i32(refs), "copies": _i32(copies),
           "missing": _i32([missing])}
    for name in ("k_cache", "v_cache"):
        cache = st[name].double()
        for src, dst, used in copies:
            if used:
                cache[:, dst, :, :used] = cache[:, src, :, :used]
        out[name] = cache
    return out
