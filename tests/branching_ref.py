"""Plain forms of the operators of decoding that branches (trees of drafted tokens, beams), on the
CPU: 64 bits, or Python integers."""
from __future__ import annotations

import math
import random

import torch


def word(v: int) -> int:
    """A pattern of 64 bits as a signed integer."""
    return v - (1 << 64) if v >> 63 & 1 else v


def words(values, dev="cpu") -> torch.Tensor:
    return torch.tensor([word(v) for v in values], dtype=torch.int64, device=dev)


def tree(rng: random.Random, n: int, reach: int = 8):
    """Masks of a random tree of n nodes."""
    mask = [1]
    for i in range(1, n):
        mask.append(mask[rng.randrange(max(0, i - reach), i)] | 1 << i)
    return mask[:n]


def chain(n: int):
    return [(2 << i) - 1 for i in range(n)]


def seen(masks, keys: int) -> torch.Tensor:
    """[nodes, keys + nodes]: what each node sees of the keys before the tree and of the tree."""
    n = len(masks)
    s = torch.ones((n, keys + n), dtype=torch.bool)
    for i, m in enumerate(masks):
        for j in range(n):
            s[i, keys + j] = bool(m >> j & 1)
    return s


def accept(targets, drafts, masks):
    """(path, count, token) of one tree."""
    paths = {}
    for i in range(min(len(targets), 64)):
        above = [j for j in range(i) if masks[i] >> j & 1]
        if i == 0:
            paths[0] = [0]
        elif above and above[-1] in paths and targets[above[-1]] == drafts[i]:
            paths[i] = paths[above[-1]] + [i]
    best = max(paths.values(), key=len, default=[])
    return sum(1 << i for i in best), len(best), targets[best[-1]] if best else -1


def compact(cache: torch.Tensor, table: torch.Tensor, lens, paths, page: int) -> torch.Tensor:
    """cache [layers, pages, heads, page, dim] (CPU) after the paths' tokens have moved."""
    out, pages = cache.clone(), cache.shape[1]

    def place(b, at):
        if at < 0 or at // page >= table.shape[1]:
            return None
        p = int(table[b, at // page])
        return (p, at % page) if 0 <= p < pages else None

    for b, (n, path) in enumerate(zip(lens, paths)):
        if n < 0:
            continue
        for j, s in enumerate([i for i in range(64) if path >> i & 1]):
            src, dst = place(b, n + s), place(b, n + j)
            if src and dst:
                out[:, dst[0], :, dst[1]] = cache[:, src[0], :, src[1]]
    return out


def beams(logits: torch.Tensor, scores: torch.Tensor, k: int):
    """(totals in 64 bits, rows, tokens) of logits [S * W, V], scores [S, W]."""
    S, W = scores.shape
    V = logits.shape[1]
    x = logits.double()
    x = torch.where(x.isnan(), -math.inf, x).view(S, W, V)
    m = x.amax(dim=2, keepdim=True)
    good = torch.isfinite(m) & torch.isfinite(scores.double())[:, :, None]
    d = torch.where(good, x - torch.where(good, m, 0.0), -math.inf)
    lse = torch.log(torch.where(good, torch.exp(d), 1.0).sum(dim=2, keepdim=True))
    total = torch.where(good & (d > -math.inf), scores.double()[:, :, None] + (d - lse), -math.inf)
    best, at = torch.sort(total.view(S, -1), dim=1, descending=True, stable=True)
    pad = max(0, k - W * V)
    best = torch.cat((best[:, :k], torch.full((S, pad), -math.inf, dtype=torch.double)), dim=1)
    at = torch.cat((at[:, :k], torch.zeros((S, pad), dtype=at.dtype)), dim=1)
    none = best == -math.inf
    rows = torch.where(none, -1, at // V + torch.arange(S)[:, None] * W)
    return best, rows.to(torch.int32), torch.where(none, -1, at % V)


def fork(table, lens, parents, refs, page: int, ahead: int = 1):
    """(table, lens, copies, missing) of lists; refs is changed in place."""
    width, pages = len(table[0]) if table else 0, len(refs)
    good = lambda p: 0 <= p < pages
    kept = lambda n: min(width, (n + ahead + page - 1) // page)
    new, new_lens = [], []
    for p in parents:
        real = 0 <= p < len(table)
        n = max(lens[p], 0) if real else 0
        row = list(table[p][:kept(n)]) if real else []
        new.append(row + [-1] * (width - len(row)))
        new_lens.append(n)
    for rows, by in ((new, 1), (table, -1)):
        for row in rows:
            for p in row:
                if good(p):
                    refs[p] += by
    places = [(i, e) for i, n in enumerate(new_lens) if 0 <= parents[i] < len(table)
              for e in range(n // page, kept(n))]
    writers = {}
    for i, e in places:
        writers.setdefault(new[i][e], []).append((i, e))
    stays = {at for p, w in writers.items() if good(p) and refs[p] == len(w) for at in w[:1]}
    free = [p for p in range(pages) if refs[p] <= 0]
    copies, missing, given = [[-1, -1, 0] for _ in parents], 0, []
    for i, e in places:
        if (i, e) in stays:
            continue
        old, fresh = new[i][e], free.pop(0) if free else -1
        if good(old):
            refs[old] -= 1
        new[i][e] = fresh
        if fresh < 0:
            missing += 1
            continue
        given.append(fresh)
        if good(old) and e == new_lens[i] // page and new_lens[i] % page:
            copies[i] = [old, fresh, new_lens[i] % page]
    for p in given:
        refs[p] = 1
    return new, new_lens, copies, missing
