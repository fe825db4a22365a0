"""Plain 64-bit forms of the batched serving operators, on the CPU, and the bounds of what the
kernels' roundings may add (bf16 rounds by at most 2^-8 of a value, fp32 by 2^-24)."""
from __future__ import annotations

import math

import torch


def rope(x: torch.Tensor, positions, inv_freq: torch.Tensor):
    """(rotated heads, bound) of x [T, heads, hd] at the positions [T]."""
    x = x.double()
    h = x.shape[-1] // 2
    ang = torch.as_tensor(positions).double()[:, None] * inv_freq.double()[None, :]
    c, s = torch.cos(ang)[:, None], torch.sin(ang)[:, None]
    a, b = x[..., :h], x[..., h:]
    y = torch.cat((a * c - b * s, b * c + a * s), dim=-1)
    # One rounding to bf16; cos and sin in fp32 from an angle of 2^-23 rad at worst, two products
    # and a sum: 2^-21 of the pair's magnitudes.
    pair = (a.abs() + b.abs()).repeat(1, 1, 2)
    return y, 2.0 ** -8 * y.abs() + 2.0 ** -21 * pair


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, scaling: float, seen=None):
    """(outputs, bound) of q [rows, hd] against k, v [keys, hd]; seen [rows, keys]: which keys a row
    sees (None: all).  A row that sees none is zeros."""
    q, k, v = q.double(), k.double(), v.double()
    n, hd = k.shape
    if n == 0:
        return torch.zeros((q.shape[0], v.shape[1]), dtype=torch.double), torch.zeros(q.shape[0], v.shape[1])
    s = q @ k.t() * scaling
    if seen is not None:
        s = torch.where(seen, s, -math.inf)
    m = s.amax(dim=1, keepdim=True)
    e = torch.exp(s - torch.where(m == -math.inf, 0.0, m))
    if seen is not None:
        e = torch.where(seen, e, 0.0)
    p = e / torch.where(e.sum(1, keepdim=True) == 0, 1.0, e.sum(1, keepdim=True))
    o = p @ v
    # Scores: hd products summed in fp32, the scaling, the difference to the maximum and the
    # exponential of up to 90 (2^-18 covers 2^-24 * 90 and the exponential's own step); weights to
    # bf16 against a sum that is not; n keys summed in fp32; the output to bf16.
    reach = ((q.abs() @ k.abs().t()).amax(dim=1, keepdim=True) * abs(scaling))
    ds = (hd + 4) * 2.0 ** -23 * reach + 2.0 ** -18
    return o, 2.0 ** -8 * o.abs() + (p @ v.abs()) * (2.0 ** -8 + 2 * ds + n * 2.0 ** -23) + 1e-30


def assert_within(got: torch.Tensor, want: torch.Tensor, bound: torch.Tensor, what: str = "") -> None:
    got = got.double().cpu()
    assert not torch.isnan(got).any(), f"{what}: NaN"
    over = (got - want).abs() - bound
    worst = int(over.argmax())
    assert over.max() <= 0, (f"{what}: off by {float((got - want).abs().flatten()[worst])} where "
                             f"{float(bound.expand_as(want).flatten()[worst])} is allowed")


def sample(x: torch.Tensor, u: float, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0) -> int:
    """The token of one row of logits (see sample_tokens), in 64 bits with a sort; the settings as
    the fp32 values that they are passed as."""
    f32 = lambda v: float(torch.tensor(v, dtype=torch.float32))
    x = torch.where(x.isnan(), -math.inf, x.double())
    top = float(x.max())
    if top == -math.inf:
        return -1
    order = torch.sort(x, descending=True, stable=True).indices
    if not f32(temperature) > 0:
        return int(order[0])
    if top == math.inf:
        w = (x == math.inf).double()
    else:
        w = torch.exp((x - top) / f32(temperature))
    n = int((x > -math.inf).sum())
    if top_k > 0:
        n = min(n, top_k)
    if f32(top_p) < 1:
        c = torch.cumsum(w[order[:n]], 0)
        n = min(n, 1 + int((c < f32(top_p) * c[-1]).sum()))
    n = max(1, min(n, int((w[order[:n]] >= f32(min_p)).sum())))
    kept = order[:n].sort().values
    c = torch.cumsum(w[kept], 0)
    return int(kept[min(int((c <= f32(u) * c[-1]).sum()), n - 1)])


class Pool:
    """A paged cache on `dev` and its sequences: pages handed out in a shuffled order."""

    def __init__(self, lens, nkv, hd, page, dev, seed=0, spare=3, width=None, interleaved=False, fill=0.0):
        g = torch.Generator().manual_seed(seed)
        counts = [(n + page - 1) // page for n in lens]
        self.pages = sum(counts) + spare
        self.page, self.nkv, self.hd, self.lens = page, nkv, hd, list(lens)
        ids = torch.randperm(self.pages, generator=g).tolist()
        self.table = torch.full((len(lens), width or max(1, max(counts, default=1))), -1, dtype=torch.int32)
        for i, c in enumerate(counts):
            self.table[i, :c] = torch.tensor([ids.pop() for _ in range(c)], dtype=torch.int32)
        if interleaved:
            both = torch.full((self.pages, 2, nkv, page, hd), fill, dtype=torch.bfloat16, device=dev)
            self.k, self.v = both[:, 0], both[:, 1]
        else:
            self.k = torch.full((self.pages, nkv, page, hd), fill, dtype=torch.bfloat16, device=dev)
            self.v = torch.full_like(self.k, fill)
        self.dev_table = self.table.to(dev)

    def put(self, i, k, v):
        """k, v [keys, nkv, hd] (CPU) as the first keys of sequence i."""
        n = k.shape[0]
        if n == 0:
            return
        page = self.table[i, torch.arange(n) // self.page].long().to(self.k.device)
        row = (torch.arange(n) % self.page).to(self.k.device)
        self.k[page, :, row] = k.to(self.k.device)
        self.v[page, :, row] = v.to(self.v.device)
