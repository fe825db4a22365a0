"""Decoding that branches over a paged cache, on the GPU against plain forms: attention for trees of
drafted tokens, their acceptance and compaction, beam selection, forked and copied pages."""
from __future__ import annotations

import glob
import math
import os
import random

import pytest
import torch

import branching_ref as ref
from serving_ref import Pool, assert_within, attention, rope

pytestmark = pytest.mark.gpu

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _bf(shape, seed, std=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * std).to(torch.bfloat16)


def _i32(v, dev):
    return torch.tensor(v, dtype=torch.int32, device=dev)


def _same(a, b):
    return torch.equal(a.cpu().contiguous().view(torch.int16), b.cpu().contiguous().view(torch.int16))


def _cuts(counts):
    cuts = [0]
    for c in counts:
        cuts.append(cuts[-1] + c)
    return cuts


# ------------------------------------------------------------------ attention of drafted tokens
class Trees:
    """Random sequences with drafted tokens behind them in a paged cache on `dev`."""

    def __init__(self, dev, lens, counts, nq, nkv, hd, page, seed=0, kind="tree", std=1.5, lead=0, behind=0, **kw):
        rng = random.Random(seed)
        self.lens, self.counts, self.nq, self.nkv, self.hd, self.dev = lens, counts, nq, nkv, hd, dev
        self.pool = Pool([a + b for a, b in zip(lens, counts)], nkv, hd, page, dev, seed=seed, fill=math.nan, **kw)
        self.k = [_bf((a + b, nkv, hd), 100 + seed + i) for i, (a, b) in enumerate(zip(lens, counts))]
        self.v = [_bf((a + b, nkv, hd), 9000 + seed + i) for i, (a, b) in enumerate(zip(lens, counts))]
        self.masks = [ref.chain(n) if kind == "chain" else ref.tree(rng, n) for n in counts]
        if kind == "any":  # no trees: any bits, none at all, bits past the nodes
            self.masks = [[rng.getrandbits(64) if i % 5 else 0 for i in range(n)] for n in counts]
        self.kind, self.lead = kind, lead
        self.cuts = [lead + c for c in _cuts(counts)]
        self.T = self.cuts[-1] + behind
        self.q = _bf((self.T, nq, hd), seed + 1, std)
        self.put()

    def put(self):
        for i, (k, v) in enumerate(zip(self.k, self.v)):
            self.pool.put(i, k, v)

    def dev_masks(self):
        if self.kind == "chain":
            return None
        full = [-1] * self.T
        for lo, m in zip(self.cuts, self.masks):
            full[lo:lo + len(m)] = [ref.word(v) for v in m]
        return torch.tensor(full, dtype=torch.int64, device=self.dev)

    def run(self, strided=False, table=None, **kw):
        from moeinfra_amd import ops

        q = self.q.to(self.dev)
        if strided:
            wide = torch.full((self.T, self.nq + 2, self.hd), math.nan, dtype=torch.bfloat16, device=self.dev)
            wide[:, :self.nq] = q
            q = wide[:, :self.nq]
        return ops.paged_tree_attention(q, self.pool.k, self.pool.v, self.pool.dev_table if table is None else table,
                                        _i32(self.lens, self.dev), _i32(self.cuts, self.dev), masks=self.dev_masks(), **kw)

    def check(self, out, scaling=None, keep=None):
        grp, out = self.nq // self.nkv, out.cpu()
        for i, (lo, n) in enumerate(zip(self.cuts, self.counts)):
            if n == 0:
                continue
            see = ref.seen(self.masks[i], self.lens[i])
            if keep is not None:
                see &= keep[i][None, :]
            for h in range(self.nkv):
                q = self.q[lo:lo + n, h * grp:(h + 1) * grp].reshape(n * grp, self.hd)
                want, tol = attention(q, self.k[i][:, h], self.v[i][:, h], self.hd ** -0.5 if scaling is None else scaling,
                                      seen=see.repeat_interleave(grp, dim=0))
                assert_within(out[lo:lo + n, h * grp:(h + 1) * grp].reshape(n * grp, self.hd), want, tol,
                              f"sequence {i} of {self.lens[i]} keys and {n} tokens, head {h}")


LENS = [0, 0, 1, 7, 8, 31, 32, 33, 63, 64, 65, 0, 127, 300, 513, 1000]
COUNTS = [1, 64, 1, 5, 64, 1, 33, 32, 2, 63, 31, 0, 17, 64, 40, 3]


@pytest.mark.parametrize("nq,nkv,hd,page,kind", [
    (32, 8, 128, 16, "tree"), (8, 2, 64, 8, "chain"), (4, 4, 128, 64, "any"), (16, 1, 128, 32, "tree"),
    (10, 2, 64, 16, "any"), (40, 2, 128, 8, "tree"), (8, 4, 256, 128, "tree"), (17, 1, 256, 16, "chain"),
    (3, 3, 64, 4096, "any"), (33, 1, 128, 64, "tree")])
def test_paged_tree_attention(cuda_device, nq, nkv, hd, page, kind):
    print(f"tree attention {nq}/{nkv} heads of {hd}, pages of {page}, {kind}", flush=True)
    t = Trees(cuda_device, LENS, COUNTS, nq, nkv, hd, page, seed=nq + hd, kind=kind, interleaved=page == 16)
    t.check(t.run(strided=nq % 2 == 0))


@pytest.mark.parametrize("lens,counts", [
    ([1], [1]), ([900], [5]), ([5000], [1]), ([20000, 3, 0, 900], [3, 64, 1, 20]), ([257] * 70, [3] * 70),
    ([40] * 300, [1 + i % 4 for i in range(300)]), ([0] * 90 + [9000] + [0] * 200, [0] * 90 + [64] + [1] * 200)])
def test_paged_tree_attention_batches(cuda_device, lens, counts):
    print(f"tree attention of {len(lens)} sequences", flush=True)
    t = Trees(cuda_device, lens, counts, 8, 2, 128, 16, seed=len(lens))
    t.check(t.run())


def test_paged_tree_attention_more_row_tiles_than_counters(cuda_device):
    print("tree attention, a workgroup for each row tile", flush=True)
    t = Trees(cuda_device, [i * 7 % 50 for i in range(2100)] + [700], [1 + i % 2 for i in range(2101)], 8, 8, 64, 16,
              seed=3)
    t.check(t.run())


@pytest.mark.parametrize("nq,nkv,hd,lens,counts", [
    (8, 8, 64, [i * 7 % 50 for i in range(2100)] + [700], [1 + i % 2 for i in range(2101)]),
    (8, 2, 128, [i * 37 % 300 for i in range(130)], [0 if i % 5 == 2 or i in (63, 64) else 1 + i * 11 % 64 for i in range(130)]),
    (16, 1, 128, [i % 70 for i in range(65)], [0] * 63 + [64, 40])])
def test_paged_tree_attention_of_many_sequences_without_a_workspace(cuda_device, nq, nkv, hd, lens, counts):
    """The C call without one: a workgroup for each sequence, KV head and row tile, also past the 64th sequence."""
    from moeinfra_amd import _lib

    print(f"tree attention of {len(lens)} sequences without a workspace", flush=True)
    dev = cuda_device
    t = Trees(dev, lens, counts, nq, nkv, hd, 16, seed=23, lead=2, behind=3)
    q, out = t.q.to(dev), torch.full_like(t.q, 9.0, device=dev)
    n, cu, masks = _i32(t.lens, dev), _i32(t.cuts, dev), t.dev_masks()
    _lib.check(_lib.lib().moe_paged_tree_attention_bf16(
        q.data_ptr(), q.stride(0), t.T, t.pool.k.data_ptr(), t.pool.v.data_ptr(), t.pool.pages, 16, t.pool.k.stride(0),
        t.pool.dev_table.data_ptr(), t.pool.dev_table.shape[1], n.data_ptr(), cu.data_ptr(), masks.data_ptr(), len(lens), nq,
        nkv, hd, hd ** -0.5, out.data_ptr(), None, 0, torch.cuda.current_stream().cuda_stream), "tree attention")
    t.check(out)
    assert bool((out[:2] == 9.0).all()) and bool((out[t.T - 3:] == 9.0).all())
    shared = t.run()
    t.check(shared)
    # With one the same within two roundings of the output and of the weights.
    got, want = out[2:t.T - 3].float(), shared[2:t.T - 3].float()
    assert float((got - want).abs().max()) <= 4 * 2.0 ** -8 * float(max(v.float().abs().max() for v in t.v if len(v)))


@pytest.mark.parametrize("nq,nkv,hd,lens,counts", [
    (8, 2, 128, [20000, 0, 8176, 5], [40, 3, 64, 1]), (8, 1, 64, [17000, 9000], [64, 2]), (8, 4, 256, [8200, 1], [33, 9]),
    (40, 2, 128, [300, 8150], [64, 64])])
def test_paged_tree_attention_without_a_workspace(cuda_device, nq, nkv, hd, lens, counts):
    """The C call without one: a workgroup for each KV head and row tile, which finds more page entries
    than it holds at a time."""
    from moeinfra_amd import _lib, ops

    print(f"tree attention {nq}/{nkv} heads of {hd} without a workspace", flush=True)
    t = Trees(cuda_device, lens, counts, nq, nkv, hd, 8, seed=21)
    q, out, dev = t.q.to(cuda_device), torch.full_like(t.q, 9.0, device=cuda_device), cuda_device
    n, cu, masks = _i32(t.lens, dev), _i32(t.cuts, dev), t.dev_masks()
    _lib.check(_lib.lib().moe_paged_tree_attention_bf16(
        q.data_ptr(), q.stride(0), t.T, t.pool.k.data_ptr(), t.pool.v.data_ptr(), t.pool.pages, 8, t.pool.k.stride(0),
        t.pool.dev_table.data_ptr(), t.pool.dev_table.shape[1], n.data_ptr(), cu.data_ptr(), masks.data_ptr(), len(lens), nq,
        nkv, hd, hd ** -0.5, out.data_ptr(), None, 0, torch.cuda.current_stream().cuda_stream), "tree attention")
    t.check(out)
    # With one the same within two roundings of the output and of the weights.
    assert float((out.float() - t.run().float()).abs().max()) <= 4 * 2.0 ** -8 * float(max(v.float().abs().max() for v in t.v))


def test_paged_tree_attention_more_kv_heads_than_workgroups_at_once(cuda_device):
    print("tree attention of 300 KV heads", flush=True)
    t = Trees(cuda_device, [70, 0, 33], [9, 64, 1], 300, 300, 64, 16, seed=22)
    t.check(t.run())


def test_far_pages(cuda_device):
    """Pages more than 2^32 bytes apart: attention, the embedding, moves and copies."""
    from moeinfra_amd import ops

    dev, nq, nkv, hd, page, apart = cuda_device, 8, 2, 64, 16, (1 << 31) + 64 * 1024
    both = torch.empty(3 * apart + 4 * nkv * page * hd, dtype=torch.bfloat16, device=dev)   # 13 GB
    shape, strides = (4, nkv, page, hd), (apart, page * hd, hd, 1)
    k, v = both.as_strided(shape, strides), both.as_strided(shape, strides, 2 * nkv * page * hd)
    keys, vals = _bf((4 * page, nkv, hd), 31), _bf((4 * page, nkv, hd), 32)
    table = _i32([[2, 0, 3, 1]], dev)
    for i, p in enumerate([2, 0, 3, 1]):
        k[p] = keys[i * page:(i + 1) * page].transpose(0, 1).to(dev)
        v[p] = vals[i * page:(i + 1) * page].transpose(0, 1).to(dev)
    q = _bf((10, nq, hd), 33, 1.5)
    out = ops.paged_tree_attention(q.to(dev), k, v, table, _i32([50], dev), _i32([0, 10], dev))
    see = ref.seen(ref.chain(10), 50).repeat_interleave(4, dim=0)
    for h in range(nkv):
        want, tol = attention(q[:, 4 * h:4 * h + 4].reshape(40, hd), keys[:60, h], vals[:60, h], hd ** -0.5, seen=see)
        assert_within(out[:, 4 * h:4 * h + 4].reshape(40, hd), want, tol, f"head {h}")
    ops.compact_paged_kv(k, v, table, _i32([15], dev), ref.words([1 << 33 | 1 << 20], dev))   # places 35, 48 to 15, 16
    assert _same(k[2, :, 15], keys[35]) and _same(v[0, :, 0], vals[48]) and _same(k[0, :, 1], keys[17])
    ops.copy_pages(k, v, _i32([[3, 1, 5]], dev))
    assert _same(k[1, :, :5], keys[32:37].transpose(0, 1)) and _same(v[1, :, 5], vals[53])
    x = _bf((1, (nq + 2 * nkv) * hd), 34)
    _, y = ops.rope_paged_kv(x.to(dev), _i32([7], dev), table, k, v, nq, _inv(hd).to(dev), want_k=True, slots=_i32([63], dev))
    assert _same(k[1, :, 15], y[0]) and _same(v[1, :, 15], x.view(-1, hd)[nq + nkv:])


def test_paged_tree_attention_rows_of_no_sequence(cuda_device):
    """Rows before the first sequence, behind the last one, and of nodes past the 64th."""
    lens, counts = [20, 300, 5], [7, 64, 70]
    t = Trees(cuda_device, lens, counts, 8, 2, 128, 16, seed=4, lead=3, behind=9, kind="chain")
    out = torch.full((t.T, 8, 128), 9.0, dtype=torch.bfloat16, device=cuda_device)
    assert t.run(out=out) is out
    left = list(range(3)) + list(range(t.T - 9 - 6, t.T))
    assert bool((out[left] == 9.0).all())
    t.counts[2], t.masks[2] = 64, t.masks[2][:64]
    t.k[2], t.v[2] = t.k[2][:69], t.v[2][:69]
    t.check(out)


def test_paged_tree_attention_workspaces(cuda_device):
    """The same bits without a workspace of the caller's, with one of another batch, and again; writes
    stay inside; what it holds before does not matter."""
    from moeinfra_amd import ops

    dev = cuda_device
    t = Trees(dev, [9000, 3, 0, 700, 5000], [64, 5, 1, 20, 33], 32, 8, 128, 16, seed=5)
    n = ops.paged_tree_attention_workspace(1, 32, 8, 128, dev).numel()
    guarded = torch.full((n + 8192,), 0x5a, dtype=torch.uint8, device=dev)
    ws = guarded[4096:4096 + n]
    a = t.run(workspace=ws)
    t.check(a)
    other = Trees(dev, [3000] * 9, [17] * 9, 32, 8, 128, 16, seed=6)
    other.check(other.run(workspace=ws))
    assert _same(a, t.run(workspace=ws)) and _same(a, t.run())
    assert bool((guarded[:4096] == 0x5a).all()) and bool((guarded[4096 + n:] == 0x5a).all())
    ws.fill_(0xff)
    assert _same(a, t.run(workspace=ws))


def test_paged_tree_attention_missing_pages_and_lengths(cuda_device):
    dev, page = cuda_device, 16
    t = Trees(dev, [100, 100, 60, 90], [20, 20, 30, 4], 8, 2, 128, page, seed=8)
    table = t.pool.dev_table.clone()
    table[0, 2] = -7                    # keys 32 .. 47
    table[1, 0] = t.pool.pages          # keys 0 .. 15
    table[1, 7] = -1                    # and the drafted 112 .. 119
    table[2, :] = -1                    # all of them
    keep = [torch.ones(a + b, dtype=torch.bool) for a, b in zip(t.lens, t.counts)]
    keep[0][32:48] = False
    keep[1][:16] = False
    keep[1][112:] = False
    keep[2][:] = False
    t.check(t.run(table=table), keep=keep)
    # A length past the table: all of its pages, no drafted keys; a negative one: drafted keys only.
    from moeinfra_amd import ops

    q = t.q[t.cuts[3]:t.cuts[3] + 4]
    for said, seen, keys in ((1 << 30, torch.ones((4, 80), dtype=torch.bool), slice(0, 80)),
                             (-5, ref.seen(t.masks[3], 0), slice(0, 4))):
        out = ops.paged_tree_attention(q.to(dev), t.pool.k, t.pool.v, t.pool.dev_table[3:4, :5].contiguous(),
                                       _i32([said], dev), _i32([0, 4], dev), masks=ref.words(t.masks[3], dev))
        for h in range(2):
            want, tol = attention(q[:, 4 * h:4 * h + 4].reshape(16, 128), t.k[3][keys, h], t.v[3][keys, h], 128 ** -0.5,
                                  seen=seen.repeat_interleave(4, dim=0))
            assert_within(out[:, 4 * h:4 * h + 4].reshape(16, 128), want, tol, f"length {said}, head {h}")
    # No pages at all: zeros.
    none = ops.paged_tree_attention(q.to(dev), t.pool.k[:0], t.pool.v[:0], t.pool.dev_table[3:4], _i32([9], dev),
                                    _i32([0, 4], dev))
    assert not bool(none.any())


@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("nq,nkv,hd,n", [(8, 2, 128, 40), (4, 4, 64, 64), (8, 4, 256, 20), (32, 1, 128, 9)])
def test_paged_tree_attention_infinities_stay_with_the_rows_that_see_them(cuda_device, nq, nkv, hd, n, value):
    """A drafted token whose keys or values have come apart changes the rows of its descendants only."""
    keys = 50
    t = Trees(cuda_device, [keys, 3], [n, n], nq, nkv, hd, 16, seed=9)
    bad = n // 3
    t.v[0][keys + bad, :, 5:9] = value
    t.k[1][3 + bad] = value
    t.put()
    out = t.run()
    rows = [[i for i in range(n) if not m[i] >> bad & 1] for m in t.masks]
    assert all(rows)
    for b in range(2):
        hit = [i for i in range(n) if t.masks[b][i] >> bad & 1]
        got = out[t.cuts[b]:t.cuts[b] + n].cpu()
        part = got[hit][:, :, 5:9] if b == 0 else got[hit]
        assert not bool(torch.isfinite(part).any())
        if b == 0:
            assert bool(torch.isfinite(got[hit][:, :, 9:]).all()) and bool(torch.isfinite(got[hit][:, :, :5]).all())
    grp = nq // nkv
    for b in range(2):
        k, v = t.k[b].clone(), t.v[b].clone()
        k[t.lens[b] + bad] = 0
        v[t.lens[b] + bad] = 0
        see = ref.seen(t.masks[b], t.lens[b])[rows[b]].repeat_interleave(grp, dim=0)
        for h in range(nkv):
            at = [t.cuts[b] + i for i in rows[b]]
            want, tol = attention(t.q[at][:, h * grp:(h + 1) * grp].reshape(-1, hd), k[:, h], v[:, h], hd ** -0.5, seen=see)
            assert_within(out[at][:, h * grp:(h + 1) * grp].reshape(-1, hd), want, tol, f"sequence {b}, head {h}")


def test_paged_tree_attention_scalings_and_large_scores(cuda_device):
    for scaling in (0.0, -0.3, 1.0, 2.0 ** -7):
        t = Trees(cuda_device, [200, 9], [30, 64], 8, 2, 128, 16, seed=11)
        t.check(t.run(scaling=scaling), scaling=scaling)
    # Scores of up to 3.2e38: neighbouring keys lie 1e36 apart, one key (or its equals) has all the weight.
    t = Trees(cuda_device, [180], [20], 4, 1, 64, 16, seed=12, kind="chain")
    t.k[0][:, 0, 1:] = 0
    t.k[0][:, 0, 0] = torch.linspace(-2.1e20, 2.1e20, 200).to(torch.bfloat16)
    t.q.zero_()
    t.q[:, :, 0] = torch.tensor([1.5e18, -1.5e18, 7.5e17, 1.0])
    t.put()
    out = t.run(scaling=1.0)
    assert not bool(torch.isnan(out).any())
    for i in range(20):
        want, _ = attention(t.q[i], t.k[0][:180 + i + 1, 0], t.v[0][:180 + i + 1, 0], 1.0)
        tol = 2.0 ** -8 * (want.abs() + t.v[0].double().abs().amax()) + 0 * want
        assert_within(out[i], want, tol, f"token {i}")


# ------------------------------------------------------------------ acceptance
@pytest.mark.parametrize("B,most,kind", [(1, 1, "tree"), (1, 64, "tree"), (5, 12, "chain"), (300, 64, "tree"),
                                         (3, 80, "chain"), (70, 64, "any")])
def test_accept_drafts(cuda_device, B, most, kind):
    from moeinfra_amd import ops

    rng = random.Random(B + most)
    counts = [rng.choice((0, 1, most, rng.randint(1, most))) for _ in range(B)]
    counts[-1] = most
    masks, drafts, targets = [], [], []
    for n in counts:
        masks.append(ref.chain(n) if kind == "chain" else ref.tree(rng, n) if kind == "tree" else
                     [rng.getrandbits(64) if i % 7 else 0 for i in range(n)])
        drafts.append([rng.randrange(4) - (1 << 40) * (i % 3 == 0) for i in range(n)])
        targets.append([rng.choice(drafts[-1]) for _ in range(n)])
    cuts = _cuts(counts)
    flat = lambda v: torch.tensor([x for r in v for x in r], dtype=torch.int64, device=cuda_device)
    m = None if kind == "chain" else ref.words([x for r in masks for x in r], cuda_device)
    paths, n, tokens = ops.accept_drafts(flat(targets), flat(drafts), _i32(cuts, cuda_device), masks=m)
    want = [ref.accept(t, d, k) for t, d, k in zip(targets, drafts, masks)]
    assert paths.tolist() == [ref.word(w[0]) for w in want]
    assert n.tolist() == [w[1] for w in want] and tokens.tolist() == [w[2] for w in want]
    assert paths.dtype is torch.int64 and n.dtype is torch.int32 and tokens.dtype is torch.int64


# ------------------------------------------------------------------ compaction, copies
def _caches(dev, layers, pages, nkv, page, hd, seed, layout):
    """(k, v) of equal values in one of the layouts that caches may have."""
    k, v = _bf((layers, pages, nkv, page, hd), seed), _bf((layers, pages, nkv, page, hd), seed + 1)
    if layout == "apart":
        return k.to(dev), v.to(dev)
    if layout == "both":     # keys and values of a page next to each other
        both = torch.empty((layers, pages, 2, nkv, page, hd), dtype=torch.bfloat16, device=dev)
        out = both[:, :, 0], both[:, :, 1]
    else:                    # the layers of a page next to each other
        both = torch.empty((2, pages, layers, nkv, page, hd), dtype=torch.bfloat16, device=dev)
        out = both[0].transpose(0, 1), both[1].transpose(0, 1)
    out[0].copy_(k)
    out[1].copy_(v)
    return out


@pytest.mark.parametrize("B,layers,nkv,page,hd,layout", [
    (1, 1, 1, 8, 8, "apart"), (7, 3, 8, 16, 128, "apart"), (20, 2, 3, 8, 80, "both"), (5, 4, 2, 64, 512, "layers"),
    (9, 1, 2, 4096, 64, "apart")])
def test_compact_paged_kv(cuda_device, B, layers, nkv, page, hd, layout):
    from moeinfra_amd import ops

    rng, dev = random.Random(B), cuda_device
    lens = [rng.choice((0, 1, page - 1, page, rng.randrange(3 * page))) for _ in range(B)]
    width = max((n + 64 + page - 1) // page for n in lens)
    pages = B * width + 2
    ids = list(range(pages))
    rng.shuffle(ids)
    table = torch.tensor([ids.pop() for _ in range(B * width)], dtype=torch.int32).view(B, width)
    patterns = [0, 1, 1 << 63, (1 << 64) - 1, ((1 << 64) - 1) ^ 1, 0b1011, 0xaaaaaaaaaaaaaaaa]
    paths = [patterns[i % 7] if i % 2 else rng.getrandbits(64) & rng.getrandbits(64) for i in range(B)]
    if B > 4:
        table[3, lens[3] // page] = -1
        table[4, -1] = pages
        lens[2] = -4
    k, v = _caches(dev, layers, pages, nkv, page, hd, 20, layout)
    want = [ref.compact(c.cpu(), table, lens, paths, page) for c in (k, v)]
    args = (table.to(dev), _i32(lens, dev), ref.words(paths, dev))
    if layers == 1:
        assert ops.compact_paged_kv(k[0], v[0], *args) is None
    else:
        ops.compact_paged_kv(k, v, *args)
    assert _same(k, want[0]) and _same(v, want[1])


def test_compact_paged_kv_past_the_table(cuda_device):
    from moeinfra_amd import ops

    k, v = _caches(cuda_device, 2, 4, 2, 8, 64, 30, "apart")
    table = torch.tensor([[2, 0], [1, 3]], dtype=torch.int32)
    lens, paths = [12, 2147483000], [0b111111010, 0b1010]
    want = [ref.compact(c.cpu(), table, lens, paths, 8) for c in (k, v)]
    ops.compact_paged_kv(k, v, table.to(cuda_device), _i32(lens, cuda_device), ref.words(paths, cuda_device))
    assert _same(k, want[0]) and _same(v, want[1])


@pytest.mark.parametrize("layers,nkv,page,hd,layout", [(1, 1, 8, 8, "apart"), (3, 8, 16, 128, "both"),
                                                       (4, 2, 64, 80, "layers"), (2, 4, 128, 256, "apart")])
def test_copy_pages(cuda_device, layers, nkv, page, hd, layout):
    from moeinfra_amd import ops

    k, v = _caches(cuda_device, layers, 12, nkv, page, hd, 40, layout)
    copies = [[0, 1, page], [0, 2, 1], [-1, -1, 0], [3, 4, page - 1], [5, 12, 3], [-2, 6, 3], [7, 7, 3], [8, 9, 0],
              [8, 10, page + 5], [11, -1, 2], [3, 5, -3]]
    want = []
    for c in (k.cpu(), v.cpu()):
        w = c.clone()
        for s, d, n in copies:
            if 0 <= s < 12 and 0 <= d < 12 and n > 0:
                w[:, d, :, :n] = c[:, s, :, :n]
        want.append(w)
    if layers == 1:
        assert ops.copy_pages(k[0], v[0], _i32(copies, cuda_device)) is None
    else:
        ops.copy_pages(k, v, _i32(copies, cuda_device))
    assert _same(k, want[0]) and _same(v, want[1])


# ------------------------------------------------------------------ beams
def _logits(rows, vocab, seed, dtype):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((rows, vocab), generator=g) * 2
    x += torch.where(torch.randn((rows, vocab), generator=g) > 3, torch.rand((rows, vocab), generator=g) * 9, 0.0)
    return x.to(dtype)


def _check_beams(got, logits, scores, k):
    best, rows, tokens = ref.beams(logits.cpu(), scores.cpu(), k)
    assert torch.equal(got[1].cpu(), rows) and torch.equal(got[2].cpu(), tokens)
    none = best == -math.inf
    assert torch.equal(got[0].cpu() == -math.inf, none)
    # Totals: one rounding to fp32, and sums in 64 bits from exponentials of 2^-40.
    err = (got[0].cpu().double() - best)[~none].abs()
    assert bool((err <= 2.0 ** -24 * best[~none].abs() + 2.0 ** -38).all())


@pytest.mark.parametrize("S,W,k,V,dtype", [
    (1, 4, 8, 32000, torch.bfloat16), (3, 4, 8, 32000, torch.float32), (2, 1, 1, 50257, torch.bfloat16),
    (5, 16, 32, 9001, torch.float32), (300, 3, 6, 1000, torch.bfloat16), (1, 16, 64, 131072, torch.bfloat16),
    (2, 256, 64, 300, torch.bfloat16), (3000, 1, 4, 301, torch.bfloat16), (1, 2, 2, 1 << 20, torch.float32),
    (7, 5, 10, 17, torch.float32)])
def test_beam_select(cuda_device, S, W, k, V, dtype):
    from moeinfra_amd import ops

    print(f"beam selection {S} x {W} x {V}, {k} best", flush=True)
    x = _logits(S * W, V, S + W, dtype).to(cuda_device)
    scores = -20 * torch.rand((S, W), generator=torch.Generator().manual_seed(V)).to(cuda_device)
    scores[S // 2, 1:] = -math.inf     # a first step
    got = ops.beam_select(x, scores, k)
    assert [t.dtype for t in got] == [torch.float32, torch.int32, torch.int64]
    _check_beams(got, x, scores, k)


@pytest.mark.parametrize("V", [1, 2, 7, 8, 9, 63, 1023, 2049, 8193])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_beam_select_odd_sizes_and_strides(cuda_device, V, dtype):
    from moeinfra_amd import ops

    S, W, k = 3, 2, 5
    base = torch.full((S * W + 1, V + 5), math.inf, dtype=dtype, device=cuda_device)
    for lead in (0, 1, 3):
        x = base[:-1, lead:lead + V]
        x.copy_(_logits(S * W, V, V + lead, dtype))
        scores = -torch.rand((S, W), generator=torch.Generator().manual_seed(V)).to(cuda_device)
        _check_beams(ops.beam_select(x, scores, k), x, scores, k)


def test_beam_select_equal_and_ordered_logits(cuda_device):
    """All equal, equal beams, rows that rise or fall, equal ones far apart, both zeros."""
    from moeinfra_amd import ops

    V, W, k = 20000, 4, 16
    g = torch.Generator().manual_seed(1)
    rise = torch.arange(V, dtype=torch.float32) / V
    rows = [torch.zeros(V), rise, rise.flip(0), torch.where(torch.arange(V) % 997 == 5, 3.0, -1.0),
            torch.where(torch.rand(V, generator=g) < 0.5, -0.0, 0.0)]
    for dtype in (torch.bfloat16, torch.float32):
        for r in rows:
            x = r.to(dtype)[None].repeat(2 * W, 1).to(cuda_device)
            for scores in (torch.zeros((2, W)), torch.tensor([[0, -1e-3, 1e-3, 0], [-5, -5, -5, -5.0]])):
                scores = scores.to(cuda_device)
                _check_beams(ops.beam_select(x, scores, k), x, scores, k)


@pytest.mark.parametrize("W,V,k", [(16, 40000, 32), (16, 131072, 16), (64, 9000, 64), (3, 300000, 64)])
def test_beam_select_more_alike_than_the_lists_hold(cuda_device, W, V, k):
    """Parts and searches with thousands of equal continuations, with few large ones among them."""
    from moeinfra_amd import ops

    print(f"{W} beams of {V} equal logits, {k} best", flush=True)
    x = torch.zeros((W, V), dtype=torch.bfloat16)
    scores = torch.zeros((1, W))
    for step in range(3):
        if step == 1:
            x[W // 2, [5, V // 2, V - 1]] = 1.0
        if step == 2:
            scores = -torch.arange(W)[None].float() / 1024
        dx, ds = x.to(cuda_device), scores.to(cuda_device)
        _check_beams(ops.beam_select(dx, ds, k), dx, ds, k)


def test_beam_select_near_totals(cuda_device):
    """Beams whose totals differ in the ninth digit only, by sums over the vocabulary."""
    from moeinfra_amd import ops

    V, W = 50000, 8
    g = torch.Generator().manual_seed(2)
    x = (torch.randn((1, V), generator=g) * 3).repeat(W, 1)
    x[:, 7] = 14.0
    low = int(x[0].argmin())
    for w in range(W):   # far below the others' sum: changes of 1e-9 of it
        x[w, low] = -6.5 + 0.02 * ((w * 5) % W)
    x = x.to(cuda_device)
    scores = torch.zeros((1, W), device=cuda_device)
    _check_beams(ops.beam_select(x, scores, 2 * W), x, scores, 2 * W)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_beam_select_masked_rows(cuda_device, dtype):
    """-inf, NaN and +inf among the logits and scores; fewer continuations than asked for; none."""
    from moeinfra_amd import ops

    S, W, V, k = 9, 3, 5000, 6
    x = _logits(S * W, V, 5, dtype)
    x[0:3] = -math.inf
    x[3:6, 2:] = -math.inf            # two tokens a beam
    x[6] = math.nan
    x[7, ::2] = math.nan
    x[9, 100] = math.inf
    x[12:15] = math.nan
    x[15, 4999], x[16, 0] = 1e30 if dtype is torch.float32 else 1e5, -1e30
    x[18:21] = -3e38
    x[21:24, 17] = 1e4
    scores = -torch.rand((S, W), generator=torch.Generator().manual_seed(6))
    scores[2, 1] = math.nan
    scores[5, 0] = math.inf
    scores[8] = -math.inf
    x, scores = x.to(cuda_device), scores.to(cuda_device)
    _check_beams(ops.beam_select(x, scores, k), x, scores, k)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_beam_select_signaling_nans(cuda_device, dtype):
    """NaNs of every kind stand for nothing, also where they share a thread with the best."""
    from moeinfra_amd import ops

    V, k = 9001, 20
    x = _logits(6, V, 8, dtype)
    bits = x.view(torch.int16 if dtype is torch.bfloat16 else torch.int32)
    nans = [0x7f81, 0xff81 - 65536, 0x7fc0] if dtype is torch.bfloat16 else [0x7f800001, 0xff80ff80 - (1 << 32), 0x7fc00000]
    for i, n in enumerate(nans):
        bits[:, 5 + i::7] = n
    x, scores = x.to(cuda_device), torch.zeros((3, 2), device=cuda_device)
    _check_beams(ops.beam_select(x, scores, k), x, scores, k)


def test_beam_select_workspaces(cuda_device):
    from moeinfra_amd import ops

    dev = cuda_device
    n = ops.beam_select_workspace(40, 4, 8, dev).numel()
    guarded = torch.full((n + 8192,), 0x5a, dtype=torch.uint8, device=dev)
    ws = guarded[4096:4096 + n]
    ws[:65536].zero_()
    for S, W, k, V in ((40, 4, 8, 3000), (1, 4, 8, 100000), (7, 2, 3, 999), (40, 4, 8, 60000)):
        x, scores = _logits(S * W, V, V, torch.bfloat16).to(dev), -torch.rand((S, W)).to(dev)
        a = ops.beam_select(x, scores, k, workspace=ws)
        _check_beams(a, x, scores, k)
        b = ops.beam_select(x, scores, k, workspace=ws)
        assert all(torch.equal(p, q) for p, q in zip(a, b))
    assert bool((guarded[:4096] == 0x5a).all()) and bool((guarded[4096 + n:] == 0x5a).all())
    assert not bool(ws[:65536].any())


def _equal_beams(W, k, x, score, dtype):
    """What W beams of equal scores and the logits x [V] give: the larger logit first, of equal ones the lower beam,
    then token.  (Totals of equal logits are equal, so a logit's tokens go beam by beam.)"""
    v, at = torch.sort(x.to(dtype).double(), descending=True, stable=True)
    want, i = [], 0
    while len(want) < k:
        same = int((v == v[i]).sum())
        want += [(w, int(t)) for w in range(W) for t in at[i:i + same][:k]]
        i += same
    return want[:k]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("V", [50257, 32001, 151669, 1999])
def test_beam_select_equal_beams_at_any_alignment(cuda_device, V, dtype):
    """Beams of the same logits and scores: in order, wherever their rows begin; the same totals from every view."""
    from moeinfra_amd import ops

    W, k = 5, 12
    for seed in range(6):
        x = _logits(1, V, seed, dtype)
        want = _equal_beams(W, k, x[0], 0.0, dtype)
        totals = []
        for lead, pad in ((0, 0), (0, 8 - V % 8), (1, 3), (3, 4), (5, 9)):
            base = torch.full((W, V + pad + lead), math.inf, dtype=dtype, device=cuda_device)
            base[:, lead:lead + V] = x.to(cuda_device)
            best, rows, tokens = ops.beam_select(base[:, lead:lead + V], torch.full((1, W), -1.5, device=cuda_device), k)
            got = list(zip(rows[0].tolist(), tokens[0].tolist()))
            assert got == want, f"seed {seed}, {lead} values before a row and {pad} behind it"
            totals.append(best)
        assert all(torch.equal(t, totals[0]) for t in totals)


@pytest.mark.parametrize("part", [0.02, 0.25, 0.5, 0.75, 0.98])
def test_beam_select_sums_tell_totals_of_two_to_the_minus_40_apart(cuda_device, part):
    """Exponentials to 2^-42: of two beams whose best totals lie 2^-40 apart the better one comes first, whatever
    places between two entries of a table of 256 powers of two the logits of one of them take."""
    from moeinfra_amd import ops

    V, unit = 2000, math.log(2) / 256
    fp32 = lambda v: torch.tensor(v, dtype=torch.float32).tolist()
    lse = lambda r: math.log(math.fsum(math.exp(v) for v in r))   # (2^-50 of itself)
    other = fp32([0.0] + [-(j - 0.001) * unit for j in range(1, V)])
    for ahead in (2.0 ** -40, -2.0 ** -40):
        row = fp32([0.0] + [-(j + 1 - part) * unit for j in range(1, V - 1)])
        # The score in steps of 2^-24 of itself, the rest by a logit far below.
        score = fp32([lse(row + [-16.0]) - lse(other) - ahead])[0]
        rest = math.exp(score + lse(other) + ahead) - math.fsum(math.exp(v) for v in row)
        row = row + fp32([math.log(rest)])
        gap = (0.0 - lse(other)) - (score - lse(row))
        assert abs(gap - ahead) < 2.0 ** -46
        x = torch.tensor([row, other], device=cuda_device)
        got = ops.beam_select(x, torch.tensor([[score, 0.0]], device=cuda_device), 2)
        assert got[1].tolist()[0] == ([1, 0] if ahead > 0 else [0, 1]) and got[2].tolist() == [[0, 0]]


@pytest.mark.parametrize("W,V,score", [(1, 40, -20.0), (2, 40, -20.0), (2, 100000, -20.0), (3, 5000, -1e20), (16, 70000, -20.0)])
def test_beam_select_logits_nearer_than_their_totals(cuda_device, W, V, score):
    """Logits that differ by less than a step of the totals: the larger one first, the lower beam's before the
    others', and the first k of them whatever k."""
    from moeinfra_amd import ops

    g = torch.Generator().manual_seed(V)
    x = torch.full((W, V), -30.0)
    at = torch.randperm(V, generator=g)[:80]
    for w in range(W):   # (the same exponentials at the same places: the same sums)
        x[w, at] = (torch.randperm(len(at), generator=g).float() + 1) * 1e-20
    scores = torch.full((1, W), score)
    x, scores = x.to(cuda_device), scores.to(cuda_device)
    order = torch.sort(x[0].double().cpu(), descending=True, stable=True).indices.tolist()
    for k in (1, 2, 3, 9, 30, min(64, V)):
        best, rows, tokens = ops.beam_select(x, scores, k)
        assert rows.tolist() == [[0] * k] and tokens.tolist() == [order[:k]], f"the best {k}"
        assert bool((best == best[0, 0]).all())


# ------------------------------------------------------------------ forked pages
def _check_fork(dev, table, lens, parents, refs, page, ahead=1, workspace=None):
    from moeinfra_amd import ops

    want_refs = list(refs)
    want = ref.fork(table, lens, parents, want_refs, page, ahead)
    r = _i32(refs, dev)
    got = ops.fork_pages(_i32(table, dev).view(len(lens), -1), _i32(lens, dev), _i32(parents, dev), r, page, ahead=ahead,
                         workspace=workspace)
    assert got[0].tolist() == want[0] and got[1].tolist() == want[1]
    assert got[2].tolist() == want[2] and got[3].tolist() == [want[3]] and r.tolist() == want_refs
    return want[0], want[1], want_refs


@pytest.mark.parametrize("rows,page,pages,ahead", [(4, 16, 40, 1), (8, 8, 200, 1), (60, 8, 3000, 20), (3, 64, 5, 1),
                                                   (33, 8, 40, 9), (256, 32, 5000, 1)])
def test_fork_pages(cuda_device, rows, page, pages, ahead):
    """Steps of random beams that grow, from one prompt; pages run out in some."""
    from moeinfra_amd import ops

    rng = random.Random(rows)
    width = 40
    ws = ops.fork_pages_workspace(pages, cuda_device)
    table, lens, refs = [[-1] * width], [0], [0] * pages
    refs[3] = 1                        # held from outside
    n = rng.randrange(4 * page)
    ids = [p for p in range(pages) if p != 3][:(n + page - 1) // page]
    for e, p in enumerate(ids):
        table[0][e] = p
        refs[p] = 1 + (e == 0)         # the first page of the prompt is kept
    lens[0] = n
    parents = [0] * rows
    for step in range(8):
        table, lens, refs = _check_fork(cuda_device, table, lens, parents, refs, page, ahead, ws)
        assert all(c >= 0 for c in refs)
        lens = [min(n + rng.randint(0, ahead), width * page) for n in lens]
        m = rows if step < 5 else max(1, rows // 2)
        parents = [rng.choice((rng.randrange(len(lens)), 0, len(lens) - 1, -1)) if step % 3 else rng.randrange(len(lens))
                   for _ in range(m)]
    assert not bool(ws.any())


def test_fork_pages_corners(cuda_device):
    dev = cuda_device
    # Full tables, lengths of any sign, pages that are not there, nothing but rows that end.
    _check_fork(dev, [[0, 1], [2, 3]], [16, 15], [0, 0, 1, 1], [1] * 4 + [0] * 9, 8)
    _check_fork(dev, [[0, 9, -1], [70, 1, -3]], [9, -4], [1, 0, 1], [1, 1, 0, 0], 8)
    _check_fork(dev, [[0, 1], [2, 3]], [16, 15], [-1, 7, 2], [1] * 4, 8)
    _check_fork(dev, [[0, 1, 2], [0, 1, 3]], [20, 17], [0, 1], [2, 2, 1, 1, 0], 8)
    # A page of two rows at different places; one page twice in a row.
    _check_fork(dev, [[5, 6, -1], [6, 7, -1]], [12, 4], [0, 1], [0, 0, 0, 0, 0, 1, 2, 1], 8)
    _check_fork(dev, [[5, 5, 1]], [12], [0, 0, 0], [0, 1, 0, 0, 0, 2], 8)
    # No page is free; no pages at all; no rows.
    _check_fork(dev, [[0, -1]], [5], [0, 0, 0], [1], 8)
    _check_fork(dev, [[0, -1]], [5], [0, 0, 0], [], 8)
    _check_fork(dev, [[0, -1]], [5], [], [1, 0], 8)
    # A length near the largest, and many tokens ahead.
    _check_fork(dev, [[0, 1]], [2147483647], [0], [1, 1, 0], 8, ahead=100)
    _check_fork(dev, [[0] + [-1] * 40], [3], [0, 0], [1] + [0] * 100, 8, ahead=300)


def test_fork_pages_most_rows(cuda_device):
    rng = random.Random(7)
    rows, pages, page = 8192, 9000, 8
    table, refs = [[i, -1] for i in range(rows)], [1] * rows + [0] * (pages - rows)
    lens = [rng.randint(0, 8) for _ in range(rows)]
    _check_fork(cuda_device, table, lens, [rng.randrange(rows) for _ in range(rows)], refs, page)


@pytest.mark.parametrize("rows,page,ahead,spare", [(2049, 8, 1, 900), (2048, 16, 1, 900), (2100, 8, 12, 2000), (1025, 8, 9, 1500),
                                                   (1024, 8, 9, 1500), (4000, 16, 1, 3000), (683, 8, 17, 700)])
def test_fork_pages_of_many_rows_step_by_step(cuda_device, rows, page, ahead, spare):
    """Around and above what is chosen in LDS (2048 rows and places): steps of random beams over prompts that many
    rows share and that are held from outside too, with one workspace, which every step leaves zero; pages run out."""
    from moeinfra_amd import ops

    print(f"{rows} rows, {ahead} tokens ahead, pages of {page}", flush=True)
    rng = random.Random(rows + ahead)
    width, prompts = 9, 40
    table, lens, refs = [], [], [0] * 3
    for i in range(rows):
        if i < prompts:                # the prompts' rows, their first pages held from outside
            n = rng.randint(1, 3 * page)
            ids = list(range(len(refs), len(refs) + (n + page - 1) // page))
            refs += [2] + [1] * (len(ids) - 1)
        else:
            j = rng.randrange(prompts)
            n, ids = lens[j], [p for p in table[j] if p >= 0]
            for p in ids:
                refs[p] += 1
        table.append(ids + [-1] * (width - len(ids)))
        lens.append(n)
    # Pages for some steps: each row's places, and what is spare.
    refs += [0] * (rows * ((ahead + page - 1) // page + 1) + spare)
    ws = ops.fork_pages_workspace(len(refs), cuda_device)
    parents, ran_out = list(range(rows)), False
    for step in range(6):
        want_missing = ref.fork([list(r) for r in table], lens, parents, list(refs), page, ahead)[3]
        ran_out |= want_missing > 0
        table, lens, refs = _check_fork(cuda_device, table, lens, parents, refs, page, ahead, ws)
        assert not bool(ws.any()), f"step {step}"
        lens = [min(n + rng.randint(0, ahead), width * page) for n in lens]
        # (Some rows end, many go on from a few, the others from themselves.)
        few = [rng.randrange(rows) for _ in range(20)]
        parents = [rng.choice((i, i, i, rng.choice(few), -1 if step == 2 else i)) for i in range(rows)]
        if step == 3:
            # No page is free but a few.
            free = [p for p, c in enumerate(refs) if c <= 0]
            for p in free[5:]:
                refs[p] = 1
    assert ran_out


# ------------------------------------------------------------------ together
def _inv(hd):
    return 1.0 / (1e6 ** (torch.arange(0, hd, 2, dtype=torch.int64).float() / hd))


def test_rope_paged_kv_slots(cuda_device):
    """A token's angle is its position's, its place its slot."""
    from moeinfra_amd import ops

    dev, nq, nkv, hd, page = cuda_device, 4, 2, 64, 8
    pool = Pool([24, 24], nkv, hd, page, dev, fill=3.0)
    #                    root, two at one position, behind the table, negative slot, padding
    pos = [5, 6, 6, 7, 9, -1]
    slot = [5, 6, 7, 24, -1, 8]
    x = _bf((6, (nq + 2 * nkv) * hd), 4)
    kc0, vc0 = pool.k.clone(), pool.v.clone()
    q_out = torch.full((6, nq * hd), 9.0, dtype=torch.bfloat16, device=dev)
    q, k = ops.rope_paged_kv(x.to(dev), _i32(pos, dev), pool.dev_table, pool.k, pool.v, nq, _inv(hd).to(dev),
                             seq_ids=_i32([1] * 6, dev), want_k=True, slots=_i32(slot, dev), q_out=q_out)
    y, tol = rope(x.view(6, -1, hd)[:, :nq + nkv], [max(p, 0) for p in pos], _inv(hd))
    assert_within(q.view(6, nq, hd)[:5], y[:5, :nq], tol[:5, :nq])
    assert_within(k[:5], y[:5, nq:], tol[:5, nq:])
    assert bool((q[5] == 9.0).all())
    for i in range(3):
        at = int(pool.table[1, slot[i] // page])
        kc0[at, :, slot[i] % page] = k[i]
        vc0[at, :, slot[i] % page] = x.view(6, -1, hd)[i, nq + nkv:].to(dev)
    assert _same(pool.k, kc0) and _same(pool.v, vc0)
    q2, k2 = ops.rope_paged_kv(x.to(dev), _i32(pos, dev), pool.dev_table, pool.k, pool.v, nq, _inv(hd).to(dev),
                               seq_ids=_i32([1] * 6, dev), want_k=True, slots=_i32(pos, dev))
    q3, k3 = ops.rope_paged_kv(x.to(dev), _i32(pos, dev), pool.dev_table, pool.k, pool.v, nq, _inv(hd).to(dev),
                               seq_ids=_i32([1] * 6, dev), want_k=True)
    assert _same(q2[:5], q3[:5]) and _same(k2[:5], k3[:5])


class Toy:
    """An embedding, one layer of attention and a head of random weights."""

    def __init__(self, dev, nq=4, nkv=2, hd=64, vocab=50):
        self.dev, self.nq, self.nkv, self.hd, self.vocab = dev, nq, nkv, hd, vocab
        self.emb, self.head = _bf((vocab, (nq + 2 * nkv) * hd), 60).to(dev), _bf((nq * hd, vocab), 61).to(dev)
        self.inv = _inv(hd).to(dev)

    def keys(self, tokens):
        """(keys, values) that a cache has to hold for these tokens, fp64 with a bound."""
        x = self.emb[tokens].cpu().view(len(tokens), -1, self.hd)
        y, tol = rope(x[:, self.nq:self.nq + self.nkv], list(range(len(tokens))), self.inv.cpu())
        return y, tol, x[:, self.nq + self.nkv:]


def _check_cache(toy, pool_k, pool_v, row, page, tokens):
    n = len(tokens)
    pages = row[[i // page for i in range(n)]].long()
    at = torch.arange(n) % page
    y, tol, v = toy.keys(tokens)
    assert_within(pool_k.cpu()[pages, :, at], y, tol, "keys")
    assert _same(pool_v.cpu()[pages, :, at], v)


def test_trees_together(cuda_device):
    """Steps of checked trees: embedding, attention, acceptance, compaction.  The cache ends with the
    accepted tokens' keys and values, each where and turned as if it had come alone, and the tokens are
    those that attention in 64 bits prefers (or nearly)."""
    from moeinfra_amd import ops

    dev, page = cuda_device, 8
    toy = Toy(dev)
    rng = random.Random(1)
    said = [[rng.randrange(toy.vocab) for _ in range(n)] for n in (1, 5, 17, 9)]   # the last is not cached yet
    B = len(said)
    pool = Pool([200] * B, toy.nkv, toy.hd, page, dev, fill=math.nan)
    ws = ops.paged_tree_attention_workspace(B, toy.nq, toy.nkv, toy.hd, dev)
    prompt = [(b, p) for b in range(B) for p in range(len(said[b]) - 1)]
    ops.rope_paged_kv(toy.emb[[said[b][p] for b, p in prompt]], _i32([p for _, p in prompt], dev), pool.dev_table, pool.k,
                      pool.v, toy.nq, toy.inv, seq_ids=_i32([b for b, _ in prompt], dev))
    cached = [len(s) - 1 for s in said]
    kept = 0
    for step in range(6):
        counts = [rng.randint(1, 40) for _ in range(B)]
        masks = [ref.tree(rng, n) for n in counts]
        drafts = [[said[b][-1]] + [rng.randrange(toy.vocab) for _ in range(counts[b] - 1)] for b in range(B)]
        depth = [[bin(m).count("1") - 1 for m in t] for t in masks]
        cu = _i32(_cuts(counts), dev)
        lens = _i32(cached, dev)
        dm = ref.words([m for t in masks for m in t], dev)
        flat = [x for d in drafts for x in d]

        def forward(flat):
            q, _ = ops.rope_paged_kv(toy.emb[flat], _i32([cached[b] + d for b in range(B) for d in depth[b]], dev),
                                     pool.dev_table, pool.k, pool.v, toy.nq, toy.inv,
                                     seq_ids=_i32([b for b in range(B) for _ in depth[b]], dev),
                                     slots=_i32([cached[b] + i for b in range(B) for i in range(counts[b])], dev))
            o = ops.paged_tree_attention(q.view(len(flat), toy.nq, toy.hd), pool.k, pool.v, pool.dev_table, lens, cu,
                                         masks=dm, workspace=ws)
            return o, (o.reshape(len(flat), -1).float() @ toy.head.float()).argmax(dim=1)

        # Drafts that the model agrees with, on one branch: each node's first child is what it chose.
        for _ in range(4):
            _, targets = forward(flat)
            cuts = _cuts(counts)
            for b in range(B):
                done = set()
                for i in range(1, counts[b]):
                    up = (masks[b][i] & ((1 << i) - 1)).bit_length() - 1
                    if up not in done and rng.random() < 0.8:
                        done.add(up)
                        flat[cuts[b] + i] = int(targets[cuts[b] + up])
        o, targets = forward(flat)
        paths, n, tokens = ops.accept_drafts(targets, torch.tensor(flat, device=dev), cu, masks=dm)
        ops.compact_paged_kv(pool.k, pool.v, pool.dev_table, lens, paths)
        for b in range(B):
            lo, hi = _cuts(counts)[b:b + 2]
            want = ref.accept(targets[lo:hi].tolist(), flat[lo:hi], masks[b])
            assert (int(paths[b]), int(n[b]), int(tokens[b])) == (ref.word(want[0]), want[1], want[2])
            path = [i for i in range(counts[b]) if want[0] >> i & 1]
            said[b] = said[b][:-1] + [flat[lo + i] for i in path] + [want[2]]
            cached[b] += len(path)
            kept += len(path) - 1
            _check_cache(toy, pool.k, pool.v, pool.table[b], page, said[b][:cached[b]])
    assert kept > 20
    # The next token by the operator for one token is the one that the trees' last pass chose.
    q, _ = ops.rope_paged_kv(toy.emb[[s[-1] for s in said]], _i32(cached, dev), pool.dev_table, pool.k, pool.v, toy.nq, toy.inv)
    q = q.view(B, toy.nq, toy.hd)
    one = ops.paged_attention(q, pool.k, pool.v, pool.dev_table, _i32([c + 1 for c in cached], dev))
    tree = ops.paged_tree_attention(q, pool.k, pool.v, pool.dev_table, _i32(cached, dev), _i32(list(range(B + 1)), dev),
                                    workspace=ws)
    # Both are within their bounds of the same values: two outputs' roundings, and the weights'.
    assert float((one.float() - tree.float()).abs().max()) <= 4 * 2.0 ** -8 * float(toy.emb.float().abs().max())


def test_beams_together(cuda_device):
    """Steps of beams: selection, pages forked and copied, embedding, attention.  Each row's pages hold
    the keys and values of its own history, and the totals are the sums of its tokens' log
    probabilities."""
    from moeinfra_amd import ops

    dev, page, W, S = cuda_device, 8, 3, 2
    toy = Toy(dev)
    rng = random.Random(2)
    prompts = [[rng.randrange(toy.vocab) for _ in range(n)] for n in (11, 16)]
    pages, width = 64, 8
    k = torch.full((pages, toy.nkv, page, toy.hd), math.nan, dtype=torch.bfloat16, device=dev)
    v = torch.full_like(k, math.nan)
    # Each prompt in its own row, the searches' other rows still empty.
    table = torch.full((S * W, width), -1, dtype=torch.int32)
    refs = torch.zeros(pages, dtype=torch.int32)
    at = 5
    for s, p in enumerate(prompts):
        for e in range((len(p) + page - 1) // page):
            table[s * W, e] = at
            refs[at] = 1
            at += 7
    table, refs = table.to(dev), refs.to(dev)
    lens = _i32([len(prompts[i // W]) if i % W == 0 else 0 for i in range(S * W)], dev)
    at = [(s * W, i) for s, p in enumerate(prompts) for i in range(len(p))]
    ops.rope_paged_kv(toy.emb[[prompts[r // W][i] for r, i in at]], _i32([i for _, i in at], dev), table, k, v, toy.nq,
                      toy.inv, seq_ids=_i32([r for r, _ in at], dev))
    history = [list(prompts[i // W]) if i % W == 0 else [] for i in range(S * W)]
    scores = torch.full((S, W), -math.inf, device=dev)
    scores[:, 0] = 0.0
    log_p = [0.0] * (S * W)
    logits = _logits(S * W, toy.vocab, 70, torch.float32).to(dev)
    bws, fws = ops.beam_select_workspace(S, W, W, dev), ops.fork_pages_workspace(pages, dev)
    for step in range(20):
        scores, rows, tokens = ops.beam_select(logits, scores, W, workspace=bws)
        lp = torch.log_softmax(logits.double().cpu(), dim=1)
        r, t = rows.flatten().tolist(), tokens.flatten().tolist()
        log_p = [log_p[p] + float(lp[p, x]) for p, x in zip(r, t)]
        # (Each step rounds the total to fp32 once.)
        assert all(abs(a - b) <= (step + 1) * 2.0 ** -24 * abs(b) + 1e-9 for a, b in zip(scores.flatten().tolist(), log_p))
        history = [history[p] for p in r]
        table, lens, copies, missing = ops.fork_pages(table, lens, rows.flatten(), refs, page, workspace=fws)
        ops.copy_pages(k, v, copies)
        assert int(missing) == 0
        q, _ = ops.rope_paged_kv(toy.emb[tokens.flatten()], lens, table, k, v, toy.nq, toy.inv)
        lens += 1
        history = [h + [x] for h, x in zip(history, t)]
        o = ops.paged_attention(q.view(S * W, toy.nq, toy.hd), k, v, table, lens)
        logits = o.reshape(S * W, -1).float() @ toy.head.float() * 0.1
        assert lens.tolist() == [len(h) for h in history]
        for i in range(S * W):
            _check_cache(toy, k, v, table[i].cpu(), page, history[i])
        count = [0] * pages
        for row in table.tolist():
            for p in row:
                if p >= 0:
                    count[p] += 1
        assert refs.tolist() == count
    # All searches end: every page is free again.
    ops.fork_pages(table, lens, _i32([-1] * S * W, dev), refs, page, workspace=fws)
    assert not bool(refs.any())


def test_beam_step_as_documented(cuda_device):
    """The documents' loop body, step after step: each row's pages hold its history, whose length `lens` is."""
    from moeinfra_amd import ops

    begin = "scores, rows, tokens = ops.beam_select("
    found = []
    for name in sorted(glob.glob(os.path.join(REPO, "*.md"))):
        with open(name) as f:
            found += f.read().split(begin)[1:]
    assert len(found) == 1
    lines = (begin + found[0].split("```")[0]).splitlines()
    at = [i for i, line in enumerate(lines) if line.startswith("q, _ =")]
    assert len(at) == 1
    dev, page_size, W, S, pages = cuda_device, 8, 3, 2, 64
    toy = Toy(dev)
    k_all, v_all = (torch.full((1, pages, toy.nkv, page_size, toy.hd), math.nan, dtype=torch.bfloat16, device=dev) for _ in range(2))
    refs = torch.zeros(pages, dtype=torch.int32, device=dev)
    table = torch.full((S * W, 6), -1, dtype=torch.int32, device=dev)
    lens = torch.zeros(S * W, dtype=torch.int32, device=dev)
    scores = torch.zeros((S, W), device=dev)
    env = dict(ops=ops, S=S, W=W, n_q=toy.nq, n_kv=toy.nkv, head_dim=toy.hd, page_size=page_size, inv_freq=toy.inv, table=table,
               lens=lens, refs=refs, scores=scores, k_all=k_all, v_all=v_all, k_cache=k_all[0], v_cache=v_all[0],
               bws=ops.beam_select_workspace(S, W, W, dev), fws=ops.fork_pages_workspace(pages, dev))
    history = [[] for _ in range(S * W)]
    for step in range(20):
        env["logits"] = _logits(S * W, toy.vocab, 200 + step, torch.float32).to(dev)
        exec("\n".join(lines[:at[0]]), env)
        env["qkv"] = toy.emb[env["tokens"].flatten()]
        exec("\n".join(lines[at[0]:]), env)
        history = [history[p] + [t] for p, t in zip(env["rows"].flatten().tolist(), env["tokens"].flatten().tolist())]
        assert env["lens"].tolist() == [step + 1] * (S * W) and int(env["missing"]) == 0
        for i in range(S * W):
            _check_cache(toy, k_all[0], v_all[0], env["table"][i].cpu(), page_size, history[i])
        q = env["q"].view(S * W, toy.nq, toy.hd)
        o = ops.paged_attention(q, k_all[0], v_all[0], env["table"], _i32([step + 1] * (S * W), dev))
        assert _same(o, env["attn"])


def _graph(run):
    """A captured `run`, after a warm-up on the capture's stream."""
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        run()
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = run()
    return g, out


def test_trees_replayed_from_a_graph(cuda_device):
    """A captured check of trees, its inputs changed in place between replays."""
    from moeinfra_amd import ops

    dev, page = cuda_device, 16
    sets = [Trees(dev, lens, counts, 8, 2, 128, page, seed=s, width=100)
            for s, (lens, counts) in enumerate([([700, 3, 0, 1200], [20, 10, 5, 13]), ([5, 900, 0, 40], [1, 0, 40, 7]),
                                                ([0, 0, 1500, 64], [0, 3, 31, 14])])]
    T = max(t.T for t in sets)
    pages = max(t.pool.pages for t in sets)
    q = torch.zeros((T, 8, 128), dtype=torch.bfloat16, device=dev)
    k, v = (torch.zeros((pages, 2, page, 128), dtype=torch.bfloat16, device=dev) for _ in range(2))
    table, lens = torch.full((4, 100), -1, dtype=torch.int32, device=dev), torch.zeros(4, dtype=torch.int32, device=dev)
    cu, masks = torch.zeros(5, dtype=torch.int32, device=dev), torch.zeros(T, dtype=torch.int64, device=dev)
    drafts, targets = (torch.zeros(T, dtype=torch.int64, device=dev) for _ in range(2))
    out, ws = torch.zeros_like(q), ops.paged_tree_attention_workspace(4, 8, 2, 128, dev)

    def step():
        ops.paged_tree_attention(q, k, v, table, lens, cu, masks=masks, out=out, workspace=ws)
        accepted = ops.accept_drafts(targets, drafts, cu, masks=masks)
        ops.compact_paged_kv(k, v, table, lens, accepted[0])
        return accepted

    def fill(t, seed):
        g = torch.Generator().manual_seed(seed)
        q[:t.T] = t.q.to(dev)
        k[:t.pool.pages], v[:t.pool.pages] = t.pool.k, t.pool.v
        table.copy_(t.pool.dev_table)
        lens.copy_(_i32(t.lens, dev))
        cu.copy_(_i32(t.cuts, dev))
        masks[:t.T] = t.dev_masks()
        drafts.copy_(torch.randint(0, 2, (T,), generator=g))
        targets.copy_(torch.randint(0, 2, (T,), generator=g))

    fill(sets[0], 0)
    g, accepted = _graph(step)
    for i in range(6):
        t = sets[i % 3]
        runs = []
        for replayed in (False, True):
            fill(t, i)
            out.zero_()
            if replayed:
                g.replay()
                got = accepted
            else:
                got = step()
            torch.cuda.synchronize()
            # (Bits: places that no token has taken hold NaN.)
            runs.append([x.clone() for x in (*got, *(c.view(torch.int16) for c in (out[:t.T], k, v)))])
            t.check(out)
        assert all(torch.equal(x, y) for x, y in zip(*runs))


def test_beams_replayed_from_a_graph(cuda_device):
    """A captured step of beams that feeds itself: what it writes is what the next replay reads."""
    from moeinfra_amd import ops

    dev, S, W, V, page, pages, width = cuda_device, 5, 4, 5000, 8, 300, 20
    x = torch.zeros((S * W, V), dtype=torch.float32, device=dev)
    scores = torch.zeros((S, W), device=dev)
    table = torch.full((S * W, width), -1, dtype=torch.int32, device=dev)
    table[:, 0] = torch.arange(S * W, dtype=torch.int32) + 4
    lens, refs = torch.full((S * W,), 3, dtype=torch.int32, device=dev), torch.zeros(pages, dtype=torch.int32, device=dev)
    refs[4:4 + S * W] = 1
    k, v = (_bf((2, pages, 2, page, 64), 80 + i).to(dev) for i in range(2))
    state = [scores, table, lens, refs, k, v]
    start = [t.clone() for t in state]
    bws, fws = ops.beam_select_workspace(S, W, W, dev), ops.fork_pages_workspace(pages, dev)

    def step():
        best, rows, tokens = ops.beam_select(x, scores, W, workspace=bws)
        new, n, copies, missing = ops.fork_pages(table, lens, rows.view(-1), refs, page, workspace=fws)
        ops.copy_pages(k, v, copies)
        scores.copy_(best)
        table.copy_(new)
        lens.copy_(n + 1)
        return rows, tokens, missing

    g, out = _graph(step)
    runs = []
    for replayed in (False, True):
        for t, s in zip(state, start):
            t.copy_(s)
        seen = []
        for i in range(10):
            x.copy_(_logits(S * W, V, 90 + i, torch.float32))
            if replayed:
                g.replay()
                got = out
            else:
                got = step()
            torch.cuda.synchronize()
            seen.append([t.clone() for t in (*got, *state)])
        runs.append(seen)
    for a, b in zip(*runs):
        assert all(torch.equal(p, q) for p, q in zip(a, b))
    assert int(runs[0][-1][2]) == 0


def test_operators_on_another_stream(cuda_device):
    from moeinfra_amd import ops

    dev = cuda_device
    t = Trees(dev, [300, 9], [20, 30], 8, 2, 128, 16, seed=13)
    x = _logits(8, 3000, 14, torch.bfloat16).to(dev)
    scores = torch.zeros((2, 4), device=dev)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        out = t.run()
        best = ops.beam_select(x, scores, 8)
    s.synchronize()
    t.check(out)
    _check_beams(best, x, scores, 8)


def test_wrappers_refuse_what_does_not_fit(cuda_device):
    from moeinfra_amd import ops

    dev = cuda_device
    bf = lambda *s: torch.zeros(s, dtype=torch.bfloat16, device=dev)
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32, device=dev)
    i64 = lambda *s: torch.zeros(s, dtype=torch.int64, device=dev)
    f32 = lambda *s: torch.zeros(s, device=dev)
    tree = lambda q=bf(5, 4, 64), k=bf(3, 2, 8, 64), v=bf(3, 2, 8, 64), table=i32(2, 3), lens=i32(2), cu=i32(3), **kw: \
        ops.paged_tree_attention(q, k, v, table, lens, cu, **kw)
    tree()
    for kw, what in ((dict(q=bf(5, 4, 128)), "head dim"), (dict(q=f32(5, 4, 64)), "must be"), (dict(table=i32(3, 3)), "rows of pages"),
                     (dict(lens=i32(3)), "lens"), (dict(cu=i64(3)), "cu_seqlens"), (dict(masks=i64(4)), "masks"),
                     (dict(masks=i32(5)), "masks"), (dict(v=bf(3, 2, 16, 64)), "differ"), (dict(out=bf(5, 4, 32)), "elements"),
                     (dict(workspace=f32(4)), "workspace"), (dict(scaling=math.nan), "NaN")):
        with pytest.raises(ValueError, match=what):
            tree(**kw)
    with pytest.raises(ValueError, match="too small"):
        tree(workspace=torch.zeros(70000, dtype=torch.uint8, device=dev))
    for args, what in (((i64(4), i64(5), i32(2)), "drafts"), ((i32(4), i64(4), i32(2)), "targets"), ((i64(4), i64(4), i32(0)), "cu_seqlens"),
                       ((i64(2, 2), i64(2, 2), i32(2)), "targets")):
        with pytest.raises(ValueError, match=what):
            ops.accept_drafts(*args)
    c = bf(2, 3, 2, 8, 64)
    for args, what in (((c, c.clone(), i32(2, 3), i32(3), i64(2)), "lens"), ((c, c.clone(), i32(2, 3), i32(2), i32(2)), "paths"),
                       ((c, c[:1], i32(2, 3), i32(2), i64(2)), "differ"), ((c, c, i32(2, 3), i32(2), i64(2)), "of their own"),
                       ((c, c.clone(), i32(6), i32(2), i64(2)), "page_table"), ((f32(2, 3, 2, 8, 64), c, i32(2, 3), i32(2), i64(2)), "must be|differ")):
        with pytest.raises(ValueError, match=what):
            ops.compact_paged_kv(*args)
    for args, what in (((c, c.clone(), i32(2, 2)), "copies"), ((c, c.clone(), i64(2, 3)), "copies")):
        with pytest.raises(ValueError, match=what):
            ops.copy_pages(*args)
    for args, what in (((bf(4, 9), f32(2, 3), 2), "scores"), ((bf(4, 9), i32(2, 2), 2), "scores"), ((i32(4, 9), f32(2, 2), 2), "logits"),
                       ((bf(4, 9), f32(2, 2), 0), "sizes"), ((bf(4, 9), f32(2, 2), 65), "sizes"), ((bf(9, 4).t(), f32(2, 2), 2), "contiguous")):
        with pytest.raises(ValueError, match=what):
            ops.beam_select(*args)
    with pytest.raises(ValueError, match="workspace"):
        ops.beam_select(bf(4, 9), f32(2, 2), 2, workspace=torch.zeros(65536, dtype=torch.uint8, device=dev))
    for args, what in (((i32(2, 3), i32(3), i32(2), i32(9), 8), "lens"), ((i32(2, 3), i32(2), i64(2), i32(9), 8), "parents"),
                       ((i32(2, 3), i32(2), i32(2), i64(9), 8), "refs"), ((i32(2, 3), i32(2), i32(2), i32(9), 12), "page size"),
                       ((i32(6), i32(2), i32(2), i32(9), 8), "page_table"), ((i32(2, 3), i32(2), i32(9000), i32(9), 8), "rows")):
        with pytest.raises(ValueError, match=what):
            ops.fork_pages(*args)
    with pytest.raises(ValueError, match="ahead|next tokens"):
        ops.fork_pages(i32(2, 3), i32(2), i32(2), i32(9), 8, ahead=0)
    t = i32(2, 3)
    with pytest.raises(ValueError, match="overlap"):
        ops.fork_pages(t, i32(2), i32(2), i32(9), 8, out=(t, i32(2), i32(2, 3), i32(1)))
    for args, what in ((((1 << 32) + 8, 1), "page_size must fit"), ((8, (1 << 32) + 1), "ahead must fit")):
        with pytest.raises(ValueError, match=what):
            ops.fork_pages(i32(2, 3), i32(2), i32(2), i32(9), args[0], ahead=args[1])
    with pytest.raises(ValueError, match="k must fit"):
        ops.beam_select(bf(4, 9), f32(2, 2), (1 << 32) + 2)
