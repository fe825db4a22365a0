"""The batched serving operators on the GPU against plain 64-bit forms: rotary embedding into a
paged cache, attention over it, attention of packed prompts, choice of tokens."""
from __future__ import annotations

import math

import pytest
import torch

from serving_ref import Pool, assert_within, attention, rope, sample

pytestmark = pytest.mark.gpu


def _bf(shape, seed, std=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * std).to(torch.bfloat16)


def _inv(hd):
    i = torch.arange(0, hd, 2, dtype=torch.int64).float()
    return 1.0 / (1e6 ** (i / hd))


def _same(a, b):
    return torch.equal(a.contiguous().view(torch.int16), b.contiguous().view(torch.int16))


# ------------------------------------------------------------------ rotary embedding, paged cache
@pytest.mark.parametrize("nq,nkv,hd,page,interleaved,padded_rows", [
    (32, 8, 128, 16, False, False), (8, 2, 64, 8, True, True), (3, 1, 16, 32, False, True),
    (4, 4, 256, 64, True, False), (6, 2, 80, 128, False, False)])
def test_rope_paged_kv(cuda_device, nq, nkv, hd, page, interleaved, padded_rows):
    from moeinfra_amd import ops

    dev = cuda_device
    # Prompts of sequences 2 and 0, a token of sequence 1 far away, one at the first place.
    lens = [page + 3, 0, 2 * page, 1]
    places = [(2, p) for p in range(2 * page)] + [(0, p) for p in range(page + 3)] + [(3, 0)]
    T = len(places)
    pool = Pool(lens, nkv, hd, page, dev, seed=1, interleaved=interleaved, fill=7.0)
    x = _bf((T, (nq + 2 * nkv) * hd + (16 if padded_rows else 0)), 2)[:, :(nq + 2 * nkv) * hd]
    inv = _inv(hd)
    kc0, vc0 = pool.k.clone(), pool.v.clone()
    xd = torch.empty((T, x.shape[1] + (16 if padded_rows else 0)), dtype=torch.bfloat16, device=dev)[:, :x.shape[1]]
    xd.copy_(x)
    seq = torch.tensor([s for s, _ in places], dtype=torch.int32, device=dev)
    pos = torch.tensor([p for _, p in places], dtype=torch.int32, device=dev)
    q, k = ops.rope_paged_kv(xd, pos, pool.dev_table, pool.k, pool.v, nq, inv.to(dev), seq_ids=seq, want_k=True)
    heads = x.reshape(T, nq + 2 * nkv, hd)
    y, tol = rope(heads[:, :nq + nkv], pos.cpu(), inv)
    assert_within(q.view(T, nq, hd), y[:, :nq], tol[:, :nq], "q")
    assert_within(k, y[:, nq:], tol[:, nq:], "k")
    # Exactly the new places changed, to k and v.
    for (s, p), kk, vv in zip(places, k, heads[:, nq + nkv:].to(dev)):
        at = int(pool.table[s, p // page])
        kc0[at, :, p % page] = kk
        vc0[at, :, p % page] = vv
    assert _same(pool.k, kc0) and _same(pool.v, vc0)


def test_rope_paged_kv_far_positions(cuda_device):
    from moeinfra_amd import ops

    nq, nkv, hd, page = 4, 2, 128, 64
    pos = [0, 1, 4095, 131071, 1048575, 16777217, 2147483583]
    inv = _inv(hd)
    x = _bf((len(pos), (nq + 2 * nkv) * hd), 3).to(cuda_device)
    pool = Pool([1] * len(pos), nkv, hd, page, cuda_device)  # a table too short for most of them
    q, k = ops.rope_paged_kv(x, torch.tensor(pos, dtype=torch.int32, device=cuda_device), pool.dev_table, pool.k,
                             pool.v, nq, inv.to(cuda_device), want_k=True)
    y, tol = rope(x.cpu().view(len(pos), -1, hd)[:, :nq + nkv], pos, inv)
    assert_within(q.view(len(pos), nq, hd), y[:, :nq], tol[:, :nq])
    assert_within(k, y[:, nq:], tol[:, nq:])


def test_rope_paged_kv_padding_and_missing_pages(cuda_device):
    from moeinfra_amd import ops

    dev, nq, nkv, hd, page = cuda_device, 4, 2, 64, 8
    pool = Pool([page] * 6, nkv, hd, page, dev, fill=3.0)
    table = pool.dev_table.clone()
    table[3, 0] = -1
    table[4, 0] = pool.pages
    #        cached, padding, past the table, page -1, page past the pool, sequences that are not there
    pos = torch.tensor([5, -1, page, 2, 2, 1, 1], dtype=torch.int32, device=dev)
    seq = torch.tensor([0, 1, 2, 3, 4, 6, -1], dtype=torch.int32, device=dev)
    x = _bf((7, (nq + 2 * nkv) * hd), 4).to(dev)
    q_out = torch.full((7, nq * hd), 9.0, dtype=torch.bfloat16, device=dev)
    kc0, vc0 = pool.k.clone(), pool.v.clone()
    q, k = ops.rope_paged_kv(x, pos, table, pool.k, pool.v, nq, _inv(hd).to(dev), seq_ids=seq, q_out=q_out, want_k=True)
    assert q is q_out and bool((q[1] == 9.0).all())
    y, tol = rope(x.cpu().view(7, -1, hd)[:, :nq + nkv], pos.cpu().clamp(min=0), _inv(hd))
    live = [0, 2, 3, 4, 5, 6]
    assert_within(q.view(7, nq, hd)[live], y[live, :nq], tol[live, :nq])
    at = int(pool.table[0, 0])
    kc0[at, :, 5] = k[0]
    vc0[at, :, 5] = x.view(7, -1, hd)[0, nq + nkv:]
    assert _same(pool.k, kc0) and _same(pool.v, vc0)


# ------------------------------------------------------------------ paged attention
def _paged(dev, lens, nq, nkv, hd, page, seed=0, scaling=None, std=1.5, strided=False, workspace="own", garbage=True,
           **kw):
    """Runs paged_attention on random sequences and checks every row; the rows of each last page
    behind the sequence hold NaN."""
    from moeinfra_amd import ops

    pool = Pool(lens, nkv, hd, page, dev, seed=seed, fill=math.nan if garbage else 0.0, **kw)
    ks = [_bf((n, nkv, hd), 100 + seed + i) for i, n in enumerate(lens)]
    vs = [_bf((n, nkv, hd), 200 + seed + i) for i, n in enumerate(lens)]
    for i, (k, v) in enumerate(zip(ks, vs)):
        pool.put(i, k, v)
    q = _bf((len(lens), nq, hd), seed, std)
    qd = q.to(dev)
    if strided:
        qd = torch.full((len(lens), nq + 2, hd), math.nan, dtype=torch.bfloat16, device=dev)[:, :nq]
        qd.copy_(q)
    ws = ops.paged_attention_workspace(len(lens), nq, nkv, hd, dev) if workspace == "own" else workspace
    out = ops.paged_attention(qd, pool.k, pool.v, pool.dev_table, torch.tensor(lens, dtype=torch.int32, device=dev),
                              scaling=scaling, workspace=ws)
    _check_paged(out, q, ks, vs, nkv, hd ** -0.5 if scaling is None else scaling)
    return out, ws


def _check_paged(out, q, ks, vs, nkv, scaling):
    grp = q.shape[1] // nkv
    for i, (k, v) in enumerate(zip(ks, vs)):
        for h in range(nkv):
            want, tol = attention(q[i, h * grp:(h + 1) * grp], k[:, h], v[:, h], scaling)
            assert_within(out[i, h * grp:(h + 1) * grp], want, tol, f"sequence {i} of {k.shape[0]} keys, head {h}")


LENS = [0, 1, 7, 8, 9, 31, 32, 33, 127, 128, 129, 255, 300, 0, 513, 1000]


@pytest.mark.parametrize("nq,nkv,hd,page", [
    (32, 8, 128, 16), (8, 2, 64, 8), (4, 4, 128, 64), (16, 1, 128, 32), (20, 1, 64, 16), (40, 2, 128, 8),
    (8, 4, 256, 128), (17, 1, 256, 16), (3, 3, 64, 4096), (33, 1, 128, 64)])
def test_paged_attention(cuda_device, nq, nkv, hd, page):
    print(f"paged attention {nq}/{nkv} heads of {hd}, pages of {page}", flush=True)
    _paged(cuda_device, LENS, nq, nkv, hd, page, seed=nq + hd, strided=nq % 2 == 0, interleaved=page == 16)


@pytest.mark.parametrize("lens", [[1], [33], [700], [5000], [20000, 3, 0, 900], [257] * 70, [40] * 300])
def test_paged_attention_batches(cuda_device, lens):
    # A lone sequence shared by many workgroups, ragged batches, more sequences than a wave has lanes.
    print(f"paged attention of {len(lens)} sequences", flush=True)
    _paged(cuda_device, lens, 8, 2, 128, 16, seed=len(lens))


@pytest.mark.parametrize("nq,nkv,hd,lens", [
    (8, 2, 64, [1 + 37 * i % 90 for i in range(1100)] + [6000, 0, 2500]),   # more sequences than workgroups at once
    (8, 8, 64, [(i * 7) % 50 for i in range(2100)] + [700]),                # ... than arrival counters: a sequence each
    (32, 8, 128, [0] * 130), (4, 1, 128, [0] * 90 + [9000] + [0] * 200 + [1])])
def test_paged_attention_large_batches(cuda_device, nq, nkv, hd, lens):
    print(f"paged attention of {len(lens)} sequences, {nq}/{nkv} heads of {hd}", flush=True)
    _paged(cuda_device, lens, nq, nkv, hd, 16, seed=7)


def test_paged_attention_shared_pages(cuda_device):
    """Sequences that begin with the same pages (a common prompt), one of them listed twice."""
    from moeinfra_amd import ops

    dev, nq, nkv, hd, page = cuda_device, 8, 2, 128, 32
    pool = Pool([100, 100], nkv, hd, page, dev, seed=15, fill=math.nan)
    k, v = [_bf((100, nkv, hd), s) for s in (150, 151)], [_bf((100, nkv, hd), s) for s in (152, 153)]
    for i in range(2):
        pool.put(i, k[i], v[i])
    table = pool.dev_table[[0, 1, 0, 0]].contiguous()
    table[1, :2] = table[0, :2]     # keys 0 .. 63 are the first one's
    k1, v1 = torch.cat((k[0][:64], k[1][64:])), torch.cat((v[0][:64], v[1][64:]))
    q = _bf((4, nq, hd), 154, 1.5)
    out = ops.paged_attention(q.to(dev), pool.k, pool.v, table, torch.tensor([100, 100, 70, 100], dtype=torch.int32, device=dev))
    _check_paged(out, q, [k[0], k1, k[0][:70], k[0]], [v[0], v1, v[0][:70], v[0]], nkv, hd ** -0.5)


def test_paged_attention_without_workspace_and_reuse(cuda_device):
    from moeinfra_amd import ops

    dev = cuda_device
    a, _ = _paged(dev, [900, 3000, 5], 8, 2, 64, 16, seed=5, workspace=None)
    # One workspace for batches of different sizes and heads, one after the other; same bits.
    ws = ops.paged_attention_workspace(64, 32, 8, 128, dev)
    b, _ = _paged(dev, [900, 3000, 5], 8, 2, 64, 16, seed=5, workspace=ws)
    _paged(dev, [3000] * 9, 32, 8, 128, 16, seed=6, workspace=ws)
    c, _ = _paged(dev, [900, 3000, 5], 8, 2, 64, 16, seed=5, workspace=ws)
    assert _same(a, b) and _same(a, c)
    assert not bool(ws[:65536].any())


@pytest.mark.parametrize("nq,nkv,hd,lens", [
    (32, 8, 128, [9000, 3, 0, 700, 5000]), (40, 2, 128, [6000, 900]), (33, 1, 128, [20000]), (8, 4, 256, [3000] * 5),
    (8, 2, 64, [1 + 37 * i % 900 for i in range(200)] + [9000])])
def test_paged_attention_stays_inside_its_workspace(cuda_device, nq, nkv, hd, lens):
    """Sequences shared by workgroups write inside the workspace of the stated size only, and leave its
    counters zero; the same call gives the same bits."""
    from moeinfra_amd import ops

    print(f"workspace of {nq}/{nkv} heads of {hd}, {len(lens)} sequences", flush=True)
    n = ops.paged_attention_workspace(len(lens), nq, nkv, hd, cuda_device).numel()
    guarded = torch.full((n + 8192,), 0x5a, dtype=torch.uint8, device=cuda_device)
    ws = guarded[4096:4096 + n]
    ws.zero_()
    a, _ = _paged(cuda_device, lens, nq, nkv, hd, 16, seed=nq, workspace=ws)
    assert bool((guarded[:4096] == 0x5a).all()) and bool((guarded[4096 + n:] == 0x5a).all())
    assert not bool(ws[:65536].any())
    b, _ = _paged(cuda_device, lens, nq, nkv, hd, 16, seed=nq, workspace=ws)
    assert _same(a, b)


def test_paged_attention_missing_pages_and_lengths(cuda_device):
    """Pages that the cache does not have weigh nothing; lengths clamp to the table."""
    from moeinfra_amd import ops

    dev, nq, nkv, hd, page = cuda_device, 8, 2, 128, 16
    lens = [100, 100, 64, 64, 40]
    pool = Pool(lens, nkv, hd, page, dev, seed=8, fill=math.nan)
    ks, vs = [_bf((n, nkv, hd), 300 + n + i) for i, n in enumerate(lens)], [_bf((n, nkv, hd), 400 + n + i) for i, n in enumerate(lens)]
    for i, (k, v) in enumerate(zip(ks, vs)):
        pool.put(i, k, v)
    table = pool.dev_table.clone()
    table[0, 2] = -7                                   # keys 32 .. 47
    table[1, 0] = pool.pages                           # keys 0 .. 15
    table[1, 6] = -1                                   # and the last ones
    table[2, :] = -1                                   # all of them
    keep = [[j for j in range(100) if not 32 <= j < 48], list(range(16, 96)), [], list(range(64)), []]
    said = torch.tensor([100, 100, 64, 64, -3], dtype=torch.int32, device=dev)
    q = _bf((5, nq, hd), 9, 1.5)
    out = ops.paged_attention(q.to(dev), pool.k, pool.v, table, said)
    _check_paged(out, q, [k[s] for k, s in zip(ks, keep)], [v[s] for v, s in zip(vs, keep)], nkv, hd ** -0.5)
    # A length past the table: all of its pages.
    full = ops.paged_attention(q[:1].to(dev), pool.k, pool.v, pool.dev_table[3:4, :4].contiguous(),
                               torch.tensor([1 << 30], dtype=torch.int32, device=dev))
    _check_paged(full, q[:1], ks[3:4], vs[3:4], nkv, hd ** -0.5)


def test_paged_attention_extremes(cuda_device):
    """Scores of every size: all equal, far apart, near the largest fp32 value."""
    from moeinfra_amd import ops

    dev, nq, nkv, hd, page, n = cuda_device, 4, 1, 64, 16, 200
    pool = Pool([n], nkv, hd, page, dev, seed=10, fill=math.nan)
    lens = torch.tensor([n], dtype=torch.int32, device=dev)
    v = _bf((n, nkv, hd), 11)
    for big in (0.0, 30.0, 1.5e18):
        k = _bf((n, nkv, hd), 12)
        k[:, 0, 1:] = 0
        q = torch.zeros((1, nq, hd), dtype=torch.bfloat16)
        q[0, :, 0] = torch.tensor([big, -big, big / 2, 1.0])
        if big > 1e9:  # scores up to 3.2e38
            k[:, 0, 0] = torch.linspace(-2.1e20, 2.1e20, n).to(torch.bfloat16)
        pool.put(0, k, v)
        out = ops.paged_attention(q.to(dev), pool.k, pool.v, pool.dev_table, lens, scaling=1.0)
        want, tol = attention(q[0], k[:, 0], v[:, 0], 1.0)
        if big > 1e9:
            # Neighbouring keys are 1e36 apart in score: one key (or several with the same bf16 key)
            # has all the weight, whatever fp32 rounds.
            tol = 2.0 ** -8 * (want.abs() + v.double().abs().amax()) + 0 * tol
            assert not torch.isnan(out).any()
            rows = [0, 1, 2]
            assert_within(out[0, rows], want[rows], tol[rows])
        else:
            assert_within(out[0], want, tol)


@pytest.mark.parametrize("n", [9, 700, 3000])
def test_paged_attention_infinite_values(cuda_device, n):
    """An infinity in a value comes through as one, also from the last of a sequence's parts."""
    from moeinfra_amd import ops

    dev, nq, nkv, hd, page = cuda_device, 4, 2, 128, 16
    pool = Pool([n], nkv, hd, page, dev, seed=18, fill=math.nan)
    k, v, q = _bf((n, nkv, hd), 180), _bf((n, nkv, hd), 181), _bf((1, nq, hd), 182)
    v[n - 1, 0, 5] = math.inf
    v[0, 1, 6] = -math.inf
    pool.put(0, k, v)
    out = ops.paged_attention(q.to(dev), pool.k, pool.v, pool.dev_table, torch.tensor([n], dtype=torch.int32, device=dev),
                              workspace=ops.paged_attention_workspace(1, nq, nkv, hd, dev)).cpu()
    assert (out[0, :2, 5] == math.inf).all() and (out[0, 2:, 6] == -math.inf).all()
    out[0, :2, 5] = out[0, 2:, 6] = v[n - 1, 0, 5] = v[0, 1, 6] = 0.0
    want = [attention(q[0, 2 * h:2 * h + 2], k[:, h], v[:, h], hd ** -0.5) for h in range(2)]
    for h, at in ((0, 5), (1, 6)):
        want[h][0][:, at] = 0.0
        assert_within(out[0, 2 * h:2 * h + 2], *want[h])


def test_paged_attention_offsets_past_32_bits(cuda_device):
    """A pool whose far pages lie more than 2^32 bytes (and 2^31 values) into the tensors."""
    from moeinfra_amd import ops

    dev, nq, nkv, hd, page, n = cuda_device, 32, 8, 128, 128, 300
    pages = (1 << 31) // (nkv * page * hd) + 9
    kc = torch.empty((pages, nkv, page, hd), dtype=torch.bfloat16, device=dev)
    vc = torch.empty_like(kc)
    ids = [pages - 1, 0, pages - 2]
    k, v, q = _bf((n, nkv, hd), 20), _bf((n, nkv, hd), 21), _bf((1, nq, hd), 22, 1.5)
    for c, at in enumerate(ids):
        m = min(page, n - c * page)
        kc[at, :, :m] = k[c * page:c * page + m].to(dev).transpose(0, 1)
        vc[at, :, :m] = v[c * page:c * page + m].to(dev).transpose(0, 1)
    table = torch.tensor([ids], dtype=torch.int32, device=dev)
    out = ops.paged_attention(q.to(dev), kc, vc, table, torch.tensor([n], dtype=torch.int32, device=dev))
    _check_paged(out, q, [k], [v], nkv, hd ** -0.5)
    # ... and a token written there.
    x = _bf((1, (nq + 2 * nkv) * hd), 23).to(dev)
    pos = torch.tensor([n], dtype=torch.int32, device=dev)
    _, kr = ops.rope_paged_kv(x, pos, table, kc, vc, nq, _inv(hd).to(dev), want_k=True)
    assert _same(kc[ids[2], :, n % page], kr[0])
    assert _same(vc[ids[2], :, n % page], x.view(1, -1, hd)[0, nq + nkv:])


# ------------------------------------------------------------------ packed attention
def _packed(dev, lens, nq, nkv, hd, seed=0, scaling=None, std=1.5, gap=0, strided=True, change=None):
    """Runs packed_attention on sequences that start behind `gap` tokens and end `gap` before the
    last one, and checks every row; rows outside hold NaN and are left alone."""
    from moeinfra_amd import ops

    cuts = [gap]
    for n in lens:
        cuts.append(cuts[-1] + n)
    T = cuts[-1] + gap
    q, k, v = _bf((T, nq, hd), seed, std), _bf((T, nkv, hd), seed + 1), _bf((T, nkv, hd), seed + 2)
    if change is not None:
        change(q, k, v, cuts)
    outside = torch.ones(T, dtype=torch.bool)
    outside[cuts[0]:cuts[-1]] = False
    for t in (q, k, v):
        t[outside] = math.nan
    dq, dk, dv = q.to(dev), k.to(dev), v.to(dev)
    if strided:  # slices of one projection's output
        row = torch.cat((q.reshape(T, -1), k.reshape(T, -1), v.reshape(T, -1)), dim=1).to(dev)
        dq = row[:, :nq * hd].view(T, nq, hd)
        dk = row[:, nq * hd:(nq + nkv) * hd].view(T, nkv, hd)
        dv = row[:, (nq + nkv) * hd:].view(T, nkv, hd)
    out = torch.full((T, nq, hd), 5.0, dtype=torch.bfloat16, device=dev)
    s = hd ** -0.5 if scaling is None else scaling
    ops.packed_attention(dq, dk, dv, torch.tensor(cuts, dtype=torch.int32, device=dev), scaling=scaling, out=out)
    assert bool((out[outside.to(dev)] == 5.0).all())
    return out, q, k, v, cuts, s


def _check_packed(out, q, k, v, cuts, scaling, rows=None):
    nq, nkv = q.shape[1], k.shape[1]
    for a, b in zip(cuts, cuts[1:]):
        n = b - a
        if n == 0:
            continue
        seen = torch.ones((n, n), dtype=torch.bool).tril()
        for h in range(nq):
            kh = h // (nq // nkv)
            want, tol = attention(q[a:b, h], k[a:b, kh], v[a:b, kh], scaling, seen)
            assert_within(out[a:b, h], want, tol, f"tokens {a} .. {b - 1}, head {h}")


@pytest.mark.parametrize("nq,nkv,hd", [(32, 8, 128), (8, 2, 64), (4, 4, 128), (6, 2, 256), (16, 1, 64), (5, 1, 128),
                                       (3, 3, 256), (40, 1, 64)])
def test_packed_attention(cuda_device, nq, nkv, hd):
    print(f"packed attention {nq}/{nkv} heads of {hd}", flush=True)
    _check_packed(*_packed(cuda_device, [1, 0, 7, 64, 65, 0, 200, 1, 130], nq, nkv, hd, seed=nq, gap=3,
                           strided=nq % 2 == 0))


@pytest.mark.parametrize("lens", [[1], [2], [31], [257], [1500], [3] * 150, [0, 0, 5, 0], [700, 1, 900]])
def test_packed_attention_batches(cuda_device, lens):
    print(f"packed attention of {len(lens)} sequences", flush=True)
    _check_packed(*_packed(cuda_device, lens, 4, 2, 128, seed=len(lens)))


@pytest.mark.parametrize("count", [31, 32, 33, 63, 64, 65, 130])
def test_packed_attention_many_sequences(cuda_device, count):
    """Batches around the numbers of sequences where the search for a workgroup's tile changes, with
    equal, empty and long ones among them."""
    print(f"packed attention of {count} sequences", flush=True)
    lens = [(0, 1, 40, 40, 7, 170)[(i * i + i // 5) % 6] for i in range(count)]
    _check_packed(*_packed(cuda_device, lens, 4, 2, 64, seed=count, gap=1))


@pytest.mark.parametrize("count,nq,nkv,hd", [(4097, 4, 4, 64), (70000, 4, 1, 128), (1 << 20, 1, 1, 64)])
def test_packed_attention_large_batches(cuda_device, count, nq, nkv, hd):
    """Batches of up to the largest number of sequences: most of one token, whose result is its own
    values, some empty, a few of several tokens (the first and the last among them)."""
    from moeinfra_amd import ops

    print(f"packed attention of {count} sequences", flush=True)
    lens = torch.ones(count, dtype=torch.int64)
    lens[5::17] = 0
    longer = [0, 1, 64, 65, 4095, 4096, count // 2, count - 1]
    lens[longer] = torch.tensor([150, 3, 33, 129, 2, 200, 65, 40])
    cuts = torch.cat((torch.tensor([2]), 2 + lens.cumsum(0)))
    T = int(cuts[-1]) + 3
    q, k, v = (torch.randn((T, n, hd), generator=torch.Generator().manual_seed(9 + n + i)).to(torch.bfloat16)
               for i, n in enumerate((nq, nkv, nkv)))
    out = torch.full((T, nq, hd), 5.0, dtype=torch.bfloat16, device=cuda_device)
    ops.packed_attention(*(t.to(cuda_device) for t in (q, k, v)), cuts.to(torch.int32).to(cuda_device), out=out)
    out = out.cpu()
    want = v.repeat_interleave(nq // nkv, dim=1)
    want[:2] = want[T - 3:] = 5.0
    for i in longer:
        a, b = int(cuts[i]), int(cuts[i + 1])
        _check_packed(out, q, k, v, [a, b], hd ** -0.5)
        want[a:b] = out[a:b]
    assert _same(out, want)


@pytest.mark.parametrize("count", [40, 3000])
def test_packed_attention_mostly_empty_batches(cuda_device, count):
    """More sequences than tokens."""
    print(f"packed attention of {count} sequences, most of them empty", flush=True)
    lens = [0] * count
    lens[0], lens[count // 2], lens[count - 3] = 1, 5, 20
    _check_packed(*_packed(cuda_device, lens, 8, 2, 128, seed=count, gap=1))


def test_packed_attention_wide_workgroups(cuda_device):
    # Enough rows for the 8-wave workgroups: 32 heads, 64 and 128 dims.
    for hd in (64, 128):
        print(f"packed attention, wide, {hd}", flush=True)
        _check_packed(*_packed(cuda_device, [700, 33, 1400], 32, 8, hd, seed=hd))


@pytest.mark.parametrize("lens,nq,nkv,hd", [([1900, 2300], 16, 16, 128), ([300, 280], 4, 1, 64), ([900], 6, 2, 256),
                                            ([600, 599, 3], 8, 1, 128)])
def test_packed_attention_kernels(cuda_device, lens, nq, nkv, hd):
    # Many rows of 16 KV heads, two key groups (few rows), the large head dim.
    print(f"packed attention {lens} {nq}/{nkv} heads of {hd}", flush=True)
    _check_packed(*_packed(cuda_device, lens, nq, nkv, hd, seed=hd))


@pytest.mark.parametrize("lens,nq,nkv", [([1030], 128, 128), ([1500, 0, 1900], 64, 64), ([2100], 64, 32), ([2051], 72, 8)])
def test_packed_attention_256_rows(cuda_device, lens, nq, nkv):
    """Long sequences of enough heads that workgroups take 256 rows: of a token, a token's two heads, nine."""
    print(f"packed attention {lens} {nq}/{nkv} heads, 256 rows", flush=True)
    _check_packed(*_packed(cuda_device, lens, nq, nkv, 128, seed=nq + nkv, gap=2))


@pytest.mark.parametrize("lens,nq,nkv", [([2100], 64, 16), ([4100], 32, 8)])
def test_packed_attention_256_rows_of_groups_of_four(cuda_device, lens, nq, nkv):
    """... and of four heads of 64 tokens; the same call gives the same bits."""
    from moeinfra_amd import ops

    print(f"packed attention {lens} {nq}/{nkv} heads, 256 rows", flush=True)
    out, q, k, v, cuts, s = _packed(cuda_device, lens, nq, nkv, 128, seed=nq)
    again = ops.packed_attention(*(t.to(cuda_device) for t in (q, k, v)),
                                 torch.tensor(cuts, dtype=torch.int32, device=cuda_device))
    assert _same(out, again)
    n = lens[0]
    seen = torch.ones((n, n), dtype=torch.bool).tril()
    for h in (0, nq // 2 + 1, nq - 1):
        want, tol = attention(q[:, h], k[:, h // 4], v[:, h // 4], s, seen)
        assert_within(out[:, h], want, tol, f"head {h}")


def test_packed_attention_256_rows_infinities(cuda_device):
    """... with an infinity and a NaN that some of a workgroup's rows see."""
    n, nq = 1030, 128

    def spoil(q, k, v, cuts):
        v[cuts[0] + 700, 3, 9] = math.inf
        v[cuts[0] + 1000, 3, 10] = math.nan

    out, q, k, v, cuts, s = _packed(cuda_device, [n], nq, nq, 128, seed=16, gap=1, change=spoil)
    o = out[1:1 + n, 3].float().cpu()
    assert torch.isinf(o[700:, 9]).all() and torch.isnan(o[1000:, 10]).all()
    v[1 + 700, 3, 9] = v[1 + 1000, 3, 10] = 0
    want, tol = attention(q[1:1 + n, 3], k[1:1 + n, 3], v[1:1 + n, 3], s, torch.ones((n, n), dtype=torch.bool).tril())
    keep = torch.ones((n, 128), dtype=torch.bool)
    keep[700:, 9] = False
    keep[1000:, 10] = False
    assert torch.isfinite(o[keep]).all()
    assert_within(torch.where(keep, o, 0.0), torch.where(keep, want, 0.0), tol)


def test_packed_attention_scalings(cuda_device):
    for scaling in (1.0, -0.125, 0.0, 2.5):
        print(f"scaling {scaling}", flush=True)
        _check_packed(*_packed(cuda_device, [70, 129], 4, 2, 64, seed=3, scaling=scaling, std=0.5))


def test_packed_attention_large_scores(cuda_device):
    """Scores up to 3e38, where a product with log2(e) would overflow."""
    def big(q, k, v, cuts):
        q[:], k[:] = 0, 0
        q[:, :, 0] = 1.5e18
        k[:, :, 0] = torch.linspace(-2e20, 2e20, k.shape[0]).to(torch.bfloat16)[:, None]

    for scaling in (1.0, 0.6):
        out, q, k, v, cuts, s = _packed(cuda_device, [90], 2, 1, 64, seed=4, scaling=scaling, change=big)
        # Keys are bf16 steps apart: the newest (of equal ones, all) has the weight.
        for t in range(90):
            same = (k[:t + 1, 0, 0] == k[t, 0, 0]).nonzero()[:, 0]
            want = v[same, 0].double().mean(0)
            tol = 2.0 ** -7 * v[same, 0].double().abs().mean(0) + 1e-6
            assert_within(out[t], want.expand(2, -1), tol.expand(2, -1), f"token {t}")


def test_packed_attention_infinities_stay_with_the_rows_that_see_them(cuda_device):
    """An infinity or NaN in a value reaches the tokens from its own on, no earlier one and no other
    sequence."""
    lens = [100, 150, 40]

    def spoil(q, k, v, cuts):
        v[cuts[1] + 70, 0, 5] = math.inf
        v[cuts[1] + 75, 1, 6] = math.nan
        v[cuts[2], :, :] = math.nan

    for hd in (64, 128, 256):
        print(f"infinities, {hd}", flush=True)
        out, q, k, v, cuts, s = _packed(cuda_device, lens, 4, 2, hd, seed=6, change=spoil)
        o = out.float().cpu()
        assert torch.isinf(o[cuts[1] + 70:cuts[2], :2, 5]).all()
        assert torch.isnan(o[cuts[1] + 75:cuts[2], 2:, 6]).all()
        assert torch.isnan(o[cuts[2]:cuts[3]]).all()
        clean = lambda t: torch.where(t.isfinite(), t, 0.0).to(torch.bfloat16)
        seen = torch.ones((150, 150), dtype=torch.bool).tril()
        for h in range(4):
            want, tol = attention(q[cuts[1]:cuts[2], h], k[cuts[1]:cuts[2], h // 2], clean(v[cuts[1]:cuts[2], h // 2]), s, seen)
            keep = torch.ones((150, hd), dtype=torch.bool)
            keep[70 if h < 2 else 75:, 5 if h < 2 else 6] = False
            got = o[cuts[1]:cuts[2], h]
            assert torch.isfinite(got[keep]).all()
            assert_within(torch.where(keep, got, 0.0), torch.where(keep, want, 0.0), tol)
        _check_packed(out, q, k, v, cuts[:2], s)


@pytest.mark.parametrize("lens,nq,nkv,hd", [
    ([1, 9, 17, 0, 33, 65, 129, 8, 64], 8, 2, 128),     # 4 heads a group: 8 n + 1
    ([1, 9, 17, 65], 4, 1, 64), ([1, 9, 33, 41], 4, 1, 256),
    ([1, 33, 65, 97, 32], 2, 2, 128), ([1, 33, 65], 3, 3, 256),      # 1: 32 n + 1
    ([1, 5, 9, 61, 64, 65], 8, 1, 64), ([2, 1, 40, 70], 40, 1, 128),  # 8: 4 n + 1; 40: a token's rows in two waves
    ([257], 4, 1, 64), ([257, 289], 4, 4, 128), ([273, 277], 16, 2, 128),  # two key groups
    ([1025], 128, 128, 128), ([2057], 64, 16, 128)])     # 256 rows
def test_packed_attention_infinities_of_last_tokens(cuda_device, lens, nq, nkv, hd):
    """An infinity in the last token's values is that token's result and no other's, whatever the
    number of rows that the sequence leaves for its last workgroup and wave."""
    print(f"infinities of last tokens, {lens} {nq}/{nkv} heads of {hd}", flush=True)

    def spoil(q, k, v, cuts):
        for a, b in zip(cuts, cuts[1:]):
            if b > a:
                v[b - 1, 0, 5] = math.inf
                v[b - 1, nkv - 1, hd - 1] = -math.inf

    out, q, k, v, cuts, s = _packed(cuda_device, lens, nq, nkv, hd, seed=nq + hd, gap=1, change=spoil)
    o, grp = out.float().cpu(), nq // nkv
    for a, b in zip(cuts, cuts[1:]):
        if b == a:
            continue
        for kh, d, x in ((0, 5, math.inf), (nkv - 1, hd - 1, -math.inf)):
            rows = o[b - 1, kh * grp:(kh + 1) * grp, d]
            assert bool((rows == x).all()), f"tokens {a} .. {b - 1}: {rows}"
            o[b - 1, kh * grp:(kh + 1) * grp, d] = 0
            v[b - 1, kh, d] = 0
    # The others', against the same values with zeros in those places (which are left out).
    for a, b in zip(cuts, cuts[1:]):
        n = b - a
        seen = torch.ones((n, n), dtype=torch.bool).tril()
        for h in sorted({0, nq // 2, nq - 1}) if n > 0 else ():
            want, tol = attention(q[a:b, h], k[a:b, h // grp], v[a:b, h // grp], s, seen)
            for kh, d in ((0, 5), (nkv - 1, hd - 1)):
                if h // grp == kh:
                    want[n - 1, d] = 0
            assert_within(o[a:b, h], want, tol, f"tokens {a} .. {b - 1}, head {h}")


@pytest.mark.parametrize("lens,nq,nkv,hd", [([300], 4, 2, 64), ([300, 310], 4, 2, 128), ([130, 300, 70], 4, 2, 256),
                                            ([130, 300, 70], 8, 2, 128)])
def test_packed_attention_nan_values_from_a_token_on(cuda_device, lens, nq, nkv, hd):
    """Values that are NaN from a token on, all of one head's (a model that has come apart): what sees
    them is NaN, the tokens before and the other head are right."""
    print(f"NaN from a token on, {lens} {nq}/{nkv} heads of {hd}", flush=True)
    at = [min(100 + 7 * i, n - 1) for i, n in enumerate(lens)]

    def spoil(q, k, v, cuts):
        for a, b, i in zip(cuts, cuts[1:], at):
            v[a + i:b, 1] = math.nan

    out, q, k, v, cuts, s = _packed(cuda_device, lens, nq, nkv, hd, seed=hd, change=spoil)
    o, grp = out.float().cpu(), nq // nkv
    for a, b, i in zip(cuts, cuts[1:], at):
        assert torch.isnan(o[a + i:b, grp:]).all()
        for h in range(nq):
            n = b - a if h < grp else i
            want, tol = attention(q[a:a + n, h], k[a:a + n, h // grp], v[a:a + n, h // grp], s,
                                  torch.ones((n, n), dtype=torch.bool).tril())
            assert_within(o[a:a + n, h], want, tol, f"tokens {a} .. {a + n - 1}, head {h}")


@pytest.mark.parametrize("n,nq,nkv,hd", [(300, 2, 1, 64), (500, 4, 4, 128), (200, 2, 1, 256)])
def test_packed_attention_large_scores_of_long_rows(cuda_device, n, nq, nkv, hd):
    """Scores up to 3e38 in rows of two key groups, and of 256 dims, and an infinity in the last
    token's values."""
    print(f"large scores, {n} tokens, {nq}/{nkv} heads of {hd}", flush=True)

    def big(q, k, v, cuts):
        q[:], k[:] = 0, 0
        q[:, :, 0] = 1.5e18
        k[:, :, 0] = torch.linspace(-2e20, 2e20, n).to(torch.bfloat16)[:, None]
        v[n - 1, 0, 3] = math.inf

    out, q, k, v, cuts, s = _packed(cuda_device, [n], nq, nkv, hd, seed=4, scaling=1.0, change=big)
    assert bool((out[n - 1, :nq // nkv, 3] == math.inf).all())
    out[n - 1, :nq // nkv, 3] = v[n - 1, 0, 3] = 0
    for t in range(n):
        # The newest key (of equal ones, all) has the weight: those are 2^60 and more apart.
        same = (k[:t + 1, 0, 0] == k[t, 0, 0]).nonzero()[:, 0]
        for h in range(nq):
            want = v[same, h // (nq // nkv)].double().mean(0)
            tol = 2.0 ** -7 * v[same, h // (nq // nkv)].double().abs().mean(0) + 1e-6
            if t == n - 1 and h < nq // nkv:
                want[3] = 0  # (checked above)
            assert_within(out[t, h], want, tol, f"token {t}, head {h}")


# ------------------------------------------------------------------ choice of tokens
SETTINGS = [dict(), dict(temperature=0.0), dict(top_k=1), dict(top_k=40), dict(top_p=0.9), dict(min_p=0.05),
            dict(temperature=0.7, top_k=50, top_p=0.9), dict(temperature=1.5, top_p=0.5, min_p=0.02),
            dict(temperature=3.0, top_k=700, top_p=0.95, min_p=0.001), dict(temperature=0.01, top_p=0.99),
            dict(top_k=10 ** 6, top_p=1.0), dict(min_p=1.0), dict(top_p=1e-6)]


def _sampled(dev, x, u, **settings):
    """sample_tokens on rows x (CPU) against the sorted form, row by row."""
    from moeinfra_amd import ops

    got = ops.sample_tokens(x.to(dev), u.to(dev), **settings).cpu().tolist()
    want = [sample(row, float(r), **settings) for row, r in zip(x, u)]
    assert got == want, settings
    return got


def _logits(rows, vocab, seed, dtype, peaks=True):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((rows, vocab), generator=g) * 2.0
    if peaks:
        x = x + torch.where(torch.rand((rows, vocab), generator=g) < 0.003, 9.0 * torch.rand((rows, vocab), generator=g), 0.0)
    return x.to(dtype), torch.rand((rows,), generator=g)


@pytest.mark.parametrize("vocab,dtype", [(32000, torch.bfloat16), (32000, torch.float32), (50257, torch.bfloat16),
                                         (131072, torch.bfloat16), (777, torch.float32), (8, torch.bfloat16)])
def test_sample_tokens(cuda_device, vocab, dtype):
    for i, settings in enumerate(SETTINGS):
        print(f"sample {vocab} {dtype} {settings}", flush=True)
        x, u = _logits(6, vocab, 10 * i + vocab, dtype, peaks=i % 2 == 0)
        _sampled(cuda_device, x, u, **settings)


@pytest.mark.parametrize("vocab", [1, 2, 7, 9, 63, 1023, 8193])
def test_sample_tokens_odd_sizes_and_strides(cuda_device, vocab):
    """Rows that start at any element of their 16 bytes, with NaN between them."""
    for dtype in (torch.bfloat16, torch.float32):
        for lead in (0, 1, 3):
            wide = torch.full((5, vocab + 2 * lead + 1), math.nan, dtype=dtype)
            x, u = _logits(5, vocab, vocab + lead, dtype)
            wide[:, lead:lead + vocab] = x
            from moeinfra_amd import ops

            got = ops.sample_tokens(wide.to(cuda_device)[:, lead:lead + vocab], u.to(cuda_device), temperature=1.3,
                                    top_p=0.8)
            assert got.cpu().tolist() == [sample(r, float(v), temperature=1.3, top_p=0.8) for r, v in zip(x, u)]


@pytest.mark.parametrize("vocab,dtype,lead", [
    (32768, torch.float32, 0), (32768, torch.float32, 1), (32769, torch.float32, 0), (40000, torch.float32, 3),
    (262147, torch.float32, 0), (32768, torch.bfloat16, 0), (32768, torch.bfloat16, 5), (300001, torch.bfloat16, 1),
    (1 << 20, torch.bfloat16, 0)])
def test_sample_tokens_long_rows(cuda_device, vocab, dtype, lead):
    """Rows that just fit a workgroup's registers, that just do not, and of the largest vocabulary."""
    from moeinfra_amd import ops

    x, u = _logits(3, vocab, vocab + lead, dtype)
    wide = torch.full((3, vocab + 2 * lead), math.nan, dtype=dtype)
    wide[:, lead:lead + vocab] = x
    d = wide.to(cuda_device)[:, lead:lead + vocab]
    for settings in (dict(), dict(temperature=0.0), dict(top_k=50, top_p=0.9), dict(top_p=0.7, min_p=0.001),
                     dict(temperature=1.4, top_k=20000)):
        print(f"sample {vocab} {dtype} {settings}", flush=True)
        got = ops.sample_tokens(d, u.to(cuda_device), **settings).cpu().tolist()
        assert got == [sample(r, float(v), **settings) for r, v in zip(x, u)], settings


def test_sample_tokens_settings_per_row(cuda_device):
    from moeinfra_amd import ops

    dev = cuda_device
    x, u = _logits(64, 5000, 31, torch.float32)
    g = torch.Generator().manual_seed(32)
    pick = lambda values, t: torch.tensor(values, dtype=t)[torch.randint(len(values), (64,), generator=g)]
    par = dict(temperature=pick([0.0, 0.4, 1.0, 2.0], torch.float32), top_k=pick([-1, 0, 1, 30, 900], torch.int32),
               top_p=pick([0.3, 0.9, 1.0, 2.0], torch.float32), min_p=pick([0.0, 0.01, 0.3], torch.float32))
    got = ops.sample_tokens(x.to(dev), u.to(dev), **{n: v.to(dev) for n, v in par.items()})
    want = [sample(x[i], float(u[i]), **{n: v[i].item() for n, v in par.items()}) for i in range(64)]
    assert got.cpu().tolist() == want


def test_sample_tokens_equal_logits(cuda_device):
    """Ties go to the lowest index: of equal logits the first are kept."""
    x = torch.zeros((9, 1000))
    u = torch.tensor([0.0, 0.1, 0.25, 0.5, 0.75, 0.9, 0.99, 0.999, 0.9999999])
    assert _sampled(cuda_device, x, u, top_k=10)[-1] == 9
    assert _sampled(cuda_device, x, u, top_p=0.25)[-1] == 249
    assert _sampled(cuda_device, x, u)[-1] == 999
    assert _sampled(cuda_device, x, u, top_k=400, top_p=0.5)[-1] == 199
    # Two levels, both zeros (equal), many of the lower one.
    x = torch.full((9, 4099), -1.0)
    x[:, 5::7] = 0.0
    x[:, 12::14] = -0.0
    for settings in (dict(top_k=3), dict(top_k=600), dict(top_p=0.2), dict(top_p=0.6), dict(min_p=0.9)):
        _sampled(cuda_device, x, u, **settings)
    _sampled(cuda_device, x.to(torch.bfloat16), u, top_k=587, top_p=0.999)


def test_sample_tokens_close_and_far_logits(cuda_device):
    """Values that differ in their last bits, in every exponent, and beyond any weight."""
    g = torch.Generator().manual_seed(40)
    u = torch.rand((6,), generator=g)
    near = 1.0 + torch.randint(0, 5000, (6, 20000), generator=g).float() * 2.0 ** -23
    far = torch.randn((6, 20000), generator=g) * 10.0 ** (torch.rand((6, 20000), generator=g) * 70 - 35)
    lowest = torch.full((6, 20000), torch.finfo(torch.float32).min)
    lowest[:, 100:103] = 3.0
    for x in (near, far, lowest, -near):
        for settings in (dict(top_k=77), dict(top_k=9000), dict(top_p=0.7), dict(temperature=1e-4, top_p=0.7),
                         dict(temperature=1e30, top_k=5000, top_p=0.5), dict(top_k=2, min_p=0.5)):
            _sampled(cuda_device, x, u, **settings)


def test_sample_tokens_values_without_a_bin(cuda_device):
    """Logits of tiny and large magnitude, and more fp32 logits in one bin (equal ones, and different
    ones that share their upper 16 bits) than are ranked at once."""
    g = torch.Generator().manual_seed(45)
    u = torch.rand((6,), generator=g)
    base = torch.randn((6, 9000), generator=g) * 2.0
    tiny, large, low, shared, equal = (base.clone() for _ in range(5))
    tiny[:, ::7] = 1e-12 * torch.randn((6, 1286), generator=g)
    large[:, ::9] += 300.0
    low[:, ::3] = -400.0 + torch.randn((6, 3000), generator=g)
    shared[:, :4000] = 5.0 + torch.rand((6, 4000), generator=g) * 2.0 ** -7
    equal[:, 3000:] = 1.25
    for x in (tiny, large, low, shared, equal):
        for settings in (dict(top_k=40), dict(top_k=3500), dict(top_p=0.7), dict(temperature=20.0, top_k=8000, top_p=0.97),
                         dict(temperature=0.05, top_p=0.9), dict(min_p=0.2)):
            _sampled(cuda_device, x, u, **settings)
            _sampled(cuda_device, x.to(torch.bfloat16), u, **settings)


def test_sample_tokens_many_fp32_rows(cuda_device):
    """Enough rows that the bin where top-p ends is guessed wrong, by one and by more: lopsided bins
    (values at one end of their 16-bit prefix), and a few heavy ones."""
    V = 4000
    x, u = _logits(96, V, 90, torch.float32)
    low = (x.view(torch.int32) & ~0xffff).view(torch.float32)            # all at their bin's small end
    x[:32] = low[:32]
    x[32:64] = (low.view(torch.int32) | 0xfff0).view(torch.float32)[32:64]
    x[64:70, 17::400] = 9.0 + torch.arange(10) * 2.0 ** -9              # ten that share two bins
    for settings in (dict(top_p=0.9), dict(top_p=0.35), dict(temperature=0.2, top_p=0.8), dict(top_k=900, top_p=0.97),
                     dict(top_p=0.6, min_p=0.002), dict(temperature=0.03, top_p=0.5)):
        _sampled(cuda_device, x, u, **settings)


def test_sample_tokens_masked_rows(cuda_device):
    """-inf and NaN are never drawn; rows of nothing else give -1; +inf takes all."""
    V = 3000
    x = torch.randn((8, V), generator=torch.Generator().manual_seed(50))
    x[0, :] = -math.inf
    x[1, :] = math.nan
    x[2, :] = -math.inf
    x[2, 1234] = -5.0
    x[3, ::2] = math.nan
    x[4, 1:] = -math.inf
    x[5, [7, 900, 2999]] = math.inf
    x[6, :2000] = torch.finfo(torch.float32).min
    x[7, :] = torch.finfo(torch.float32).min
    u = torch.linspace(0.05, 0.95, 8)
    for settings in (dict(), dict(top_k=2), dict(top_p=0.5), dict(temperature=0.0), dict(temperature=0.5, top_k=20, top_p=0.8, min_p=0.1)):
        got = _sampled(cuda_device, x, u, **settings)
        assert got[:3] == [-1, -1, 1234] and got[4] == 0 and got[5] in (7, 900, 2999)
        _sampled(cuda_device, x.to(torch.bfloat16), u, **settings)


def test_sample_tokens_random_numbers_at_the_ends(cuda_device):
    """u of 0 and next to 1, and numbers outside [0, 1), which take the first and the last kept."""
    from moeinfra_amd import ops

    x = torch.randn((1, 4000), generator=torch.Generator().manual_seed(51))
    kept = torch.sort(x[0], descending=True).indices[:25].sort().values
    for u, at in ((0.0, 0), (1.0 - 2.0 ** -24, 24), (1.0, 24), (7.5, 24), (-1.0, 0), (math.nan, 0)):
        got = ops.sample_tokens(x.to(cuda_device), torch.tensor([u], device=cuda_device), top_k=25)
        assert int(got) == int(kept[at])


# ------------------------------------------------------------------ together
class _Server:
    """A layer's attention of a batch of sequences: prompts in one packed pass, then steps, and a
    choice of tokens; the state that a server keeps."""

    def __init__(self, dev, lens, steps, nq=8, nkv=2, hd=64, page=16, vocab=500):
        from moeinfra_amd import ops

        self.dev, self.nq, self.nkv, self.hd, self.lens = dev, nq, nkv, hd, list(lens)
        self.pool = Pool([n + steps for n in lens], nkv, hd, page, dev, seed=60, fill=math.nan)
        self.inv = _inv(hd).to(dev)
        self.ws = ops.paged_attention_workspace(len(lens), nq, nkv, hd, dev)
        self.pos = torch.tensor(lens, dtype=torch.int32, device=dev)       # of the next token; -1: padding
        self.seen = self.pos + 1
        g = torch.Generator().manual_seed(61)
        self.embed = (torch.randn((vocab, (nq + 2 * nkv) * hd), generator=g)).to(torch.bfloat16).to(dev)
        self.head = (torch.randn((nq * hd, vocab), generator=g) * 0.1).to(torch.bfloat16).to(dev)
        self.tok = torch.zeros((len(lens),), dtype=torch.int64, device=dev)
        self.u = torch.zeros((len(lens),), device=dev)
        self.x = torch.empty((len(lens), self.embed.shape[1]), dtype=torch.bfloat16, device=dev)
        self.attn = torch.empty((len(lens), nq, hd), dtype=torch.bfloat16, device=dev)

    def prompts(self, qkv):
        from moeinfra_amd import ops

        lens = self.lens
        seq = torch.tensor([i for i, n in enumerate(lens) for _ in range(n)], dtype=torch.int32, device=self.dev)
        pos = torch.tensor([p for n in lens for p in range(n)], dtype=torch.int32, device=self.dev)
        cu = torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32, device=self.dev)
        q, k = ops.rope_paged_kv(qkv, pos, self.pool.dev_table, self.pool.k, self.pool.v, self.nq, self.inv,
                                 seq_ids=seq, want_k=True)
        v = qkv[:, (self.nq + self.nkv) * self.hd:].view(-1, self.nkv, self.hd)
        return ops.packed_attention(q.view(-1, self.nq, self.hd), k, v, cu)

    def step(self):
        """One token of each sequence: embedding, rotation into the cache, attention, logits, the
        next token; positions advance (padding rows stay at -1)."""
        from moeinfra_amd import ops

        torch.index_select(self.embed, 0, self.tok, out=self.x)
        q, _ = ops.rope_paged_kv(self.x, self.pos, self.pool.dev_table, self.pool.k, self.pool.v, self.nq, self.inv)
        ops.paged_attention(q.view(-1, self.nq, self.hd), self.pool.k, self.pool.v, self.pool.dev_table, self.seen,
                            out=self.attn, workspace=self.ws)
        logits = self.attn.view(len(self.lens), -1) @ self.head
        ops.sample_tokens(logits, self.u, temperature=0.9, top_k=100, top_p=0.95, out=self.tok)
        live = (self.pos >= 0).to(torch.int32)
        self.pos += live
        self.seen += live
        return logits


def test_prompts_and_steps_together(cuda_device):
    """Packed prompts into the cache, then steps over it, against the 64-bit forms fed with the
    bf16 tensors that pass between the operators."""
    dev, lens, steps = cuda_device, [37, 1, 130], 4
    sv = _Server(dev, lens, steps)
    nq, nkv, hd = sv.nq, sv.nkv, sv.hd
    qkv = _bf((sum(lens), (nq + 2 * nkv) * hd), 62).to(dev)
    out = sv.prompts(qkv)
    heads = qkv.cpu().view(-1, nq + 2 * nkv, hd)
    pos = [p for n in lens for p in range(n)]
    rot, _ = rope(heads[:, :nq + nkv], pos, _inv(hd))
    rot = rot.to(torch.bfloat16)
    # (A rotated value next to a tie may be rounded to the other side than here: a step of 2^-7 of one
    # product of about 9 at most, times the scaling of 1/8, moves a score by 2^-7 and a weight by
    # twice that.  Such values are 2^-13 of all, more than one in a score hardly ever.)
    slack = 2.0 ** -6
    ks, vs, at = [], [], 0
    for i, n in enumerate(lens):
        ks.append(rot[at:at + n, nq:])
        vs.append(heads[at:at + n, nq + nkv:])
        for h in range(nq):
            seen = torch.ones((n, n), dtype=torch.bool).tril()
            want, tol = attention(rot[at:at + n, h], ks[i][:, h // (nq // nkv)], vs[i][:, h // (nq // nkv)], hd ** -0.5, seen)
            assert_within(out[at:at + n, h], want, tol + slack * vs[i].double().abs().amax(), f"prompt {i}")
        at += n
    g = torch.Generator().manual_seed(63)
    for s in range(steps):
        tok = sv.tok.cpu()
        sv.u.copy_(torch.rand((3,), generator=g))
        u = sv.u.cpu()
        logits = sv.step()
        x = sv.embed[tok.to(dev)].cpu().view(3, nq + 2 * nkv, hd)
        r, _ = rope(x[:, :nq + nkv], [n + s for n in lens], _inv(hd))
        r = r.to(torch.bfloat16)
        for i in range(3):
            ks[i] = torch.cat((ks[i], r[i:i + 1, nq:]))
            vs[i] = torch.cat((vs[i], x[i:i + 1, nq + nkv:]))
            for h in range(nq):
                want, tol = attention(r[i, h:h + 1], ks[i][:, h // (nq // nkv)], vs[i][:, h // (nq // nkv)], hd ** -0.5)
                assert_within(sv.attn[i, h:h + 1], want, tol + slack * vs[i].double().abs().amax(), f"step {s}")
        assert sv.tok.cpu().tolist() == [sample(logits[i].float().cpu(), float(u[i]), temperature=0.9, top_k=100, top_p=0.95)
                                         for i in range(3)]


def test_prompts_and_steps_by_what_passes_between_them(cuda_device):
    """Prompts and steps as above, each operator's result against the 64-bit form of what it was given:
    the rotated queries and keys that the call before it returned, and the cache's own rows."""
    from moeinfra_amd import ops

    dev, lens, steps = cuda_device, [37, 1, 130, 300], 3
    sv = _Server(dev, lens, steps)
    nq, nkv, hd, page = sv.nq, sv.nkv, sv.hd, sv.pool.page
    qkv = _bf((sum(lens), (nq + 2 * nkv) * hd), 66).to(dev)
    seq = torch.tensor([i for i, n in enumerate(lens) for _ in range(n)], dtype=torch.int32, device=dev)
    pos = torch.tensor([p for n in lens for p in range(n)], dtype=torch.int32, device=dev)
    cuts = [sum(lens[:i]) for i in range(len(lens) + 1)]
    q, k = ops.rope_paged_kv(qkv, pos, sv.pool.dev_table, sv.pool.k, sv.pool.v, nq, sv.inv, seq_ids=seq, want_k=True)
    heads = qkv.cpu().view(-1, nq + 2 * nkv, hd)
    y, tol = rope(heads[:, :nq + nkv], pos.cpu(), _inv(hd))
    q = q.view(-1, nq, hd)
    assert_within(q, y[:, :nq], tol[:, :nq], "q")
    assert_within(k, y[:, nq:], tol[:, nq:], "k")
    out = ops.packed_attention(q, k, qkv[:, (nq + nkv) * hd:].view(-1, nkv, hd),
                               torch.tensor(cuts, dtype=torch.int32, device=dev))
    _check_packed(out, q.cpu(), k.cpu(), heads[:, nq + nkv:], cuts, hd ** -0.5)

    def cached(i, n):  # the first n rows of sequence i, from the cache
        at = torch.arange(n)
        p = sv.pool.table[i, at // page].long()
        return sv.pool.k.cpu()[p, :, at % page], sv.pool.v.cpu()[p, :, at % page]

    for i, n in enumerate(lens):
        kc, vc = cached(i, n)
        assert _same(kc, k[cuts[i]:cuts[i + 1]].cpu()) and _same(vc, heads[cuts[i]:cuts[i + 1], nq + nkv:])
    g = torch.Generator().manual_seed(67)
    for s in range(steps):
        x = (torch.randn((len(lens), (nq + 2 * nkv) * hd), generator=g)).to(torch.bfloat16)
        at = torch.tensor([n + s for n in lens], dtype=torch.int32)
        q, _ = ops.rope_paged_kv(x.to(dev), at.to(dev), sv.pool.dev_table, sv.pool.k, sv.pool.v, nq, sv.inv)
        q = q.view(-1, nq, hd)
        y, tol = rope(x.view(len(lens), -1, hd)[:, :nq + nkv], at, _inv(hd))
        assert_within(q, y[:, :nq], tol[:, :nq], f"step {s}, q")
        both = [cached(i, n + s + 1) for i, n in enumerate(lens)]
        for i, (kc, vc) in enumerate(both):
            assert_within(kc[-1], y[i, nq:], tol[i, nq:], f"step {s}, k")
            assert _same(vc[-1], x[i].view(-1, hd)[nq + nkv:])
        out = ops.paged_attention(q, sv.pool.k, sv.pool.v, sv.pool.dev_table, (at + 1).to(dev), workspace=sv.ws)
        _check_paged(out, q.cpu(), [kc for kc, _ in both], [vc for _, vc in both], nkv, hd ** -0.5)
        logits, u = (out.view(len(lens), -1) @ sv.head).float(), torch.rand((len(lens),), generator=g)
        _sampled(dev, logits.cpu(), u, temperature=0.9, top_k=100, top_p=0.95)


def test_steps_replayed_from_a_graph(cuda_device):
    """The step captured once (a batch with padding rows) and replayed, against eager steps, with
    eager work on the same workspace between the replays."""
    dev, lens, steps = cuda_device, [37, 700, 5, 1], 6
    runs = []
    for captured in (False, True):
        sv = _Server(dev, lens, steps + 2)
        sv.prompts(_bf((sum(lens), (sv.nq + 2 * sv.nkv) * sv.hd), 64).to(dev))
        sv.pos[2] = -1       # padding from here on
        sv.seen[2] = 0
        g = torch.Generator().manual_seed(65)
        got = []
        graph = None
        if captured:
            state = [t.clone() for t in (sv.pos, sv.seen, sv.tok, sv.pool.k, sv.pool.v)]
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                sv.step()
            torch.cuda.current_stream().wait_stream(side)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                sv.step()
            for t, saved in zip((sv.pos, sv.seen, sv.tok, sv.pool.k, sv.pool.v), state):
                t.copy_(saved)
        for s in range(steps):
            sv.u.copy_(torch.rand((4,), generator=g))
            if captured:
                graph.replay()
            else:
                sv.step()
            got.append((sv.tok.cpu().tolist(), sv.attn.clone()))
            _paged(dev, [300 + s, 2, 90], sv.nq, sv.nkv, sv.hd, 16, seed=s, workspace=sv.ws)
        assert not bool(sv.ws[:65536].any())
        assert bool((sv.attn[2] == 0).all())
        runs.append(got)
    for (a, x), (b, y) in zip(*runs):
        assert a == b and _same(x, y)


def test_operators_on_another_stream(cuda_device):
    """Each operator on a side stream, its inputs made there."""
    from moeinfra_amd import ops

    dev = cuda_device
    main = _paged(dev, [50, 600], 8, 2, 64, 16, seed=70)[0]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _paged(dev, [50, 600], 8, 2, 64, 16, seed=70)[0]
        assert _same(main, got)
        _check_packed(*_packed(dev, [70, 3], 4, 2, 64, seed=71))
        x, u = _logits(3, 900, 72, torch.float32)
        _sampled(dev, x, u, top_p=0.9)
    side.synchronize()


def test_wrappers_refuse_what_does_not_fit(cuda_device):
    from moeinfra_amd import ops

    dev = cuda_device
    bf = lambda *s: torch.zeros(s, dtype=torch.bfloat16, device=dev)
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32, device=dev)
    f32 = lambda *s: torch.zeros(s, device=dev)
    kc, table = bf(4, 2, 16, 64), i32(3, 2)
    vc = bf(4, 2, 16, 64)
    bad = [
        (lambda: ops.rope_paged_kv(bf(3, 768), i32(4), table, kc, vc, 8, f32(32)), "positions"),
        (lambda: ops.rope_paged_kv(bf(3, 760), i32(3), table, kc, vc, 8, f32(32)), "qkv rows"),
        (lambda: ops.rope_paged_kv(bf(3, 768), i32(3), table, kc, vc, 8, f32(31)), "inv_freq"),
        (lambda: ops.rope_paged_kv(bf(3, 768), i32(3), table, kc, bf(5, 2, 16, 64), 8, f32(32)), "differ"),
        (lambda: ops.rope_paged_kv(bf(3, 768).float(), i32(3), table, kc, vc, 8, f32(32)), "bfloat16"),
        (lambda: ops.rope_paged_kv(bf(3, 768), i32(3).long(), table, kc, vc, 8, f32(32)), "int32"),
        (lambda: ops.rope_paged_kv(bf(3, 768), i32(3), table, kc, kc, 8, f32(32)), "caches of their own"),
        (lambda: ops.rope_paged_kv(bf(3, 768), i32(3), table, kc, vc, 8, f32(32), seq_ids=i32(2)), "seq_ids"),
        (lambda: ops.paged_attention(bf(3, 8, 64), kc, vc, table, i32(2)), "lens must be"),
        (lambda: ops.paged_attention(bf(3, 8, 128), kc, vc, table, i32(3)), "head dim"),
        (lambda: ops.paged_attention(bf(3, 7, 64), kc, vc, table, i32(3)), "invalid attention sizes"),
        (lambda: ops.paged_attention(bf(3, 64, 8).transpose(1, 2), kc, vc, table, i32(3)), "contiguous rows"),
        (lambda: ops.paged_attention(bf(3, 8, 64), kc, vc, table, i32(3), workspace=f32(4).to(torch.uint8)), "too small"),
        (lambda: ops.paged_attention(bf(3, 8, 64), kc.transpose(1, 2), vc.transpose(1, 2), table, i32(3)), "contiguous rows"),
        (lambda: ops.packed_attention(bf(5, 8, 64), bf(5, 2, 64), bf(4, 2, 64), i32(2)), "do not fit"),
        (lambda: ops.packed_attention(bf(5, 8, 64), bf(5, 3, 64), bf(5, 3, 64), i32(2)), "multiple"),
        (lambda: ops.packed_attention(bf(5, 8, 96), bf(5, 2, 96), bf(5, 2, 96), i32(2)), "head dim"),
        (lambda: ops.packed_attention(bf(5, 8, 64), bf(5, 2, 64), bf(5, 2, 64), i32(2, 2)), "cu_seqlens"),
        (lambda: ops.sample_tokens(bf(3, 10).half(), f32(3)), "bfloat16"),
        (lambda: ops.sample_tokens(bf(10, 3).t(), f32(3)), "contiguous rows"),
        (lambda: ops.sample_tokens(bf(3, 10), f32(2)), "u must be"),
        (lambda: ops.sample_tokens(bf(3, 10), f32(3), top_k=f32(3)), "top_k"),
        (lambda: ops.sample_tokens(bf(3, 10), f32(3), top_p=f32(2)), "top_p"),
        (lambda: ops.sample_tokens(bf(3, 10), f32(3), top_p=0.0), "top-p"),
        (lambda: ops.sample_tokens(bf(3, 10), f32(3), out=i32(3)), "out"),
    ]
    for call, needle in bad:
        with pytest.raises(ValueError, match=needle):
            call()
    # Nothing to do.
    assert ops.packed_attention(bf(0, 8, 64), bf(0, 2, 64), bf(0, 2, 64), i32(1)).shape == (0, 8, 64)
    assert ops.paged_attention(bf(0, 8, 64), kc, vc, i32(0, 2), i32(0)).shape == (0, 8, 64)
    assert ops.sample_tokens(bf(0, 10), f32(0)).shape == (0,)
    assert ops.rope_paged_kv(bf(0, 768), i32(0), table, kc, vc, 8, f32(32))[0].shape == (0, 512)
    # A pool without pages: no keys.
    none = ops.paged_attention(bf(3, 8, 64), kc[:0], vc[:0], table, i32(3) + 20)
    assert bool((none == 0).all())
