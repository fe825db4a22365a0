"""Refusals of the batched serving operators, without a GPU: what the C entry points and their
torch wrappers reject before any launch."""
from __future__ import annotations

import pytest
import torch

from moeinfra_amd import _lib, ops

# Addresses that are never read: far apart, 16-byte aligned.
A, B, C, D, E, F, G, H = (i << 40 for i in range(1, 9))


def _append(**kw):
    a = dict(qkv=A, stride=768, T=4, nq=8, nkv=2, hd=64, inv=B, pos=C, seq=None, table=D, n_seqs=4, width=8,
             pages=32, page=16, page_stride=2 * 16 * 64, q=E, k=None, kc=F, vc=G, stream=None)
    a.update(kw)
    return _lib.lib().moe_rope_paged_kv_bf16(*a.values())


def _paged(**kw):
    a = dict(q=A, stride=512, kc=F, vc=G, pages=32, page=16, page_stride=2 * 16 * 64, table=D, width=8, lens=C, B=4,
             nq=8, nkv=2, hd=64, scaling=0.125, out=E, ws=None, ws_bytes=0, stream=None)
    a.update(kw)
    return _lib.lib().moe_paged_attention_bf16(*a.values())


def _packed(**kw):
    a = dict(q=A, q_stride=512, k=B, k_stride=128, v=C, v_stride=128, T=10, cu=D, B=3, nq=8, nkv=2, hd=64,
             scaling=0.125, out=E, stream=None)
    a.update(kw)
    return _lib.lib().moe_packed_attention_bf16(*a.values())


def _sample(**kw):
    a = dict(logits=A, f32=0, stride=1000, B=4, V=1000, u=B, t=None, temperature=1.0, k=None, top_k=0, p=None,
             top_p=1.0, mp=None, min_p=0.0, token=C, stream=None)
    a.update(kw)
    return _lib.lib().moe_sample_tokens(*a.values())


REFUSED = [
    (_append, dict(hd=24), "head dim"),
    (_append, dict(hd=528), "head dim"),
    (_append, dict(page=4), "page size"),
    (_append, dict(page=24), "page size"),
    (_append, dict(page=8192), "page size"),
    (_append, dict(page_stride=2040), "page stride"),
    (_append, dict(page_stride=2052), "page stride"),
    (_append, dict(stride=760), "qkv rows"),
    (_append, dict(stride=772), "qkv rows"),
    (_append, dict(T=-1), "bad sizes"),
    (_append, dict(T=1 << 31), "bad sizes"),
    (_append, dict(T=1 << 24), "bad sizes"),
    (_append, dict(nq=0), "bad sizes"),
    (_append, dict(pages=-1), "bad sizes"),
    (_append, dict(pages=1 << 31), "bad sizes"),
    (_append, dict(qkv=None), "null"),
    (_append, dict(pos=None), "null"),
    (_append, dict(table=None), "null"),
    (_append, dict(vc=None), "null"),
    (_append, dict(q=E + 8), "aligned"),
    (_append, dict(kc=F + 2), "aligned"),
    (_append, dict(q=A + 64), "overlap"),
    (_append, dict(k=E + 64), "overlap"),
    (_append, dict(q=F + 4096), "overlap"),
    (_append, dict(vc=F), "caches of their own"),
    (_paged, dict(nq=7), "multiple"),
    (_paged, dict(nkv=0), "multiple"),
    (_paged, dict(hd=96), "head dim"),
    (_paged, dict(hd=32), "head dim"),
    (_paged, dict(page=4), "page size"),
    (_paged, dict(page=48), "page size"),
    (_paged, dict(page_stride=1024), "page stride"),
    (_paged, dict(B=-1), "bad sizes"),
    (_paged, dict(pages=1 << 31), "bad sizes"),
    (_paged, dict(B=1 << 20, nq=64, nkv=64, stride=4096, page_stride=64 * 16 * 64), "bad sizes"),
    (_paged, dict(width=1 << 28), "too long"),
    (_paged, dict(width=1 << 20, B=1 << 20), "too long"),
    (_paged, dict(stride=504), "q rows"),
    (_paged, dict(lens=None), "null"),
    (_paged, dict(kc=None), "null"),
    (_paged, dict(q=A + 2), "aligned"),
    (_paged, dict(out=A), "overlap"),
    (_paged, dict(out=G + 64), "overlap"),
    (_paged, dict(ws=H, ws_bytes=4096), "workspace too small"),
    (_paged, dict(ws=H + 8, ws_bytes=1 << 30), "workspace must be"),
    (_packed, dict(nq=9), "multiple"),
    (_packed, dict(hd=80), "head dim"),
    (_packed, dict(scaling=float("nan")), "NaN"),
    (_packed, dict(T=-1), "bad sizes"),
    (_packed, dict(T=1 << 30), "bad sizes"),
    (_packed, dict(B=-1), "bad sizes"),
    (_packed, dict(T=1 << 23, B=1 << 20, nq=1 << 12, nkv=1 << 12, q_stride=1 << 18, k_stride=1 << 18, v_stride=1 << 18,
                   q=1 << 56, k=2 << 56, v=3 << 56, out=4 << 56), "bad sizes"),
    (_packed, dict(q_stride=504), "apart"),
    (_packed, dict(k_stride=132), "aligned"),
    (_packed, dict(v_stride=64), "apart"),
    (_packed, dict(k_stride=1 << 31), "values apart"),
    (_packed, dict(v_stride=1 << 40), "values apart"),
    (_packed, dict(cu=None), "null"),
    (_packed, dict(v=C + 8), "aligned"),
    (_packed, dict(out=E + 4), "aligned"),
    (_packed, dict(out=A + 1024), "overlap"),
    (_packed, dict(out=C - 1024), "overlap"),
    (_sample, dict(f32=2), "bf16"),
    (_sample, dict(B=-1), "bad sizes"),
    (_sample, dict(B=1 << 22), "bad sizes"),
    (_sample, dict(V=0), "logits"),
    (_sample, dict(V=(1 << 20) + 1, stride=1 << 21), "logits"),
    (_sample, dict(stride=999), "apart"),
    (_sample, dict(temperature=-1.0), "temperature"),
    (_sample, dict(temperature=float("nan")), "temperature"),
    (_sample, dict(top_k=-1), "top-k"),
    (_sample, dict(top_p=0.0), "top-p"),
    (_sample, dict(top_p=1.5), "top-p"),
    (_sample, dict(min_p=-0.1), "min-p"),
    (_sample, dict(min_p=1.1), "min-p"),
    (_sample, dict(u=None), "null"),
    (_sample, dict(f32=1, logits=A + 2), "aligned"),
    (_sample, dict(token=C + 4), "aligned"),
    (_sample, dict(token=A + 800), "overlap"),
]


@pytest.mark.parametrize("call,change,needle", REFUSED, ids=[f"{c.__name__[1:]}-{k}" for c, k, _ in REFUSED])
def test_refused_before_any_launch(call, change, needle):
    assert call(**change) == _lib.MOE_STATUS_INVALID_ARGUMENT
    assert needle in _lib.lib().moe_last_error().decode()


def test_empty_calls_do_nothing():
    assert _append(T=0, qkv=None, q=None, table=None, kc=None, vc=None) == 0
    assert _paged(B=0, q=None, out=None, lens=None) == 0
    assert _packed(T=0, q=None, k=None, v=None, cu=None, out=None) == 0
    assert _packed(B=0, cu=None) == 0
    assert _sample(B=0, logits=None, u=None, token=None) == 0


def test_paged_attention_workspace_grows_with_the_batch():
    f = _lib.lib().moe_paged_attention_workspace_bytes
    sizes = [f(b, 32, 8, 128) for b in (0, 1, 8, 256, 5000, 1 << 20)]
    assert sizes == sorted(sizes) and sizes[0] >= 65536
    assert f(-1, 32, 8, 128) == -1 and f(1, 32, 8, 96) == -1 and f(1, 9, 2, 128) == -1


@pytest.mark.parametrize("nq,nkv,hd", [(32, 8, 128), (8, 2, 64), (40, 2, 128), (33, 1, 128), (8, 4, 256), (4, 4, 128),
                                       (1 << 16, 1, 256)])
def test_paged_attention_workspace_is_one_size_for_all_batches(nq, nkv, hd):
    """One size for every batch (a workspace made for one serves any other of the same heads): the
    counters, and two places of a partial result for each workgroup that runs at once."""
    f = _lib.lib().moe_paged_attention_workspace_bytes
    sizes = {f(b, nq, nkv, hd) for b in (0, 1, 7, 64, 256, 5000, 1 << 20)}
    assert len(sizes) == 1
    grp = nq // nkv
    place = min(grp, 16) * (hd + 2) * 4
    units = nkv * -(-grp // 16)
    places, rest = divmod(sizes.pop() - 65536, place)
    assert rest == 0 and places % (2 * units) == 0 and places >= 2 * units


def test_wrappers_take_gpu_tensors_only():
    bf = lambda *s: torch.zeros(s, dtype=torch.bfloat16)
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32)
    with pytest.raises(ValueError, match="GPU tensor"):
        ops.rope_paged_kv(bf(4, 768), i32(4), i32(4, 8), bf(32, 2, 16, 64), bf(32, 2, 16, 64), 8, torch.zeros(32))
    with pytest.raises(ValueError, match="GPU tensor"):
        ops.paged_attention(bf(4, 8, 64), bf(32, 2, 16, 64), bf(32, 2, 16, 64), i32(4, 8), i32(4))
    with pytest.raises(ValueError, match="GPU tensor"):
        ops.packed_attention(bf(4, 8, 64), bf(4, 2, 64), bf(4, 2, 64), i32(2))
    with pytest.raises(ValueError, match="GPU tensor"):
        ops.sample_tokens(bf(4, 100), torch.zeros(4))
    with pytest.raises(ValueError, match="invalid attention sizes"):
        ops.paged_attention_workspace(4, 8, 2, 96, "cpu")
