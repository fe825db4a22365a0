"""Refusals of the operators of decoding that branches, without a GPU: what the C entry points and
their torch wrappers reject before any launch."""
from __future__ import annotations

import pytest
import torch

from moeinfra_amd import _lib, ops

# Addresses that are never read: far apart, 16-byte aligned.
A, B, C, D, E, F, G, H, I, J = (i << 40 for i in range(1, 11))


def _slots(**kw):
    a = dict(qkv=A, stride=768, T=4, nq=8, nkv=2, hd=64, inv=B, pos=C, slots=I, seq=None, table=D, n_seqs=4, width=8,
             pages=32, page=16, page_stride=2 * 16 * 64, q=E, k=None, kc=F, vc=G, stream=None)
    a.update(kw)
    return _lib.lib().moe_rope_paged_kv_slots_bf16(*a.values())


def _tree(**kw):
    a = dict(q=A, stride=512, T=20, kc=F, vc=G, pages=32, page=16, page_stride=2 * 16 * 64, table=D, width=8, lens=C, cu=B,
             masks=I, B=4, nq=8, nkv=2, hd=64, scaling=0.125, out=E, ws=None, ws_bytes=0, stream=None)
    a.update(kw)
    return _lib.lib().moe_paged_tree_attention_bf16(*a.values())


def _accept(**kw):
    a = dict(targets=A, drafts=B, masks=C, cu=D, T=20, B=4, paths=E, counts=F, tokens=G, stream=None)
    a.update(kw)
    return _lib.lib().moe_accept_drafts(*a.values())


def _compact(**kw):
    a = dict(kc=A, vc=B, layers=3, layer_stride=32 * 2048, pages=32, page=16, page_stride=2048, nkv=2, hd=64, table=C,
             n_seqs=4, width=8, lens=D, paths=E, stream=None)
    a.update(kw)
    return _lib.lib().moe_compact_paged_kv_bf16(*a.values())


def _copy(**kw):
    a = dict(kc=A, vc=B, layers=3, layer_stride=32 * 2048, pages=32, page=16, page_stride=2048, nkv=2, hd=64, copies=C,
             n=4, stream=None)
    a.update(kw)
    return _lib.lib().moe_copy_pages_bf16(*a.values())


def _beam(**kw):
    a = dict(logits=A, f32=0, stride=1000, S=4, W=3, V=1000, scores=B, k=6, best=C, rows=D, tokens=E, ws=F, ws_bytes=1 << 24,
             stream=None)
    a.update(kw)
    return _lib.lib().moe_beam_select(*a.values())


def _fork(**kw):
    a = dict(table=A, lens=B, n_seqs=4, width=8, parents=C, n_new=6, refs=D, pages=32, page=16, ahead=1, new_table=E,
             new_lens=F, copies=G, missing=H, ws=I, ws_bytes=256, stream=None)
    a.update(kw)
    return _lib.lib().moe_fork_pages(*a.values())


REFUSED = [
    (_slots, dict(slots=None), "null"),
    (_slots, dict(hd=24), "head dim"),
    (_slots, dict(page=4), "page size"),
    (_slots, dict(T=-1), "bad sizes"),
    (_slots, dict(vc=F), "caches of their own"),
    (_tree, dict(nq=7), "multiple"),
    (_tree, dict(nkv=0), "multiple"),
    (_tree, dict(hd=96), "head dim"),
    (_tree, dict(scaling=float("nan")), "NaN"),
    (_tree, dict(page=4), "page size"),
    (_tree, dict(page=48), "page size"),
    (_tree, dict(page=8192), "page size"),
    (_tree, dict(page_stride=1024), "page stride"),
    (_tree, dict(page_stride=2052), "page stride"),
    (_tree, dict(B=-1), "bad sizes"),
    (_tree, dict(T=-1), "bad sizes"),
    (_tree, dict(T=1 << 31), "bad sizes"),
    (_tree, dict(pages=1 << 31), "bad sizes"),
    (_tree, dict(width=-1), "bad sizes"),
    (_tree, dict(nq=1 << 17, nkv=1 << 17), "bad sizes"),
    (_tree, dict(width=1 << 28), "too long"),
    (_tree, dict(width=1 << 20, B=1 << 20), "too long"),
    (_tree, dict(width=0, B=1 << 20, nq=1 << 16, nkv=1, stride=1 << 22), "too long"),
    (_tree, dict(stride=504), "q rows"),
    (_tree, dict(stride=516), "q rows"),
    (_tree, dict(q=None), "null"),
    (_tree, dict(lens=None), "null"),
    (_tree, dict(cu=None), "null"),
    (_tree, dict(table=None), "null"),
    (_tree, dict(kc=None), "null"),
    (_tree, dict(q=A + 2), "aligned"),
    (_tree, dict(vc=G + 8), "aligned"),
    (_tree, dict(out=E + 4), "aligned"),
    (_tree, dict(masks=I + 4), "aligned"),
    (_tree, dict(lens=C + 2), "aligned"),
    (_tree, dict(out=A), "overlap"),
    (_tree, dict(out=G + 64), "overlap"),
    (_tree, dict(ws=H, ws_bytes=4096), "workspace too small"),
    (_tree, dict(ws=H + 8, ws_bytes=1 << 32), "workspace must be"),
    (_accept, dict(T=-1), "bad sizes"),
    (_accept, dict(T=1 << 31), "bad sizes"),
    (_accept, dict(B=(1 << 20) + 1), "bad sizes"),
    (_accept, dict(targets=None), "null"),
    (_accept, dict(cu=None), "null"),
    (_accept, dict(counts=None), "null"),
    (_accept, dict(masks=C + 4), "aligned"),
    (_accept, dict(counts=F + 2), "aligned"),
    (_accept, dict(paths=A + 32), "overlap"),
    (_accept, dict(tokens=D), "overlap"),
    (_accept, dict(counts=E + 8), "overlap"),
    (_compact, dict(hd=12), "head dim"),
    (_compact, dict(hd=520), "head dim"),
    (_compact, dict(page=4), "page size"),
    (_compact, dict(page=24), "page size"),
    (_compact, dict(page_stride=2040), "page stride"),
    (_compact, dict(page_stride=2052), "page stride"),
    (_compact, dict(layers=-1), "bad sizes"),
    (_compact, dict(nkv=0), "bad sizes"),
    (_compact, dict(pages=1 << 31), "bad sizes"),
    (_compact, dict(n_seqs=-1), "bad sizes"),
    (_compact, dict(n_seqs=1 << 24), "bad sizes"),
    (_compact, dict(layer_stride=2048), "apart"),
    (_compact, dict(layer_stride=32 * 2048 + 4), "apart"),
    (_compact, dict(kc=None), "null"),
    (_compact, dict(lens=None), "null"),
    (_compact, dict(vc=A), "caches of their own"),
    (_compact, dict(vc=B + 8), "aligned"),
    (_compact, dict(paths=E + 4), "aligned"),
    (_copy, dict(hd=0), "head dim"),
    (_copy, dict(page=12), "page size"),
    (_copy, dict(layer_stride=0), "apart"),
    (_copy, dict(n=-1), "bad sizes"),
    (_copy, dict(n=1 << 24), "bad sizes"),
    (_copy, dict(copies=None), "null"),
    (_copy, dict(copies=C + 2), "aligned"),
    (_copy, dict(vc=A), "caches of their own"),
    (_beam, dict(f32=2), "bf16"),
    (_beam, dict(W=0), "beams"),
    (_beam, dict(W=257), "beams"),
    (_beam, dict(k=0), "continuations"),
    (_beam, dict(k=65), "continuations"),
    (_beam, dict(S=-1), "searches"),
    (_beam, dict(S=16385), "searches"),
    (_beam, dict(V=0), "logits"),
    (_beam, dict(V=(1 << 20) + 1, stride=1 << 21), "logits"),
    (_beam, dict(stride=999), "apart"),
    (_beam, dict(logits=None), "null"),
    (_beam, dict(tokens=None), "null"),
    (_beam, dict(ws=None), "workspace too small"),
    (_beam, dict(ws_bytes=65536), "workspace too small"),
    (_beam, dict(ws=F + 8), "workspace must be"),
    (_beam, dict(f32=1, logits=A + 2), "aligned"),
    (_beam, dict(tokens=E + 4), "aligned"),
    (_beam, dict(best=A + 16), "overlap"),
    (_beam, dict(rows=C + 4), "overlap"),
    (_beam, dict(scores=F + 128), "overlap"),
    (_fork, dict(page=4), "page size"),
    (_fork, dict(page=20), "page size"),
    (_fork, dict(n_seqs=8193), "rows"),
    (_fork, dict(n_new=-1), "rows"),
    (_fork, dict(width=-1), "bad sizes"),
    (_fork, dict(width=1 << 28), "bad sizes"),
    (_fork, dict(pages=-1), "bad sizes"),
    (_fork, dict(ahead=0), "next tokens"),
    (_fork, dict(ahead=(1 << 20) + 1), "next tokens"),
    (_fork, dict(n_new=8192, ahead=3), "written to"),
    (_fork, dict(ahead=1 << 20), "written to"),
    (_fork, dict(parents=None), "null"),
    (_fork, dict(missing=None), "null"),
    (_fork, dict(refs=None), "null"),
    (_fork, dict(ws=None), "workspace too small"),
    (_fork, dict(ws_bytes=252), "workspace too small"),
    (_fork, dict(lens=B + 2), "aligned"),
    (_fork, dict(new_table=A), "overlap"),
    (_fork, dict(new_lens=C + 4), "overlap"),
    (_fork, dict(refs=A + 4), "overlap"),
    (_fork, dict(missing=G), "overlap"),
    (_fork, dict(ws=D), "overlap"),
]


@pytest.mark.parametrize("call,change,needle", REFUSED, ids=[f"{c.__name__[1:]}-{k}" for c, k, _ in REFUSED])
def test_refused_before_any_launch(call, change, needle):
    assert call(**change) == _lib.MOE_STATUS_INVALID_ARGUMENT
    assert needle in _lib.lib().moe_last_error().decode()


@pytest.mark.parametrize("kw", [dict(ws=A), dict(ws=A - 4096), dict(ws=E), dict(ws=E + 64), dict(ws=F), dict(ws=G), dict(ws=C - 64),
                                dict(ws=B), dict(ws=D), dict(ws=I), dict(out=C - 8), dict(out=B), dict(out=D), dict(out=I)])
def test_tree_attention_refuses_a_workspace_or_output_in_its_inputs(kw):
    """What the workgroups write while others still read: the workspace and out, against all inputs and each other."""
    assert _tree(**{"ws": H, "ws_bytes": 1 << 36, **kw}) == _lib.MOE_STATUS_INVALID_ARGUMENT
    assert "overlap" in _lib.lib().moe_last_error().decode()


@pytest.mark.parametrize("n", [(1 << 31) - 1, (1 << 30) + (1 << 20)])
def test_copies_beyond_64_bits_are_refused(n):
    """Copies times layers times groups of heads wrap around 64 bits: too many, not few."""
    big = dict(layers=1 << 16, layer_stride=1 << 40, pages=1, page=512, nkv=65535, hd=256, page_stride=1 << 33, n=n)
    assert _copy(**big) == _lib.MOE_STATUS_INVALID_ARGUMENT
    assert "bad sizes" in _lib.lib().moe_last_error().decode()


def test_empty_calls_do_nothing():
    assert _slots(T=0, qkv=None, q=None, slots=None) == 0
    assert _tree(B=0, cu=None, lens=None) == 0
    assert _tree(T=0, q=None, out=None) == 0
    assert _accept(B=0, cu=None, paths=None) == 0
    assert _compact(n_seqs=0, table=None, lens=None, paths=None) == 0
    assert _compact(layers=0, kc=None, vc=None) == 0
    assert _compact(pages=0, kc=None, vc=None) == 0
    assert _copy(n=0, copies=None) == 0
    assert _beam(S=0, logits=None, scores=None, best=None, ws=None) == 0


def test_workspaces_are_host_functions():
    tree = _lib.lib().moe_paged_tree_attention_workspace_bytes
    assert len({tree(b, 32, 8, 128) for b in (0, 1, 64, 1 << 20)}) == 1 and tree(1, 32, 8, 128) > 65536
    assert tree(-1, 32, 8, 128) == -1 and tree(1, 32, 8, 96) == -1 and tree(1, 9, 2, 128) == -1
    beam = _lib.lib().moe_beam_select_workspace_bytes
    sizes = [beam(s, 4, 8) for s in (0, 1, 64, 1000, 16384)]
    assert sizes == sorted(sizes) and sizes[0] > 65536 and beam(1, 4, 16) > beam(1, 4, 8)
    assert beam(16385, 1, 1) == -1 and beam(1, 257, 1) == -1 and beam(1, 1, 65) == -1 and beam(1, 1, 0) == -1
    fork = _lib.lib().moe_fork_pages_workspace_bytes
    assert fork(100) >= 800 and fork(-1) == -1 and fork(0) > 0


def test_wrappers_take_gpu_tensors_only():
    bf = lambda *s: torch.zeros(s, dtype=torch.bfloat16)
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32)
    i64 = lambda *s: torch.zeros(s, dtype=torch.int64)
    with pytest.raises(ValueError, match="GPU tensor"):
        ops.paged_tree_attention(bf(4, 8, 64), bf(32, 2, 16, 64), bf(32, 2, 16, 64), i32(2, 8), i32(2), i32(3))
    with pytest.raises(ValueError, match="GPU tensor"):
        ops.accept_drafts(i64(4), i64(4), i32(2))
    with pytest.raises(ValueError, match="GPU tensor"):
        ops.compact_paged_kv(bf(3, 32, 2, 16, 64), bf(3, 32, 2, 16, 64), i32(2, 8), i32(2), i64(2))
    with pytest.raises(ValueError, match="GPU tensor"):
        ops.beam_select(bf(4, 100), torch.zeros(2, 2), 4)
    with pytest.raises(ValueError, match="GPU tensor"):
        ops.fork_pages(i32(2, 8), i32(2), i32(2), i32(30), 16)
    with pytest.raises(ValueError, match="GPU tensor"):
        ops.copy_pages(bf(32, 2, 16, 64), bf(32, 2, 16, 64), i32(2, 3))
    with pytest.raises(ValueError, match="invalid attention sizes"):
        ops.paged_tree_attention_workspace(4, 8, 2, 96, "cpu")
    with pytest.raises(ValueError, match="invalid sizes"):
        ops.beam_select_workspace(4, 8, 65, "cpu")
    with pytest.raises(ValueError, match="invalid number of pages"):
        ops.fork_pages_workspace(-1, "cpu")
    # Numbers are refused where they would lose their upper bits on the way.
    with pytest.raises(ValueError, match="k must fit"):
        ops.beam_select_workspace(4, 8, (1 << 32) + 4, "cpu")
    with pytest.raises(ValueError, match="head_dim must fit"):
        ops.paged_tree_attention_workspace(4, 8, 2, (1 << 32) + 64, "cpu")
