"""Torch-tensor wrappers over the C ABI of ``libmoeinfra_hip.so``.

Every function validates dtype, shape and device first and raises ``ValueError`` the way
the reference does; kernels are enqueued on the current HIP stream of the tensors'
device (``torch.cuda.current_stream``).  Nothing here synchronises with the host, and
there is no non-HIP implementation: CPU tensors are rejected.
"""
from __future__ import annotations

import ctypes
from typing import Optional, Sequence

import torch

from . import _lib
from ._lib import MoeNf4Expert, check, lib
from .nf4 import NF4_BLOCKSIZE, nf4_code_tensor


def _stream(device: torch.device) -> int:
    return torch.cuda.current_stream(device).cuda_stream


def _require_cuda(t: torch.Tensor, name: str) -> None:
    if not isinstance(t, torch.Tensor):
        raise ValueError(f"{name} must be a torch.Tensor")
    if t.device.type != "cuda":
        raise ValueError(f"{name} must be a GPU tensor (got device {t.device}); "
                         "the MoE path runs only on the HIP device")


def _require(t: torch.Tensor, name: str, dtype: torch.dtype, device: torch.device) -> None:
    _require_cuda(t, name)
    if t.dtype != dtype:
        raise ValueError(f"{name} must be {dtype} (got {t.dtype})")
    if t.device != device:
        raise ValueError(f"{name} device {t.device} != {device}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


# ----------------------------------------------------------------------------- K1
def nf4_expand_absmax(absmax_q: torch.Tensor, absmax2: torch.Tensor, code2: torch.Tensor,
                      offset, blocksize2: int) -> torch.Tensor:
    """fp32 block scales of a nested (double-quantised) NF4 state:
    ``code2[absmax_q[i]] * absmax2[i // blocksize2] + offset`` (bitsandbytes'
    dequantize_blockwise of the absmax, then ``+= offset``)."""
    dev = absmax_q.device
    _require(absmax_q, "absmax_q", torch.uint8, dev)
    _require(absmax2, "absmax2", torch.float32, dev)
    _require(code2, "code2", torch.float32, dev)
    if code2.numel() != 256:
        raise ValueError("the nested code must have 256 entries")
    n = absmax_q.numel()
    if absmax2.numel() * int(blocksize2) < n:
        raise ValueError(f"absmax2 has {absmax2.numel()} groups, {n} values need "
                         f"{(n + blocksize2 - 1) // blocksize2}")
    off = 0.0 if offset is None else float(offset)
    out = torch.empty(absmax_q.shape, dtype=torch.float32, device=dev)
    check(lib().moe_nf4_expand_absmax(absmax_q.data_ptr(), absmax2.data_ptr(), code2.data_ptr(), off,
                                      n, int(blocksize2), out.data_ptr(),
                                      torch.cuda.current_stream(dev).cuda_stream),
          "moe_nf4_expand_absmax")
    return out


def nf4_dequant(packed: torch.Tensor, absmax: torch.Tensor, code: torch.Tensor,
                shape: Sequence[int], blocksize: int = NF4_BLOCKSIZE,
                out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Packed NF4 -> bf16 tensor of ``shape`` (bitsandbytes ``dequantize_4bit`` semantics:
    ``bf16(code[q] * absmax[i // blocksize])``, high nibble first)."""
    dev = packed.device
    _require(packed, "packed", torch.uint8, dev)
    _require(absmax, "absmax", torch.float32, dev)
    _require(code, "code", torch.float32, dev)
    numel = 1
    for s in shape:
        numel *= int(s)
    if code.numel() != 16:
        raise ValueError("NF4 code must have 16 entries")
    if packed.numel() * 2 < numel:
        raise ValueError(f"packed has {packed.numel()} bytes, shape needs {(numel + 1) // 2}")
    if absmax.numel() * blocksize < numel:
        raise ValueError(f"absmax has {absmax.numel()} blocks, shape needs "
                         f"{(numel + blocksize - 1) // blocksize}")
    if out is None:
        out = torch.empty(tuple(int(s) for s in shape), dtype=torch.bfloat16, device=dev)
    else:
        _require(out, "out", torch.bfloat16, dev)
        if out.numel() != numel:
            raise ValueError("out has the wrong number of elements")
    check(lib().moe_nf4_dequant_bf16(packed.data_ptr(), absmax.data_ptr(), code.data_ptr(),
                                     out.data_ptr(), numel, blocksize, _stream(dev)),
          "nf4_dequant")
    return out


# ----------------------------------------------------------------------------- K0
def nf4_quantize(w: torch.Tensor, blocksize: int = NF4_BLOCKSIZE,
                 code: Optional[torch.Tensor] = None, own_code: bool = False):
    """bf16 weight -> (packed uint8 [numel//2, 1], absmax fp32 [nblocks], code fp32 [16]).
    ``own_code``: the returned code is a new tensor that the launch fills, not the shared one."""
    dev = w.device
    _require_cuda(w, "weight")
    if w.dtype != torch.bfloat16:
        raise ValueError(f"Expected BF16 weights, got {w.dtype}")
    w = w.contiguous()
    if code is None:
        code = nf4_code_tensor(dev)
    _require(code, "code", torch.float32, dev)
    numel = w.numel()
    if numel % 2:
        raise ValueError("NF4 packing needs an even number of values")
    packed = torch.empty((numel // 2, 1), dtype=torch.uint8, device=dev)
    absmax = torch.empty(((numel + blocksize - 1) // blocksize,), dtype=torch.float32, device=dev)
    # (an empty weight launches nothing, so its code is copied)
    mine = torch.empty_like(code) if own_code and numel else None
    check(lib().moe_nf4_quantize_state_bf16(w.data_ptr(), numel, blocksize, code.data_ptr(),
                                            packed.data_ptr(), absmax.data_ptr(), _ptr(mine),
                                            _stream(dev)), "nf4_quantize")
    if own_code:
        return packed, absmax, code.clone() if mine is None else mine
    return packed, absmax, code


# ----------------------------------------------------------------------------- K2
def router_topk(x: torch.Tensor, gate: torch.Tensor, k: int,
                bias: Optional[torch.Tensor] = None, want_logits: bool = True,
                idx32_out: Optional[torch.Tensor] = None):
    """(logits bf16 [T,E] | None, weights fp32 [T,k], indices int64 [T,k])."""
    dev = x.device
    _require(x, "hidden_states", torch.bfloat16, dev)
    _require(gate, "gate_weight", torch.bfloat16, dev)
    if x.ndim != 2 or gate.ndim != 2 or x.shape[1] != gate.shape[1]:
        raise ValueError(f"shape mismatch: hidden {tuple(x.shape)} vs gate {tuple(gate.shape)}")
    T, H = x.shape
    E = gate.shape[0]
    if bias is not None:
        _require(bias, "bias", torch.float32, dev)
        if bias.numel() != E:
            raise ValueError("bias must have one value per expert")
    logits = torch.empty((T, E), dtype=torch.bfloat16, device=dev) if want_logits else None
    w = torch.empty((T, k), dtype=torch.float32, device=dev)
    idx = torch.empty((T, k), dtype=torch.int64, device=dev)
    if idx32_out is not None:
        _require(idx32_out, "idx32_out", torch.int32, dev)
    check(lib().moe_router_topk(x.data_ptr(), gate.data_ptr(), _ptr(bias), T, H, E, k,
                                _ptr(logits), w.data_ptr(), idx.data_ptr(), _ptr(idx32_out),
                                _stream(dev)), "router_topk")
    return logits, w, idx


# ----------------------------------------------------------------------------- K3
def permute(idx32: torch.Tensor, num_experts: int):
    """Expert-sorted grouping of routing slots.  Returns a dict of int32 device tensors:
    counts [E], offsets [E+1], perm_tok [T*k], slot_pos [T*k], active [E+1]."""
    dev = idx32.device
    _require(idx32, "idx32", torch.int32, dev)
    if idx32.ndim != 2:
        raise ValueError("idx32 must be [T, k]")
    T, k = idx32.shape
    E = int(num_experts)
    i32 = dict(dtype=torch.int32, device=dev)
    r = {
        "counts": torch.empty((E,), **i32),
        "offsets": torch.empty((E + 1,), **i32),
        "perm_tok": torch.empty((T * k,), **i32),
        "slot_pos": torch.empty((T * k,), **i32),
        "active": torch.empty((E + 1,), **i32),
    }
    check(lib().moe_permute(idx32.data_ptr(), T, k, E, r["counts"].data_ptr(),
                            r["offsets"].data_ptr(), r["perm_tok"].data_ptr(),
                            r["slot_pos"].data_ptr(), r["active"].data_ptr(), _stream(dev)),
          "permute")
    return r


# ----------------------------------------------------------------------------- K4/K5
def expert_table(experts: Sequence[Optional[MoeNf4Expert]]):
    """ctypes array of ``moe_nf4_expert_t`` (None -> an all-null, absent expert)."""
    if len(experts) > _lib.MOE_MAX_EXPERTS:
        raise ValueError(f"at most {_lib.MOE_MAX_EXPERTS} experts per call")
    arr = (MoeNf4Expert * max(1, len(experts)))()
    for i, e in enumerate(experts):
        if e is not None:
            arr[i] = e
    return arr


def choose_nsplit(T: int, k: int, E: int, H: int, F: int) -> int:
    """The library's default number of down-projection K splits (ypart planes) for a layer
    of T tokens, top-k k, E experts and hidden/FFN sizes H/F."""
    n = lib().moe_layer_down_splits(T, k, E, H, F)
    if n < 1:
        raise ValueError(f"invalid layer sizes T={T} k={k} E={E} H={H} F={F}")
    return n


def expert_ffn(table, num_experts: int, x: torch.Tensor, k: int, hidden: int, inter: int,
               route: dict, nsplit: Optional[int] = None):
    """K4 on routed rows: returns (h bf16 [T*k, F], ypart fp32 [nsplit, T*k, H])."""
    dev = x.device
    _require(x, "hidden_states", torch.bfloat16, dev)
    T = x.shape[0]
    if nsplit is None:
        nsplit = choose_nsplit(T, k, num_experts, hidden, inter)
    h = torch.empty((T * k, inter), dtype=torch.bfloat16, device=dev)
    ypart = torch.empty((nsplit, T * k, hidden), dtype=torch.float32, device=dev)
    check(lib().moe_expert_ffn_nf4(table, num_experts, x.data_ptr(), T, k, hidden, inter,
                                   route["counts"].data_ptr(), route["offsets"].data_ptr(),
                                   route["perm_tok"].data_ptr(), route["active"].data_ptr(),
                                   h.data_ptr(), ypart.data_ptr(), nsplit, _stream(dev)),
          "expert_ffn")
    return h, ypart


def combine(ypart: torch.Tensor, weights: torch.Tensor, idx32: torch.Tensor,
            slot_pos: torch.Tensor, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """K5: ascending-expert weighted combine into a bf16 [T, H] output."""
    dev = ypart.device
    _require(ypart, "ypart", torch.float32, dev)
    _require(weights, "weights", torch.float32, dev)
    _require(idx32, "idx32", torch.int32, dev)
    _require(slot_pos, "slot_pos", torch.int32, dev)
    nsplit, rows, H = ypart.shape
    T, k = weights.shape
    if out is None:
        out = torch.empty((T, H), dtype=torch.bfloat16, device=dev)
    check(lib().moe_combine(ypart.data_ptr(), nsplit, weights.data_ptr(), idx32.data_ptr(),
                            slot_pos.data_ptr(), T, k, H, out.data_ptr(), _stream(dev)),
          "combine")
    return out


def expert_swiglu(expert: MoeNf4Expert, x: torch.Tensor, hidden: int, inter: int) -> torch.Tensor:
    """One expert on all rows of x (bf16 [T, H]) -> bf16 [T, H]."""
    dev = x.device
    _require(x, "x", torch.bfloat16, dev)
    if x.ndim != 2 or x.shape[1] != hidden:
        raise ValueError(f"x must be [T, {hidden}] (got {tuple(x.shape)})")
    T = x.shape[0]
    y = torch.empty((T, hidden), dtype=torch.bfloat16, device=dev)
    if T == 0:
        return y
    ws_bytes = lib().moe_expert_workspace_bytes(T, hidden, inter)
    ws = torch.empty((ws_bytes,), dtype=torch.uint8, device=dev)
    one = (MoeNf4Expert * 1)(expert)
    check(lib().moe_expert_swiglu_nf4(one, x.data_ptr(), T, hidden, inter, y.data_ptr(),
                                      ws.data_ptr(), ws_bytes, _stream(dev)), "expert_swiglu")
    return y


def layer_forward(table, num_experts: int, gate: torch.Tensor, x: torch.Tensor, k: int,
                  inter: int, bias: Optional[torch.Tensor] = None, want_logits: bool = False,
                  out: Optional[torch.Tensor] = None, workspace: Optional[torch.Tensor] = None):
    """Whole MoE layer (K2->K3->K4->K5) on resident experts.

    Returns (out bf16 [T,H], logits bf16 [T,E] | None, weights fp32 [T,k], idx int64 [T,k]).
    """
    dev = x.device
    _require(x, "hidden_states", torch.bfloat16, dev)
    _require(gate, "gate_weight", torch.bfloat16, dev)
    T, H = x.shape
    E = int(num_experts)
    if gate.shape != (E, H):
        raise ValueError(f"gate must be [{E}, {H}] (got {tuple(gate.shape)})")
    if bias is not None:
        _require(bias, "bias", torch.float32, dev)
    ws_bytes = lib().moe_layer_workspace_bytes(T, k, E, H, inter)
    if workspace is None or workspace.numel() < ws_bytes:
        workspace = torch.empty((max(ws_bytes, 1),), dtype=torch.uint8, device=dev)
    if out is None:
        out = torch.empty((T, H), dtype=torch.bfloat16, device=dev)
    logits = torch.empty((T, E), dtype=torch.bfloat16, device=dev) if want_logits else None
    w = torch.empty((T, k), dtype=torch.float32, device=dev)
    idx = torch.empty((T, k), dtype=torch.int64, device=dev)
    check(lib().moe_layer_forward_nf4(table, E, gate.data_ptr(), _ptr(bias), x.data_ptr(), T, H,
                                      inter, k, out.data_ptr(), _ptr(logits), w.data_ptr(),
                                      idx.data_ptr(), workspace.data_ptr(), workspace.numel(),
                                      _stream(dev)), "layer_forward")
    return out, logits, w, idx


# ----------------------------------------------------------------------------- batched serving
# These calls are short (a decode step makes dozens, most of a few us on the device), so their
# checks are written for the host's time: what is right takes one expression per tensor, and only
# what is not goes through the functions that say why.  The stream is the raw handle of
# torch.cuda.current_stream, without the Python object around it (0.1 instead of 1.9 us).  Of the
# 8 to 10 us of a call, the launch takes 4.
_BF16, _F32, _I32 = torch.bfloat16, torch.float32, torch.int32


def _launch(fn, what: str, dev: torch.device, *args) -> None:
    """Calls an entry point with the current stream of ``dev``, on that device (whose sizes the
    launch is planned for, and whose default stream it may be)."""
    index = dev.index
    if torch._C._cuda_getDevice() == index:
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    if rc:
        check(rc, what)


def _plain(t: torch.Tensor, name: str, dtype: torch.dtype, dev: torch.device, shape=None) -> int:
    """The address of a contiguous tensor of this type, device and (unless None) shape."""
    if not (isinstance(t, torch.Tensor) and t.dtype is dtype and t.device == dev and t.is_contiguous()):
        _require(t, name, dtype, dev)
    if shape is not None and t.shape != shape:
        raise ValueError(f"{name} must be {list(shape)} (got {tuple(t.shape)})")
    return t.data_ptr()


def _rows(t: torch.Tensor, name: str, dev: torch.device, ndim: int) -> int:
    """The stride of the rows of a bf16 tensor [rows, ...] whose rows are contiguous, but not
    necessarily next to each other (a slice of a projection's output)."""
    if isinstance(t, torch.Tensor) and t.dtype is _BF16 and t.device == dev and t.ndim == ndim and t.is_contiguous():
        n = t.shape[0]
        if n > 1:
            return t.stride(0)
        if n == 1:
            return (t.numel() + 7) // 8 * 8  # (there is no other row)
    _require_cuda(t, name)
    if t.dtype is not _BF16:
        raise ValueError(f"{name} must be {_BF16} (got {t.dtype})")
    if t.device != dev:
        raise ValueError(f"{name} device {t.device} != {dev}")
    shape, strides = t.shape, t.stride()
    if len(shape) != ndim:
        raise ValueError(f"{name} must have {ndim} dimensions (got {tuple(shape)})")
    row = 1
    for n, stride in zip(shape[:0:-1], strides[:0:-1]):
        if stride != row and n > 1:
            raise ValueError(f"{name} must have contiguous rows (got strides {strides})")
        row *= n
    return strides[0] if shape[0] > 1 else (row + 7) // 8 * 8


def _pages(k_cache: torch.Tensor, v_cache: torch.Tensor, dev: torch.device):
    """(page stride, shape) of a paged cache (k and v [pages, kv heads, page size, head dim], whole
    pages at one stride)."""
    if (isinstance(k_cache, torch.Tensor) and isinstance(v_cache, torch.Tensor) and k_cache.dtype is _BF16
            and v_cache.dtype is _BF16 and k_cache.device == dev and v_cache.device == dev
            and k_cache.is_contiguous() and v_cache.is_contiguous()):
        shape = k_cache.shape
        if len(shape) == 4 and shape[0] > 1 and v_cache.shape == shape:
            _, heads, size, hd = shape
            return heads * size * hd, shape
    stride = _rows(k_cache, "k_cache", dev, 4)
    if _rows(v_cache, "v_cache", dev, 4) != stride or k_cache.shape != v_cache.shape:
        raise ValueError(f"k_cache {tuple(k_cache.shape)} of page stride {stride} and v_cache {tuple(v_cache.shape)} of "
                         f"page stride {v_cache.stride(0)} differ")
    return stride, k_cache.shape


def _out(out: Optional[torch.Tensor], name: str, like: torch.Tensor, *shape) -> torch.Tensor:
    """A caller's output, checked for its number of elements, or a new one (new_empty with sizes of
    its own takes 1.2 us, torch.empty 1.6)."""
    if out is None:
        return like.new_empty(*shape)
    _plain(out, name, like.dtype, like.device)
    n = 1
    for s in shape:
        n *= s
    if out.numel() != n:
        raise ValueError(f"{name} has the wrong number of elements")
    return out


def rope_paged_kv(qkv: torch.Tensor, positions: torch.Tensor, page_table: torch.Tensor, k_cache: torch.Tensor,
                  v_cache: torch.Tensor, n_q_heads: int, inv_freq: torch.Tensor,
                  seq_ids: Optional[torch.Tensor] = None, q_out: Optional[torch.Tensor] = None,
                  want_k: bool = False, slots: Optional[torch.Tensor] = None):
    """Rotary embedding of new tokens of many sequences, their keys and values written to the
    sequences' pages (``k_cache`` / ``v_cache`` [pages, kv heads, page size, head dim], bf16;
    ``page_table`` int32 [sequences, pages per sequence]).

    ``qkv`` bf16 [T, (q heads + 2 kv heads) * head dim]; token t stands at ``positions[t]`` (int32)
    of sequence ``seq_ids[t]`` (int32; None: sequence t), its key and value at place ``slots[t]``
    (int32; None: its position; the tokens of a drafted tree lie one behind the other, several of
    them at one position).  ``inv_freq`` fp32 [head dim / 2].
    Returns (rotated q bf16 [T, q heads * head dim], rotated k bf16 [T, kv heads, head dim] | None).
    Tokens at negative positions are padding: their rows, here and in the cache, are left as they
    were.  A token whose page the table (or the cache) does not have is rotated, not cached.  No
    two tokens of a call may have one place."""
    _require_cuda(qkv, "qkv")
    dev = qkv.device
    stride = _rows(qkv, "qkv", dev, 2)
    page_stride, (pages, nkv, size, hd) = _pages(k_cache, v_cache, dev)
    T, row = qkv.shape
    nq = int(n_q_heads)
    if row != (nq + 2 * nkv) * hd:
        raise ValueError(f"qkv rows have {row} values, {nq} query and {nkv} KV heads of {hd} need {(nq + 2 * nkv) * hd}")
    table = _plain(page_table, "page_table", _I32, dev)
    table_shape = page_table.shape
    if len(table_shape) != 2:
        raise ValueError("page_table must be [sequences, pages]")
    n_seqs, width = table_shape
    pos = _plain(positions, "positions", _I32, dev, (T,))
    freq = _plain(inv_freq, "inv_freq", _F32, dev, (hd // 2,))
    seqs = None if seq_ids is None else _plain(seq_ids, "seq_ids", _I32, dev, (T,))
    q_out = _out(q_out, "q_out", qkv, T, nq * hd)
    k_out = qkv.new_empty(T, nkv, hd) if want_k else None
    if slots is not None:
        _launch(lib().moe_rope_paged_kv_slots_bf16, "rope_paged_kv", dev, qkv.data_ptr(), stride, T, nq, nkv, hd, freq,
                pos, _plain(slots, "slots", _I32, dev, (T,)), seqs, table, n_seqs, width, pages, size, page_stride,
                q_out.data_ptr(), _ptr(k_out), k_cache.data_ptr(), v_cache.data_ptr())
        return q_out, k_out
    _launch(lib().moe_rope_paged_kv_bf16, "rope_paged_kv", dev, qkv.data_ptr(), stride, T, nq, nkv, hd, freq, pos, seqs,
            table, n_seqs, width, pages, size, page_stride, q_out.data_ptr(), _ptr(k_out), k_cache.data_ptr(),
            v_cache.data_ptr())
    return q_out, k_out


def paged_attention_workspace(batch: int, n_q_heads: int, n_kv_heads: int, head_dim: int, device) -> torch.Tensor:
    """Workspace of ``paged_attention`` for batches of up to ``batch`` sequences: made once, then
    shared by calls that run one after the other (one stream)."""
    n = lib().moe_paged_attention_workspace_bytes(batch, n_q_heads, n_kv_heads, head_dim)
    if n < 0:
        raise ValueError(f"invalid attention sizes batch={batch} heads={n_q_heads}/{n_kv_heads} head_dim={head_dim}")
    return torch.zeros((n,), dtype=torch.uint8, device=device)


def paged_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, page_table: torch.Tensor,
                    lens: torch.Tensor, scaling: Optional[float] = None, out: Optional[torch.Tensor] = None,
                    workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of one new token per sequence, ``q`` bf16 [B, q heads, head dim], against the first
    ``lens[b]`` (int32) keys of its pages; bf16 [B, q heads, head dim].  ``scaling`` defaults to
    head_dim ** -0.5.  Rows without keys (padding of a batch) are zeros.  ``workspace``
    (``paged_attention_workspace``) saves the call making one."""
    _require_cuda(q, "q")
    dev = q.device
    stride = _rows(q, "q", dev, 3)
    page_stride, (pages, nkv, size, hd) = _pages(k_cache, v_cache, dev)
    B, nq, q_dim = q.shape
    if q_dim != hd:
        raise ValueError(f"q has head dim {q_dim}, the cache {hd}")
    table = _plain(page_table, "page_table", _I32, dev)
    table_shape = page_table.shape
    if len(table_shape) != 2 or table_shape[0] != B:
        raise ValueError(f"page_table must have {B} rows of pages (got {tuple(table_shape)})")
    n = _plain(lens, "lens", _I32, dev, (B,))
    out = _out(out, "out", q, B, nq, hd)
    if workspace is None:
        workspace = paged_attention_workspace(B, nq, nkv, hd, dev)
    _launch(lib().moe_paged_attention_bf16, "paged_attention", dev, q.data_ptr(), stride, k_cache.data_ptr(),
            v_cache.data_ptr(), pages, size, page_stride, table, table_shape[1], n, B, nq, nkv, hd,
            hd ** -0.5 if scaling is None else scaling, out.data_ptr(),
            _plain(workspace, "workspace", torch.uint8, dev), workspace.numel())
    return out


def packed_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens: torch.Tensor,
                     scaling: Optional[float] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Causal attention of whole sequences packed one behind the other: sequence b is tokens
    ``cu_seqlens[b] .. cu_seqlens[b + 1] - 1`` (int32 [B + 1], not decreasing) of ``q`` bf16
    [T, q heads, head dim] and ``k``, ``v`` [T, kv heads, head dim], whose rows may lie apart (slices of
    a projection's output); bf16 [T, q heads, head dim].  ``scaling`` defaults to head_dim ** -0.5.
    Tokens of no sequence are left as they were in ``out`` (without one they hold anything)."""
    _require_cuda(q, "q")
    dev = q.device
    q_stride, k_stride, v_stride = _rows(q, "q", dev, 3), _rows(k, "k", dev, 3), _rows(v, "v", dev, 3)
    T, nq, hd = q.shape
    if k.shape != v.shape or k.shape[0] != T or k.shape[2] != hd:
        raise ValueError(f"q {tuple(q.shape)}, k {tuple(k.shape)} and v {tuple(v.shape)} do not fit")
    cu = _plain(cu_seqlens, "cu_seqlens", _I32, dev)
    if cu_seqlens.ndim != 1 or cu_seqlens.numel() < 1:
        raise ValueError(f"cu_seqlens must be [sequences + 1] (got {tuple(cu_seqlens.shape)})")
    out = _out(out, "out", q, T, nq, hd)
    _launch(lib().moe_packed_attention_bf16, "packed_attention", dev, q.data_ptr(), q_stride, k.data_ptr(), k_stride,
            v.data_ptr(), v_stride, T, cu, cu_seqlens.numel() - 1, nq, k.shape[1], hd,
            hd ** -0.5 if scaling is None else scaling, out.data_ptr())
    return out


def sample_tokens(logits: torch.Tensor, u: torch.Tensor, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0,
                  out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The next token (int64 [B]) of each row of ``logits`` (bf16 or fp32 [B, V], rows may lie apart),
    drawn by the row's random number ``u`` (fp32 [B], in [0, 1)).

    Weights are e^((x - max) / temperature).  By falling logit (equal ones by rising index) the first
    ``top_k`` tokens are kept (0: all), of those the shortest prefix that reaches ``top_p`` of their
    weight, of those the ones of at least ``min_p`` times the largest; the token is the first, by
    rising index, at which the kept weights add up to more than ``u`` of their sum.  Temperature 0
    gives the largest logit.  -inf and NaN are never drawn; a row of nothing else gives -1.  Each
    setting is a number, or a tensor with a value per row (fp32; ``top_k`` int32)."""
    _require_cuda(logits, "logits")
    dev, f32 = logits.device, logits.dtype is _F32
    if not f32 and logits.dtype is not _BF16:
        raise ValueError(f"logits must be {_BF16} or {_F32} (got {logits.dtype})")
    if logits.ndim != 2 or (logits.stride(1) != 1 and logits.shape[1] > 1):
        raise ValueError(f"logits must be [rows, vocabulary] with contiguous rows (got {tuple(logits.shape)}, "
                         f"strides {logits.stride()})")
    B, V = logits.shape
    shape = (B,)
    numbers = _plain(u, "u", _F32, dev, shape)
    if out is None:
        out = torch.empty(shape, dtype=torch.int64, device=dev)
    else:
        _plain(out, "out", torch.int64, dev)
        if out.numel() != B:
            raise ValueError("out has the wrong number of elements")
    tensor = torch.Tensor
    t = k = p = m = None
    if isinstance(temperature, tensor):
        t, temperature = _plain(temperature, "temperature", _F32, dev, shape), 1.0
    if isinstance(top_k, tensor):
        k, top_k = _plain(top_k, "top_k", _I32, dev, shape), 0
    if isinstance(top_p, tensor):
        p, top_p = _plain(top_p, "top_p", _F32, dev, shape), 1.0
    if isinstance(min_p, tensor):
        m, min_p = _plain(min_p, "min_p", _F32, dev, shape), 0.0
    _launch(lib().moe_sample_tokens, "sample_tokens", dev, logits.data_ptr(), int(f32), logits.stride(0) if B > 1 else V,
            B, V, numbers, t, temperature, k, top_k, p, top_p, m, min_p, out.data_ptr())
    return out


# ----------------------------------------------------------------------------- decoding that branches
_I64 = torch.int64


def _int32(v, name: str) -> int:
    """A number that an entry point takes in 32 bits."""
    v = int(v)
    if not -1 << 31 <= v < 1 << 31:
        raise ValueError(f"{name} must fit 32 bits (got {v})")
    return v


def _layers(k_cache: torch.Tensor, v_cache: torch.Tensor):
    """(layers, layer stride, page stride, shape of a layer) of paged caches: of one layer as in
    ``_pages``, or of several ([layers, pages, kv heads, page size, head dim])."""
    if (isinstance(k_cache, torch.Tensor) and isinstance(v_cache, torch.Tensor) and k_cache.ndim == 5 and k_cache.is_cuda
            and k_cache.dtype is _BF16 and v_cache.dtype is _BF16 and k_cache.device == v_cache.device
            and k_cache.is_contiguous() and v_cache.is_contiguous()):
        shape = k_cache.shape
        if v_cache.shape == shape:
            layers, pages, heads, size, hd = shape
            row = heads * size * hd
            return layers, pages * row, row, (pages, heads, size, hd)
    _require_cuda(k_cache, "k_cache")
    dev, ndim = k_cache.device, k_cache.ndim
    if ndim == 4:
        stride, shape = _pages(k_cache, v_cache, dev)
        return 1, 0, stride, shape
    if ndim != 5:
        raise ValueError(f"k_cache must have 4 or 5 dimensions (got {tuple(k_cache.shape)})")
    _require_cuda(v_cache, "v_cache")
    if v_cache.dtype is not _BF16 or v_cache.device != dev:
        raise ValueError(f"v_cache must be {_BF16} on {dev} (got {v_cache.dtype} on {v_cache.device})")
    if k_cache.shape != v_cache.shape or k_cache.stride() != v_cache.stride():
        raise ValueError(f"k_cache {tuple(k_cache.shape)} of strides {k_cache.stride()} and v_cache "
                         f"{tuple(v_cache.shape)} of strides {v_cache.stride()} differ")
    shape = k_cache.shape[1:]
    if k_cache.shape[0] == 0:
        return 0, 0, shape[1] * shape[2] * shape[3], shape
    return k_cache.shape[0], k_cache.stride(0), _rows(k_cache[0], "k_cache", dev, 4), shape


def paged_tree_attention_workspace(batch: int, n_q_heads: int, n_kv_heads: int, head_dim: int, device) -> torch.Tensor:
    """Workspace of ``paged_tree_attention`` for batches of any size: made once, then shared by calls
    that run one after the other (one stream)."""
    n = lib().moe_paged_tree_attention_workspace_bytes(batch, _int32(n_q_heads, "n_q_heads"),
                                                       _int32(n_kv_heads, "n_kv_heads"), _int32(head_dim, "head_dim"))
    if n < 0:
        raise ValueError(f"invalid attention sizes batch={batch} heads={n_q_heads}/{n_kv_heads} head_dim={head_dim}")
    return torch.empty((n,), dtype=torch.uint8, device=device)


def paged_tree_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, page_table: torch.Tensor,
                         lens: torch.Tensor, cu_seqlens: torch.Tensor, masks: Optional[torch.Tensor] = None,
                         scaling: Optional[float] = None, out: Optional[torch.Tensor] = None,
                         workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of drafted tokens, ``q`` bf16 [T, q heads, head dim], against the paged keys of their
    sequences; bf16 [T, q heads, head dim].  Sequence b's (up to 64) are rows ``cu_seqlens[b] ..
    cu_seqlens[b + 1] - 1`` (int32 [B + 1]); each sees the sequence's first ``lens[b]`` (int32) keys, and
    the key at place ``lens[b] + j`` if bit j of its mask is set (``masks`` int64 [T]; None: a chain,
    each sees the drafted ones up to itself).  ``scaling`` defaults to head_dim ** -0.5.  Rows without
    keys are zeros, rows of no sequence are left as they were in ``out`` (without one they hold
    anything).  ``workspace`` (``paged_tree_attention_workspace``) saves the call making one."""
    _require_cuda(q, "q")
    dev = q.device
    stride = _rows(q, "q", dev, 3)
    page_stride, (pages, nkv, size, hd) = _pages(k_cache, v_cache, dev)
    T, nq, q_dim = q.shape
    if q_dim != hd:
        raise ValueError(f"q has head dim {q_dim}, the cache {hd}")
    cu = _plain(cu_seqlens, "cu_seqlens", _I32, dev)
    if cu_seqlens.ndim != 1 or cu_seqlens.numel() < 1:
        raise ValueError(f"cu_seqlens must be [sequences + 1] (got {tuple(cu_seqlens.shape)})")
    B = cu_seqlens.numel() - 1
    table = _plain(page_table, "page_table", _I32, dev)
    table_shape = page_table.shape
    if len(table_shape) != 2 or table_shape[0] != B:
        raise ValueError(f"page_table must have {B} rows of pages (got {tuple(table_shape)})")
    n = _plain(lens, "lens", _I32, dev, (B,))
    seen = None if masks is None else _plain(masks, "masks", _I64, dev, (T,))
    out = _out(out, "out", q, T, nq, hd)
    if workspace is None:
        workspace = paged_tree_attention_workspace(B, nq, nkv, hd, dev)
    _launch(lib().moe_paged_tree_attention_bf16, "paged_tree_attention", dev, q.data_ptr(), stride, T,
            k_cache.data_ptr(), v_cache.data_ptr(), pages, size, page_stride, table, table_shape[1], n, cu, seen, B, nq,
            nkv, hd, hd ** -0.5 if scaling is None else scaling, out.data_ptr(),
            _plain(workspace, "workspace", torch.uint8, dev), workspace.numel())
    return out


def accept_drafts(targets: torch.Tensor, drafts: torch.Tensor, cu_seqlens: torch.Tensor,
                  masks: Optional[torch.Tensor] = None):
    """Which drafted tokens the model itself would have chosen: ``targets`` (int64 [T]) are its choices
    after each, ``drafts`` (int64 [T]) the tokens, ``cu_seqlens`` and ``masks`` as in
    ``paged_tree_attention``; a token's parent is the last one before it in its mask.  The first of a
    sequence is accepted, another one if its parent is and its token is the choice after the parent.
    Returns, for the first of the longest accepted paths, (its tokens as bits int64 [B], their number
    int32 [B], the choice after the last of them int64 [B]); 0, 0, -1 for sequences without tokens."""
    _require_cuda(targets, "targets")
    dev = targets.device
    if targets.ndim != 1:
        raise ValueError(f"targets must be [tokens] (got {tuple(targets.shape)})")
    t = _plain(targets, "targets", _I64, dev)
    shape = targets.shape
    d = _plain(drafts, "drafts", _I64, dev, shape)
    m = None if masks is None else _plain(masks, "masks", _I64, dev, shape)
    cu = _plain(cu_seqlens, "cu_seqlens", _I32, dev)
    if cu_seqlens.ndim != 1 or cu_seqlens.numel() < 1:
        raise ValueError(f"cu_seqlens must be [sequences + 1] (got {tuple(cu_seqlens.shape)})")
    B = cu_seqlens.numel() - 1
    paths, counts, tokens = targets.new_empty(B), cu_seqlens.new_empty(B), targets.new_empty(B)
    _launch(lib().moe_accept_drafts, "accept_drafts", dev, t, d, m, cu, shape[0], B, paths.data_ptr(),
            counts.data_ptr(), tokens.data_ptr())
    return paths, counts, tokens


def compact_paged_kv(k_cache: torch.Tensor, v_cache: torch.Tensor, page_table: torch.Tensor, lens: torch.Tensor,
                     paths: torch.Tensor) -> None:
    """Keys and values of accepted tokens moved to where they belong, in place: of the set bits s_0 < s_1
    < .. of ``paths[b]`` (int64 [B], from ``accept_drafts``), place ``lens[b] + s_j`` (int32 [B]) of
    sequence b goes to place ``lens[b] + j``.  The caches are of one layer, or of all ([layers, pages,
    kv heads, page size, head dim], pages and layers at strides of their own)."""
    layers, layer_stride, page_stride, (pages, nkv, size, hd) = _layers(k_cache, v_cache)
    dev = k_cache.device
    table = _plain(page_table, "page_table", _I32, dev)
    table_shape = page_table.shape
    if len(table_shape) != 2:
        raise ValueError("page_table must be [sequences, pages]")
    B = table_shape[0]
    _launch(lib().moe_compact_paged_kv_bf16, "compact_paged_kv", dev, k_cache.data_ptr(), v_cache.data_ptr(), layers,
            layer_stride, pages, size, page_stride, nkv, hd, table, B, table_shape[1],
            _plain(lens, "lens", _I32, dev, (B,)), _plain(paths, "paths", _I64, dev, (B,)))


def beam_select_workspace(searches: int, beams: int, k: int, device) -> torch.Tensor:
    """Workspace of ``beam_select`` for so many searches: made once, then shared by calls that run one
    after the other (one stream)."""
    n = lib().moe_beam_select_workspace_bytes(searches, beams, _int32(k, "k"))
    if n < 0:
        raise ValueError(f"invalid sizes searches={searches} beams={beams} k={k}")
    ws = torch.empty((n,), dtype=torch.uint8, device=device)
    ws[:65536].zero_()
    return ws


def beam_select(logits: torch.Tensor, scores: torch.Tensor, k: int, workspace: Optional[torch.Tensor] = None):
    """The ``k`` best continuations of each search: of all its beams and all tokens those of the largest
    ``scores[s, w] + log_softmax(logits[s * W + w])``; ``logits`` bf16 or fp32 [S * W, V] (rows may lie
    apart), ``scores`` fp32 [S, W], sums over the vocabulary in 64 bits.  Returns (totals fp32 [S, k],
    falling; the rows of ``logits`` that go on, int32 [S, k]; tokens int64 [S, k]).  Equal ones go by beam,
    inside it by logit, then token.  -inf and NaN are never chosen; a score of -inf is no beam (a search's
    first step has one), nor is a beam whose logits hold +inf; what there is too little for is -inf, -1, -1."""
    _require_cuda(logits, "logits")
    dev, f32 = logits.device, logits.dtype is _F32
    if not f32 and logits.dtype is not _BF16:
        raise ValueError(f"logits must be {_BF16} or {_F32} (got {logits.dtype})")
    if logits.ndim != 2 or (logits.stride(1) != 1 and logits.shape[1] > 1):
        raise ValueError(f"logits must be [rows, vocabulary] with contiguous rows (got {tuple(logits.shape)}, "
                         f"strides {logits.stride()})")
    base = _plain(scores, "scores", _F32, dev)
    if scores.ndim != 2 or scores.numel() != logits.shape[0]:
        raise ValueError(f"scores must be [searches, beams] of {logits.shape[0]} rows (got {tuple(scores.shape)})")
    (S, W), (rows, V) = scores.shape, logits.shape
    k = _int32(k, "k")
    if workspace is None:
        workspace = beam_select_workspace(S, W, k, dev)
    best = scores.new_empty(S, max(k, 0))
    beam = torch.empty((S, max(k, 0)), dtype=_I32, device=dev)
    token = torch.empty((S, max(k, 0)), dtype=_I64, device=dev)
    _launch(lib().moe_beam_select, "beam_select", dev, logits.data_ptr(), int(f32), logits.stride(0) if rows > 1 else V,
            S, W, V, base, k, best.data_ptr(), beam.data_ptr(), token.data_ptr(),
            _plain(workspace, "workspace", torch.uint8, dev), workspace.numel())
    return best, beam, token


def fork_pages_workspace(pages: int, device) -> torch.Tensor:
    """Workspace of ``fork_pages`` for a cache of so many pages: made once, then shared by calls that run
    one after the other (one stream)."""
    n = lib().moe_fork_pages_workspace_bytes(pages)
    if n < 0:
        raise ValueError(f"invalid number of pages {pages}")
    return torch.zeros((n,), dtype=torch.uint8, device=device)


def fork_pages(page_table: torch.Tensor, lens: torch.Tensor, parents: torch.Tensor, refs: torch.Tensor,
               page_size: int, ahead: int = 1, out=None, workspace: Optional[torch.Tensor] = None):
    """Page table rows taken over by the sequences that continue (beams reordered, forked, dropped):
    new row i goes on from row ``parents[i]`` (int32 [N]) of ``page_table`` (int32 [B, width]) and ``lens``
    (int32 [B]); any other number than a row's makes an empty one.  ``refs`` (int32 [pages], in place)
    counts the holders of each page; pages of no holder are free.  The places of the next ``ahead``
    positions become each row's alone: what others hold too is replaced by the lowest free page.

    Returns (table int32 [N, width], lens int32 [N], copies int32 [N, 3], missing int32 [1]); ``out`` is
    such a tuple to write to.  ``copies`` are for ``copy_pages``: (page, new page, positions in use), or
    (-1, -1, 0).  ``missing`` counts places for which no page was free: -1 in the table
    (also where the row shared a partly filled page: its keys there are lost to it)."""
    _require_cuda(page_table, "page_table")
    dev = page_table.device
    table = _plain(page_table, "page_table", _I32, dev)
    if page_table.ndim != 2 or parents.ndim != 1 or refs.ndim != 1:
        raise ValueError(f"page_table must be [sequences, pages], parents [rows], refs [pages] (got "
                         f"{tuple(page_table.shape)}, {tuple(parents.shape)}, {tuple(refs.shape)})")
    B, width = page_table.shape
    N, pages = parents.shape[0], refs.shape[0]
    n = _plain(lens, "lens", _I32, dev, (B,))
    page_size, ahead = _int32(page_size, "page_size"), _int32(ahead, "ahead")
    if out is None:
        out = (page_table.new_empty(N, width), page_table.new_empty(N), page_table.new_empty(N, 3),
               page_table.new_empty(1))
    if workspace is None:
        workspace = fork_pages_workspace(pages, dev)
    _launch(lib().moe_fork_pages, "fork_pages", dev, table, n, B, width, _plain(parents, "parents", _I32, dev), N,
            _plain(refs, "refs", _I32, dev), pages, page_size, ahead, _plain(out[0], "table", _I32, dev, (N, width)),
            _plain(out[1], "lens", _I32, dev, (N,)), _plain(out[2], "copies", _I32, dev, (N, 3)),
            _plain(out[3], "missing", _I32, dev, (1,)), _plain(workspace, "workspace", torch.uint8, dev),
            workspace.numel())
    return out


def copy_pages(k_cache: torch.Tensor, v_cache: torch.Tensor, copies: torch.Tensor) -> None:
    """The first ``copies[i, 2]`` positions of page ``copies[i, 0]`` copied to page ``copies[i, 1]`` (int32
    [N, 3], from ``fork_pages``; pairs of pages that are not there are none), keys and values, in all
    layers (caches as in ``compact_paged_kv``)."""
    layers, layer_stride, page_stride, (pages, nkv, size, hd) = _layers(k_cache, v_cache)
    dev = k_cache.device
    pairs = _plain(copies, "copies", _I32, dev)
    if copies.ndim != 2 or copies.shape[1] != 3:
        raise ValueError(f"copies must be [copies, 3] (got {tuple(copies.shape)})")
    _launch(lib().moe_copy_pages_bf16, "copy_pages", dev, k_cache.data_ptr(), v_cache.data_ptr(), layers, layer_stride,
            pages, size, page_stride, nkv, hd, pairs, copies.shape[0])
