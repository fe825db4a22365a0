"""Performance cases of the batched serving operators: what a program that serves many
sequences at once has the framework do between its projections, each operator in its plain
form (elementary torch operations) and through the framework's own entry points.

Kinds of case:
  append  rope_paged_kv: the rotary embedding of new tokens' queries and keys, keys and values
          written to the sequences' pages.
  paged   paged_attention: one new token per sequence against its paged keys and values.
  packed  packed_attention: causal attention of whole prompts of different lengths, packed one
          behind the other.
  sample  sample_tokens: the next token of each row of logits, by temperature, top-k, top-p and
          min-p from a given random number.
"""
from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

DEV = "cuda:0"
THETA = 1e6


# ------------------------------------------------------------------ cases
def listed():
    mix = {"q_heads": 32, "kv_heads": 8, "head_dim": 128}   # the benchmark model's attention
    small = {"q_heads": 8, "kv_heads": 2, "head_dim": 64}   # a small model's
    return [
        # A step of a few conversations: one token each, where the launch is what it costs.
        {"name": "append_step_8", "kind": "append", "seqs": 8, "tokens": 8, "page": 16, "far": 4000,
         "with_k": False, **mix},
        # A step of a full server, far into long conversations.
        {"name": "append_step_256", "kind": "append", "seqs": 256, "tokens": 256, "page": 64, "far": 131072,
         "with_k": False, **mix},
        # Prompts of different lengths on their way into the cache, their keys also kept packed.
        {"name": "append_prompts_8192", "kind": "append", "seqs": 7, "tokens": 8192, "page": 64, "far": 0,
         "with_k": True, **mix},
        # One conversation, short context: latency.
        {"name": "paged_1x700", "kind": "paged", "seqs": 1, "longest": 700, "ragged": 0, "pad": 0, "page": 16, **mix},
        # A batch of very different lengths, rows of padding among them (a step captured for 40).
        {"name": "paged_40_ragged", "kind": "paged", "seqs": 40, "longest": 9001, "ragged": 3, "pad": 5,
         "page": 16, **mix},
        # Long contexts: the bandwidth of the device.
        {"name": "paged_16x32768", "kind": "paged", "seqs": 16, "longest": 32768, "ragged": 0, "pad": 0,
         "page": 64, **mix},
        # Three questions of a small model.
        {"name": "packed_41", "kind": "packed", "tokens": 41, "seqs": 3, "ragged": 5, **small},
        # Prompts of a paragraph to a few pages.
        {"name": "packed_3333", "kind": "packed", "tokens": 3333, "seqs": 9, "ragged": 11, **mix},
        # Documents.
        {"name": "packed_16384", "kind": "packed", "tokens": 16384, "seqs": 3, "ragged": 2, **mix},
        # One conversation's token.
        {"name": "sample_1_topk", "kind": "sample", "rows": 1, "vocab": 32000, "dtype": "bf16", "flat": 0.0,
         "top_k": 50, "top_p": 0.9, "min_p": 0.0, "mixed": False},
        # A batch with nucleus sampling, logits in 32 bits.
        {"name": "sample_64_nucleus", "kind": "sample", "rows": 64, "vocab": 32000, "dtype": "fp32", "flat": 0.0,
         "top_k": 0, "top_p": 0.95, "min_p": 0.0, "mixed": False},
        # A full server, a large vocabulary, every request with settings of its own.
        {"name": "sample_256_mixed", "kind": "sample", "rows": 256, "vocab": 131072, "dtype": "bf16", "flat": 0.5,
         "top_k": 0, "top_p": 1.0, "min_p": 0.0, "mixed": True},
    ]


HEADS = ((32, 8, 128), (32, 8, 128), (8, 2, 64), (16, 16, 64), (32, 4, 128), (24, 8, 128), (16, 1, 128), (8, 4, 256),
         (40, 2, 128), (12, 4, 64))


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("append", "paged", "packed", "sample"))
    nq, nkv, hd = rng.choice(HEADS)
    heads = {"q_heads": nq, "kv_heads": nkv, "head_dim": hd}
    if kind == "append":
        if rng.random() < 0.5:  # a step
            n = _log(rng, 1, 256)
            return {"kind": kind, "seqs": n, "tokens": n, "page": rng.choice((8, 16, 32, 64, 128)),
                    "far": _log(rng, 10, 131072), "with_k": False, **heads}
        most = max(1, 8192 * 48 * 128 // ((nq + 2 * nkv) * hd))
        n = _log(rng, 1, min(most, 8192))
        return {"kind": kind, "seqs": rng.randint(1, min(n, 12)), "tokens": n,
                "page": rng.choice((8, 16, 32, 64, 128)), "far": 0, "with_k": rng.random() < 0.7, **heads}
    if kind == "paged":
        seqs = _log(rng, 1, 128)
        most = max(1, (1 << 31) // (seqs * nkv * hd * 4))
        longest = _log(rng, 1, min(32768, most))
        return {"kind": kind, "seqs": seqs, "longest": longest, "ragged": rng.randint(0, 99),
                "pad": rng.randint(0, seqs // 4), "page": rng.choice((8, 16, 32, 64, 128)), **heads}
    if kind == "packed":
        seqs = _log(rng, 1, 16)
        most = int(math.sqrt(1.4e8 * 32 * 128 / (nq * hd)))  # one sequence of all of them costs no more than the largest
        return {"kind": kind, "tokens": _log(rng, max(seqs, 2), min(most, 16384)), "seqs": seqs,
                "ragged": rng.randint(1, 99), **heads}
    vocab = _log(rng, 300, 131072)
    return {"kind": kind, "rows": _log(rng, 1, 256), "vocab": vocab, "dtype": rng.choice(("bf16", "fp32")) if vocab <= 65536 else "bf16",
            "flat": rng.choice((0.0, 0.5, 1.0)), "top_k": rng.choice((0, 0, 1, 20, 50, 200, 1000)),
            "top_p": rng.choice((1.0, 0.95, 0.9, 0.5)), "min_p": rng.choice((0.0, 0.0, 0.05, 0.2)),
            "mixed": rng.random() < 0.4}


def _paged_lens(case):
    """Keys of each sequence: all the longest, or spread below it; rows of padding have none."""
    n, longest = case["seqs"], case["longest"]
    if not case["ragged"]:
        lens = [longest] * n
    else:
        r = random.Random(case["ragged"])
        lens = [1 + int((longest - 1) * r.random() ** 2) for _ in range(n)]
        lens[r.randrange(n)] = longest
    return [0 if i >= n - case["pad"] else v for i, v in enumerate(lens)]


def _packed_lens(tokens, seqs, seed):
    """Lengths of `seqs` sequences, one token at least, that add up to `tokens`."""
    seqs = min(seqs, tokens)
    r = random.Random(seed)
    cuts = sorted(r.sample(range(1, tokens), seqs - 1)) if seqs > 1 else []
    return [b - a for a, b in zip([0] + cuts, cuts + [tokens])]


# ------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(shape, g, std=1.0):
    return (torch.randn(shape, generator=g, device=DEV) * std).to(torch.bfloat16)


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _inv_freq(hd):
    i = torch.arange(0, hd, 2, dtype=torch.int64).float()
    return (1.0 / (THETA ** (i / hd))).to(DEV)


def prepare(case, seed):
    g = _gen(seed)
    rng = random.Random(seed)
    kind = case["kind"]
    if kind == "sample":
        return _prepare_sample(case, g, rng)
    nq, nkv, hd = case["q_heads"], case["kv_heads"], case["head_dim"]
    st = {"kind": kind, "nq": nq, "nkv": nkv, "hd": hd, "scaling": float(hd ** -0.5)}
    if kind == "append":
        P, n, T = case["page"], case["seqs"], case["tokens"]
        if case["far"]:  # a step: one token per sequence, somewhere
            pos = [rng.randrange(case["far"]) for _ in range(n)]
            owner = list(range(n))
            width = case["far"] // P + 1
            # The pool holds the pages that the step writes (and some others); pages of earlier
            # positions are not read here.
            need = [(i, pos[i] // P) for i in range(n)]
        else:  # whole prompts from position 0
            lens = _packed_lens(T, n, 7 * n + T)
            pos = [p for m in lens for p in range(m)]
            owner = [i for i, m in enumerate(lens) for _ in range(m)]
            width = max(lens) // P + 1
            need = [(i, p) for i, m in enumerate(lens) for p in range((m + P - 1) // P)]
        pages = len(need) + 3
        ids = list(range(pages))
        rng.shuffle(ids)
        table = torch.full((n, width), -1, dtype=torch.int32)
        for (i, p), page in zip(need, ids):
            table[i, p] = page
        st.update(qkv=_randn((T, (nq + 2 * nkv) * hd), g), positions=_i32(pos),
                  seq_ids=None if case["far"] else _i32(owner), table=table.to(DEV), page=P,
                  k_cache=_randn((pages, nkv, P, hd), g), v_cache=_randn((pages, nkv, P, hd), g),
                  inv_freq=_inv_freq(hd), with_k=case["with_k"])
        return st
    if kind == "paged":
        P, lens = case["page"], _paged_lens(case)
        counts = [(v + P - 1) // P for v in lens]
        pages = max(1, sum(counts))
        ids = list(range(pages))
        rng.shuffle(ids)
        table = torch.full((len(lens), max(1, max(counts))), -1, dtype=torch.int32)
        at = 0
        for i, c in enumerate(counts):
            table[i, :c] = torch.tensor(ids[at:at + c], dtype=torch.int32)
            at += c
        # Keys that some queries like better than others: scores with a spread of a few units.
        st.update(q=_randn((len(lens), nq, hd), g, 1.5), k_cache=_randn((pages, nkv, P, hd), g),
                  v_cache=_randn((pages, nkv, P, hd), g), table=table.to(DEV), lens=_i32(lens),
                  host_lens=lens, page=P, workspace=None)
        if own:
            from moeinfra_amd import ops

            st["workspace"] = ops.paged_attention_workspace(len(lens), nq, nkv, hd, DEV)
        return st
    T, lens = case["tokens"], _packed_lens(case["tokens"], case["seqs"], case["ragged"])
    cuts = [0]
    for v in lens:
        cuts.append(cuts[-1] + v)
    qkv = _randn((T, (nq + 2 * nkv) * hd), g)
    # Rotated queries and keys come packed; the values still lie in the projection's output.
    st.update(q=_randn((T, nq, hd), g, 1.5), k=_randn((T, nkv, hd), g),
              v=qkv[:, (nq + nkv) * hd:].view(T, nkv, hd), cu=_i32(cuts), cuts=cuts)
    return st


def _prepare_sample(case, g, rng):
    B, V = case["rows"], case["vocab"]
    # A model's logits: a broad bulk and a few tokens far above it; "flat" is the share of rows
    # without such tokens.
    x = torch.randn((B, V), generator=g, device=DEV) * 2.0
    peaks = torch.randn((B, V), generator=g, device=DEV) > 3.2
    x = x + torch.where(peaks, torch.rand((B, V), generator=g, device=DEV) * 9.0, 0.0) * (
        torch.rand((B, 1), generator=g, device=DEV) >= case["flat"])
    # Some rows may say only part of the vocabulary (a grammar's mask).
    masked = torch.rand((B, 1), generator=g, device=DEV) < 0.25
    gone = torch.rand((B, V), generator=g, device=DEV) < 0.9
    x = torch.where(masked & gone, -math.inf, x)
    x = x.to(torch.bfloat16 if case["dtype"] == "bf16" else torch.float32)
    st = {"kind": "sample", "logits": x, "u": torch.rand((B,), generator=g, device=DEV)}
    if case["mixed"]:
        pick = lambda values, t: torch.tensor([rng.choice(values) for _ in range(B)], dtype=t, device=DEV)
        st.update(temperature=pick((0.0, 0.3, 0.7, 1.0, 1.0, 1.3), torch.float32),
                  top_k=pick((0, 0, 1, 40, 400), torch.int32),
                  top_p=pick((1.0, 1.0, 0.95, 0.8), torch.float32),
                  min_p=pick((0.0, 0.0, 0.1), torch.float32))
    else:
        st.update(temperature=0.8, top_k=case["top_k"], top_p=case["top_p"], min_p=case["min_p"])
    return st


# ------------------------------------------------------------------ one pass
def run(st):
    kind = st["kind"]
    if own:
        from moeinfra_amd import ops

        if kind == "append":
            q, k = ops.rope_paged_kv(st["qkv"], st["positions"], st["table"], st["k_cache"], st["v_cache"],
                                     st["nq"], st["inv_freq"], seq_ids=st["seq_ids"], want_k=st["with_k"])
            out = {"q": q, "k_cache": st["k_cache"], "v_cache": st["v_cache"]}
            return {**out, "k": k} if st["with_k"] else out
        if kind == "paged":
            return ops.paged_attention(st["q"], st["k_cache"], st["v_cache"], st["table"], st["lens"],
                                       scaling=st["scaling"], workspace=st["workspace"])
        if kind == "packed":
            return ops.packed_attention(st["q"], st["k"], st["v"], st["cu"], scaling=st["scaling"])
        return ops.sample_tokens(st["logits"], st["u"], temperature=st["temperature"], top_k=st["top_k"],
                                 top_p=st["top_p"], min_p=st["min_p"])
    return {"append": _plain_append, "paged": _plain_paged, "packed": _plain_packed,
            "sample": _plain_sample}[kind](st)


def _plain_append(st):
    nq, nkv, hd, P = st["nq"], st["nkv"], st["hd"], st["page"]
    x = st["qkv"].float().view(-1, nq + 2 * nkv, hd)
    pos = st["positions"].long()
    # Angles in 64 bits: of far positions 32 bits keep too few digits below a turn.
    ang = pos.double()[:, None] * st["inv_freq"].double()
    cos, sin = torch.cos(ang).float()[:, None], torch.sin(ang).float()[:, None]
    a, b = x[:, :nq + nkv, :hd // 2], x[:, :nq + nkv, hd // 2:]
    r = torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1).to(torch.bfloat16)
    q, k = r[:, :nq].reshape(-1, nq * hd), r[:, nq:]
    owner = torch.arange(x.shape[0], device=DEV) if st["seq_ids"] is None else st["seq_ids"].long()
    page = st["table"][owner, pos // P].long()
    st["k_cache"][page, :, pos % P] = k
    st["v_cache"][page, :, pos % P] = st["qkv"].view(-1, nq + 2 * nkv, hd)[:, nq + nkv:]
    out = {"q": q, "k_cache": st["k_cache"], "v_cache": st["v_cache"]}
    return {**out, "k": k.contiguous()} if st["with_k"] else out


def _plain_paged(st):
    nq, nkv, hd = st["nq"], st["nkv"], st["hd"]
    out = torch.zeros((len(st["host_lens"]), nq, hd), dtype=torch.bfloat16, device=DEV)
    for i, n in enumerate(st["host_lens"]):
        if n == 0:
            continue
        pages = st["table"][i, :(n + st["page"] - 1) // st["page"]].long()
        k = st["k_cache"][pages].transpose(0, 1).reshape(nkv, -1, hd)[:, :n].float()
        v = st["v_cache"][pages].transpose(0, 1).reshape(nkv, -1, hd)[:, :n].float()
        s = torch.matmul(st["q"][i].float().view(nkv, nq // nkv, hd), k.transpose(1, 2)) * st["scaling"]
        e = torch.exp(s - s.amax(dim=-1, keepdim=True))
        o = torch.matmul(e, v) / e.sum(dim=-1, keepdim=True)
        out[i] = o.reshape(nq, hd).to(torch.bfloat16)
    return out


def _plain_packed(st):
    nq, nkv, hd = st["nq"], st["nkv"], st["hd"]
    out = torch.empty_like(st["q"])
    for lo, hi in zip(st["cuts"], st["cuts"][1:]):
        k = st["k"][lo:hi].float().transpose(0, 1)[:, None]                 # [nkv, 1, n, hd]
        v = st["v"][lo:hi].float().transpose(0, 1)[:, None]
        for a in range(lo, hi, 1024):                                       # queries, some at a time
            b = min(a + 1024, hi)
            q = st["q"][a:b].float().view(b - a, nkv, nq // nkv, hd).permute(1, 2, 0, 3)
            s = torch.matmul(q, k[:, :, :b - lo].transpose(2, 3)) * st["scaling"]
            seen = torch.arange(lo, b, device=DEV)[None, :] <= torch.arange(a, b, device=DEV)[:, None]
            s = torch.where(seen, s, -math.inf)
            e = torch.exp(s - s.amax(dim=-1, keepdim=True))
            o = torch.matmul(e, v[:, :, :b - lo]) / e.sum(dim=-1, keepdim=True)
            out[a:b] = o.permute(2, 0, 1, 3).reshape(b - a, nq, hd).to(torch.bfloat16)
    return out


def _plain_sample(st):
    x = st["logits"].double()
    B, V = x.shape
    # (Plain numbers pass through the call in 32 bits.)
    col = lambda v: (v if torch.is_tensor(v) else torch.full((B,), float(v), device=DEV)).double()[:, None]
    T, k, p, mp = (col(st[n]) for n in ("temperature", "top_k", "top_p", "min_p"))
    m = x.amax(dim=1, keepdim=True)
    w = torch.exp((x - m) / torch.where(T > 0, T, 1.0))
    order = torch.sort(x, dim=1, descending=True, stable=True).indices      # ties: lowest index first
    ws = w.gather(1, order)
    rank = torch.arange(V, device=DEV)[None, :]
    ws = torch.where(rank < torch.where(k > 0, k, float(V)), ws, 0.0)
    cum = torch.cumsum(ws, dim=1)
    keep = (cum - ws < p * cum[:, -1:]) & (ws >= mp)
    # Temperature 0 is the first of the order, and so is what lets nothing else through.
    keep = torch.where(T > 0, keep, False) | (rank == 0)
    c = torch.cumsum(torch.zeros_like(w).scatter_(1, order, torch.where(keep, ws, 0.0)), dim=1)
    return (c <= st["u"].double()[:, None] * c[:, -1:]).sum(dim=1)


# ------------------------------------------------------------------ work
def work(case):
    kind = case["kind"]
    if kind == "sample":
        size = 2 if case["dtype"] == "bf16" else 4
        # One difference, one scale, one exponential and one sum per value.
        return {"bytes": case["rows"] * (case["vocab"] * size + 12), "flops": 4 * case["rows"] * case["vocab"]}
    nq, nkv, hd = case["q_heads"], case["kv_heads"], case["head_dim"]
    if kind == "append":
        T = case["tokens"]
        values = T * (2 * (nq + 2 * nkv) + (nkv if case["with_k"] else 0)) * hd
        return {"bytes": 2 * values + 12 * T, "flops": 3 * T * (nq + nkv) * hd}
    if kind == "paged":
        lens = _paged_lens(case)
        return {"bytes": sum(lens) * nkv * hd * 4 + len(lens) * nq * hd * 4, "flops": 4 * nq * hd * sum(lens)}
    lens = _packed_lens(case["tokens"], case["seqs"], case["ragged"])
    return {"bytes": case["tokens"] * (2 * nq + 2 * nkv) * hd * 2,
            "flops": 4 * nq * hd * sum(n * (n + 1) // 2 for n in lens)}


# ------------------------------------------------------------------ the definition in 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    return {"append": _exact_append, "paged": _exact_paged, "packed": _exact_packed,
            "sample": _exact_sample}[case["kind"]](st)


def _exact_append(st):
    nq, nkv, hd, P = st["nq"], st["nkv"], st["hd"], st["page"]
    T, h = st["qkv"].shape[0], hd // 2
    x = st["qkv"].double().reshape(T, nq + 2 * nkv, 2, h)
    pos = st["positions"].cpu().tolist()
    owner = list(range(T)) if st["seq_ids"] is None else st["seq_ids"].cpu().tolist()
    turn = torch.polar(torch.ones((T, h), dtype=torch.double, device=DEV),
                       torch.outer(st["positions"].double(), st["inv_freq"].double()))
    z = torch.complex(x[:, :nq + nkv, 0], x[:, :nq + nkv, 1]) * turn[:, None]
    y = torch.cat((z.real, z.imag), dim=-1)
    kc, vc, table = st["k_cache"].double(), st["v_cache"].double(), st["table"].cpu()
    rows = torch.tensor([int(table[s, t // P]) * P + t % P for s, t in zip(owner, pos)], device=DEV)
    for cache, new in ((kc, y[:, nq:]), (vc, x[:, nq + nkv:].reshape(T, nkv, hd))):
        for n in range(nkv):
            flat = cache[:, n].reshape(-1, hd)
            flat[rows] = new[:, n]
            cache[:, n] = flat.view(-1, P, hd)
    out = {"q": y[:, :nq].reshape(T, nq * hd), "k_cache": kc, "v_cache": vc}
    return {**out, "k": y[:, nq:].contiguous()} if st["with_k"] else out


def _exact_paged(st):
    nq, nkv, hd, P = st["nq"], st["nkv"], st["hd"], st["page"]
    out = torch.zeros((len(st["host_lens"]), nq, hd), dtype=torch.double, device=DEV)
    for i, n in enumerate(st["host_lens"]):
        if n == 0:
            continue
        j = torch.arange(n, device=DEV)
        page = st["table"][i].long()[j // P]
        for h in range(nkv):
            k, v = st["k_cache"][page, h, j % P].double(), st["v_cache"][page, h, j % P].double()
            heads = slice(h * (nq // nkv), (h + 1) * (nq // nkv))
            out[i, heads] = torch.softmax(st["q"][i, heads].double() @ k.t() * st["scaling"], dim=-1) @ v
    return out


def _exact_packed(st):
    nq, nkv, hd = st["nq"], st["nkv"], st["hd"]
    out = torch.empty(st["q"].shape, dtype=torch.double, device=DEV)
    for lo, hi in zip(st["cuts"], st["cuts"][1:]):
        for h in range(nq):
            k, v = (st[n][lo:hi, h // (nq // nkv)].double() for n in ("k", "v"))
            for a in range(lo, hi, 4096):
                b = min(a + 4096, hi)
                s = st["q"][a:b, h].double() @ k[:b - lo].t() * st["scaling"]
                s = s.masked_fill(torch.ones_like(s, dtype=torch.bool).triu(a - lo + 1), -math.inf)
                out[a:b, h] = torch.softmax(s, dim=-1) @ v[:b - lo]
    return out


def _exact_sample(st):
    x = st["logits"].double().cpu().numpy()
    u = st["u"].double().cpu().numpy()
    B, V = x.shape
    par = [v.double().cpu().numpy() if torch.is_tensor(v) else np.full(B, float(v))
           for v in (st["temperature"], st["top_k"], st["top_p"], st["min_p"])]
    # (Scalars pass through the call as fp32 values.)
    par = [np.float32(v).astype(np.float64) if i != 1 else v for i, v in enumerate(par)]
    out = np.empty(B, dtype=np.int64)
    for r in range(B):
        T, k, p, mp = (v[r] for v in par)
        if T <= 0:
            out[r] = int(np.argmax(x[r]))
            continue
        order = np.argsort(-x[r], kind="stable")
        w = np.exp((x[r][order] - x[r][order[0]]) / T)
        if k > 0:
            order, w = order[:int(k)], w[:int(k)]
        c = np.cumsum(w)
        n = 1 + int(np.searchsorted(c, p * c[-1], side="left"))
        n = max(1, min(n, len(w), int((w >= mp).sum())))
        kept = np.sort(order[:n])
        c = np.cumsum(np.exp((x[r][kept] - x[r][order[0]]) / T))
        out[r] = kept[min(int(np.searchsorted(c, u[r] * c[-1], side="right")), len(kept) - 1)]
    return torch.from_numpy(out).to(DEV)
