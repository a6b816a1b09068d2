"""The operators of a serving loop over a paged key/value cache: what is measured, their plain forms, and what they have to give.

A pool holds the pages of one layer's cache: keys and values [pages, kv_heads, page_size, head_dim], and for every slot of a
page the attention weight that its position has received so far, [pages, kv_heads, page_size].  A sequence owns a list of pages;
its position p lives in slot p % page_size of page table[p // page_size].

Kinds of case
  append   the projections of the step's new tokens, rows of one fused product [tokens, (heads + 2 kv_heads) * head_dim]:
           RMS norm of every query and key head (where the model has one), rotation by the tables of cosines and sines,
           queries out in the cache's type, keys and values into their slots
  attend   attention of every sequence's new tokens over its pages: a single token, a few, or a chunk of a prompt
  observe  the same, and the weights that the cached positions received are added to what they had
  evict    the positions of every sequence and key head that received most weight, and its last ones, go to new pages

Ranges: the head layouts of this repository's models (TinyLlama 32 / 4 heads of 64, Llama-2 7B 32 / 32 of 128, Qwen3 8B 32 / 8
of 128) and a group of seven; pages of 16 to 128 positions; one to 64 sequences; one to 2048 new tokens; contexts of one to
16384 positions; a cache of 16 bits and one of 32.
"""
from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False
DEV = "cuda:0"
EPS = 1e-6
HEADS = {"tinyllama": (32, 4, 64), "llama2_7b": (32, 32, 128), "qwen3_8b": (32, 8, 128), "sevens": (28, 4, 128)}
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
MAX_POSITIONS = 16384


def listed() -> list:
    return [
        # one decode step of a full serving batch: a token of each of 64 sequences, queries and keys normed per head
        dict(name="append_step", kind="append", heads="qwen3_8b", dtype="bf16", page=64, seqs=64, q_lo=1, q_hi=1, kv_lo=200, kv_hi=8000, norm=True),
        # prompts of several users read at once
        dict(name="append_prompts", kind="append", heads="qwen3_8b", dtype="bf16", page=64, seqs=5, q_lo=900, q_hi=2048, kv_lo=900, kv_hi=6000, norm=True),
        # the first answer token of one short chat: the smallest call, all latency
        dict(name="attend_one", kind="attend", heads="tinyllama", dtype="bf16", page=16, seqs=1, q_lo=1, q_hi=1, kv_lo=37, kv_hi=37),
        # one decode step of 64 sequences of very different lengths
        dict(name="attend_step", kind="attend", heads="qwen3_8b", dtype="bf16", page=64, seqs=64, q_lo=1, q_hi=1, kv_lo=1000, kv_hi=8000),
        # one user far into a long conversation, cache of 32 bits
        dict(name="attend_long_f32", kind="attend", heads="tinyllama", dtype="f32", page=32, seqs=1, q_lo=1, q_hi=1, kv_lo=16001, kv_hi=16001),
        # drafted tokens of a dozen users, checked at once: a few tokens each
        dict(name="attend_drafts", kind="attend", heads="sevens", dtype="bf16", page=32, seqs=12, q_lo=2, q_hi=9, kv_lo=300, kv_hi=5000),
        # a chunk of a prompt in 32 bits
        dict(name="attend_chunk_f32", kind="attend", heads="tinyllama", dtype="f32", page=64, seqs=2, q_lo=300, q_hi=509, kv_lo=700, kv_hi=4000),
        # a chunk of 2048 tokens of a long document: the most work of all
        dict(name="attend_chunk", kind="attend", heads="qwen3_8b", dtype="bf16", page=128, seqs=1, q_lo=2048, q_hi=2048, kv_lo=16384, kv_hi=16384),
        # decode steps that keep count of what is looked at
        dict(name="observe_step", kind="observe", heads="qwen3_8b", dtype="bf16", page=64, seqs=16, q_lo=1, q_hi=1, kv_lo=2000, kv_hi=8000),
        # the end of a prompt, whose queries say what of it will be needed
        dict(name="observe_chunk", kind="observe", heads="qwen3_8b", dtype="bf16", page=64, seqs=2, q_lo=200, q_hi=512, kv_lo=3000, kv_hi=6500),
        # four caches shrink to an eighth
        dict(name="evict_long", kind="evict", heads="qwen3_8b", dtype="bf16", page=64, seqs=4, kv_lo=12000, kv_hi=16384, keep=0.125, recent=256),
        # one long chat in 32 bits gives up a tenth of its positions
        dict(name="evict_f32", kind="evict", heads="tinyllama", dtype="f32", page=32, seqs=1, kv_lo=2047, kv_hi=2047, keep=0.9, recent=64),
    ]


def _log(rng, lo, hi) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng) -> dict:
    kind = rng.choice(["append", "attend", "attend", "observe", "evict"])
    heads = rng.choice(list(HEADS))
    case = dict(kind=kind, heads=heads, dtype=rng.choice(["bf16", "bf16", "f32"]), page=rng.choice([16, 32, 64, 128]))
    heads_q, heads_kv, dim = HEADS[heads]
    if kind == "evict":
        kv_hi = _log(rng, 64, MAX_POSITIONS)
        seqs = max(1, min(_log(rng, 1, 16), (4 * MAX_POSITIONS * 8 * 128) // (kv_hi * heads_kv * dim)))
        kv_lo = max(1, int(kv_hi * rng.uniform(0.3, 1.0)))
        return dict(case, seqs=seqs, kv_lo=kv_lo, kv_hi=kv_hi, keep=rng.choice([0.125, 0.25, 0.5, 0.9]), recent=_log(rng, 1, max(2, kv_lo // 8)))
    q_hi = rng.choice([1, _log(rng, 1, 16), _log(rng, 16, 2048)])
    q_lo = max(1, int(q_hi * rng.uniform(0.3, 1.0)))
    kv_hi = max(q_hi, _log(rng, 1, MAX_POSITIONS))
    kv_lo = max(1, int(kv_hi * rng.uniform(0.3, 1.0)))
    seqs = _log(rng, 1, 64)
    most = 32 * 2048 * 16384 if kind != "append" else 1 << 62  # scores of the plain form
    seqs = max(1, min(seqs, most // (heads_q * q_hi * kv_hi), (64 * 4500 * 8 * 128) // (kv_hi * heads_kv * dim)))
    if kind == "append":
        seqs = max(1, min(seqs, 8192 // q_hi))
        return dict(case, seqs=seqs, q_lo=q_lo, q_hi=q_hi, kv_lo=kv_lo, kv_hi=kv_hi, norm=rng.random() < 0.6)
    while heads_q * q_hi * kv_hi > most:  # the draw costs no more than the largest listed case
        kv_hi, q_hi = max(1, kv_hi // 2), max(1, min(q_hi, kv_hi // 2))
    return dict(case, seqs=seqs, q_lo=min(q_lo, q_hi), q_hi=q_hi, kv_lo=min(kv_lo, kv_hi), kv_hi=kv_hi)


# ---- inputs ---------------------------------------------------------------------------------------------------
def _lengths(case: dict) -> tuple:
    """New tokens and cached positions (the new ones among them) of every sequence: by the case alone; a single one has the upper ends."""
    rng = random.Random(f"{case['seqs']}/{case['kv_lo']}/{case['kv_hi']}")
    n = case["seqs"]
    kv = [case["kv_hi"]] + [rng.randint(case["kv_lo"], case["kv_hi"]) for _ in range(n - 1)]
    if case["kind"] == "evict":
        q = [max(1, int(k * case["keep"])) for k in kv]  # positions that stay
    else:
        q = [min(kv[0], case["q_hi"])] + [min(k, rng.randint(case["q_lo"], case["q_hi"])) for k in kv[1:]]
    return q, kv


def _pages(case: dict) -> tuple:
    """Pages that the sequences need, and those of the kept positions (evict)."""
    q, kv = _lengths(case)
    page = case["page"]
    return [-(-k // page) for k in kv], [-(-k // page) for k in q] if case["kind"] == "evict" else []


def _tables(case: dict, seed: int) -> tuple:
    """Tables [seqs, most pages] of page numbers, drawn without replacement, zeros behind the last page."""
    need, kept = _pages(case)
    total = sum(need) + sum(kept) + 3
    order = np.random.default_rng(seed).permutation(total).astype(np.int32)

    def table(counts, first):
        ends = first + np.cumsum(counts)
        cols = np.arange(max(counts))
        at = (ends - counts)[:, None] + cols[None, :]
        return np.where(cols[None, :] < np.asarray(counts)[:, None], order[np.minimum(at, total - 1)], 0).astype(np.int32)

    return total, table(need, 0), table(kept, sum(need)) if kept else None


def _rope(dim: int) -> tuple:
    """Cosines and sines [positions, dim / 2], angles in 64 bits."""
    angle = np.arange(MAX_POSITIONS)[:, None] * 10000.0 ** (-np.arange(0, dim, 2) / dim)
    return np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32)


class _Memory:
    """Device memory of a pool, for torch to look at; what looks at it keeps the pool."""

    def __init__(self, pool, ptr, shape, typestr):
        self.pool = pool
        self.__cuda_array_interface__ = dict(data=(ptr, False), shape=shape, typestr=typestr, version=3)


def _handles(case: dict, s: dict) -> None:
    """The pool, plans and tables that a program on the framework keeps."""
    import lumen_b200 as L
    ctx = L.default_context()
    heads_q, heads_kv, dim = HEADS[case["heads"]]
    half = case["dtype"] == "bf16"
    pool = L.PagePool(s["k"].shape[0], case["page"], heads_kv, dim, L.BF16 if half else L.F32, ctx)
    ctx.synchronize()
    for name, ptr in (("k", pool.k_ptr), ("v", pool.v_ptr), ("mass", pool.mass_ptr)):
        if name in s:
            x = s[name]
            there = torch.as_tensor(_Memory(pool, ptr, tuple(x.shape), "<i2" if x.dtype == torch.bfloat16 else "<f4"), device=DEV).view(x.dtype)
            there.copy_(x)
            s[name] = there
    q, kv = s["q_lens"], s["kv_lens"]
    if case["kind"] == "evict":
        s["from"] = L.PageBatch(pool, heads_q, [0] * len(kv), kv, s["host_tables"])
        s["to"] = L.PageBatch(pool, heads_q, [0] * len(kv), q, s["host_kept_tables"])
    else:
        s["batch"] = L.PageBatch(pool, heads_q, q, kv, s["host_tables"])
    if case["kind"] == "append":
        s["rope"] = L.RotaryEmbedding.from_tables(s["cos"].cpu().numpy(), s["sin"].cpu().numpy(), ctx)
    s["pool"], s["L"], s["ctx"] = pool, L, ctx
    ctx.synchronize()


def prepare(case: dict, seed: int) -> dict:
    heads_q, heads_kv, dim = HEADS[case["heads"]]
    t = TYPES[case["dtype"]]
    g = torch.Generator(device=DEV).manual_seed(seed * 7919 + 17)
    q_lens, kv_lens = _lengths(case)
    pages, tables, kept_tables = _tables(case, seed)
    rnd = lambda *shape: torch.randn(shape, generator=g, device=DEV)  # noqa: E731
    s = dict(case=case, q_lens=q_lens, kv_lens=kv_lens, host_tables=tables, host_kept_tables=kept_tables)
    s["k"] = rnd(pages, heads_kv, case["page"], dim).to(t)
    s["v"] = rnd(pages, heads_kv, case["page"], dim).to(t)
    s["tables"] = torch.from_numpy(tables).to(DEV).long()
    kv, ql = np.asarray(kv_lens), np.asarray(q_lens)
    s["kv"], s["ql"] = torch.from_numpy(kv).to(DEV), torch.from_numpy(ql).to(DEV)
    if case["kind"] == "evict":
        # weights that long tails have: few positions hold most, many nothing at all (ties)
        s["mass"] = torch.relu(rnd(pages, heads_kv, case["page"])) ** 4
        s["kept_tables"] = torch.from_numpy(kept_tables).to(DEV).long()
        s["kept"] = torch.full((case["seqs"], heads_kv, max(q_lens)), -1, dtype=torch.int32, device=DEV)
    else:
        tokens = int(ql.sum())
        seq = np.repeat(np.arange(len(ql)), ql)
        within = np.arange(tokens) - np.repeat(np.cumsum(ql) - ql, ql)
        pos = kv[seq] - ql[seq] + within
        s["seq"], s["within"], s["pos"] = (torch.from_numpy(x).to(DEV) for x in (seq, within, pos))
        if case["kind"] == "append":
            s["qkv"] = rnd(tokens, (heads_q + 2 * heads_kv) * dim)
            s["q"] = torch.empty(tokens, heads_q, dim, dtype=t, device=DEV)
            if case["norm"]:
                s["q_norm"], s["k_norm"] = 1 + 0.1 * rnd(dim), 1 + 0.1 * rnd(dim)
            s["cos"], s["sin"] = (torch.from_numpy(x).to(DEV) for x in _rope(dim))
        else:
            s["q"] = (1.5 * rnd(tokens, heads_q, dim)).to(t)
            s["out"] = torch.empty(tokens, heads_q, dim, dtype=t, device=DEV)
            first = np.cumsum(ql) - ql
            s["padded"] = torch.from_numpy(np.minimum(first[:, None] + np.arange(ql.max())[None, :], tokens - 1)).to(DEV)
            if case["kind"] == "observe":
                s["lse"] = torch.empty(tokens, heads_q, device=DEV)
                s["mass"] = torch.rand((pages, heads_kv, case["page"]), generator=g, device=DEV)
    if own:
        _handles(case, s)
    torch.cuda.synchronize()
    return s


# ---- the plain forms ----------------------------------------------------------------------------------------------
def _plain_append(s: dict) -> list:
    case = s["case"]
    heads_q, heads_kv, dim = HEADS[case["heads"]]
    x = s["qkv"].view(-1, heads_q + 2 * heads_kv, dim)
    q, k, v = x[:, :heads_q], x[:, heads_q: heads_q + heads_kv], x[:, heads_q + heads_kv:]
    cos, sin = s["cos"][s["pos"]][:, None], s["sin"][s["pos"]][:, None]

    def normed(x, w):
        return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w if case["norm"] else x

    def turned(x):
        a, b = x[..., : dim // 2], x[..., dim // 2:]
        return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)

    q, k = turned(normed(q, s.get("q_norm"))), turned(normed(k, s.get("k_norm")))
    page = s["tables"][s["seq"], s["pos"] // case["page"]]
    s["q"].copy_(q)
    s["k"][page, :, s["pos"] % case["page"]] = k.to(s["k"].dtype)
    s["v"][page, :, s["pos"] % case["page"]] = v.to(s["v"].dtype)
    return [s["q"], s["k"], s["v"]]


def _plain_attend(s: dict) -> tuple:
    """Outputs [tokens, heads, dim], log of the sum of weights [tokens, heads], and the weights [seqs, kv_heads, group, tokens, positions]."""
    case = s["case"]
    heads_q, heads_kv, dim = HEADS[case["heads"]]
    n, group, most = case["seqs"], heads_q // heads_kv, s["padded"].shape[1]
    k, v = (s[x][s["tables"]].transpose(1, 2).reshape(n, heads_kv, -1, dim).float() for x in "kv")
    q = s["q"].float()[s["padded"]].view(n, most, heads_kv, group, dim).permute(0, 2, 3, 1, 4).reshape(n, heads_kv, group * most, dim)
    w = torch.matmul(q, k.transpose(-1, -2)).view(n, heads_kv, group, most, -1)
    w *= dim ** -0.5
    i, j = torch.arange(most, device=DEV), torch.arange(k.shape[2], device=DEV)
    hidden = j[None, None, :] > (s["kv"] - s["ql"])[:, None, None] + i[None, :, None]
    w.masked_fill_(hidden[:, None, None], -math.inf)
    top = w.amax(-1, keepdim=True)
    w -= top
    w.exp_()
    total = w.sum(-1, keepdim=True)
    w /= total
    live = (j[None, :] < s["kv"][:, None])[:, None, :, None]
    out = torch.matmul(w.view(n, heads_kv, group * most, -1), torch.where(live, v, 0)).view(n, heads_kv, group, most, dim)
    out = out.permute(0, 3, 1, 2, 4).reshape(n, most, heads_q, dim)[s["seq"], s["within"]]
    lse = (top + total.log()).squeeze(-1).permute(0, 3, 1, 2).reshape(n, most, heads_q)[s["seq"], s["within"]]
    return out.to(s["q"].dtype), lse, w


def _plain_observe(s: dict) -> list:
    out, lse, w = _plain_attend(s)
    case = s["case"]
    real = torch.arange(w.shape[3], device=DEV)[None, :] < s["ql"][:, None]
    gained = (w * real[:, None, None, :, None]).sum((2, 3))  # [seqs, kv_heads, positions]
    live = torch.arange(w.shape[4], device=DEV)[None, :] < s["kv"][:, None]
    gained = torch.where(live[:, None], gained, 0).view(case["seqs"], w.shape[1], -1, case["page"]).transpose(1, 2)
    s["mass"].index_add_(0, s["tables"].reshape(-1), gained.reshape(-1, w.shape[1], case["page"]))
    return [out, lse, s["mass"]]


def _plain_evict(s: dict) -> list:
    case = s["case"]
    heads_q, heads_kv, dim = HEADS[case["heads"]]
    n, page = case["seqs"], case["page"]
    m = s["mass"][s["tables"]].transpose(1, 2).reshape(n, heads_kv, -1)
    j = torch.arange(m.shape[2], device=DEV)[None, None]
    recent = torch.minimum(s["ql"], torch.full_like(s["ql"], case["recent"]))[:, None, None]
    kv, keep = s["kv"][:, None, None], s["ql"][:, None, None]
    key = torch.where(j >= kv, -math.inf, torch.where(j >= kv - recent, math.inf, m))
    order = torch.sort(key, dim=-1, descending=True, stable=True).indices
    chosen = torch.where(j < keep, order, m.shape[2]).sort(-1).values[..., : s["kept"].shape[2]]
    slots = torch.arange(chosen.shape[2], device=DEV)
    real = slots[None, None] < keep
    s["kept"].copy_(torch.where(real, chosen, s["kept"].long()))
    b, h, i = torch.nonzero(real.expand(n, heads_kv, -1), as_tuple=True)
    p = chosen[b, h, i]
    source = (s["tables"][b, p // page], h, p % page)
    goal = (s["kept_tables"][b, i // page], h, i % page)
    for name in ("k", "v", "mass"):
        s[name][goal] = s[name][source]
    return [s["kept"], s["k"], s["v"], s["mass"]]


# ---- one pass -----------------------------------------------------------------------------------------------------
def run(s: dict):
    kind = s["case"]["kind"]
    if not own:
        if kind == "append":
            return _plain_append(s)
        if kind == "attend":
            return _plain_attend(s)[0]
        return _plain_observe(s) if kind == "observe" else _plain_evict(s)
    L, pool = s["L"], s["pool"]
    if kind == "evict":
        L.paged_evict(pool, s["from"], s["to"], s["case"]["recent"], s["kept"].data_ptr(), s["kept"].shape[2])
        return [s["kept"], s["k"], s["v"], s["mass"]]
    heads_q, heads_kv, dim = HEADS[s["case"]["heads"]]
    if kind == "append":
        at, row = s["qkv"].data_ptr(), s["qkv"].shape[1]
        norms = dict(q_norm_ptr=s["q_norm"].data_ptr(), k_norm_ptr=s["k_norm"].data_ptr(), eps=EPS) if s["case"]["norm"] else {}
        L.paged_append(pool, s["batch"], at, at + 4 * heads_q * dim, at + 4 * (heads_q + heads_kv) * dim, row, row, s["q"].data_ptr(), rope=s["rope"], **norms)
        return [s["q"], s["k"], s["v"]]
    lse = s["lse"].data_ptr() if kind == "observe" else 0
    L.paged_attention(pool, s["batch"], s["q"].data_ptr(), dim ** -0.5, s["out"].data_ptr(), lse_ptr=lse)
    if kind == "attend":
        return s["out"]
    L.paged_attention_mass(pool, s["batch"], s["q"].data_ptr(), dim ** -0.5, lse)
    return [s["out"], s["lse"], s["mass"]]


# ---- what a pass cannot do without ----------------------------------------------------------------------------------
def work(case: dict) -> dict:
    heads_q, heads_kv, dim = HEADS[case["heads"]]
    e = 2 if case["dtype"] == "bf16" else 4
    q, kv = _lengths(case)
    if case["kind"] == "append":
        rows = sum(q)
        tables = rows * dim * 4
        return dict(bytes=rows * (heads_q + 2 * heads_kv) * dim * (4 + e) + tables, flops=rows * (heads_q + heads_kv) * dim * (7.0 if case["norm"] else 3.0))
    if case["kind"] == "evict":  # weights of all positions read once; the kept rows read and written
        return dict(bytes=sum(kv) * heads_kv * 4 + sum(q) * heads_kv * (2 * 2 * dim * e + 4 + 4), flops=float(sum(kv) * heads_kv))
    seen = sum(n * (k - n) + n * (n + 1) // 2 for n, k in zip(q, kv))  # pairs of a query and a position
    once = dict(bytes=2 * sum(q) * heads_q * dim * e + 2 * sum(kv) * heads_kv * dim * e, flops=4.0 * seen * heads_q * dim)
    if case["kind"] == "observe":  # and the weights' sums, of scores that are there once they are computed
        once = dict(bytes=once["bytes"] + sum(kv) * heads_kv * 8 + sum(q) * heads_q * 4, flops=once["flops"] + seen * heads_q)
    return once


# ---- in 64 bits, from the definitions ---------------------------------------------------------------------------------
def exact(case: dict, seed: int):
    global own
    kept, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = kept
    heads_q, heads_kv, dim = HEADS[case["heads"]]
    page, group = case["page"], heads_q // heads_kv
    q_lens, kv_lens = s["q_lens"], s["kv_lens"]

    def rows(pool, table, n):  # the first n positions: [n, kv_heads, ...]
        return pool[table].transpose(1, 2).reshape(len(table) * page, *pool.shape[1:2], *pool.shape[3:])[:n]

    def places(table, positions):  # flat slot numbers
        return table[positions // page] * page + positions % page

    if case["kind"] == "append":
        k, v, q, t = s["k"].double(), s["v"].double(), [], 0
        for b, n in enumerate(q_lens):
            pos = torch.arange(kv_lens[b] - n, kv_lens[b], device=DEV)
            x = s["qkv"][t: t + n].double().view(n, -1, dim)
            t += n
            z = torch.complex(s["cos"][pos].double(), s["sin"][pos].double())[:, None]

            def head(y, w):
                if case["norm"]:
                    y = y / ((y * y).sum(-1, keepdim=True) / dim + EPS).sqrt() * s[w].double()
                y = torch.complex(y[..., : dim // 2].contiguous(), y[..., dim // 2:].contiguous()) * z
                return torch.cat([y.real, y.imag], -1)

            q.append(head(x[:, :heads_q], "q_norm"))
            at = places(s["tables"][b], pos)
            k.transpose(1, 2)[at // page, at % page] = head(x[:, heads_q: heads_q + heads_kv], "k_norm")
            v.transpose(1, 2)[at // page, at % page] = x[:, heads_q + heads_kv:]
        return [torch.cat(q), k, v]
    if case["kind"] == "evict":
        kept, pools = s["kept"].clone(), [s[x].clone() for x in ("k", "v", "mass")]
        for b, keep in enumerate(q_lens):
            n = kv_lens[b]
            table, goal = s["tables"][b], s["kept_tables"][b]
            m = rows(s["mass"], table, n).cpu().numpy()
            last = min(keep, case["recent"])
            for h in range(heads_kv):
                old = np.lexsort((np.arange(n - last), -m[: n - last, h]))[: keep - last]
                stay = torch.from_numpy(np.sort(np.concatenate([old, np.arange(n - last, n)])).astype(np.int64)).to(DEV)
                kept[b, h, :keep] = stay.int()
                a, z = places(table, stay), places(goal, torch.arange(keep, device=DEV))
                for x in pools:
                    x[z // page, h, z % page] = x[a // page, h, a % page]
        return [kept, pools[0].double(), pools[1].double(), pools[2].double()]
    out, lse, t = [], [], 0
    mass = s["mass"].double() if case["kind"] == "observe" else None
    for b, n in enumerate(q_lens):
        length = kv_lens[b]
        table = s["tables"][b]
        k, v = (rows(s[x], table, length).double() for x in "kv")
        o, l = torch.empty(n, heads_q, dim, dtype=torch.float64, device=DEV), torch.empty(n, heads_q, dtype=torch.float64, device=DEV)
        ahead = torch.ones(n, length, dtype=torch.bool, device=DEV).triu(length - n + 1)
        for h in range(heads_q):
            z = s["q"][t: t + n, h].double() @ k[:, h // group].T / math.sqrt(dim)
            z[ahead] = -math.inf
            l[:, h] = torch.logsumexp(z, -1)
            p = torch.softmax(z, -1)
            o[:, h] = p @ v[:, h // group]
            if mass is not None:
                at = places(table, torch.arange(length, device=DEV))
                mass[at // page, h // group, at % page] += p.sum(0)
        t += n
        out.append(o)
        lse.append(l)
    return torch.cat(out) if case["kind"] == "attend" else [torch.cat(out), torch.cat(lse), mass]
