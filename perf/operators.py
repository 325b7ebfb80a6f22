"""Serving operators: writing a paged key-value cache, attention over it, moving its pages.

``listed()`` names the cases, ``draw(rng)`` gives further ones of the same ranges, ``prepare(case, seed)`` builds what a
serving program holds before the call, ``run(state)`` is one pass (in elementary torch operations, or through the
framework's entry points where ``own`` is set), ``exact(case, seed)`` the same from the definitions in 64 bits and
``work(case)`` the bytes and operations a pass cannot do without.

A cache layer is a pair of tensors ``[pages, kv_heads, page_size, head_dim]``; position ``j`` of sequence ``s`` lives in
page ``table[s, j // page_size]`` at slot ``j % page_size``.  ``lengths[s]`` counts the tokens of a sequence with its new
ones; the new tokens of all sequences are packed rows, those of sequence ``s`` at ``offsets[s] .. offsets[s + 1]``.

Kinds of cases:

* ``append``: new tokens enter the cache: queries and keys are rotated to their positions, keys and values written into
  the pages;
* ``decode``: attention of one new token per sequence over its cached tokens;
* ``prompt``: causal attention of packed runs of new tokens over their sequences' cached tokens;
* ``copy``: pages of all layers copied inside the cache, as forking and compacting sequences do.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEVICE = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


# ------------------------------------------------------------------------------------------------------------- cases
def listed() -> list[dict]:
    return [
        # one generation step of a full batch of the 1.1B Llama's heads: 256 conversations at any point up to its context
        {"name": "append_step", "kind": "append", "dtype": "bf16", "heads": 32, "kv_heads": 4, "head_dim": 64, "page": 64,
         "seqs": 256, "new": 256, "past": 4000, "theta": 10000.0},
        # prompts of seven users written at once, with far positions behind a long shared prefix
        {"name": "append_prompts", "kind": "append", "dtype": "bf16", "heads": 24, "kv_heads": 8, "head_dim": 128, "page": 16,
         "seqs": 7, "new": 8190, "past": 100000, "theta": 500000.0},
        # the smallest call: one short GPT-2-small text
        {"name": "decode_one_short", "kind": "decode", "dtype": "fp16", "heads": 12, "kv_heads": 12, "head_dim": 64, "page": 16,
         "seqs": 1, "longest": 77},
        # an ordinary serving batch of the 1.1B Llama
        {"name": "decode_batch", "kind": "decode", "dtype": "bf16", "heads": 32, "kv_heads": 4, "head_dim": 64, "page": 64,
         "seqs": 64, "longest": 4096},
        # one conversation over a book: the work has to be split over the cache's length
        {"name": "decode_long", "kind": "decode", "dtype": "bf16", "heads": 24, "kv_heads": 8, "head_dim": 128, "page": 128,
         "seqs": 1, "longest": 131071},
        # a full batch of the 3B Llama's heads: the largest cache
        {"name": "decode_full", "kind": "decode", "dtype": "bf16", "heads": 24, "kv_heads": 8, "head_dim": 128, "page": 16,
         "seqs": 128, "longest": 8192},
        # a short question
        {"name": "prompt_one_short", "kind": "prompt", "dtype": "bf16", "heads": 12, "kv_heads": 12, "head_dim": 64, "page": 16,
         "seqs": 1, "new": 37, "past": 0},
        # a batch of prompts of different lengths, some behind cached turns
        {"name": "prompt_packed", "kind": "prompt", "dtype": "bf16", "heads": 32, "kv_heads": 4, "head_dim": 64, "page": 64,
         "seqs": 16, "new": 8000, "past": 500},
        # a few hundred new tokens behind a long document
        {"name": "prompt_chunk", "kind": "prompt", "dtype": "fp16", "heads": 24, "kv_heads": 8, "head_dim": 128, "page": 16,
         "seqs": 1, "new": 256, "past": 32768},
        # a whole document of odd length
        {"name": "prompt_long", "kind": "prompt", "dtype": "bf16", "heads": 24, "kv_heads": 8, "head_dim": 128, "page": 64,
         "seqs": 1, "new": 8191, "past": 0},
        # one conversation forked: its open page copied in all layers of the 1.1B Llama
        {"name": "copy_fork", "kind": "copy", "dtype": "bf16", "layers": 22, "kv_heads": 4, "head_dim": 64, "page": 64,
         "pages": 64, "pairs": 1},
        # a cache of the 3B Llama's heads compacted after half of its conversations ended
        {"name": "copy_compact", "kind": "copy", "dtype": "bf16", "layers": 26, "kv_heads": 8, "head_dim": 128, "page": 16,
         "pages": 2000, "pairs": 777},
    ]


# the heads of the repository's models and benchmarks, and one key head for all queries
_HEADS = [(12, 12, 64), (32, 4, 64), (24, 8, 128), (4, 2, 64), (32, 32, 128), (16, 1, 128)]


def _log_int(rng, lo: int, hi: int) -> int:
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return min(max(int(round(v)), lo), hi)


def draw(rng) -> dict:
    kind = rng.choice(["append", "decode", "decode", "prompt", "prompt", "copy"])
    heads, kv_heads, head_dim = rng.choice(_HEADS)
    case = {"kind": kind, "dtype": rng.choice(["bf16", "bf16", "fp16"]), "heads": heads, "kv_heads": kv_heads,
            "head_dim": head_dim, "page": rng.choice([16, 32, 64, 128])}
    if kind == "append":
        seqs = _log_int(rng, 1, 256)
        return {**case, "seqs": seqs, "new": max(seqs, _log_int(rng, 1, 8190)), "past": rng.choice([0, _log_int(rng, 1, 100000)]),
                "theta": rng.choice([0.0, 10000.0, 500000.0])}
    if kind == "decode":
        longest = _log_int(rng, 1, 131071)
        # no more cache than the largest listed case: about half of the longest times the sequences
        room = 128 * 8192 * 8 * 128 // (longest * kv_heads * head_dim)
        return {**case, "seqs": _log_int(rng, 1, max(1, min(256, room))), "longest": longest}
    if kind == "prompt":
        seqs = _log_int(rng, 1, 32)
        new = max(seqs, _log_int(rng, 1, 8191))
        # no more scores than the whole document's, heads included
        room = int(24 * 128 * 8191 * 4096 / (heads * head_dim * new)) - new
        return {**case, "seqs": seqs, "new": new, "past": rng.choice([0, _log_int(rng, 1, max(1, min(32768, room)))]) if room > 0 else 0}
    case.pop("heads")
    layers = rng.randint(2, 26)
    page_elems = 2 * layers * kv_heads * case["page"] * head_dim
    most = 2 * 26 * 8 * 16 * 128 * 777 // page_elems
    pairs = _log_int(rng, 1, max(1, min(777, most)))
    return {**case, "layers": layers, "pages": 2 * pairs + rng.randint(1, pairs + 16), "pairs": pairs}


def _shares(case: dict) -> tuple[list[int], list[int]]:
    """New tokens and total lengths of the sequences of a case; set by its sizes alone."""
    n = case["seqs"]
    rng = random.Random(n * 1000003 + case.get("new", 0) * 101 + case.get("longest", 0) + case.get("past", 0) * 7)
    if case["kind"] == "decode":
        lengths = [case["longest"]] + [rng.randint(1, case["longest"]) for _ in range(n - 1)]
        return [1] * n, lengths
    cuts = sorted(rng.sample(range(1, case["new"]), n - 1)) if n > 1 else []
    new = [b - a for a, b in zip([0] + cuts, cuts + [case["new"]])]
    past = [case["past"]] + [rng.randint(0, case["past"]) for _ in range(n - 1)]
    return new, [a + b for a, b in zip(new, past)]


# ----------------------------------------------------------------------------------------------------------- prepare
def prepare(case: dict, seed: int) -> dict:
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    host = torch.Generator().manual_seed(seed)
    dtype, P, Hkv, D = DTYPES[case["dtype"]], case["page"], case["kv_heads"], case["head_dim"]

    def randn(*shape):
        out = torch.empty(shape, dtype=dtype, device=DEVICE)
        return out.normal_(generator=gen)

    if case["kind"] == "copy":
        order = torch.randperm(case["pages"], generator=host).to(torch.int32)
        n = case["pairs"]
        return {"case": case, "storage": randn(case["layers"], 2, case["pages"], Hkv, P, D),
                "src": order[:n].to(DEVICE), "dst": order[n:2 * n].to(DEVICE)}
    new, lengths = _shares(case)
    width = max((n + P - 1) // P for n in lengths)
    # the pages a call touches are scattered over the cache; a long prefix that only an append passes over is one page
    # that all its sequences share
    first = [(t - n) // P if case["kind"] == "append" else 0 for n, t in zip(new, lengths)]
    used = [(t + P - 1) // P - f for t, f in zip(lengths, first)]
    pages = 1 + sum(used)
    order = (torch.randperm(pages - 1, generator=host) + 1).to(torch.int32)
    table = torch.full((len(new), width), -1, dtype=torch.int32)
    at = 0
    for s, (f, u) in enumerate(zip(first, used)):
        table[s, :f] = 0
        table[s, f:f + u] = order[at:at + u]
        at += u
    offsets = [0]
    for n in new:
        offsets.append(offsets[-1] + n)
    state = {"case": case, "k_pages": randn(pages, Hkv, P, D), "v_pages": randn(pages, Hkv, P, D), "table": table.to(DEVICE),
             "lengths": torch.tensor(lengths, dtype=torch.int32, device=DEVICE),
             "offsets": torch.tensor(offsets, dtype=torch.int32, device=DEVICE), "new": new, "total": lengths}
    if case["kind"] == "append":
        state["qkv"] = randn(offsets[-1], (case["heads"] + 2 * Hkv) * D)
    else:
        state["q"] = randn(offsets[-1], case["heads"], D)
    return state


# --------------------------------------------------------------------------------------------------------------- run
def run(state: dict):
    case = state["case"]
    if own:
        from incin_b200.ops import functional as F
        if case["kind"] == "copy":
            return F.copy_pages(state["storage"], state["src"], state["dst"])
        cache = (state["k_pages"], state["v_pages"], state["table"], state["lengths"])
        if case["kind"] == "append":
            q = F.kv_append(state["qkv"], *cache, state["offsets"], n_heads=case["heads"], theta=case["theta"] or None)
            return q, state["k_pages"], state["v_pages"]
        if case["kind"] == "decode":
            return F.decode_attention(state["q"], *cache)
        return F.prompt_attention(state["q"], *cache, state["offsets"])
    if case["kind"] == "copy":
        storage = state["storage"]
        storage[:, :, state["dst"].long()] = storage[:, :, state["src"].long()]
        return storage
    if case["kind"] == "append":
        return _append_plain(state)
    return _attention_plain(state)


def _append_plain(state: dict):
    case, qkv = state["case"], state["qkv"]
    H, Hkv, D, P = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    x = qkv.view(-1, H + 2 * Hkv, D)
    rows = torch.arange(x.shape[0], device=x.device)
    seq = (rows[:, None] >= state["offsets"][None, 1:]).sum(1)
    pos = state["lengths"].long()[seq] - state["offsets"].long()[seq + 1] + rows
    rot = x[:, :H + Hkv].float()
    if case["theta"]:
        freq = case["theta"] ** (-2.0 * torch.arange(D // 2, dtype=torch.float64, device=x.device) / D)
        angle = pos.double()[:, None] * freq                      # far positions need more than 32 bits
        cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
        a, b = rot[..., :D // 2], rot[..., D // 2:]
        rot = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    rot = rot.to(x.dtype)
    page, slot = state["table"].long()[seq, pos // P], pos % P
    state["k_pages"][page, :, slot] = rot[:, H:]
    state["v_pages"][page, :, slot] = x[:, H + Hkv:]
    return rot[:, :H].contiguous(), state["k_pages"], state["v_pages"]


def _attention_plain(state: dict):
    case, q = state["case"], state["q"]
    H, Hkv, D, P = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    out, at = torch.empty_like(q), 0
    for s, (n, total) in enumerate(zip(state["new"], state["total"])):
        pages = state["table"][s, :(total + P - 1) // P].long()
        k, v = (t[pages].transpose(0, 1).reshape(Hkv, -1, D)[:, :total].float() for t in (state["k_pages"], state["v_pages"]))
        qs = q[at:at + n].float().view(n, Hkv, H // Hkv, D).permute(1, 2, 0, 3).reshape(Hkv, -1, D)
        scores = qs @ k.transpose(1, 2) * D ** -0.5
        if n > 1:
            last = torch.arange(total - n, total, device=q.device).repeat(H // Hkv)
            scores.masked_fill_(torch.arange(total, device=q.device) > last[:, None], -math.inf)
        p = (scores - scores.amax(-1, keepdim=True)).exp()
        o = (p @ v) / p.sum(-1, keepdim=True)
        out[at:at + n] = o.view(Hkv, H // Hkv, n, D).permute(2, 0, 1, 3).reshape(n, H, D).to(q.dtype)
        at += n
    return out


# ------------------------------------------------------------------------------------------------------------- exact
def exact(case: dict, seed: int):
    state = prepare(case, seed)
    if case["kind"] == "copy":
        storage = state["storage"]
        for a, b in zip(state["src"].tolist(), state["dst"].tolist()):
            storage[:, :, b].copy_(storage[:, :, a])
        return storage
    H, Hkv, D, P = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    table = state["table"].cpu()
    if case["kind"] == "append":
        k, v = state["k_pages"].double(), state["v_pages"].double()
        x = state["qkv"].double().view(-1, H + 2 * Hkv, D)
        q = x[:, :H].clone()
        at = 0
        for s, (n, total) in enumerate(zip(state["new"], state["total"])):
            pos = torch.arange(total - n, total)
            rows = x[at:at + n]
            if case["theta"]:
                pairs = torch.arange(D // 2, dtype=torch.float64)
                angle = pos.double()[:, None] * torch.exp(-2.0 * pairs / D * math.log(case["theta"]))
                turn = torch.polar(torch.ones_like(angle), angle).to(x.device)[:, None]
                z = torch.complex(rows[:, :H + Hkv, :D // 2], rows[:, :H + Hkv, D // 2:]) * turn
                rows = torch.cat([torch.cat([z.real, z.imag], -1), rows[:, H + Hkv:]], 1)
            q[at:at + n] = rows[:, :H]
            where = table[s, pos // P].long() * P + pos % P
            for pages, part in ((k, rows[:, H:H + Hkv]), (v, rows[:, H + Hkv:])):
                flat = pages.transpose(1, 2).reshape(-1, Hkv, D)
                flat[where.to(x.device)] = part
                pages.copy_(flat.view(-1, P, Hkv, D).transpose(1, 2))
            at += n
        return q, k, v
    q = state["q"]
    out, at = torch.empty(q.shape, dtype=torch.float64, device=q.device), 0
    for s, (n, total) in enumerate(zip(state["new"], state["total"])):
        where = torch.arange(total)
        page, slot = table[s, where // P].long().to(q.device), (where % P).to(q.device)
        for h in range(Hkv):
            k, v = state["k_pages"][page, h, slot].double(), state["v_pages"][page, h, slot].double()
            for g in range(h * (H // Hkv), (h + 1) * (H // Hkv)):
                z = torch.einsum("nd,ld->nl", q[at:at + n, g].double(), k) / math.sqrt(D)
                if n > 1:
                    z += torch.full((n, total), -math.inf, dtype=torch.float64, device=q.device).triu_(total - n + 1)
                out[at:at + n, g] = torch.softmax(z, 1) @ v
        at += n
    return out


# -------------------------------------------------------------------------------------------------------------- work
def work(case: dict) -> dict:
    Hkv, D = case["kv_heads"], case["head_dim"]
    if case["kind"] == "copy":
        return {"bytes": 2 * case["pairs"] * case["layers"] * 2 * Hkv * case["page"] * D * 2, "flops": 0}
    H = case["heads"]
    new, lengths = _shares(case)
    rows, tokens = sum(new), sum(lengths)
    if case["kind"] == "append":
        row = (H + 2 * Hkv) * D * 2
        return {"bytes": 2 * rows * row, "flops": rows * (H + Hkv) * D * 3 if case["theta"] else 0}
    seen = sum((t - n) * n + n * (n + 1) // 2 for n, t in zip(new, lengths))
    return {"bytes": 2 * rows * H * D * 2 + 2 * tokens * Hkv * D * 2, "flops": 4 * seen * H * D}
