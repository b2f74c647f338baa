"""Workloads of the operators for several sequences at once: attention of packed prompts, the paged cache (append and the
attention of a chunk of new tokens over it) and the log probabilities of given tokens.

`prepare` makes what a program has in hand before the call (inputs, the page pool, its table, the device's lengths and,
on the host, the lengths that the program's scheduler knows), `run` makes one pass: with `own` the calls of
byteprof_amd.optim.attention and byteprof_amd.optim.logprobs, without it the same operators in elementary float32 torch.
`exact` restates a pass in float64. The paths:

  packed    causal (or full) attention of whole prompts, one after another in [tokens, heads, head_dim], grouped heads;
            rows that belong to no sequence (the padding of a fixed-size batch) come out as zeros
  paged     a chunk of new tokens of each sequence (one for a decode step, several for a verify round, many for a part of
            a prompt) over its cache in pages; the chunk's own keys are in the cache already
  append    the chunk's keys and values into their pages
  logprobs  log softmax at the given tokens, the entropy, and the `top` most likely tokens of every row
"""

from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed() -> list[dict]:
    return [
        # four short prompts of a decoder of 16 heads of 128, q | k | v as slices of one projection: latency
        {"name": "packed short prompts", "path": "packed", "lens": "17,1,64,160", "hq": 16, "hk": 16, "d": 128,
         "dtype": "bf16", "causal": True, "pad": 0, "fused": True},
        # a batch of ragged prompts, four query heads to a key head
        {"name": "packed ragged batch", "path": "packed", "lens": "1531,256,4000,77,900,1024,333,71", "hq": 32, "hk": 8,
         "d": 128, "dtype": "bf16", "causal": True, "pad": 0, "fused": False},
        # one long document, as many key heads as query heads
        {"name": "packed long document", "path": "packed", "lens": "16384", "hq": 16, "hk": 16, "d": 128,
         "dtype": "bf16", "causal": True, "pad": 0, "fused": True},
        # fp16 heads of 64 in a batch padded to a fixed size
        {"name": "packed fp16 heads of 64", "path": "packed", "lens": "511,2047,1,1300", "hq": 12, "hk": 4, "d": 64,
         "dtype": "fp16", "causal": True, "pad": 237, "fused": False},
        # one token of one sequence behind a short prompt: the smallest decode step
        {"name": "paged one token", "path": "paged", "lens": "161", "chunks": "1", "page": 16, "hq": 16, "hk": 16,
         "d": 128, "dtype": "bf16"},
        # a decode step of many sequences of all lengths
        {"name": "paged decode batch", "path": "paged",
         "lens": ",".join(str(64 + (i * 2659) % 8111) for i in range(64)), "chunks": ",".join(["1"] * 64), "page": 16,
         "hq": 32, "hk": 8, "d": 128, "dtype": "bf16"},
        # a verify round: 8 drafts + 1 of six sequences, one of them long
        {"name": "paged verify round", "path": "paged", "lens": "40961,900,2500,130,7777,512", "chunks": "9,9,9,9,9,9",
         "page": 64, "hq": 16, "hk": 4, "d": 128, "dtype": "fp16"},
        # parts of prompts behind what the cache holds of them
        {"name": "paged prompt chunks", "path": "paged", "lens": "8192,4500,700,2049", "chunks": "512,512,511,1",
         "page": 32, "hq": 32, "hk": 8, "d": 128, "dtype": "bf16"},
        # the keys and values of one decoded token, and of whole prompts
        {"name": "append one token", "path": "append", "lens": "161", "chunks": "1", "page": 16, "hk": 16, "d": 128,
         "dtype": "bf16"},
        {"name": "append prompts", "path": "append", "lens": "4096,1777,16,2300", "chunks": "4096,1777,16,2000",
         "page": 16, "hk": 16, "d": 128, "dtype": "bf16"},
        # a decoded token's probability with the alternatives that an interface shows
        {"name": "logprobs one row", "path": "logprobs", "rows": 1, "vocab": 100352, "pad": 0, "top": 5, "dtype": "bf16",
         "banned": 0},
        # a document scored token by token
        {"name": "logprobs document", "path": "logprobs", "rows": 2048, "vocab": 100278, "pad": 74, "top": 20,
         "dtype": "bf16", "banned": 40},
    ]


def _log(rng: random.Random, lo: int, hi: int) -> int:
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


HEADS = ((16, 16), (32, 8), (12, 4), (8, 1), (6, 6), (10, 2), (4, 4), (28, 4), (16, 2), (5, 1))
HEAD_DIMS = (64, 128, 128, 128, 256, 80, 96, 40)


def draw(rng: random.Random) -> dict:
    path = rng.choice(("packed", "packed", "paged", "paged", "paged", "append", "logprobs", "logprobs"))
    if path == "logprobs":
        rows, vocab = _log(rng, 1, 2048), _log(rng, 200, 160000)
        return {"path": path, "rows": rows, "vocab": vocab, "pad": rng.choice((0, 0, -vocab % 64)),
                "top": rng.choice((0, 1, 5, 20, 32)), "dtype": rng.choice(("bf16", "bf16", "fp16", "fp32")),
                "banned": rng.choice((0, 0, vocab // 50))}
    hq, hk = rng.choice(HEADS)
    d, dtype = rng.choice(HEAD_DIMS), rng.choice(("bf16", "bf16", "fp16"))
    count = _log(rng, 1, 64)
    if path == "packed":
        mean = _log(rng, 8, 8192)
        lens = [max(1, round(mean * rng.uniform(0.1, 1.9))) for _ in range(count)]
        while sum(lens) > 16384 or sum(n * n for n in lens) * hq * d > 2.5e11:
            lens = lens[:-1] if len(lens) > 1 else [lens[0] // 2]
        return {"path": path, "lens": ",".join(map(str, lens)), "hq": hq, "hk": hk, "d": d, "dtype": dtype,
                "causal": rng.random() < 0.8, "pad": rng.choice((0, 0, rng.randint(1, 200))),
                "fused": rng.random() < 0.5}
    mean, chunk = _log(rng, 8, 32768), _log(rng, 1, 512) if rng.random() < 0.6 else 1
    lens = [max(1, round(mean * rng.uniform(0.1, 1.9))) for _ in range(count)]
    while sum(lens) * hk * d > 2.5e8:
        lens = lens[:-1] if len(lens) > 1 else [lens[0] // 2]
    chunks = [min(n, chunk if rng.random() < 0.7 else rng.randint(1, chunk)) for n in lens]
    while sum(c * n for c, n in zip(chunks, lens)) * hq * d > 2.5e11:
        lens, chunks = (lens[:-1], chunks[:-1]) if len(lens) > 1 else (lens, [chunks[0] // 2])
    case = {"path": path, "lens": ",".join(map(str, lens)), "chunks": ",".join(map(str, chunks)),
            "page": rng.choice((8, 16, 16, 32, 64, 128, 256)), "hk": hk, "d": d, "dtype": dtype}
    if path == "paged":
        case["hq"] = hq
    return case


def _ints(text: str) -> list[int]:
    return [int(x) for x in text.split(",")]


def _offsets(lens: list[int]) -> list[int]:
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return out


def prepare(case: dict, seed: int) -> dict:
    g = torch.Generator(device=DEV).manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def randn(*shape: int) -> torch.Tensor:
        return torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32).to(dt)

    if case["path"] == "logprobs":
        rows, vocab = case["rows"], case["vocab"]
        # an LM head's rows: a broad normal body with a few likely tokens far above it
        logits = torch.randn(rows, vocab + case["pad"], generator=g, device=DEV, dtype=torch.float32) * 2.0
        likely = torch.randint(0, vocab, (rows, 12), generator=g, device=DEV)
        boost = torch.rand(rows, 12, generator=g, device=DEV) * 12.0
        logits.scatter_add_(1, likely, boost)
        logits = logits.to(dt)[:, :vocab]
        targets = torch.randint(0, vocab, (rows,), generator=g, device=DEV)
        pick = torch.rand(rows, generator=g, device=DEV) < 0.7  # mostly a likely token
        targets = torch.where(pick, likely[:, 0], targets)
        if case["banned"]:  # tokens that a program forbids; the given token is never one of them
            given = torch.gather(logits, 1, targets[:, None])
            logits[:, torch.randint(0, vocab, (case["banned"],), generator=g, device=DEV)] = -math.inf
            logits.scatter_(1, targets[:, None], given)
        return {"case": case, "logits": logits, "targets": targets}

    lens, hk, d = _ints(case["lens"]), case["hk"], case["d"]
    i32 = lambda xs: torch.tensor(xs, dtype=torch.int32, device=DEV)  # noqa: E731
    if case["path"] == "packed":
        hq, total = case["hq"], sum(lens) + case["pad"]
        if case["fused"]:
            qkv = randn(total, (hq + 2 * hk) * d).view(total, hq + 2 * hk, d)
            q, k, v = qkv[:, :hq], qkv[:, hq:hq + hk], qkv[:, hq + hk:]
        else:
            q, k, v = randn(total, hq, d), randn(total, hk, d), randn(total, hk, d)
        return {"case": case, "q": q, "k": k, "v": v, "cu": i32(_offsets(lens)), "offsets": _offsets(lens)}

    chunks, page = _ints(case["chunks"]), case["page"]
    pages = [-(-n // page) for n in lens]
    pool = sum(pages) + 3
    # the pool's pages go to the sequences in no order; the table's unused entries are -1
    order = torch.randperm(pool, generator=g, device=DEV).to(torch.int32)
    table = torch.full((len(lens), max(pages)), -1, dtype=torch.int32, device=DEV)
    used = 0
    for b, n in enumerate(pages):
        table[b, :n] = order[used:used + n]
        used += n
    state = {"case": case, "k_pages": randn(pool, page, hk, d), "v_pages": randn(pool, page, hk, d), "table": table,
             "lengths": i32(lens), "cu": i32(_offsets(chunks)), "offsets": _offsets(chunks), "lens": lens}
    if case["path"] == "paged":
        state["q"] = randn(sum(chunks), case["hq"], d)
    else:
        state["k"], state["v"] = randn(sum(chunks), hk, d), randn(sum(chunks), hk, d)
    return state


def run(state: dict):
    return _own(state) if own else _plain(state)


def _own(state: dict):
    path = state["case"]["path"]
    if path == "logprobs":
        from byteprof_amd.optim.logprobs import token_logprobs

        out = token_logprobs(state["logits"], state["targets"], top=state["case"]["top"])
        return [out.logprob, out.entropy, out.top_ids, out.top_logprobs]
    from byteprof_amd.optim import attention

    if path == "packed":
        return attention.packed_attention(state["q"], state["k"], state["v"], state["cu"],
                                          causal=state["case"]["causal"])
    if path == "paged":
        return attention.paged_attention(state["q"], state["k_pages"], state["v_pages"], state["table"],
                                         state["lengths"], state["cu"])
    attention.paged_append(state["k"], state["v"], state["k_pages"], state["v_pages"], state["table"], state["lengths"],
                           state["cu"])
    return [state["k_pages"], state["v_pages"]]


def _plain_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, first: int | None) -> torch.Tensor:
    """q [n, Hq, D] over k, v [m, Hk, D] in float32; query i sees keys 0 .. first + i (first None: all of them). A row
    that sees nothing gives zeros."""
    n, hq, d = q.shape
    m, hk = k.shape[:2]
    group = hq // hk
    kf, vf = k.float().permute(1, 2, 0), v.float().permute(1, 0, 2)  # [Hk, D, m], [Hk, m, D]
    out = torch.empty(n, hq, d, dtype=torch.float32, device=q.device)
    step = max(1, min(n, (1 << 28) // max(1, hq * m)))
    for a in range(0, n, step):
        b = min(n, a + step)
        top = m if first is None else max(0, min(m, first + b))  # keys that any of these rows sees
        qf = q[a:b].float().reshape(b - a, hk, group, d).permute(1, 2, 0, 3).reshape(hk, group * (b - a), d)
        s = torch.matmul(qf, kf[:, :, :top]).view(hk, group, b - a, top) * d ** -0.5
        if first is not None:
            seen = torch.arange(top, device=q.device)[None, :] <= torch.arange(first + a, first + b, device=q.device)[:, None]
            s = torch.where(seen, s, -math.inf)
        p = torch.exp(s - s.amax(-1, keepdim=True).clamp_min(-3e38)) if top else s
        total = p.sum(-1, keepdim=True)
        p = torch.where(total > 0, p / total, 0.0)
        o = torch.matmul(p.reshape(hk, group * (b - a), top), vf[:, :top])
        out[a:b] = o.view(hk, group, b - a, d).permute(2, 0, 1, 3).reshape(b - a, hq, d)
    return out.to(q.dtype)


def _plain(state: dict):
    case = state["case"]
    path = case["path"]
    if path == "logprobs":
        return _plain_logprobs(state["logits"], state["targets"], case["top"])
    off = state["offsets"]
    if path == "packed":
        q, k, v = state["q"], state["k"], state["v"]
        out = torch.zeros(q.shape, dtype=q.dtype, device=q.device)
        for a, b in zip(off, off[1:]):
            out[a:b] = _plain_attention(q[a:b], k[a:b], v[a:b], 0 if case["causal"] else None)
        return out
    kp, vp, table, page = state["k_pages"], state["v_pages"], state["table"], case["page"]
    hk, d = case["hk"], case["d"]
    if path == "append":
        for b, (lo, hi) in enumerate(zip(off, off[1:])):
            at = torch.arange(state["lens"][b] - (hi - lo), state["lens"][b], device=DEV)
            slots = table[b, at // page].long() * page + at % page
            kp.view(-1, hk, d)[slots] = state["k"][lo:hi]
            vp.view(-1, hk, d)[slots] = state["v"][lo:hi]
        return [kp, vp]
    q = state["q"]
    out = torch.empty_like(q)
    for b, (lo, hi) in enumerate(zip(off, off[1:])):
        n = state["lens"][b]
        ids = table[b, :-(-n // page)].long()
        k, v = kp[ids].reshape(-1, hk, d)[:n], vp[ids].reshape(-1, hk, d)[:n]
        out[lo:hi] = _plain_attention(q[lo:hi], k, v, n - (hi - lo))
    return out


def _plain_logprobs(logits: torch.Tensor, targets: torch.Tensor, top: int):
    """In float32, some rows at a time; the order of equal logits is that of their ids."""
    rows, vocab = logits.shape
    parts = []
    step = max(1, (1 << 27) // vocab)
    for a in range(0, rows, step):
        x = logits[a:a + step].float() + 0.0  # -0 becomes +0: the two are equal
        m = x.amax(-1, keepdim=True)
        d = x - m
        e = torch.exp(d)
        z = e.sum(-1, keepdim=True)
        lz = torch.log(z)
        lp = torch.gather(d, 1, targets[a:a + step, None]) - lz
        h = lz - torch.where(e > 0, e * d, 0.0).sum(-1, keepdim=True) / z
        bits = x.view(torch.int32)
        rank = (bits ^ ((bits >> 31) & 0x7FFFFFFF)).long() * (1 << 32) + (vocab - 1 - torch.arange(vocab, device=x.device))
        ids = vocab - 1 - (torch.topk(rank, top, dim=-1, sorted=True).values & 0xFFFFFFFF)
        parts.append((lp[:, 0], h[:, 0], ids, torch.gather(d, 1, ids) - lz))
    return [torch.cat(p) for p in zip(*parts)]


def exact(case: dict, seed: int):
    state = prepare(case, seed)
    path = case["path"]
    if path == "logprobs":
        outs = []
        for x, t in zip(state["logits"].split(256), state["targets"].split(256)):
            x = x.double()
            lse = torch.logsumexp(x, -1)
            p = torch.exp(x - lse[:, None])
            ent = -(p * torch.where(p > 0, x - lse[:, None], 0.0)).sum(-1)
            vals, ids = torch.sort(x, dim=-1, descending=True, stable=True)
            outs.append((x[torch.arange(len(t), device=x.device), t] - lse, ent, ids[:, :case["top"]],
                         vals[:, :case["top"]] - lse[:, None]))
        return [torch.cat(o) for o in zip(*outs)]
    off, hk = state["offsets"], case["hk"]
    if path == "append":
        want = [state["k_pages"].clone(), state["v_pages"].clone()]
        for b, (lo, hi) in enumerate(zip(off, off[1:])):
            rows = state["table"][b].tolist()
            for i in range(lo, hi):
                at = state["lens"][b] - hi + i
                for pool, new in zip(want, (state["k"], state["v"])):
                    pool[rows[at // case["page"]], at % case["page"]] = new[i]
        return [w.double() for w in want]
    q = state["q"]
    group = case["hq"] // hk
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    for b, (lo, hi) in enumerate(zip(off, off[1:])):
        if path == "packed":
            k, v, before = state["k"][lo:hi], state["v"][lo:hi], 0
        else:
            n = state["lens"][b]
            at = torch.arange(n, device=q.device)
            where = (state["table"][b][at // case["page"]].long(), at % case["page"])
            k, v, before = state["k_pages"][where], state["v_pages"][where], n - (hi - lo)
        causal = path == "paged" or case["causal"]
        for h in range(case["hq"]):
            kh, vh = k[:, h // group].double(), v[:, h // group].double()
            for a in range(lo, hi, 4096):
                z = min(hi, a + 4096)
                s = q[a:z, h].double() @ kh.T / math.sqrt(case["d"])
                if causal:
                    last = before + torch.arange(a - lo, z - lo, device=q.device)
                    s.masked_fill_(torch.arange(len(kh), device=q.device)[None, :] > last[:, None], -math.inf)
                out[a:z, h] = torch.softmax(s, -1) @ vh
    return out


def work(case: dict) -> dict:
    size = {"bf16": 2, "fp16": 2, "fp32": 4}[case["dtype"]]
    if case["path"] == "logprobs":
        n = case["rows"] * case["vocab"]
        # an exponential, two sums and a maximum an element
        return {"bytes": n * size + case["rows"] * (16 + 12 * case["top"]), "flops": 5 * n}
    lens, hk, d = _ints(case["lens"]), case["hk"], case["d"]
    if case["path"] == "append":
        tokens = sum(_ints(case["chunks"]))
        return {"bytes": 4 * tokens * hk * d * size, "flops": 0}
    hq = case["hq"]
    if case["path"] == "packed":
        pairs = sum(n * (n + 1) // 2 if case["causal"] else n * n for n in lens)
        tokens = sum(lens)
        return {"bytes": size * d * (tokens * (hq + 2 * hk) + (tokens + case["pad"]) * hq), "flops": 4 * d * hq * pairs}
    chunks = _ints(case["chunks"])
    pairs = sum(c * (n - c) + c * (c + 1) // 2 for n, c in zip(lens, chunks))
    return {"bytes": size * d * (2 * hq * sum(chunks) + 2 * hk * sum(lens)), "flops": 4 * d * hq * pairs}
