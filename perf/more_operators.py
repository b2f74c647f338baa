"""Workloads of the operators around a paged cache held in 8 bits, and of rotary positions.

`prepare` makes what a program has in hand before the call (inputs, the page pool with its scales, the table, the device's
lengths), `run` makes one pass: with `own` the calls of byteprof_amd.optim.attention and byteprof_amd.optim.rotary, without it
the same operators in elementary torch. `exact` restates a pass in float64. The paths:

  rotary     q and k [tokens, heads, head_dim] turned by position x frequency, the angles right at any position; half or
             interleaved pairs, the whole head or its first columns
  append     a chunk's keys and values into their pages as 8-bit codes (e4m3 or int8) with a power of two for each block of
             tokens and head, then the sequences read back, so that the pass returns the values that the cache now stands for.
             A block that already holds tokens keeps its scale or takes a greater one, and its codes are rounded again
  read       the last positions of each sequence out of the pages, as values
  attention  a chunk of new tokens of each sequence (one for a decode step, several for a verify round, many for a part of a
             prompt) over its 8-bit cache; the chunk's own keys are in the cache already
"""

from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
CODES = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}


def listed() -> list[dict]:
    return [
        # one decoded token of a decoder of 16 heads of 128, q | k | v as slices of one projection: latency
        {"name": "rotary one token", "path": "rotary", "tokens": 1, "hq": 16, "hk": 16, "d": 128, "rot": 128,
         "interleaved": False, "dtype": "bf16", "fused": True, "far": 4000, "stretch": 1.0},
        # a batch of prompts, positions stretched for a long context
        {"name": "rotary prompts", "path": "rotary", "tokens": 8192, "hq": 32, "hk": 8, "d": 128, "rot": 128,
         "interleaved": False, "dtype": "bf16", "fused": True, "far": 131072, "stretch": 8.0},
        # interleaved pairs in a part of each head, an odd number of tokens at far positions
        {"name": "rotary part of the head", "path": "rotary", "tokens": 1537, "hq": 12, "hk": 4, "d": 80, "rot": 32,
         "interleaved": True, "dtype": "fp16", "fused": False, "far": 1 << 20, "stretch": 1.0},
        # one decoded token into the middle of a block, whose earlier codes may have to be rounded again
        {"name": "append one token", "path": "append", "lens": "155", "chunks": "1", "page": 16, "block": 16, "hk": 16, "d": 128,
         "kind": "int8", "dtype": "bf16"},
        # whole prompts and a later part of one
        {"name": "append prompts", "path": "append", "lens": "4096,1777,16,2300", "chunks": "4096,1777,16,2000", "page": 16,
         "block": 16, "hk": 16, "d": 128, "kind": "e4m3", "dtype": "bf16"},
        # a cached beginning of a prompt handed to a program that wants it in 16 bits
        {"name": "read one prefix", "path": "read", "lens": "161", "chunks": "161", "page": 16, "block": 16, "hk": 16, "d": 128,
         "kind": "e4m3", "dtype": "bf16"},
        # many sequences moved out of a cache of small heads
        {"name": "read many sequences", "path": "read", "lens": "8191,4500,700,2049,12000,333", "chunks": "8191,4500,700,2049,9000,1",
         "page": 64, "block": 32, "hk": 12, "d": 64, "kind": "int8", "dtype": "fp16"},
        # one token of one sequence behind a short prompt: the smallest decode step
        {"name": "attention one token", "path": "attention", "lens": "161", "chunks": "1", "page": 16, "block": 16, "hq": 16,
         "hk": 16, "d": 128, "kind": "e4m3", "dtype": "bf16"},
        # a decode step of many sequences of all lengths
        {"name": "attention decode batch", "path": "attention", "lens": ",".join(str(64 + (i * 2659) % 8111) for i in range(64)),
         "chunks": ",".join(["1"] * 64), "page": 16, "block": 16, "hq": 32, "hk": 8, "d": 128, "kind": "e4m3", "dtype": "bf16"},
        # a decode step over a few long contexts, as many query heads as key heads
        {"name": "attention long contexts", "path": "attention", "lens": "40000,65537,9000", "chunks": "1,1,1", "page": 128,
         "block": 64, "hq": 16, "hk": 16, "d": 64, "kind": "int8", "dtype": "bf16"},
        # a verify round: 8 drafts + 1 of six sequences, one of them long
        {"name": "attention verify round", "path": "attention", "lens": "40961,900,2500,130,7777,512", "chunks": "9,9,9,9,9,9",
         "page": 64, "block": 32, "hq": 16, "hk": 4, "d": 128, "kind": "int8", "dtype": "fp16"},
        # parts of prompts behind what the cache holds of them
        {"name": "attention prompt chunks", "path": "attention", "lens": "8192,4500,700,2049", "chunks": "512,512,511,1",
         "page": 32, "block": 32, "hq": 32, "hk": 8, "d": 128, "kind": "e4m3", "dtype": "bf16"},
    ]


def _log(rng: random.Random, lo: int, hi: int) -> int:
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


HEADS = ((16, 16), (32, 8), (12, 4), (8, 1), (6, 6), (10, 2), (4, 4), (28, 4), (16, 2), (5, 1))
HEAD_DIMS = (64, 128, 128, 128, 256, 80, 96, 40)


def draw(rng: random.Random) -> dict:
    path = rng.choice(("rotary", "rotary", "append", "append", "read", "attention", "attention", "attention"))
    hq, hk = rng.choice(HEADS)
    d = rng.choice(HEAD_DIMS)
    if path == "rotary":
        tokens = _log(rng, 1, 8192)
        while tokens * (hq + hk) * d > 4.2e7:
            tokens //= 2
        return {"path": path, "tokens": tokens, "hq": hq, "hk": hk, "d": d, "rot": rng.choice((d, d, d // 2, 2 * rng.randint(1, d // 2))),
                "interleaved": rng.random() < 0.4, "dtype": rng.choice(("bf16", "bf16", "fp16", "fp32")),
                "fused": rng.random() < 0.5, "far": _log(rng, 2, 1 << 22), "stretch": rng.choice((1.0, 4.0, 32.0))}
    page = rng.choice((8, 16, 16, 32, 64, 128, 256))
    block = rng.choice([b for b in (4, 8, 16, 32, 64, page) if page % b == 0 and (b >= 8 or rng.random() < 0.3)])
    case = {"path": path, "page": page, "block": block, "hk": hk, "d": d, "kind": rng.choice(("e4m3", "int8")),
            "dtype": rng.choice(("bf16", "bf16", "fp16"))}
    count = _log(rng, 1, 64)
    if path == "attention":
        mean, chunk = _log(rng, 8, 32768), _log(rng, 1, 512) if rng.random() < 0.5 else 1
    else:
        mean, chunk = _log(rng, 8, 4096), _log(rng, 1, 4096)
    lens = [max(1, round(mean * rng.uniform(0.1, 1.9))) for _ in range(count)]
    chunks = [min(n, chunk if rng.random() < 0.7 else rng.randint(1, chunk)) for n in lens]
    while (max(lens) * len(lens) * hk * d > 2.6e8 or (path != "attention" and sum(lens) * hk * d > 1.6e7)
           or (path == "attention" and len(lens) * max(chunks) * max(lens) * hq > 5e8)):
        lens, chunks = (lens[:-1], chunks[:-1]) if len(lens) > 1 else ([lens[0] // 2], [max(1, min(lens[0], chunks[0]) // 2)])
    case["lens"], case["chunks"] = ",".join(map(str, lens)), ",".join(map(str, chunks))
    if path == "attention":
        case["hq"] = hq
    return case


def _ints(text: str) -> list[int]:
    return [int(x) for x in text.split(",")]


def _offsets(lens: list[int]) -> list[int]:
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return out


def _frequencies(rot: int, stretch: float) -> tuple[torch.Tensor, float]:
    """Frequencies 10000^(-2i / rot); stretched: those that turn fewer than once in 4096 positions divided by `stretch`, those
    that turn more than 32 times as they are, a ramp between, and the factor that goes with it on cosine and sine."""
    f = 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    if stretch == 1.0:
        return f.float().to(DEV), 1.0
    keep = ((4096 * f / (2 * math.pi) - 1) / 31).clamp(0, 1)
    return (f * keep + f / stretch * (1 - keep)).float().to(DEV), 0.1 * math.log(stretch) + 1


def _scale_bytes(amax: torch.Tensor, kind: str) -> torch.Tensor:
    """The exponent byte (bias 127) of the least power of two that amax, in float32, divided by is at most 448 or 127: the
    exponent of amax less that of the greatest code, one more where amax has the greater significand."""
    bits = amax.view(torch.int32)
    byte = ((bits + 0x1FFFFF) >> 23) - 8 if kind == "e4m3" else ((bits + 0x01FFFF) >> 23) - 6
    return byte.clamp_min(0)


def _power(byte: torch.Tensor) -> torch.Tensor:
    """2 ** (byte - 127) in float32."""
    byte = byte.to(torch.int32)
    return torch.where(byte == 0, 0x400000, byte << 23).view(torch.float32)


def _encode(x: torch.Tensor, byte: torch.Tensor, kind: str) -> torch.Tensor:
    x = x * _power(254 - byte)
    return x.to(torch.float8_e4m3fn) if kind == "e4m3" else torch.round(x).to(torch.int8)


def prepare(case: dict, seed: int) -> dict:
    g = torch.Generator(device=DEV).manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def randn(*shape: int) -> torch.Tensor:
        return torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32)

    hk, d = case["hk"], case["d"]
    if case["path"] == "rotary":
        tokens, hq = case["tokens"], case["hq"]
        if case["fused"]:
            qkv = randn(tokens, (hq + 2 * hk) * d).to(dt).view(tokens, hq + 2 * hk, d)
            q, k = qkv[:, :hq], qkv[:, hq:hq + hk]
        else:
            q, k = randn(tokens, hq, d).to(dt), randn(tokens, hk, d).to(dt)
        # sequences of 500 tokens that begin anywhere
        begin = torch.randint(0, case["far"], (tokens // 500 + 1,), generator=g, device=DEV)
        at = torch.arange(tokens, device=DEV)
        inv_freq, factor = _frequencies(case["rot"], case["stretch"])
        return {"case": case, "q": q, "k": k, "positions": (begin[at // 500] + at) % case["far"], "inv_freq": inv_freq,
                "factor": factor}

    lens, chunks, page, block, kind = _ints(case["lens"]), _ints(case["chunks"]), case["page"], case["block"], case["kind"]
    i32 = lambda xs: torch.tensor(xs, dtype=torch.int32, device=DEV)  # noqa: E731
    pages = [-(-n // page) for n in lens]
    pool = sum(pages) + 3
    # the pool's pages go to the sequences in no order; the table's unused entries are -1
    order = torch.randperm(pool, generator=g, device=DEV).to(torch.int32)
    table = torch.full((len(lens), max(pages)), -1, dtype=torch.int32, device=DEV)
    used = 0
    for b, n in enumerate(pages):
        table[b, :n] = order[used:used + n]
        used += n
    state = {"case": case, "table": table, "lengths": i32(lens), "cu": i32(_offsets(chunks)), "tokens": sum(chunks),
             "all": i32(_offsets(lens)), "lens": lens, "chunks": chunks}
    for name in ("k", "v"):
        # blocks of different magnitudes
        x = randn(pool, page // block, block, hk, d) * torch.exp2(0.7 * randn(pool, page // block, 1, hk, 1))
        byte = _scale_bytes(x.abs().amax((2, 4)), kind)
        state[name + "_pages"] = _encode(x, byte[:, :, None, :, None], kind).view(pool, page, hk, d)
        state[name + "_scales"] = byte.to(torch.uint8).view(torch.float8_e8m0fnu)
    if case["path"] == "attention":
        state["q"] = randn(sum(chunks), case["hq"], d).to(dt)
    elif case["path"] == "append":
        state["k"], state["v"] = randn(sum(chunks), hk, d).to(dt), randn(sum(chunks), hk, d).to(dt)
    return state


def run(state: dict):
    return _own(state) if own else _plain(state)


def _own(state: dict):
    case = state["case"]
    if case["path"] == "rotary":
        from byteprof_amd.optim.rotary import rotary

        return rotary(state["q"], state["k"], state["positions"], state["inv_freq"], interleaved=case["interleaved"],
                      factor=state["factor"])
    from byteprof_amd.optim import attention

    where = (state["k_pages"], state["v_pages"], state["table"], state["lengths"])
    scales = {"k_scales": state["k_scales"], "v_scales": state["v_scales"]}
    if case["path"] == "attention":
        return attention.paged_attention(state["q"], *where, state["cu"], **scales)
    if case["path"] == "read":
        return attention.paged_read(*where, state["cu"], state["tokens"], dtype=DTYPES[case["dtype"]], **scales)
    attention.paged_append(state["k"], state["v"], *where, state["cu"], **scales)
    return attention.paged_read(*where, state["all"], sum(state["lens"]), dtype=DTYPES[case["dtype"]], **scales)


def _plain(state: dict):
    path = state["case"]["path"]
    if path == "rotary":
        return [_plain_rotary(state, state["q"]), _plain_rotary(state, state["k"])]
    if path == "attention":
        return _plain_attention(state)
    if path == "append":
        _plain_append(state, "k")
        _plain_append(state, "v")
        return [_plain_read(state, "k", state["all"], sum(state["lens"])), _plain_read(state, "v", state["all"], sum(state["lens"]))]
    return [_plain_read(state, "k", state["cu"], state["tokens"]), _plain_read(state, "v", state["cu"], state["tokens"])]


def _plain_rotary(state: dict, x: torch.Tensor) -> torch.Tensor:
    case = state["case"]
    angle = state["positions"].double()[:, None] * state["inv_freq"].double()
    cos, sin = (angle.cos() * state["factor"]).float()[:, None], (angle.sin() * state["factor"]).float()[:, None]
    turned, rest = x[..., :case["rot"]].float(), x[..., case["rot"]:]
    if case["interleaved"]:
        a, b = turned[..., ::2], turned[..., 1::2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = turned.chunk(2, -1)
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([turned.to(x.dtype), rest], -1)


def _places(state: dict, cu: torch.Tensor, tokens: int) -> tuple[torch.Tensor, ...]:
    """Of every token of the chunks: its page, its place in the page, its sequence and its position."""
    at = torch.arange(tokens, device=DEV)
    b = torch.bucketize(at, cu[1:].long(), right=True)
    pos = (state["lengths"] - cu[1:]).long()[b] + at
    page = state["case"]["page"]
    return state["table"].long()[b, pos // page], pos % page, b, pos


def _plain_read(state: dict, name: str, cu: torch.Tensor, tokens: int) -> torch.Tensor:
    page, slot, _, _ = _places(state, cu, tokens)
    byte = state[name + "_scales"].view(torch.uint8)[page, slot // state["case"]["block"]]
    return (state[name + "_pages"][page, slot].float() * _power(byte)[..., None]).to(DTYPES[state["case"]["dtype"]])


def _plain_append(state: dict, name: str) -> None:
    case, cu = state["case"], state["cu"].long()
    kind, block, hk, d = case["kind"], case["block"], case["hk"], case["d"]
    x = state[name].float()
    page, slot, b, pos = _places(state, state["cu"], state["tokens"])
    blocks = case["page"] // block
    unit = page * blocks + slot // block
    scales = state[name + "_scales"].view(torch.uint8).view(-1, hk)
    codes = state[name + "_pages"].view(-1, block, hk, d)
    # the least scale that the new tokens of each block need
    amax = torch.zeros(len(scales), hk, device=DEV)
    amax.scatter_reduce_(0, unit[:, None].expand(-1, hk), x.abs().amax(-1), "amax")
    need = _scale_bytes(amax, kind)[unit]
    # the blocks that hold tokens from before the chunk: each chunk's first, if the chunk does not begin it
    first = cu[:-1]
    old = unit[first]
    held = pos[first] - (pos[first] - pos[first] % case["page"] + slot[first] // block * block)  # tokens of it before the chunk
    had = scales[old].int()
    grown = torch.where(held[:, None] > 0, torch.maximum(had, need[first]), need[first])
    again = _encode(codes[old].float() * _power(had)[:, None, :, None], grown[:, None, :, None], kind)
    keep = torch.arange(block, device=DEV)[None, :] < held[:, None]
    raw = codes.view(torch.uint8)
    raw[old] = torch.where(keep[:, :, None, None], again.view(torch.uint8), raw[old])
    byte = torch.where((unit == old[b])[:, None], grown[b], need)
    scales[unit] = byte.to(torch.uint8)
    raw[unit, slot % block] = _encode(x, byte[:, :, None], kind).view(torch.uint8)


def _plain_attention(state: dict) -> torch.Tensor:
    """In float32, the sequences side by side, each padded to the longest; a padded key counts as one that comes later."""
    case, q, cu = state["case"], state["q"], state["cu"].long()
    page, block, hk, hq, d = case["page"], case["block"], case["hk"], case["hq"], case["d"]
    seqs, most, chunk = len(state["lens"]), max(state["lens"]), max(state["chunks"])
    ids = state["table"].long().clamp_min(0)

    def values(name: str) -> torch.Tensor:  # [sequences, Hk, keys, D]
        scale = _power(state[name + "_scales"].view(torch.uint8)[ids])
        x = state[name + "_pages"][ids].float().view(*ids.shape, page // block, block, hk, d) * scale[:, :, :, None, :, None]
        return x.view(seqs, -1, hk, d)[:, :most].permute(0, 2, 1, 3)

    b = torch.bucketize(torch.arange(len(q), device=DEV), cu[1:], right=True)
    i = torch.arange(len(q), device=DEV) - cu[b]
    padded = torch.zeros(seqs, chunk, hq, d, device=DEV)
    padded[b, i] = q.float()
    rows = padded.view(seqs, chunk, hk, hq // hk, d).permute(0, 2, 1, 3, 4).reshape(seqs, hk, chunk * (hq // hk), d)
    s = torch.matmul(rows, values("k").transpose(2, 3).contiguous()).view(seqs, hk, chunk, hq // hk, most) * d ** -0.5
    first = (state["lengths"].long() - cu[1:] + cu[:-1])[:, None] + torch.arange(chunk, device=DEV)
    unseen = torch.arange(most, device=DEV)[None, None, :] > torch.minimum(first, state["lengths"].long()[:, None] - 1)[:, :, None]
    s.masked_fill_(unseen[:, None, :, None, :], -math.inf)
    s -= s.amax(-1, keepdim=True)
    s.exp_()
    s /= s.sum(-1, keepdim=True)
    o = torch.matmul(s.view(seqs, hk, -1, most), values("v").contiguous()).view(seqs, hk, chunk, hq // hk, d)
    return o.permute(0, 2, 1, 3, 4).reshape(seqs, chunk, hq, d)[b, i].to(q.dtype)


def exact(case: dict, seed: int):
    state = prepare(case, seed)
    if case["path"] == "rotary":
        outs, rot = [], case["rot"]
        theta = state["positions"].to(torch.float64).reshape(-1, 1, 1) * state["inv_freq"].to(torch.float64)
        turn = torch.polar(torch.full_like(theta, state["factor"]), theta)
        for x in (state["q"], state["k"]):
            y = x.to(torch.float64).clone()
            if case["interleaved"]:
                re, im = y[..., 0:rot:2].clone(), y[..., 1:rot:2].clone()
            else:
                re, im = y[..., :rot // 2].clone(), y[..., rot // 2:rot].clone()
            z = torch.complex(re, im) * turn
            if case["interleaved"]:
                y[..., 0:rot:2], y[..., 1:rot:2] = z.real, z.imag
            else:
                y[..., :rot // 2], y[..., rot // 2:rot] = z.real, z.imag
            outs.append(y)
        return outs
    page, block, hk = case["page"], case["block"], case["hk"]
    lens, chunks, rows = state["lens"], state["chunks"], state["table"].tolist()

    def cached(name: str, b: int) -> torch.Tensor:
        """The values that the cache stands for of sequence b, before the pass: [length, Hk, D]."""
        ids = torch.tensor(rows[b][:-(-lens[b] // page)], device=DEV)
        codes = state[name + "_pages"][ids].to(torch.float64)
        exponent = state[name + "_scales"].view(torch.uint8)[ids].to(torch.float64) - 127
        return (codes * torch.exp2(exponent).repeat_interleave(block, 1)[..., None]).reshape(-1, hk, case["d"])[:lens[b]]

    def step(x: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
        """x to the nearest multiple of what a code at scale can hold."""
        if case["kind"] == "int8":
            return torch.round(x / scale) * scale
        least = torch.full_like(x, 2.0 ** -6)
        power = torch.exp2(torch.floor(torch.log2(torch.maximum((x / scale).abs(), least))) - 3) * scale
        return torch.round(x / power) * power

    if case["path"] in ("append", "read"):
        outs = []
        for name in ("k", "v"):
            parts = []
            for b, (n, c) in enumerate(zip(lens, chunks)):
                x = cached(name, b)
                if case["path"] == "read":
                    parts.append(x[n - c:])
                    continue
                off = sum(chunks[:b])
                new, start = state[name][off:off + c].to(torch.float64), n - c
                greatest = 448.0 if case["kind"] == "e4m3" else 127.0
                for at in range(start // block * block, n, block):
                    lo, hi = max(at, start), min(at + block, n)
                    amax = new[lo - start:hi - start].abs().amax((0, 2))
                    scale = torch.exp2(torch.ceil(torch.log2(amax / greatest)).clamp_min(-127))
                    if at < start:
                        had = state[name + "_scales"].view(torch.uint8)[rows[b][at // page], at % page // block]
                        scale = torch.maximum(scale, torch.exp2(had.to(torch.float64) - 127))
                        x[at:start] = step(x[at:start], scale[:, None])
                    x[lo:hi] = step(new[lo - start:hi - start], scale[:, None])
                parts.append(x)
            outs.append(torch.cat(parts))
        return outs
    q, off = state["q"], _offsets(chunks)
    group = case["hq"] // hk
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    for b, (lo, hi) in enumerate(zip(off, off[1:])):
        k, v, before = cached("k", b), cached("v", b), lens[b] - (hi - lo)
        for h in range(case["hq"]):
            s = q[lo:hi, h].double() @ k[:, h // group].T / math.sqrt(case["d"])
            last = before + torch.arange(hi - lo, device=q.device)
            s.masked_fill_(torch.arange(len(k), device=q.device)[None, :] > last[:, None], -math.inf)
            out[lo:hi, h] = torch.softmax(s, -1) @ v[:, h // group]
    return out


def work(case: dict) -> dict:
    size, hk, d = {"bf16": 2, "fp16": 2, "fp32": 4}[case["dtype"]], case["hk"], case["d"]
    if case["path"] == "rotary":
        n = case["tokens"] * (case["hq"] + hk)
        return {"bytes": 2 * size * n * d + 8 * case["tokens"], "flops": 3 * n * case["rot"]}
    lens, chunks = _ints(case["lens"]), _ints(case["chunks"])
    held = 2 * hk * (d + 1 / case["block"])  # bytes of a cached position
    if case["path"] == "read":
        return {"bytes": sum(chunks) * (held + 2 * size * hk * d), "flops": 0}
    if case["path"] == "append":
        # the chunks in and their codes out, then all codes in and their values out
        return {"bytes": sum(chunks) * (held + 2 * size * hk * d) + sum(lens) * (held + 2 * size * hk * d), "flops": 0}
    pairs = sum(c * (n - c) + c * (c + 1) // 2 for n, c in zip(lens, chunks))
    return {"bytes": 2 * size * d * case["hq"] * sum(chunks) + sum(lens) * held, "flops": 4 * d * case["hq"] * pairs}
