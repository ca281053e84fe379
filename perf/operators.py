"""What serving with a paged key/value cache has the framework do, as cases that can be timed.

A server keeps the attention keys and values of many sequences in pages of a few tokens that any sequence may hold in any
order, as bf16 values or in 4 bits.  Its three calls on them:

  append  new tokens: queries and keys normalised and rotated to their positions, keys and values stored in their pages.
          In 4 bits the stored rows are read back as well, as a server does that moves a sequence or checks what it holds.
  attend  attention of the new tokens' queries over the pages: one token of every sequence, a few (guessed ahead), or
          whole prompts of different lengths side by side; optionally with scores capped by a tanh, a bias by distance,
          a prefix that every row sees, and the model's output gate.
  read    rows of the cache as plain values (a sequence that is moved to another machine, or to disk).

Layout: pages [num_pages, 2 (keys, values), kv_heads, page_size, head_dim]; in 4 bits two codes to a byte (the even
dimension in the low half, code + 8) beside scales [num_pages, 2, kv_heads, page_size, head_dim / 32] in f16.  Sequence b
owns rows q_start[b] to q_start[b + 1] - 1 of the call; they are its last tokens of kv_len[b].
"""
import math
import random

import torch

own = False

# (heads, kv_heads, head_dim, rotated dimensions): the framework's default model, then generic ones.
SHAPES = [(16, 4, 256, 64), (32, 8, 128, 128), (16, 2, 128, 32), (20, 4, 128, 64), (8, 8, 64, 64), (24, 8, 64, 32), (16, 1, 64, 64)]
BASE = dict(bits=16, page=16, ragged=True, norm=False, gate=False, cap=0.0, slopes=False, prefix=False)


def case(name, kind, shape, sequences, new, cached, **more):
    heads, kv_heads, dim, rot = shape
    out = dict(kind=kind, heads=heads, kv_heads=kv_heads, dim=dim, rot=rot, sequences=sequences, new=new, cached=cached, **dict(BASE, **more))
    return dict(out, name=name) if name else out


def listed():
    model, wide, five, small, one = SHAPES[0], SHAPES[1], SHAPES[3], SHAPES[4], SHAPES[6]
    return [
        # One token of one sequence: the smallest call there is.
        case("append_1", "append", model, 1, 1, 1023, norm=True),
        # The prompts of a few users arrive together and are kept in 4 bits.
        case("append_prompts_4bit", "append", wide, 5, 2500, 300, bits=4, page=32),
        # The first answer tokens of one short chat.
        case("step_1", "attend", model, 1, 1, 700, gate=True),
        # The benchmark's batch: 64 sequences decoded together, of different lengths.
        case("step_64", "attend", model, 64, 1, 8191, gate=True, page=64),
        # One very long document in 4 bits, one token at a time.
        case("step_long_4bit", "attend", model, 1, 1, 131000, bits=4, page=64, gate=True),
        # Many sequences in 4 bits, three tokens each (two of them guessed ahead), an odd group of heads.
        case("guess_96_4bit", "attend", five, 96, 3, 5000, bits=4, page=32),
        # Prompts of different lengths side by side, as a scheduler packs them.
        case("prompts", "attend", model, 4, 2048, 0, gate=True, page=64),
        # The next piece of a long prompt whose beginning is in the cache, in 4 bits.
        case("piece_4bit", "attend", wide, 2, 1024, 7000, bits=4, page=64, ragged=False),
        # Capped scores and a bias by distance, an odd length, small heads without sharing.
        case("capped", "attend", small, 3, 1501, 77, cap=30.0, slopes=True),
        # A prefix (an image, an instruction) that every row sees, many heads on one.
        case("prefix", "attend", one, 8, 700, 0, prefix=True, page=128),
        # A long sequence leaves the machine, and one in 4 bits.
        case("read", "read", model, 1, 30001, 0, page=64),
        case("read_4bit", "read", wide, 7, 6000, 0, bits=4),
    ]


def draw(rng):
    """Any kind, shape, format and page size; lengths spread over their logarithm, held to the listed cases' cost."""
    def spread(low, high):
        return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))

    shape = rng.choice(SHAPES)
    common = dict(bits=rng.choice((4, 16)), page=rng.choice((16, 32, 64, 128, 256)), ragged=rng.random() < 0.7)
    kind = rng.choice(("append", "step", "step", "prompt", "prompt", "read"))
    if kind in ("append", "read"):
        sequences = spread(1, 64)
        new = spread(1, max(2, 16000 // sequences))
        return case(None, kind, shape, sequences, new, spread(1, 4000) if kind == "append" else 0, norm=rng.random() < 0.5, **common)
    common.update(gate=rng.random() < 0.5, cap=rng.choice((0.0, 0.0, 30.0, 50.0)), slopes=rng.random() < 0.25, prefix=rng.random() < 0.25)
    if kind == "step":
        sequences = spread(1, 128)
        return case(None, "attend", shape, sequences, rng.choice((1, 1, 1, 2, 4)), spread(1, 200000 // sequences), **common)
    sequences = spread(1, 16)
    new = spread(5, 2200 // sequences)
    return case(None, "attend", shape, sequences, new, rng.choice((0, spread(1, 4500 // sequences))), **common)


def lengths(c):
    """(new tokens, tokens in the cache with them) of every sequence; the first has the case's own figures."""
    r = random.Random(c["sequences"] * 7919 + c["new"] * 31 + c["cached"])
    new, total = [], []
    for b in range(c["sequences"]):
        some = c["ragged"] and b > 0
        n = r.randint((c["new"] + 1) // 2, c["new"]) if some else c["new"]
        old = r.randint(c["cached"] // 4, c["cached"]) if some else c["cached"]
        new.append(n)
        total.append(old + n)
    return new, total


def prefixes(c):
    """A prefix for every sequence, some of them past its end or of no length."""
    _, total = lengths(c)
    r = random.Random(c["sequences"] + c["cached"])
    return [r.choice((0, t // 4, t // 2, t + 5)) for t in total]


def prepare(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    H, G, D, P, R = c["heads"], c["kv_heads"], c["dim"], c["page"], c["rot"]
    new, total = lengths(c)
    tokens, held = sum(new), [-(-t // P) for t in total]
    count = sum(held) + 3  # some pages are nobody's
    order, width = torch.randperm(count, generator=g, device="cuda").to(torch.int32), max(held)
    first = torch.tensor([sum(held[:b]) for b in range(len(held))], device="cuda")[:, None] + torch.arange(width, device="cuda")[None]
    s = dict(c, max_q=max(new), max_kv=max(total), tokens=tokens)
    s["page_table"] = order[first.clamp(max=count - 1)].contiguous()
    s["q_start"] = torch.tensor([sum(new[:b]) for b in range(len(new) + 1)], dtype=torch.int32, device="cuda")
    s["kv_len"] = torch.tensor(total, dtype=torch.int32, device="cuda")

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)

    # channels of a trained model's keys differ in size; values do so less
    channel = torch.exp(0.4 * normal(2, G, 1, D))
    s["pages"], s["scales"] = (torch.empty(count, 2, G, P, D if c["bits"] == 16 else D // 2, device="cuda", dtype=torch.bfloat16 if c["bits"] == 16 else torch.uint8), None)
    if c["bits"] == 4:
        s["scales"] = torch.empty(count, 2, G, P, D // 32, device="cuda", dtype=torch.float16)
    step = max(1, (1 << 26) // (2 * G * P * D))
    for at in range(0, count, step):
        n = min(step, count - at)
        rows = (normal(n, 2, G, P, D) * channel).to(torch.bfloat16)
        if c["bits"] == 16:
            s["pages"][at:at + n] = rows
        else:
            s["pages"][at:at + n], s["scales"][at:at + n] = quantised(rows)
    if c["kind"] == "append":
        s["qg"] = normal(tokens, H, 2, D).to(torch.bfloat16)  # queries and output gates of a head side by side, as projected
        s["k"] = (normal(tokens, G, D) * channel[0, :, 0]).to(torch.bfloat16)
        s["v"] = (normal(tokens, G, D) * channel[1, :, 0]).to(torch.bfloat16)
        angle = torch.arange(max(total), device="cuda", dtype=torch.float64)[:, None] * 1e7 ** (-torch.arange(R // 2, device="cuda", dtype=torch.float64)[None] * 2 / R)
        s["cos"], s["sin"] = (torch.cat((f(angle), f(angle)), 1).float().contiguous() for f in (torch.cos, torch.sin))
        s["q_norm"], s["k_norm"] = ((0.1 * normal(D)).to(torch.bfloat16) if c["norm"] else None for _ in range(2))
    elif c["kind"] == "attend":
        s["q"] = normal(tokens, H, D).to(torch.bfloat16)
        s["gate"] = normal(tokens, H, 2, D).to(torch.bfloat16)[:, :, 1] if c["gate"] else None
        s["slopes"] = (2.0 ** (-8.0 * torch.arange(1, H + 1, device="cuda") / H)).float() if c["slopes"] else None
        s["prefix"] = torch.tensor(prefixes(c), dtype=torch.int32, device="cuda") if c["prefix"] else None
    return s


# ---- the plain form ------------------------------------------------------------------------------------------------------


def quantised(rows):
    """bf16 rows [..., dim] -> codes [..., dim / 2], scales [..., dim / 32]: blocks of 32 with scale largest / 7."""
    x = rows.float().unflatten(-1, (-1, 32))
    scale = (x.abs().amax(-1) / 7).clamp(max=65504).half()
    d = scale.float()[..., None]
    codes = torch.where(d > 0, torch.round(x / d), torch.zeros_like(x)).clamp(-7, 7).add(8).to(torch.uint8).flatten(-2)
    return codes[..., 0::2] | codes[..., 1::2] << 4, scale


def values(codes, scales):
    """What codes and scales stand for, in 32 bits (exact)."""
    c = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).float() - 8
    return (c.unflatten(-1, (-1, 32)) * scales.float()[..., None]).flatten(-2)


def once_rounded(x):
    """f64 -> bf16 in one rounding (through f32, which is moved off the middle where its own rounding put it there)."""
    f = x.float()
    middle = (f.view(torch.int32) & 0xffff == 0x8000) & (f.double() != x)
    away = torch.where(x > f.double(), math.inf, -math.inf).float()
    return torch.where(middle, torch.nextafter(f, away), f).to(torch.bfloat16)


def places(s):
    """Sequence and position of every row of the call."""
    t = torch.arange(s["tokens"], device="cuda")
    b = torch.searchsorted(s["q_start"][1:].long(), t, right=True)
    return b, s["kv_len"][b].long() - s["q_start"][b + 1].long() + t


def slots(s, b, position):
    return s["page_table"][b, position // s["page"]].long(), position % s["page"]


def rotated(x, norm, s, position):
    """Normalised (where the model has weights for it) and rotated, in 64 bits: angles and values next to a rounding border."""
    x = x.double()
    if norm is not None:
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + 1e-6) * (1 + norm.double())
    r = s["rot"]
    c, n = s["cos"][position].double()[:, None], s["sin"][position].double()[:, None]
    a, b, rest = x[..., :r // 2], x[..., r // 2:r], x[..., r:]
    return once_rounded(torch.cat((a * c[..., :r // 2] - b * n[..., :r // 2], b * c[..., r // 2:] + a * n[..., r // 2:], rest), -1))


def plain_append(s):
    b, position = places(s)
    page, slot = slots(s, b, position)
    q = rotated(s["qg"][:, :, 0], s["q_norm"], s, position)
    for which, rows in enumerate((rotated(s["k"], s["k_norm"], s, position), s["v"])):
        if s["bits"] == 16:
            s["pages"][page, which, :, slot] = rows
        else:
            s["pages"][page, which, :, slot], s["scales"][page, which, :, slot] = quantised(rows)
    return q


def plain_read(s):
    b, position = places(s)
    page, slot = slots(s, b, position)
    got = (s["pages"][page, :, :, slot] if s["bits"] == 16 else values(s["pages"][page, :, :, slot], s["scales"][page, :, :, slot]).to(torch.bfloat16))
    return got[:, 0].contiguous(), got[:, 1].contiguous()


def plain_attend(s):
    B, H, G, D = s["sequences"], s["heads"], s["kv_heads"], s["dim"]
    S = H // G
    length, start = s["kv_len"].long()[:, None], s["q_start"].long()
    i, j = torch.arange(s["max_q"], device="cuda")[None], torch.arange(s["max_kv"], device="cuda")[None]
    count = (start[1:] - start[:-1])[:, None]
    row = torch.minimum(start[:-1, None] + i, start[1:, None] - 1)
    page, slot = slots(s, torch.arange(B, device="cuda")[:, None], torch.minimum(j, length - 1))
    kv = s["pages"][page, :, :, slot]
    kv = kv.float() if s["bits"] == 16 else values(kv, s["scales"][page, :, :, slot])  # B, keys, 2, G, D
    k, v = kv[:, :, 0].permute(0, 2, 3, 1), kv[:, :, 1].transpose(1, 2)
    q = s["q"][row].float().unflatten(2, (G, S)).permute(0, 2, 3, 1, 4).reshape(B, G, S * s["max_q"], D)
    x = (q @ k * D ** -0.5).unflatten(2, (S, s["max_q"]))
    if s["cap"]:
        x = s["cap"] * torch.tanh(x / s["cap"])
    position = (length - count + i)[:, :, None]
    away = j[:, None] - position
    if s["slopes"] is not None:
        x = x - s["slopes"].view(1, G, S, 1, 1) * away.abs()[:, None, None]
    seen = away <= 0
    if s["prefix"] is not None:
        seen = seen | (j < s["prefix"].long()[:, None])[:, None]
    seen = (seen & (j < length)[:, None])[:, None, None]
    x = torch.where(seen, x, -math.inf)
    top = x.amax(-1, keepdim=True)
    x = torch.where(seen, torch.exp(x - top), 0)
    total = x.sum(-1, keepdim=True)
    out = (x.flatten(2, 3) @ v).unflatten(2, (S, s["max_q"]))
    out = torch.where(total > 0, out / total, 0).permute(0, 3, 1, 2, 4).flatten(2, 3)[(i < count)]  # tokens, H, D
    if s["gate"] is not None:
        out = out * torch.sigmoid(s["gate"].float())
    return out.to(torch.bfloat16)


# ---- one pass ------------------------------------------------------------------------------------------------------------


def run(s):
    if own:
        from llmcp_b200 import paged
        cache = paged.Cache(s["pages"], s["scales"])
        batch = paged.Batch(s["q_start"], s["kv_len"], s["page_table"], s["max_q"], s["max_kv"])
        if s["kind"] == "append":
            q = paged.append(cache, batch, s["qg"][:, :, 0], s["k"], s["v"], s["cos"], s["sin"], q_norm=s["q_norm"], k_norm=s["k_norm"])
            if s["bits"] == 16:
                return {"q": q, "pages": s["pages"]}
            k, v = paged.read(cache, batch, s["tokens"])
            return {"q": q, "k": k, "v": v}
        if s["kind"] == "read":
            k, v = paged.read(cache, batch, s["tokens"])
            return {"k": k, "v": v}
        return {"out": paged.attention(cache, batch, s["q"], softcap=s["cap"], slopes=s["slopes"], prefix=s["prefix"], gate=s["gate"])}
    if s["kind"] == "append":
        q = plain_append(s)
        if s["bits"] == 16:
            return {"q": q, "pages": s["pages"]}
        k, v = plain_read(s)
        return {"q": q, "k": k, "v": v}
    if s["kind"] == "read":
        k, v = plain_read(s)
        return {"k": k, "v": v}
    return {"out": plain_attend(s)}


def row_bytes(c):
    """Bytes of one key or value of one head in the cache."""
    return 2 * c["dim"] if c["bits"] == 16 else c["dim"] // 2 + c["dim"] // 16


def work(c):
    new, total = lengths(c)
    tokens, H, G, D = sum(new), c["heads"], c["kv_heads"], c["dim"]
    tables = 4 * (2 * c["sequences"] + 1 + sum(-(-t // c["page"]) for t in total))
    if c["kind"] == "append":
        # queries in and out, keys and values in, rows of the cache out (in 4 bits also in again and out as values)
        moved = tokens * (4 * H * D + 4 * G * D + 2 * G * row_bytes(c)) + 8 * c["rot"] * tokens
        moved += 0 if c["bits"] == 16 else tokens * 2 * G * (row_bytes(c) + 2 * D)
        return {"bytes": tables + moved, "flops": tokens * (H + G) * (3 * c["rot"] + (4 * D if c["norm"] else 0))}
    if c["kind"] == "read":
        return {"bytes": tables + tokens * 2 * G * (row_bytes(c) + 2 * D), "flops": 0 if c["bits"] == 16 else tokens * 2 * G * D}
    front = prefixes(c) if c["prefix"] else [0] * len(new)
    pairs = sum(sum(min(t, max(t - n + i + 1, f)) for i in range(n)) for n, t, f in zip(new, total, front))
    return {"bytes": tables + sum(total) * 2 * G * row_bytes(c) + tokens * H * D * (6 if c["gate"] else 4), "flops": 4 * D * H * pairs}


# ---- the definition in 64 bits, a sequence at a time -----------------------------------------------------------------------


def nearest(x, bits, least):
    """Round to `bits` significant bits, ties to even, with steps no finer than 2^least."""
    _, e = torch.frexp(x)
    unit = torch.ldexp(torch.ones_like(x), torch.clamp(e - bits, min=least))
    return torch.round(x / unit) * unit


def exact_rows(s, rows):
    """What the cache holds for rows given in 64 bits."""
    rows = nearest(rows, 8, -133)
    if s["bits"] == 16:
        return rows
    blocks = rows.reshape(*rows.shape[:-1], -1, 32)
    scale = torch.clamp(nearest(blocks.abs().amax(-1, keepdim=True) / 7, 11, -24), max=65504.0)
    codes = torch.clamp(torch.round(blocks / torch.where(scale == 0, 1.0, scale)), -7, 7) * (scale != 0)
    return (codes * scale).reshape(rows.shape)


def held(s, b, which, first, last):
    """Keys (0) or values (1) `first` to `last` - 1 of sequence b from the pages, in 64 bits: [keys, kv_heads, dim]."""
    at = torch.arange(first, last, device=s["pages"].device)
    rows = (s["page_table"].long()[b][at // s["page"]], which, slice(None), at % s["page"])
    raw = s["pages"][rows]
    if s["bits"] == 16:
        return raw.double()
    unpacked = torch.empty(*raw.shape[:2], s["dim"], dtype=torch.float64, device=raw.device)
    unpacked[..., 0::2], unpacked[..., 1::2] = (raw % 16).double() - 8, (raw // 16).double() - 8
    return unpacked * s["scales"][rows].double().repeat_interleave(32, -1)


def exact(c, seed):
    s = prepare(c, seed)
    new, total = lengths(c)
    G, D, R = c["kv_heads"], c["dim"], c["rot"]
    firsts = [sum(new[:b]) for b in range(len(new))]

    def turned(x, weight, n, t):
        x = x.double()
        if weight is not None:
            x = x * torch.rsqrt((x * x).sum(-1, keepdim=True) / D + 1e-6) * (weight.double() + 1)
        turn = torch.complex(s["cos"][t - n:t, :R // 2].double(), s["sin"][t - n:t, :R // 2].double())[:, None]
        z = torch.complex(x[..., :R // 2], x[..., R // 2:R]) * turn
        return torch.cat((z.real, z.imag, x[..., R:]), -1)

    if c["kind"] == "append":
        part = [slice(f, f + n) for f, n in zip(firsts, new)]
        q = torch.cat([turned(s["qg"][p, :, 0], s["q_norm"], n, t) for p, n, t in zip(part, new, total)])
        k = exact_rows(s, torch.cat([turned(s["k"][p], s["k_norm"], n, t) for p, n, t in zip(part, new, total)]))
        v = exact_rows(s, s["v"].double())
        if c["bits"] == 4:
            return {"q": q, "k": k, "v": v}
        pages = s["pages"].double()
        for b, (p, n, t) in enumerate(zip(part, new, total)):
            at = torch.arange(t - n, t, device=pages.device)
            where = s["page_table"].long()[b][at // s["page"]]
            pages[where, 0, :, at % s["page"]], pages[where, 1, :, at % s["page"]] = k[p], v[p]
        return {"q": q, "pages": pages}
    if c["kind"] == "read":
        return {name: torch.cat([held(s, b, which, t - n, t) for b, (n, t) in enumerate(zip(new, total))]) for which, name in enumerate("kv")}
    front = prefixes(c) if c["prefix"] else [0] * len(new)
    outs = []
    for b, (f, n, t) in enumerate(zip(firsts, new, total)):
        k, v = held(s, b, 0, 0, t), held(s, b, 1, 0, t)
        position = torch.arange(t - n, t, device=k.device)
        keys = torch.arange(t, device=k.device)
        last = torch.clamp(torch.clamp(position + 1, min=front[b]), max=t)  # keys 0 .. last - 1 are seen
        heads = []
        for h in range(c["heads"]):
            z = s["q"][f:f + n, h].double() @ k[:, h * G // c["heads"]].T / math.sqrt(D)
            if c["cap"]:
                z = torch.tanh(z / c["cap"]) * c["cap"]
            if c["slopes"]:
                z = z - (position[:, None] - keys[None]).abs() * float(s["slopes"][h])
            heads.append(torch.softmax(z.masked_fill(keys[None] >= last[:, None], -math.inf), -1) @ v[:, h * G // c["heads"]])
        outs.append(torch.stack(heads, 1))
    out = torch.cat(outs)
    return {"out": out if s["gate"] is None else out / (1 + torch.exp(-s["gate"].double()))}
