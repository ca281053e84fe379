"""The paged key/value cache in plain 64-bit arithmetic on the CPU: what tests/test_paged.py and tests/test_gpu_paged.py compare with."""
import math

import torch

NAN16 = 0x7E00


def bf16_round(x):
    """float64 -> the nearest bf16 value (ties to even), as float64; steps end at the subnormal one, 2^-133."""
    _, e = torch.frexp(x)
    unit = torch.ldexp(torch.ones_like(x), torch.clamp(e - 8, min=-133))
    return torch.where(torch.isfinite(x), torch.round(x / unit) * unit, x)


def quantise(y):
    """bf16 rows as float64 [..., dim] -> (codes -7..7 [..., dim], scales [..., dim / 32] float16)."""
    blocks = y.unflatten(-1, (-1, 32))
    top = blocks.abs().amax(-1)
    scale = (top / 7).clamp(max=65504).to(torch.float16)  # from float64, via float32: 7 times a middle of f16 is no bf16 value
    scale = torch.where(blocks.isnan().any(-1), torch.full_like(scale, math.nan), scale)
    d = scale.double()[..., None]
    codes = torch.where(d > 0, torch.round(blocks / d), torch.zeros_like(blocks)).clamp(-7, 7)
    return codes.flatten(-2), scale


def rotate(x, weight, cos, sin, eps=1e-6):
    """x [tokens, heads, dim] -> normalised and rotated, float64; cos and sin [tokens, rot]."""
    x = x.double()
    if weight is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * (1 + weight.double())
    if cos is None:
        return x
    half = cos.shape[1] // 2
    c, s = cos.double()[:, None], sin.double()[:, None]
    a, b = x[..., :half], x[..., half:2 * half]
    return torch.cat((a * c[..., :half] - b * s[..., :half], b * c[..., half:] + a * s[..., half:], x[..., 2 * half:]), -1)


def tables(batch, page_size, spare, seed, bad=-7):
    """(q_start, kv_len, page_table, number of pages) of [(new, total)] with pages in random order; unused entries are `bad`."""
    g = torch.Generator().manual_seed(seed)
    held = [-(-t // page_size) for _, t in batch]
    count = sum(held) + spare
    order = torch.randperm(count, generator=g).to(torch.int32)
    table = torch.full((len(batch), max(held + [1])), bad, dtype=torch.int32)
    at = 0
    for b, n in enumerate(held):
        table[b, :n] = order[at:at + n]
        at += n
    starts = [0]
    for n, _ in batch:
        starts.append(starts[-1] + n)
    return torch.tensor(starts, dtype=torch.int32), torch.tensor([t for _, t in batch], dtype=torch.int32), table, count


def unpack(pages, scales):
    """The values a 4-bit cache stands for, float64."""
    codes = torch.stack((pages & 15, pages >> 4), -1).flatten(-2).double() - 8
    return (codes.unflatten(-1, (-1, 32)) * scales.double()[..., None]).flatten(-2)


def sequence_rows(values, table, b, which, total):
    """Keys or values of sequence b: [total, kv_heads, dim] from values [pages, 2, heads, size, dim]."""
    size = values.shape[3]
    j = torch.arange(total)
    return values[table[b, j // size].long(), which, :, j % size]


def attention(q, values, q_start, kv_len, table, scale, softcap=0.0, slopes=None, prefix=None, gate=None, rows=None):
    """(out, weight, (reach, span)) in float64: out as defined, weight = sum p |v| * gate (what a relative error of the weights
    moves out by at most); per [row, head] reach = the largest sum |q k scale| among the seen keys, and span = their number
    times the largest |v| among them (what an absolute error of the weights moves out by)."""
    tokens, heads, dim = q.shape
    out, weight = torch.zeros(tokens, heads, dim, dtype=torch.float64), torch.zeros(tokens, heads, dim, dtype=torch.float64)
    reach, span = torch.zeros(tokens, heads, 1, dtype=torch.float64), torch.zeros(tokens, heads, 1, dtype=torch.float64)
    for b in range(len(kv_len)):
        first, end, total = int(q_start[b]), int(q_start[b + 1]), int(kv_len[b])
        if end == first or total == 0:
            continue
        k, v = (sequence_rows(values, table, b, which, total).double() for which in (0, 1))
        position = torch.arange(first, end) - end + total
        j = torch.arange(total)
        seen = j[None] <= position[:, None]
        if prefix is not None:
            seen |= (j < int(prefix[b]))[None]
        for h in range(heads):
            g = h // (heads // k.shape[1])
            x = q[first:end, h].double() @ k[:, g].T * scale
            far = q[first:end, h].double().abs() @ k[:, g].abs().T * abs(scale)
            if softcap:
                x = softcap * torch.tanh(x / softcap)
            if slopes is not None:
                x = x - float(slopes[h]) * (position[:, None] - j[None]).abs()
            x = x.masked_fill(~seen, -math.inf)
            p = torch.nan_to_num(torch.softmax(x, -1), nan=0.0)
            out[first:end, h], weight[first:end, h] = p @ v[:, g], p @ v[:, g].abs()
            reach[first:end, h, 0] = (far * seen).amax(-1)
            span[first:end, h, 0] = seen.sum(-1) * v[:, g].abs().max()
    if gate is not None:
        s = torch.sigmoid(gate.double())
        out, weight = out * s, weight * s
    return out, weight, (reach, span)


def attention_bound(out, weight, extent, bits, softcap=0.0):
    """How far a kernel may be from attention()'s out.  Half a step of bf16 (2^-8) for the result.  Weights: rounded to bf16
    (2^-8) over bf16 pages, to f16 (2^-11) over 4-bit pages; there the values' and keys' f16 forms too (2^-11 each, the
    keys' as a change of the score, which moves a weight and the sum by its size: twice).  f32 sums: 2^-20 of what is
    added up; exp, tanh and the score's scaling 2^-18 beside them, and 2^-20 of the cap.

    Over 4-bit pages a weight has f16's range too: below 2^-14 its steps are 2^-24, so it is off by up to 2^-25 there.  With
    the row's largest weight held at 2^7 or more (times the largest value scale, which goes into the weights or stays with
    the values), that is 2^-32 of the largest weight for each key, and as much of the largest value for the result, which
    the sum of the weights (at least the largest) divides.  It shows where a heavy key's value is 0 and only weights below
    2^-21 of the largest are left."""
    reach, span = extent
    relative = 2.0 ** -8 if bits == 16 else 2.0 ** -10
    score = reach * (2.0 ** -20 + (0 if bits == 16 else 2.0 ** -11)) + softcap * 2.0 ** -20
    return 2.0 ** -8 * out.abs() + weight * (relative + 2 * score + 2.0 ** -17) * (1 + 2.0 ** -7) + (0 if bits == 16 else span * 2.0 ** -32) + 1e-30
