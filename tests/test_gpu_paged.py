"""The paged key/value cache on a B200 against plain 64-bit arithmetic (tests/paged_reference.py).

What append stores and what read returns has to be the correctly rounded value, bit for bit; attention stays within the
bound that paged_reference.attention_bound derives.  Everything that must not matter is NaN: cache rows from a sequence's
length on, rows behind the last sequence, pages nobody owns."""
import math

import numpy as np
import pytest
import torch

import llmcp_b200 as L
import paged_reference as R
from llmcp_b200 import paged

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def cuda(*tensors):
    out = [None if t is None else t.cuda() for t in tensors]
    return out if len(out) > 1 else out[0]


def empty_cache(count, heads, size, dim, bits):
    """A cache of NaN: (pages, scales) on the GPU."""
    if bits == 16:
        return torch.full((count, 2, heads, size, dim), math.nan, dtype=BF, device="cuda"), None
    return (torch.full((count, 2, heads, size, dim // 2), 0xF1, dtype=torch.uint8, device="cuda"),
            torch.full((count, 2, heads, size, dim // 32), math.nan, dtype=torch.float16, device="cuda"))


def filled_cache(seed, batch, table, count, heads, size, dim, bits, scale=1.0):
    """A cache whose owned rows hold random values, everything else NaN: (pages, scales, values float32 on the CPU)."""
    g = torch.Generator().manual_seed(seed)
    pages, scales = empty_cache(count, heads, size, dim, bits)
    values = torch.zeros(count, 2, heads, size, dim)
    host, host_scales = pages.cpu(), None if scales is None else scales.cpu()
    for b, (_, total) in enumerate(batch):
        for p in range(-(-total // size)):
            n, page = min(size, total - p * size), int(table[b, p])
            y = R.bf16_round(scale * torch.randn(2, heads, n, dim, generator=g, dtype=torch.float64))
            if bits == 16:
                host[page, :, :, :n] = y.to(BF)
                values[page, :, :, :n] = y.float()
            else:
                codes, d = R.quantise(y)
                code8 = (codes + 8).to(torch.uint8)
                host[page, :, :, :n] = code8[..., 0::2] | code8[..., 1::2] << 4
                host_scales[page, :, :, :n] = d
                values[page, :, :, :n] = ((codes.unflatten(-1, (-1, 32)) * d.double()[..., None]).flatten(-2)).float()
    pages.copy_(host)
    if scales is not None:
        scales.copy_(host_scales)
    return pages, scales, values


def make_batch(q_start, kv_len, table, batch, **changes):
    a = dict(max_q=max([n for n, _ in batch] + [0]), max_kv=max([t for _, t in batch] + [0]))
    a.update(changes)
    return paged.Batch(*cuda(q_start, kv_len, table), a["max_q"], a["max_kv"])


# ---- append and read -----------------------------------------------------------------------------------------------------

SHAPES = [(4, 2, 64, 64), (5, 1, 128, 32), (16, 4, 256, 64), (3, 3, 256, 256), (6, 2, 64, 4), (0, 2, 128, 128), (2, 1, 64, 0)]
BATCHES = [[(1, 1)], [(1, 17), (1, 16), (1, 33)], [(5, 5), (0, 9), (1, 40), (20, 33)], [(130, 131), (17, 300)]]


@pytest.mark.parametrize("batch", BATCHES)
@pytest.mark.parametrize("heads,groups,dim,rot", SHAPES)
@pytest.mark.parametrize("bits", [16, 4])
def test_append_and_read(batch, heads, groups, dim, rot, bits):
    _append_and_read(batch, heads, groups, dim, rot, bits, 16 if dim != 128 else 64, norm=heads % 2 == 0)


def test_append_and_read_many_rows():
    """Enough rows for the kernels that take several heads per warp, and a number of heads that is no multiple of theirs."""
    _append_and_read([(700, 1000), (1500, 1500), (1300, 1311)], 11, 1, 128, 128, 4, 256, norm=True)
    _append_and_read([(3000, 3500), (2201, 2201)], 5, 5, 64, 32, 16, 32, norm=False)


def _append_and_read(batch, heads, groups, dim, rot, bits, size, norm):
    g = torch.Generator().manual_seed(len(batch) * 1000 + dim + rot + bits)
    q_start, kv_len, table, count = R.tables(batch, size, 2, 3)
    tokens, padded = int(q_start[-1]), int(q_start[-1]) + 3
    spread = torch.exp(torch.randn(padded, 1, 1, generator=g))
    qg = (torch.randn(padded, max(heads, 1), 2, dim, generator=g) * spread[..., None]).to(BF)
    k, v = ((torch.randn(padded, groups, dim, generator=g) * spread).to(BF) for _ in range(2))
    k[0, 0, :32] = 0  # a block of zeros
    q_norm, k_norm = ((0.2 * torch.randn(dim, generator=g)).to(BF) if norm else None for _ in range(2))
    longest = max(t for _, t in batch)
    angle = torch.arange(longest)[:, None] * torch.rand(1, max(rot // 2, 1), generator=g)
    cos, sin = ((torch.cat((f(angle), f(angle)), 1).float()[:, :rot].contiguous() if rot else None) for f in (torch.cos, torch.sin))
    pages, scales = empty_cache(count, groups, size, dim, bits)
    before = pages.clone(), None if scales is None else scales.clone()
    cache, call = paged.Cache(pages, scales), make_batch(q_start, kv_len, table, batch)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    q_out = torch.full((padded, heads, dim), 7.0, dtype=BF, device="cuda") if heads else None
    q_dev = cuda(qg)[:, :heads, 0] if heads else None
    got = paged.append(cache, call, q_dev, *cuda(k, v, cos, sin), q_norm=cuda(q_norm), k_norm=cuda(k_norm), q_out=q_out, status=status)
    k_read, v_read = paged.read(cache, call, padded, dtype=torch.float32, status=status)
    k16, v16 = paged.read(cache, call, padded)
    assert int(status) == 0
    position = torch.cat([torch.arange(t - n, t) for n, t in batch])
    rows = (cos[position], sin[position]) if rot else (None, None)
    if heads:
        want = R.bf16_round(R.rotate(qg[:tokens, :, 0], q_norm, *rows)).to(BF)
        assert torch.equal(got[:tokens].cpu(), want)
        assert (got[tokens:] == 7.0).all()  # rows behind the last sequence
    owner = torch.cat([torch.full((n,), b) for b, (n, _) in enumerate(batch)])
    page, slot = table[owner, position // size].long(), position % size
    expected = [t.cpu() for t in before if t is not None]
    for which, (x, weight) in enumerate(((k, k_norm), (v, None))):
        y = R.bf16_round(R.rotate(x[:tokens], weight, *rows) if which == 0 else x[:tokens].double())
        if bits == 16:
            expected[0][page, which, :, slot] = y.to(BF)
            held = y
        else:
            codes, d = R.quantise(y)
            code8 = (codes + 8).to(torch.uint8)
            expected[0][page, which, :, slot] = code8[..., 0::2] | code8[..., 1::2] << 4
            expected[1][page, which, :, slot] = d
            held = (codes.unflatten(-1, (-1, 32)) * d.double()[..., None]).flatten(-2)
        assert torch.equal((k_read, v_read)[which][:tokens].cpu(), held.float())
        assert torch.equal((k16, v16)[which][:tokens].cpu(), R.bf16_round(held).to(BF))
    for tensor, want in zip([t for t in (pages, scales) if t is not None], expected):
        assert torch.equal(tensor.cpu().view(torch.uint8), want.view(torch.uint8))  # the rows written, and no others


def test_append_rows_off_a_16_byte_boundary():
    """Rows that start two bytes off, with odd strides, give the values of dense ones."""
    g = torch.Generator().manual_seed(5)
    batch = [(3, 20), (2, 2)]
    q_start, kv_len, table, count = R.tables(batch, 16, 1, 1)
    flat = torch.randn(5 * 1000, generator=g).to(BF).cuda()
    views = [torch.as_strided(flat, (5, h, 128), (997, 133, 1), 1 + 2 * i) for i, h in enumerate((4, 2, 2))]
    call, results = make_batch(q_start, kv_len, table, batch), []
    for tensors in (views, [t.contiguous() for t in views]):
        pages, _ = empty_cache(count, 2, 16, 128, 16)
        results.append((paged.append(paged.Cache(pages), call, *tensors), pages))
    assert torch.equal(results[0][0], results[1][0])
    assert torch.equal(results[0][1].view(torch.int16), results[1][1].view(torch.int16))


def test_append_extreme_values_in_4_bits():
    """Middles between codes, infinities, values past 7 * 65504, subnormal scales, NaN: as the definition has them."""
    y = torch.zeros(8, 1, 64, dtype=torch.float64)
    y[0, 0, :14] = torch.tensor([s * (c + 0.5) for c in range(7) for s in (1, -1)])  # scale 1 with the next line
    y[0, 0, 31] = 7.0
    y[1, 0, 3], y[1, 0, 4] = math.inf, 1.0
    y[2, 0, :2] = torch.tensor([3e38, -500000.0])
    y[3, 0, :4] = torch.tensor([3e-7, -2e-7, 1e-7, 4e-8])
    y[4, 0, :2] = torch.tensor([1e-30, -1e-38])
    y[5, 0, 40] = math.nan
    y[6, 0] = torch.linspace(-3, 3, 64)
    y = R.bf16_round(y)
    pages, scales = empty_cache(1, 1, 16, 64, 4)
    cache = paged.Cache(pages, scales)
    call = make_batch(torch.tensor([0, 8], dtype=torch.int32), torch.tensor([8], dtype=torch.int32), torch.zeros(1, 1, dtype=torch.int32), [(8, 8)])
    x = y.to(BF).cuda()
    paged.append(cache, call, None, x, x)
    codes, d = R.quantise(y)
    want = (codes.unflatten(-1, (-1, 32)) * d.double()[..., None]).flatten(-2).float()
    for got in paged.read(cache, call, 8, dtype=torch.float32):
        assert torch.equal(got.cpu().isnan(), want.isnan())
        assert torch.equal(got.cpu().nan_to_num(), want.nan_to_num())
    assert want[0, 0, :4].tolist() == [0.0, 0.0, 2.0, -2.0]  # 0.5 and 1.5 go to the even code


def test_append_leaves_out_what_does_not_fit():
    """Pages that do not exist, positions past the rotation's table, lengths past the bounds: reported, nothing written."""
    pages, _ = empty_cache(2, 1, 16, 64, 16)
    cache, x = paged.Cache(pages), torch.ones(3, 1, 64, dtype=BF, device="cuda")
    table = torch.tensor([[0], [1], [2]], dtype=torch.int32)  # page 2 does not exist
    starts, lengths = torch.arange(4, dtype=torch.int32), torch.tensor([4, 5, 6], dtype=torch.int32)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    tables = torch.ones(8, 64, device="cuda")
    for change, written in ((dict(), {(0, 3), (1, 4)}), (dict(max_kv=5), {(0, 3), (1, 4)}), (dict(max_kv=4), {(0, 3)}), (dict(rows=5), {(0, 3), (1, 4)}),
                            (dict(rows=4), {(0, 3)}), (dict(max_q=0), set())):
        pages.fill_(math.nan)
        status.zero_()
        rows = change.pop("rows", 8)
        call = make_batch(starts, lengths, table, [(1, 6)], **change)
        paged.append(cache, call, None, x, x, tables[:rows], tables[:rows], status=status)
        assert int(status) == (4 if change.get("max_q") != 0 else 0)
        done = (~pages[:, 0, 0, :, 0].isnan()).nonzero().tolist()
        assert {tuple(p) for p in done} == written
        k, _ = paged.read(cache, call, 3)  # refuses the same rows
        torch.cuda.synchronize()


# ---- attention -----------------------------------------------------------------------------------------------------------

ATTENTION_BATCHES = [[(1, 1)], [(1, 0), (1, 15)], [(1, 16), (0, 9), (1, 17), (1, 300)], [(3, 40), (2, 2), (1, 700)], [(5, 3), (4, 64)],
                     [(33, 33), (1, 65)], [(130, 130), (1, 65), (64, 200)], [(257, 700), (40, 41)]]
ATTENTION_SHAPES = [(4, 2, 64), (5, 1, 128), (8, 2, 256), (16, 1, 64), (3, 3, 128), (16, 4, 256), (14, 2, 64), (40, 2, 128)]


def check_attention(batch, heads, groups, dim, bits, size, softcap=0.0, slopes=False, prefix=None, gate=False, scale=None, spread=1.0):
    g = torch.Generator().manual_seed(sum(n * 7 + t for n, t in batch) + dim + heads)
    q_start, kv_len, table, count = R.tables(batch, size, 2, 11)
    tokens, padded = int(q_start[-1]), int(q_start[-1]) + 2
    pages, scales, values = filled_cache(1, batch, table, count, groups, size, dim, bits)
    q = (spread * torch.randn(padded, heads, dim, generator=g)).to(BF)
    q[tokens:] = math.nan
    gates = torch.randn(padded, heads, 2, dim, generator=g).to(BF)[:, :, 1] if gate else None
    slope = torch.rand(heads, generator=g) * 0.5 if slopes else None
    front = None if prefix is None else torch.tensor(prefix[:len(batch)], dtype=torch.int32)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = torch.full((padded, heads, dim), 7.0, dtype=BF, device="cuda")
    cache, call = paged.Cache(pages, scales), make_batch(q_start, kv_len, table, batch)
    gates_dev = None if gates is None else torch.stack((gates, gates), 2).cuda()[:, :, 1]
    paged.attention(cache, call, cuda(q), scale=scale, softcap=softcap, slopes=cuda(slope), prefix=cuda(front), gate=gates_dev, out=out, status=status)
    assert int(status) == 0
    scale = dim ** -0.5 if scale is None else scale
    want, weight, reach = R.attention(q[:tokens], values, q_start, kv_len, table, scale, softcap, slope, front, None if gates is None else gates[:tokens])
    got = out[:tokens].cpu().double()
    off = (got - want).abs() / R.attention_bound(want, weight, reach, bits, softcap)
    assert not got.isnan().any() and off.max() <= 1, f"{off.max():.3f} of the bound at {np.unravel_index(int(off.argmax()), off.shape)}"
    assert (out[tokens:] == 7.0).all()  # rows behind the last sequence


@pytest.mark.parametrize("batch", ATTENTION_BATCHES)
@pytest.mark.parametrize("heads,groups,dim", ATTENTION_SHAPES)
@pytest.mark.parametrize("bits", [16, 4])
def test_attention(batch, heads, groups, dim, bits):
    check_attention(batch, heads, groups, dim, bits, {64: 16, 128: 64, 256: 32}[dim])


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("size", [16, 32, 64, 128, 256])
def test_attention_page_sizes(size, bits):
    check_attention([(1, 1000), (1, 255), (1, 257)], 8, 2, 128, bits, size)
    check_attention([(100, 513), (70, 255)], 8, 2, 128, bits, size)


@pytest.mark.parametrize("options", [dict(softcap=2.0), dict(softcap=30.0, gate=True), dict(slopes=True), dict(prefix=[5, 0, 300, 64, 1]),
                                     dict(gate=True), dict(softcap=5.0, slopes=True, prefix=[40, 1000, 3, 0, 2], gate=True), dict(scale=0.5),
                                     dict(spread=30.0), dict(scale=-0.1), dict(scale=0.0)], ids=str)
@pytest.mark.parametrize("batch", [[(1, 40), (1, 333), (1, 3)], [(5, 40), (2, 130), (7, 3)], [(150, 333), (5, 64), (64, 100)]])
@pytest.mark.parametrize("heads,groups,dim,bits", [(8, 2, 256, 16), (4, 2, 64, 4), (6, 2, 128, 16), (5, 1, 128, 4), (4, 1, 256, 4)])
def test_attention_options(batch, heads, groups, dim, bits, options):
    check_attention(batch, heads, groups, dim, bits, 32, **options)


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_attention_over_long_caches(bits, dim):
    """Few rows over many keys (the work of a row is split), beside short sequences, and a piece of a prompt on a long cache."""
    check_attention([(1, 20011), (1, 5), (3, 9000)], 4, 2, dim, bits, 64)
    check_attention([(20, 6000)], 8, 2, dim, bits, 32, slopes=True)


@pytest.mark.parametrize("bits", [16, 4])
def test_attention_many_sequences(bits):
    check_attention([(1, 1 + 37 * b % 400) for b in range(150)], 8, 2, 128, bits, 16, gate=True)


@pytest.mark.parametrize("rows", [1, 70])
def test_attention_scores_that_grow_along_the_keys(rows):
    """Every key outdoes those before it by more than the last: the running maximum moves all the way."""
    size, total, dim = 64, 600, 128
    q_start, kv_len, table, count = R.tables([(rows, total)], size, 0, 1)
    values = torch.zeros(count, 2, 1, size, dim)
    j = torch.arange(total)
    key = (j.double() * 0.5)[:, None, None].expand(-1, 1, dim) / dim
    values[table[0, j // size].long(), 0, :, j % size] = R.bf16_round(key).float()
    values[table[0, j // size].long(), 1, :, j % size] = torch.randn(total, 1, dim, generator=torch.Generator().manual_seed(1)).to(BF).float()
    q = torch.full((rows, 2, dim), 2.0, dtype=BF)
    got = paged.attention(paged.Cache(values.to(BF).cuda()), make_batch(q_start, kv_len, table, [(rows, total)]), q.cuda(), scale=1.0)
    want, weight, reach = R.attention(q, values, q_start, kv_len, table, 1.0)
    assert ((got.cpu().double() - want).abs() <= R.attention_bound(want, weight, reach, 16)).all()


@pytest.mark.parametrize("rows", [1, 40])
@pytest.mark.parametrize("bits", [16, 4])
def test_attention_leaves_out_what_does_not_fit(rows, bits):
    """A page that does not exist counts as zeros, a length past the bounds leaves its rows; both are reported."""
    batch = [(rows, 100), (rows, 90)]
    q_start, kv_len, table, count = R.tables(batch, 32, 1, 2)
    pages, scales, values = filled_cache(3, batch, table, count, 2, 32, 64, bits)
    q = torch.randn(2 * rows, 4, 64, generator=torch.Generator().manual_seed(1)).to(BF)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    for bad in (-1, count, 2 ** 31 - 1, -2 ** 31):
        broken, shown = table.clone(), values.clone()
        broken[0, 1], shown[table[0, 1].long()] = bad, 0
        status.zero_()
        got = paged.attention(paged.Cache(pages, scales), make_batch(q_start, kv_len, broken, batch), q.cuda(), status=status)
        want, weight, reach = R.attention(q, shown, q_start, kv_len, table, 0.125)
        assert int(status) == 4
        assert ((got.cpu().double() - want).abs() <= R.attention_bound(want, weight, reach, bits)).all()
    for change in (dict(max_kv=95), dict(lengths=[100, 129]), dict(lengths=[-5, 90]), dict(starts=[0, -1, 2 * rows]), dict(starts=[0, rows, 5000]), dict(max_q=0 if rows == 1 else rows - 1)):
        status.zero_()
        lengths, starts = change.pop("lengths", [100, 90]), change.pop("starts", q_start.tolist())
        call = make_batch(torch.tensor(starts, dtype=torch.int32), torch.tensor(lengths, dtype=torch.int32), table, batch, **dict(dict(max_kv=2000), **change))
        out = torch.full((2 * rows, 4, 64), 7.0, dtype=BF, device="cuda")
        paged.attention(paged.Cache(pages, scales), call, q.cuda(), out=out, status=status)
        assert int(status) == (0 if change.get("max_q") == 0 else 4)


def test_attention_far_into_a_large_cache():
    """Rows past 2^31 elements from the start of the cache, in both formats."""
    for bits, dim in ((16, 256), (4, 256)):
        size, heads = 64, 4
        count = (1 << 31) // (2 * heads * size * (dim if bits == 16 else dim // 2)) + 40
        batch = [(1, 500), (30, 300)]
        q_start, kv_len, table, small = R.tables(batch, size, 0, 4)
        pages, scales, values = filled_cache(9, batch, table, small, heads, size, dim, bits)
        large = torch.empty((count, *pages.shape[1:]), dtype=pages.dtype, device="cuda")
        large[count - small:] = pages
        large_scales = None
        if bits == 4:
            large_scales = torch.empty((count, *scales.shape[1:]), dtype=scales.dtype, device="cuda")
            large_scales[count - small:] = scales
        cache, call = paged.Cache(large, large_scales), make_batch(q_start, kv_len, (table + count - small) * (table >= 0), batch)
        q = torch.randn(31, 8, dim, generator=torch.Generator().manual_seed(1)).to(BF)
        want, weight, reach = R.attention(q, values, q_start, kv_len, table, dim ** -0.5)
        assert ((paged.attention(cache, call, q.cuda()).cpu().double() - want).abs() <= R.attention_bound(want, weight, reach, bits)).all()
        x = torch.randn(31, heads, dim, generator=torch.Generator().manual_seed(2)).to(BF).cuda()
        paged.append(cache, call, None, x, x)
        k, v = paged.read(cache, call, 31)
        if bits == 16:
            assert torch.equal(k, x) and torch.equal(v, x)
        else:
            assert torch.equal(k, v) and (k.float() - x.float()).abs().max() < 0.5


# ---- together ------------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("bits", [16, 4])
def test_a_conversation_in_one_captured_graph(bits):
    """Append and attention of a step are captured once; lengths move between replays, a padded slot stays empty; every
    step equals the plain result, and a second graph with a workspace of its own runs beside it on another stream."""
    heads, groups, dim, size, slots, steps = 8, 2, 256, 16, 4, 20
    g = torch.Generator().manual_seed(3)
    lengths0 = [37, 1, 300]
    batch = [(1, t + steps) for t in lengths0]
    q_start, _, table, count = R.tables(batch, size, 1, 8)
    table = torch.cat((table, torch.zeros(1, table.shape[1], dtype=torch.int32)))  # the padded slot
    pages, scales, values = filled_cache(5, [(1, t) for t in lengths0], table, count, groups, size, dim, bits)
    start = torch.tensor([0, 1, 2, 3, 3], dtype=torch.int32).cuda()  # three sequences in four slots
    lengths = torch.tensor(lengths0 + [0], dtype=torch.int32).cuda()
    states = []
    for _ in range(2):
        p, s = pages.clone(), None if scales is None else scales.clone()
        x = [torch.zeros(slots, h, dim, dtype=BF, device="cuda") for h in (heads, groups, groups)]
        cache, call = paged.Cache(p, s), paged.Batch(start, lengths, cuda(table), 1, 400)
        ws = torch.full((paged.workspace_bytes(cache, call, slots, heads) + 16,), 0xFF, dtype=torch.uint8, device="cuda")
        out = torch.full((slots, heads, dim), 7.0, dtype=BF, device="cuda")
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        paged.attention(cache, call, paged.append(cache, call, *x, status=status), out=out, workspace=ws, status=status)  # loads the kernels
        p.copy_(pages)
        if s is not None:
            s.copy_(scales)
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            paged.attention(cache, call, paged.append(cache, call, *x, status=status), out=out, workspace=ws, status=status)
        states.append((graph, x, out, cache, call, ws, status))  # a graph holds addresses: what it reads has to live
    side = torch.cuda.Stream()
    host_lengths = list(lengths0)
    for step in range(steps):
        host_lengths = [t + 1 for t in host_lengths]
        lengths.copy_(torch.tensor(host_lengths + [0], dtype=torch.int32))
        fresh = [torch.randn(slots, h, dim, generator=g).to(BF) for h in (heads, groups, groups)]
        for graph, x, out, *_ in states:
            for a, b in zip(x, fresh):
                a.copy_(b)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            states[1][0].replay()
        states[0][0].replay()
        torch.cuda.synchronize()
        for b, t in enumerate(host_lengths):
            where = (int(table[b, (t - 1) // size]), slice(None), slice(None), (t - 1) % size)
            row = torch.stack(fresh[1:])[:, b].double()
            if bits == 4:
                codes, d = R.quantise(row)
                row = (codes.unflatten(-1, (-1, 32)) * d.double()[..., None]).flatten(-2)
            values[where] = row.float()
        want, weight, reach = R.attention(fresh[0][:3], values, [0, 1, 2, 3], host_lengths, table, dim ** -0.5)
        for _, _, out, *_, status in states:
            assert int(status) == 0
            assert ((out[:3].cpu().double() - want).abs() <= R.attention_bound(want, weight, reach, bits)).all()
            assert (out[3] == 7.0).all()
    assert torch.equal(states[0][2], states[1][2])  # the same steps give the same bits


def test_same_call_gives_the_same_bits():
    batch = [(1, 9000), (1, 77), (2, 2500)]
    q_start, kv_len, table, count = R.tables(batch, 64, 0, 4)
    pages, scales, _ = filled_cache(2, batch, table, count, 2, 64, 128, 4)
    cache, call = paged.Cache(pages, scales), make_batch(q_start, kv_len, table, batch)
    q = torch.randn(4, 8, 128, generator=torch.Generator().manual_seed(6)).to(BF).cuda()
    first = paged.attention(cache, call, q)
    for _ in range(5):
        assert torch.equal(paged.attention(cache, call, q), first)


@pytest.mark.parametrize("S,position", [(1, 40), (50, 17)])
def test_layer_equals_the_frameworks_attention(S, position):
    """Append and attention over pages against llmcp_op_attention (exact mode) over its contiguous cache: the model's
    layer with its norms, rotation and gate.  Keys differ by at most their rounding (f64 here, f32 there)."""
    nh, nkv, hd, rot, cap, size = 16, 4, 256, 64, 96, 16
    g = torch.Generator().manual_seed(S)
    bits = lambda t: t.contiguous().view(torch.int16).numpy().view(np.uint16)
    qg, k, v = (torch.randn(S, n, generator=g).to(BF) for n in (nh * 2 * hd, nkv * hd, nkv * hd))
    q_norm, k_norm = ((0.1 * torch.randn(hd, generator=g)).to(BF) for _ in range(2))
    old = torch.randn(2, nkv, position, hd, generator=g).to(BF)
    cache = torch.zeros(2, nkv, cap, hd, dtype=BF)
    cache[:, :, :position] = old
    tables = [np.stack([L.make_cos_sin(p)[i] for p in range(cap)]) for i in (0, 1)]
    rows = slice(position, position + S)
    want, after = L.ops.attention(bits(qg), bits(k), bits(v), bits(q_norm), bits(k_norm), tables[0][rows], tables[1][rows], bits(cache),
                                  position, nh, nkv, hd, rot)
    to_float = lambda a: torch.from_numpy(np.ascontiguousarray(a).view(np.int16)).view(BF).double()
    want, after = to_float(want).view(S, nh, hd), to_float(after)
    total = position + S
    q_start, kv_len, table, count = R.tables([(S, total)], size, 1, 2)
    pages, _ = empty_cache(count, nkv, size, hd, 16)
    j = torch.arange(position)
    pages[cuda(table)[0, j // size].long(), :, :, j.cuda() % size] = old.permute(2, 0, 1, 3).cuda()
    c, call = paged.Cache(pages), make_batch(q_start, kv_len, table, [(S, total)])
    split = cuda(qg).view(S, nh, 2, hd)
    q = paged.append(c, call, split[:, :, 0], cuda(k).view(S, nkv, hd), cuda(v).view(S, nkv, hd), *(torch.from_numpy(t).cuda() for t in tables),
                     q_norm=cuda(q_norm), k_norm=cuda(k_norm))
    out = paged.attention(c, call, q, gate=split[:, :, 1]).cpu().double()
    whole = paged.Batch(torch.tensor([0, total], dtype=torch.int32).cuda(), *cuda(kv_len, table), total, total)
    keys, vals = (t.cpu().double() for t in paged.read(c, whole, total))
    assert ((keys.transpose(0, 1) - after[0, :, :total]).abs() <= 2.0 ** -7 * after[0, :, :total].abs() + 1e-30).all()
    assert torch.equal(vals.transpose(0, 1), after[1, :, :total])
    values = torch.zeros(count, 2, nkv, size, hd)
    at = torch.arange(total)
    values[table[0, at // size].long(), :, :, at % size] = after[:, :, :total].permute(2, 0, 1, 3).float()
    _, weight, (reach, span) = R.attention(q.cpu(), values, q_start, kv_len, table, hd ** -0.5, gate=split[:, :, 1].cpu())
    # beside the kernel's own bound: half a step of the other result, and scores that a step of a key or query (2^-7 in
    # 2^-7 * reach each, and hardly ever) may have moved
    assert ((out - want).abs() <= R.attention_bound(out, weight, (reach, span), 16) + 2.0 ** -8 * want.abs() + weight * reach * 2.0 ** -11).all()


def test_other_devices_streams_and_types_are_refused():
    pages, _ = empty_cache(2, 1, 16, 64, 16)
    cache = paged.Cache(pages)
    call = make_batch(*R.tables([(1, 3)], 16, 0, 1)[:3], [(1, 3)])
    q = torch.zeros(1, 2, 64, dtype=BF, device="cuda")
    for change, word in ((dict(q=q.float()), "bfloat16"), (dict(q=q.cpu()), "lie on"), (dict(q=q[..., ::2]), "dense"), (dict(q=q[:, :, :32]), "head_dim"),
                         (dict(slopes=torch.zeros(3, device="cuda")), "per head"), (dict(prefix=torch.zeros(1, device="cuda")), "int32"),
                         (dict(gate=q[:, :1]), "shape"), (dict(out=q.float()), "bfloat16"), (dict(workspace=q), "uint8"),
                         (dict(status=torch.zeros(1, device="cuda")), "int32")):
        arguments = dict(dict(q=q), **change)
        with pytest.raises(L.LlmcpError, match=word):
            paged.attention(cache, call, arguments.pop("q"), **arguments)
    with pytest.raises(L.LlmcpError, match="uint8"):
        paged.Cache(pages, torch.zeros(2, 2, 1, 16, 2, dtype=torch.float16, device="cuda"))
    with pytest.raises(L.LlmcpError, match="page sizes"):
        paged.Cache(torch.zeros(2, 2, 1, 24, 64, dtype=BF, device="cuda"))


def test_a_call_on_another_stream_follows_that_stream():
    batch = [(1, 3000)]
    q_start, kv_len, table, count = R.tables(batch, 64, 0, 4)
    pages, scales, _ = filled_cache(2, batch, table, count, 2, 64, 128, 16)
    cache, call = paged.Cache(pages), make_batch(q_start, kv_len, table, batch)
    q = torch.randn(1, 8, 128, generator=torch.Generator().manual_seed(6)).to(BF).cuda()
    first = paged.attention(cache, call, q)
    torch.cuda.synchronize()
    side, late = torch.cuda.Stream(), torch.zeros_like(q)
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)
        late.copy_(q)  # comes after the sleep; a call on the default stream would read zeros
        second = paged.attention(cache, call, late)
    side.synchronize()
    assert torch.equal(first, second)


def test_append_in_place_and_rows_past_the_range_of_f32():
    """q_out may be q; rows whose squares leave f32's range, zeros without eps, infinities and NaN are as the definition has them."""
    heads, dim, rot = 3, 128, 128
    g = torch.Generator().manual_seed(8)
    size = torch.tensor([1.0, 1e-30, 1e-38, 1e25, 2e37, 0.0, 1.0, 1.0])
    batch = [(8, 20)]
    q_start, kv_len, table, count = R.tables(batch, 16, 0, 1)
    for eps in (1e-6, 0.0):
        x = (torch.randn(8, heads, dim, generator=g) * size[:, None, None]).to(BF)
        x[6, :, 5], x[7, :, 70] = math.inf, math.nan
        weight = (0.2 * torch.randn(dim, generator=g)).to(BF)
        angle = torch.rand(20, rot // 2, generator=g) * 6
        cos, sin = (torch.cat((f(angle), f(angle)), 1).contiguous() for f in (torch.cos, torch.sin))
        want = R.bf16_round(R.rotate(x, weight, cos[12:], sin[12:], eps))
        pages, _ = empty_cache(count, heads, 16, dim, 16)
        cache, call, q = paged.Cache(pages), make_batch(q_start, kv_len, table, batch), x.cuda()
        got = paged.append(cache, call, q, *cuda(x, x, cos, sin), q_norm=weight.cuda(), k_norm=weight.cuda(), eps=eps, q_out=q)
        assert got is q
        k, v = paged.read(cache, call, 8)
        assert torch.equal(v.cpu().view(torch.int16), x.view(torch.int16))
        for y in (q, k):
            assert torch.equal(y.cpu().isnan(), want.isnan())
            assert torch.equal(y.cpu().double().nan_to_num(), want.nan_to_num())


@pytest.mark.parametrize("rows", [1, 3, 60])
@pytest.mark.parametrize("heads,groups,dim,bits", [(8, 2, 256, 16), (4, 2, 64, 4), (6, 2, 128, 4), (1, 1, 128, 16)])
def test_attention_of_queries_with_strides(rows, heads, groups, dim, bits):
    """Queries and gates as the projection leaves them, and with tokens next to each other, give what dense ones give."""
    batch = [(rows, 200), (rows, 61)]
    q_start, kv_len, table, count = R.tables(batch, 32, 1, 2)
    pages, scales, _ = filled_cache(3, batch, table, count, groups, 32, dim, bits)
    cache, call = paged.Cache(pages, scales), make_batch(q_start, kv_len, table, batch)
    qg = torch.randn(2 * rows, heads, 2, dim, generator=torch.Generator().manual_seed(1)).to(BF).cuda()
    dense = paged.attention(cache, call, qg[:, :, 0].contiguous(), gate=qg[:, :, 1].contiguous())
    assert torch.equal(paged.attention(cache, call, qg[:, :, 0], gate=qg[:, :, 1]), dense)
    turned = qg.permute(2, 1, 0, 3).contiguous()  # [2, heads, tokens, dim]
    assert torch.equal(paged.attention(cache, call, turned[0].transpose(0, 1), gate=turned[1].transpose(0, 1)), dense)
    assert torch.equal(paged.attention(cache, call, turned[0].transpose(0, 1), gate=qg[:, :, 1]), dense)


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("heads,groups,dim", [(128, 1, 64), (128, 1, 256), (256, 2, 128), (96, 2, 64), (33, 1, 256), (17, 1, 128)])
def test_attention_many_heads_on_one_key(heads, groups, dim, bits):
    check_attention([(1, 150), (3, 40)], heads, groups, dim, bits, 32, gate=True)


def test_workspaces_that_are_refused():
    batch = [(1, 5000)]
    q_start, kv_len, table, count = R.tables(batch, 64, 0, 1)
    pages, scales, _ = filled_cache(1, batch, table, count, 2, 64, 64, 16)
    cache, call = paged.Cache(pages, scales), make_batch(q_start, kv_len, table, batch)
    q = torch.randn(1, 4, 64, generator=torch.Generator().manual_seed(1)).to(BF).cuda()
    size = paged.workspace_bytes(cache, call, 1, 4)
    assert size > 16  # one row over many keys is split
    whole = torch.empty(size + 16, dtype=torch.uint8, device="cuda")
    for bad in (whole[:size - 1], whole[8:], whole[:0]):
        with pytest.raises(L.LlmcpError, match="workspace"):
            paged.attention(cache, call, q, workspace=bad)
    assert torch.equal(paged.attention(cache, call, q, workspace=whole[:size]), paged.attention(cache, call, q))


@pytest.mark.parametrize("dim,bits", [(64, 16), (128, 4), (256, 16), (256, 4)])
def test_prompts_in_captured_graphs(dim, bits):
    """The pieces of prompts of changing lengths through one captured append and attention, twice at the same time on two
    streams with workspaces of their own."""
    heads, groups, size, most = 4, 2, 32, 400
    g = torch.Generator().manual_seed(4)
    _, _, table, count = R.tables([(1, most)] * 3, size, 0, 8)
    start, lengths = torch.zeros(4, dtype=torch.int32, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda")
    tokens, states = 160, []
    for _ in range(2):
        pages, scales = empty_cache(count, groups, size, dim, bits)
        x = [torch.zeros(tokens, h, dim, dtype=BF, device="cuda") for h in (heads, groups, groups)]
        cache, call = paged.Cache(pages, scales), paged.Batch(start, lengths, cuda(table), 150, most)
        ws = torch.full((paged.workspace_bytes(cache, call, tokens, heads) + 16,), 0xFF, dtype=torch.uint8, device="cuda")
        out, status = torch.full((tokens, heads, dim), 7.0, dtype=BF, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
        paged.attention(cache, call, paged.append(cache, call, *x, status=status), out=out, workspace=ws, status=status)  # loads the kernels
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            paged.attention(cache, call, paged.append(cache, call, *x, status=status), out=out, workspace=ws, status=status)
        states.append((graph, x, out, cache, call, ws, status))
    values, held, side = torch.zeros(count, 2, groups, size, dim), [0, 0, 0], torch.cuda.Stream()
    for news in ((100, 1, 40), (1, 150, 0), (3, 2, 77), (0, 0, 0), (150, 5, 5)):
        held = [t + n for t, n in zip(held, news)]
        starts = [0, *torch.tensor(news).cumsum(0).tolist()]
        start.copy_(torch.tensor(starts, dtype=torch.int32))
        lengths.copy_(torch.tensor(held, dtype=torch.int32))
        fresh = [torch.randn(tokens, h, dim, generator=g).to(BF) for h in (heads, groups, groups)]
        for _, x, out, *_ in states:
            out.fill_(7.0)
            for a, b in zip(x, fresh):
                a.copy_(b)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            states[1][0].replay()
        states[0][0].replay()
        torch.cuda.synchronize()
        for b, (n, t) in enumerate(zip(news, held)):
            j = torch.arange(t - n, t)
            for which in (0, 1):
                rows = fresh[1 + which][starts[b]:starts[b + 1]].double()
                if bits == 4:
                    codes, d = R.quantise(rows)
                    rows = (codes.unflatten(-1, (-1, 32)) * d.double()[..., None]).flatten(-2)
                values[table[b, j // size].long(), which, :, j % size] = rows.float()
        used = starts[-1]
        want, weight, reach = R.attention(fresh[0][:used], values, starts, held, table, dim ** -0.5)
        for _, _, out, *_, status in states:
            assert int(status) == 0
            assert ((out[:used].cpu().double() - want).abs() <= R.attention_bound(want, weight, reach, bits)).all()
            assert (out[used:] == 7.0).all()


@pytest.mark.parametrize("rows,bits", [(1, 4), (200, 4), (200, 16)])
def test_two_calls_at_once(rows, bits):
    """Calls on two streams whose workspaces come from torch's allocator do not touch each other's."""
    batch = [(rows, 3000), (rows, 1234)]
    q_start, kv_len, table, count = R.tables(batch, 64, 0, 1)
    pages, scales, _ = filled_cache(1, batch, table, count, 2, 64, 128, bits)
    cache, call = paged.Cache(pages, scales), make_batch(q_start, kv_len, table, batch)
    queries = [torch.randn(2 * rows, 8, 128, generator=torch.Generator().manual_seed(s)).to(BF).cuda() for s in range(2)]
    want = [paged.attention(cache, call, q) for q in queries]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], [[], []]
    for _ in range(10):
        for q, stream, results in zip(queries, streams, got):
            with torch.cuda.stream(stream):
                results.append(paged.attention(cache, call, q))
    torch.cuda.synchronize()
    for w, results in zip(want, got):
        assert all(torch.equal(w, r) for r in results)


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("batch", [[(1, 1)], [(1, 300), (2, 40)], [(70, 300), (5, 40)]])
def test_bounds_far_above_the_lengths(batch, bits):
    """max_q and max_kv of 2^30 lay out no more than rows and pages allow, and the results are as ever."""
    q_start, kv_len, table, count = R.tables(batch, 32, 0, 2)
    pages, scales, values = filled_cache(3, batch, table, count, 2, 32, 128, bits)
    tokens = int(q_start[-1])
    q = torch.randn(tokens, 256, 128, generator=torch.Generator().manual_seed(1)).to(BF)
    cache, call = paged.Cache(pages, scales), make_batch(q_start, kv_len, table, batch, max_q=1 << 30, max_kv=1 << 30)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    for heads in (8, 256):
        assert paged.workspace_bytes(cache, call, tokens, heads) < 1 << 28
        got = paged.attention(cache, call, q[:, :heads].cuda(), status=status).cpu().double()
        want, weight, reach = R.attention(q[:, :heads], values, q_start, kv_len, table, 128 ** -0.5)
        assert int(status) == 0
        assert ((got - want).abs() <= R.attention_bound(want, weight, reach, bits)).all()
    k, v = paged.read(cache, call, tokens)
    again = paged.read(cache, make_batch(q_start, kv_len, table, batch), tokens)
    assert torch.equal(k, again[0]) and torch.equal(v, again[1])
