"""The paged key/value cache at the ends of its ranges: sizes of values, gates and caps, positions past 2^24, rows without keys.
Compared with plain 64-bit arithmetic (tests/paged_reference.py), as tests/test_gpu_paged.py is."""
import math

import pytest
import torch

import paged_reference as R
from llmcp_b200 import paged
from test_gpu_paged import BF, cuda, empty_cache, filled_cache, make_batch

pytestmark = pytest.mark.gpu


def pack(values):
    """float64 [pages, 2, heads, size, dim] -> 4-bit (pages, scales, the values that they stand for) on the CPU."""
    codes, d = R.quantise(R.bf16_round(values))
    code8 = (codes + 8).to(torch.uint8)
    return code8[..., 0::2] | code8[..., 1::2] << 4, d, (codes.unflatten(-1, (-1, 32)) * d.double()[..., None]).flatten(-2)


def within(got, want, bound):
    off = (got.cpu().double() - want).abs() / bound
    assert not off.isnan().any() and off.max() <= 1, f"{off.max():.3f} of the bound"


# ---- 4-bit values of any size --------------------------------------------------------------------------------------------

STEPS, PROMPTS = [(1, 300), (2, 70), (1, 6000)], [(150, 333), (40, 41), (20, 4000)]
SHAPES_4BIT = [(4, 2, 64), (6, 2, 128), (4, 1, 256)]


@pytest.mark.parametrize("size", [1e-2, 1e-3, 1e-4, 1e-5, 2e-6, 1e5])
@pytest.mark.parametrize("batch", [STEPS, PROMPTS], ids=["steps", "prompts"])
@pytest.mark.parametrize("heads,groups,dim", SHAPES_4BIT)
def test_attention_over_4_bit_values_of_any_size(heads, groups, dim, batch, size):
    """From scales that are f16's last bits to values past f16's end; queries as much larger keep the scores' size."""
    g = torch.Generator().manual_seed(dim)
    q_start, kv_len, table, count = R.tables(batch, 64, 1, 5)
    pages, scales, values = filled_cache(7, batch, table, count, groups, 64, dim, 4, scale=size)
    q = (torch.randn(int(q_start[-1]), heads, dim, generator=g) / size).to(BF)
    got = paged.attention(paged.Cache(pages, scales), make_batch(q_start, kv_len, table, batch), q.cuda())
    want, weight, extent = R.attention(q, values, q_start, kv_len, table, dim ** -0.5)
    within(got, want, R.attention_bound(want, weight, extent, 4))


@pytest.mark.parametrize("largest", [3.0, 3e5])
@pytest.mark.parametrize("batch", [STEPS, PROMPTS], ids=["steps", "prompts"])
@pytest.mark.parametrize("heads,groups,dim", SHAPES_4BIT)
def test_attention_over_4_bit_blocks_of_mixed_sizes(heads, groups, dim, batch, largest):
    """Blocks between 1e-6 and `largest` side by side; only one sequence, one head, keys or values has the largest ones."""
    g = torch.Generator().manual_seed(dim + 1)
    q_start, kv_len, table, count = R.tables(batch, 64, 1, 5)
    blocks = 10.0 ** (-6 + 6.4 * torch.rand(count, 2, groups, 64, dim // 32, 1, generator=g, dtype=torch.float64))
    raw = (blocks * torch.rand(count, 2, groups, 64, dim // 32, 32, generator=g, dtype=torch.float64).sub(0.5)).flatten(-2)
    raw[table[0, 2].long(), 1, groups - 1, 5] *= largest / raw[table[0, 2].long(), 1, groups - 1, 5].abs().max()
    raw[table[1, 0].long(), 0, 0, 9] *= largest / raw[table[1, 0].long(), 0, 0, 9].abs().max()
    pages, scales, values = pack(raw)
    q = torch.randn(int(q_start[-1]), heads, dim, generator=g).to(BF)
    scale = dim ** -0.5 / largest
    got = paged.attention(paged.Cache(*cuda(pages, scales)), make_batch(q_start, kv_len, table, batch), q.cuda(), scale=scale)
    want, weight, extent = R.attention(q, values, q_start, kv_len, table, scale)
    within(got, want, R.attention_bound(want, weight, extent, 4))


# ---- light weights over small 4-bit values ---------------------------------------------------------------------------------


@pytest.mark.parametrize("size", [1e4, 1.0, 1e-1, 1e-2, 1e-3, 1e-4, 1e-5, 2e-6])
@pytest.mark.parametrize("batch", [[(1, 40), (3, 9), (2, 2)], [(1, 700), (2, 6000)], [(40, 90), (70, 333)]], ids=str)
@pytest.mark.parametrize("heads,groups,dim", SHAPES_4BIT)
def test_light_weights_over_4_bit_values_of_any_size(heads, groups, dim, batch, size):
    """Scores that one key dominates: where its value is 0, what is left comes from light weights.

    Few rows: a weight p (the row's largest at least 2^7) and its product with the value's scale d, times 2^j, are rounded to
    f16, which below 2^-14 is off by up to 2^-25.  Codes are at most 7 and the weights' sum at least 2^7, so a key moves the
    result by up to 7 (2^-25 d + 2^-25 2^-j) / 2^7 = 7 2^-32 (d + 2^-j).  j brings the largest d to [1/2, 1) but is at most 14 and
    not negative: 2^-j <= max(2^-14, min(1, 2 d)).  For d of 1 and more the weights are kept lower instead, by less than 2 d."""
    g = torch.Generator().manual_seed(dim + 7)
    q_start, kv_len, table, count = R.tables(batch, 64, 1, 5)
    pages, scales, values = filled_cache(7, batch, table, count, groups, 64, dim, 4, scale=size)
    q = (10 / size * torch.randn(int(q_start[-1]), heads, dim, generator=g)).to(BF)
    got = paged.attention(paged.Cache(pages, scales), make_batch(q_start, kv_len, table, batch), q.cuda())
    want, weight, extent = R.attention(q, values, q_start, kv_len, table, dim ** -0.5)
    d, keys = float(scales.nan_to_num().max()), torch.cat([torch.arange(t - n, t) + 1 for n, t in batch])[:, None, None]
    light = keys * 7 * 2.0 ** -32 * max(1.0, 2 * d) * (d + max(2.0 ** -14, min(1.0, 2 * d)))
    within(got, want, R.attention_bound(want, weight, extent, 4) + light)


# ---- rows without keys ---------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("rows", [1, 40])
@pytest.mark.parametrize("width,most", [(0, 0), (0, 100), (4, 0)])
def test_rows_of_sequences_without_keys_are_zeros(width, most, rows, dim, bits):
    pages, scales = empty_cache(2, 2, 16, dim, bits)
    starts, lengths = torch.tensor([0, rows, 2 * rows], dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    call = paged.Batch(*cuda(starts, lengths, torch.zeros(2, width, dtype=torch.int32)), rows, most)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    q = torch.randn(2 * rows + 1, 4, dim, device="cuda").to(BF)
    for gate in (None, q):
        out = torch.full_like(q, 7.0)
        paged.attention(paged.Cache(pages, scales), call, q, gate=gate, out=out, status=status)
        assert int(status) == 0
        assert (out[:2 * rows] == 0).all() and (out[2 * rows:] == 7.0).all()


# ---- positions that f32 does not hold --------------------------------------------------------------------------------------


@pytest.mark.parametrize("rows,heads,dim,bits", [(1, 2, 64, 4), (3, 2, 64, 16), (1, 2, 256, 16), (20, 2, 64, 16), (20, 2, 256, 16)])
def test_bias_by_distance_past_2_to_the_24_keys(rows, heads, dim, bits):
    """The bias leaves nothing of keys some thousands away, so that the last ones are the whole answer."""
    size, count, near = 256, 40, 4096
    total = (1 << 24) + 2817
    g = torch.Generator().manual_seed(dim + rows)
    table = torch.randint(0, count, (1, -(-total // size)), generator=g, dtype=torch.int32)  # pages may be a sequence's more than once
    pages, scales, values = filled_cache(3, [(0, count * size)], torch.arange(count, dtype=torch.int32)[None], count, 1, size, dim, bits)
    q = torch.randn(rows, heads, dim, generator=g).to(BF)
    slopes = torch.tensor([0.25, 1.0])
    starts = torch.tensor([0, rows], dtype=torch.int32)
    call = paged.Batch(*cuda(starts, torch.tensor([total], dtype=torch.int32), table), rows, total)
    got = paged.attention(paged.Cache(pages, scales), call, q.cuda(), slopes=slopes.cuda())
    first = total // size * size - near
    want, weight, (reach, span) = R.attention(q, values, [0, rows], [total - first], table[:, first // size:], dim ** -0.5, slopes=slopes)
    within(got, want, R.attention_bound(want, weight, (reach, span), bits))


# ---- caps -----------------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("cap", [1e-39, 1e-30, 3.0, 1e4, 1e6, 1e30])
@pytest.mark.parametrize("batch", [[(1, 300), (2, 70)], [(150, 333), (40, 41)]], ids=["steps", "prompts"])
@pytest.mark.parametrize("heads,groups,dim,bits", [(4, 2, 64, 16), (6, 2, 128, 4), (4, 1, 256, 16), (4, 1, 256, 4)])
@pytest.mark.parametrize("spread", [1.0, 8.0])
def test_caps_of_any_size(heads, groups, dim, bits, batch, cap, spread):
    """tanh keeps the scores' relative precision: 2^-20 (exp and reciprocal 2^-21.5 each of a tanh of 0.46 at least, the
    polynomial below that 2^-21), so a cap far above them changes nothing."""
    g = torch.Generator().manual_seed(dim + 3)
    q_start, kv_len, table, count = R.tables(batch, 64, 1, 5)
    pages, scales, values = filled_cache(7, batch, table, count, groups, 64, dim, bits)
    q = (spread * torch.randn(int(q_start[-1]), heads, dim, generator=g)).to(BF)
    q[0] = 0  # scores of 0, beside a cap whose reciprocal is past f32's end
    got = paged.attention(paged.Cache(pages, scales), make_batch(q_start, kv_len, table, batch), q.cuda(), softcap=cap)
    want, weight, extent = R.attention(q, values, q_start, kv_len, table, dim ** -0.5, softcap=float(torch.tensor(cap)))
    bound = R.attention_bound(want, weight, extent, bits) + weight * 2 * extent[0] * 2.0 ** -20
    within(got, want, bound)


# ---- gates ----------------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("batch", [[(1, 40), (1, 3)], [(1, 20011)], [(2, 3000)] * 20, [(150, 333), (40, 41)], [(20, 6000)]], ids=str)
@pytest.mark.parametrize("heads,groups,dim,bits", [(8, 2, 64, 16), (8, 2, 128, 4), (8, 2, 256, 16)])
def test_gates_that_close(heads, groups, dim, bits, batch):
    """Sigmoids of gates down to -87 keep their relative precision, from f32's normal range on (2^-126) nothing is left,
    -infinity closes, infinity opens, NaN stays."""
    g = torch.Generator().manual_seed(dim + 4)
    q_start, kv_len, table, count = R.tables(batch, 64, 1, 5)
    pages, scales, values = filled_cache(7, batch, table, count, groups, 64, dim, bits)
    tokens = int(q_start[-1])
    q = torch.randn(tokens, heads, dim, generator=g).to(BF)
    choices = torch.tensor([-math.inf, math.inf, math.nan, -60.0, -79.5, -80.5, -83.0, -86.5, -95.0, -3e38, 3e38, 0.0])
    gate = choices[torch.randint(0, len(choices), (tokens, heads, dim), generator=g)].to(BF)
    got = paged.attention(paged.Cache(pages, scales), make_batch(q_start, kv_len, table, batch), q.cuda(), gate=gate.cuda()).cpu().double()
    want, weight, extent = R.attention(q, values, q_start, kv_len, table, dim ** -0.5)
    s = torch.sigmoid(gate.double())
    assert torch.equal(got.isnan(), gate.isnan())
    assert (got[gate == -math.inf] == 0).all()
    bound = (R.attention_bound(want, weight, extent, bits) - 1e-30) * s + weight * (2.0 ** -126 + s * 2.0 ** -17)
    near = (got - want * s).abs() <= bound  # both 0 behind a closed gate where a row's only value is 0
    assert near[~gate.isnan() & (gate != -math.inf)].all()


# ---- gates beside large values -------------------------------------------------------------------------------------------


@pytest.mark.parametrize("batch", [[(1, 40), (1, 3)], [(1, 20011)], [(2, 3000)] * 20, [(150, 333), (40, 41)], [(20, 6000)]], ids=str)
@pytest.mark.parametrize("heads,groups,dim", [(8, 2, 64), (8, 2, 128), (8, 2, 256)])
def test_gates_that_nearly_close_large_values(heads, groups, dim, batch):
    """A sigmoid below f32's range times a value of 1e20 is an ordinary number.  Its exponent, gate log2 e, is rounded to f32: at
    130 off by 2^-17 and 130 2^-24 (the constant), times ln 2, and the two halves' powers by 2^-22 each: below 2^-16."""
    g = torch.Generator().manual_seed(dim + 8)
    q_start, kv_len, table, count = R.tables(batch, 64, 1, 5)
    pages, scales, values = filled_cache(7, batch, table, count, groups, 64, dim, 16, scale=1e20)
    tokens = int(q_start[-1])
    q = (torch.randn(tokens, heads, dim, generator=g) * 1e-20).to(BF)
    choices = torch.tensor([-60.0, -79.5, -86.5, -88.0, -95.0, -110.0, -130.0, -180.0, -math.inf, 3.0])
    gate = choices[torch.randint(0, len(choices), (tokens, heads, dim), generator=g)].to(BF)
    got = paged.attention(paged.Cache(pages), make_batch(q_start, kv_len, table, batch), q.cuda(), gate=gate.cuda()).cpu().double()
    want, weight, extent = R.attention(q, values, q_start, kv_len, table, dim ** -0.5)
    s = torch.sigmoid(gate.double())
    bound = R.attention_bound(want, weight, extent, 16) * s + weight * s * 2.0 ** -16 + 2.0 ** -133  # the last: steps of a subnormal result
    assert ((got - want * s).abs() <= bound).all()
    assert (got[gate == -math.inf] == 0).all()


# ---- queries -----------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("batch", [[(1, 300), (2, 70)], [(150, 333), (40, 41)]], ids=["steps", "prompts"])
@pytest.mark.parametrize("heads,groups,dim", SHAPES_4BIT)
def test_queries_next_to_the_end_of_their_type(heads, groups, dim, batch):
    g = torch.Generator().manual_seed(dim + 5)
    q_start, kv_len, table, count = R.tables(batch, 64, 1, 5)
    pages, scales, values = filled_cache(7, batch, table, count, groups, 64, dim, 4, scale=1e-3)
    q = (torch.rand(int(q_start[-1]), heads, dim, generator=g, dtype=torch.float64).sub(0.5) * 2.0 ** 122).to(BF)
    scale = 2.0 ** -112
    got = paged.attention(paged.Cache(pages, scales), make_batch(q_start, kv_len, table, batch), q.cuda(), scale=scale)
    want, weight, extent = R.attention(q, values, q_start, kv_len, table, scale)
    within(got, want, R.attention_bound(want, weight, extent, 4))


# ---- scales ------------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("batch", [STEPS, PROMPTS], ids=["steps", "prompts"])
@pytest.mark.parametrize("heads,groups,dim", SHAPES_4BIT)
def test_scales_below_zero(heads, groups, dim, batch):
    """append writes none, but a cache may come from elsewhere: they multiply codes like any other."""
    g = torch.Generator().manual_seed(dim + 6)
    q_start, kv_len, table, count = R.tables(batch, 64, 1, 5)
    pages, scales, _ = filled_cache(7, batch, table, count, groups, 64, dim, 4)
    sign = torch.where(torch.rand(scales.shape, generator=g) < 0.5, -1.0, 1.0)
    scales *= sign.half().cuda()
    values = R.unpack(pages.cpu(), scales.cpu()).nan_to_num()
    q = torch.randn(int(q_start[-1]), heads, dim, generator=g).to(BF)
    got = paged.attention(paged.Cache(pages, scales), make_batch(q_start, kv_len, table, batch), q.cuda())
    want, weight, extent = R.attention(q, values, q_start, kv_len, table, dim ** -0.5)
    within(got, want, R.attention_bound(want, weight, extent, 4))


# ---- bounds ------------------------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("bits", [16, 4])
def test_a_bound_above_the_calls_rows_changes_nothing(bits):
    """No sequence has more rows than the call: max_q past them takes no other kernel and no more memory."""
    batch = [(1, 3000), (1, 50)]
    q_start, kv_len, table, count = R.tables(batch, 64, 1, 5)
    pages, scales, _ = filled_cache(7, batch, table, count, 2, 64, 128, bits)
    cache, q = paged.Cache(pages, scales), torch.randn(2, 8, 128, device="cuda").to(BF)
    tight, wide = (make_batch(q_start, kv_len, table, batch, max_q=most) for most in (2, 1 << 30))
    assert paged.workspace_bytes(cache, wide, 2, 8) == paged.workspace_bytes(cache, tight, 2, 8)
    assert torch.equal(paged.attention(cache, wide, q), paged.attention(cache, tight, q))


# ---- refused rows ----------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("rows", [1, 40])
@pytest.mark.parametrize("dim,bits", [(64, 16), (64, 4), (256, 16), (256, 4)])
def test_refused_sequences_leave_their_rows_and_no_others(rows, dim, bits):
    batch = [(rows, 100), (rows, 90)]
    q_start, kv_len, table, count = R.tables(batch, 32, 1, 2)
    pages, scales, values = filled_cache(3, batch, table, count, 2, 32, dim, bits)
    q = torch.randn(2 * rows, 4, dim, generator=torch.Generator().manual_seed(1)).to(BF)
    want, weight, extent = R.attention(q, values, q_start, kv_len, table, dim ** -0.5)
    bound = R.attention_bound(want, weight, extent, bits)
    cache = paged.Cache(pages, scales)
    for change, valid in ((dict(max_kv=95), [1]), (dict(lengths=[100, 129]), [0]), (dict(lengths=[-5, 90]), [1]), (dict(starts=[0, -1, 2 * rows]), []),
                          (dict(starts=[0, rows, 5000]), [0]), (dict(starts=[0, 5000, 2 * rows]), [])):
        change = dict(change)
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        lengths, starts = change.pop("lengths", [100, 90]), change.pop("starts", q_start.tolist())
        call = make_batch(torch.tensor(starts, dtype=torch.int32), torch.tensor(lengths, dtype=torch.int32), table, batch, **dict(dict(max_kv=2000), **change))
        out = torch.full((2 * rows, 4, dim), 7.0, dtype=BF, device="cuda")
        paged.attention(cache, call, q.cuda(), out=out, status=status)
        assert int(status) == 4
        for b in range(2):
            part = slice(b * rows, (b + 1) * rows)
            if b in valid:
                within(out[part], want[part], bound[part])
            else:
                assert (out[part] == 7.0).all()


@pytest.mark.parametrize("bits,dtype", [(16, torch.float32), (16, BF), (4, torch.float32), (4, BF)])
def test_read_leaves_refused_rows(bits, dtype):
    """Through the C entry, into buffers that show what was written."""
    batch = [(3, 20), (2, 40), (1, 5), (4, 4)]
    q_start, kv_len, table, count = R.tables(batch, 16, 1, 2)
    pages, scales, values = filled_cache(3, batch, table, count, 2, 16, 64, bits)
    broken = table.clone()
    broken[0, 1] = count  # the page of the first sequence's last rows
    cache, call = paged.Cache(pages, scales), make_batch(q_start, kv_len, broken, batch, max_kv=39)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = torch.full((2, 12, 2, 64), 7.0, dtype=dtype, device="cuda")
    assert paged._library().llmcp_dev_paged_read(cache._c, call._c(cache, 12), out[0].data_ptr(), out[1].data_ptr(), 0 if dtype is torch.float32 else 1,
                                                 status.data_ptr(), None) == 0
    torch.cuda.synchronize()
    assert int(status) == 4
    assert (out[:, :5] == 7.0).all() and (out[:, 10:] == 7.0).all()
    for which in (0, 1):
        rows = torch.cat([R.sequence_rows(values, table, b, which, t)[t - n:] for b, (n, t) in list(enumerate(batch))[2:]]).double()
        assert torch.equal(out[which, 5:10].cpu().double(), rows if dtype is torch.float32 else R.bf16_round(rows))


# ---- results in place ------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("batch", [[(1, 40), (1, 3)], [(1, 20011), (2, 60)], [(2, 3000)] * 20, [(150, 333), (40, 41)], [(20, 6000)]], ids=str)
@pytest.mark.parametrize("heads,groups,dim,bits", [(8, 2, 64, 16), (10, 2, 128, 4), (8, 2, 256, 16), (8, 2, 256, 4)])
def test_results_in_place_of_queries_or_gates(heads, groups, dim, bits, batch):
    q_start, kv_len, table, count = R.tables(batch, 64, 1, 5)
    pages, scales, _ = filled_cache(7, batch, table, count, groups, 64, dim, bits)
    cache, call, tokens = paged.Cache(pages, scales), make_batch(q_start, kv_len, table, batch), int(q_start[-1])
    q, gate = torch.randn(2, tokens, heads, dim, device="cuda", generator=torch.Generator("cuda").manual_seed(1)).to(BF)
    want = paged.attention(cache, call, q, gate=gate)
    over_q, over_gate = q.clone(), gate.clone()
    assert paged.attention(cache, call, over_q, gate=gate, out=over_q) is over_q and torch.equal(over_q, want)
    assert paged.attention(cache, call, q, gate=over_gate, out=over_gate) is over_gate and torch.equal(over_gate, want)


# ---- append ---------------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("heads,dim,rot", [(16, 128, 128), (8, 64, 4), (8, 256, 64)])
def test_append_rounds_products_below_f32s_range_once(heads, dim, rot, norm):
    """Values whose f32 products are subnormal (all of a row's without norm, every other one's beside ordinary ones with it)
    come out as the correctly rounded value like any other."""
    g = torch.Generator().manual_seed(dim)
    tokens = 3000
    x = torch.randn(tokens, heads, dim, generator=g, dtype=torch.float64)
    tiny = 2.0 ** -(119 + 14 * torch.rand(tokens, heads, dim, generator=g, dtype=torch.float64))
    x = (torch.where(torch.arange(dim) % 2 == 0, x, x * tiny) if norm else x * tiny).to(BF)
    weight = (0.2 * torch.randn(dim, generator=g)).to(BF) if norm else None
    angle = torch.rand(tokens, rot // 2, generator=g) * 6
    if norm:  # partners are both ordinary or both tiny; a rotation by next to nothing keeps them apart from each other
        angle = angle * 0 + 1e-3
    cos, sin = (torch.cat((f(angle), f(angle)), 1).contiguous() for f in (torch.cos, torch.sin))
    want = R.bf16_round(R.rotate(x, weight, cos, sin)).to(BF)
    pages, _ = empty_cache(-(-tokens // 256), heads, 256, dim, 16)
    table = torch.arange(pages.shape[0], dtype=torch.int32)[None]
    call = make_batch(torch.tensor([0, tokens], dtype=torch.int32), torch.tensor([tokens], dtype=torch.int32), table, [(tokens, tokens)])
    cache = paged.Cache(pages)
    got = paged.append(cache, call, *cuda(x, x, x, cos, sin), q_norm=cuda(weight), k_norm=cuda(weight))
    k, _ = paged.read(cache, call, tokens)
    for y in (got, k):
        assert torch.equal(y.cpu().double(), want.double())


# ---- ties -----------------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dim,equal", [(64, 1), (64, 4), (128, 2), (128, 32), (256, 1), (256, 64)])
def test_append_rounds_exact_middles_to_even(dim, equal):
    """Rows of a few values of one size, whose norm is a power of two times it, with weights that put the result exactly half way
    between two bf16 values."""
    g = torch.Generator().manual_seed(dim + equal)
    tokens, heads = 64, 5
    order = torch.rand(tokens, heads, dim, generator=g).argsort(-1)
    size = 2.0 ** torch.randint(-8, 9, (tokens, heads, 1), generator=g) * (1 + torch.randint(0, 128, (tokens, heads, 1), generator=g) / 128)
    sign = torch.randint(0, 2, (tokens, heads, dim), generator=g) * 2 - 1
    x = torch.where(order < equal, sign * size, 0.0).to(BF)
    weight = ((2 * torch.randint(0, 128, (dim,), generator=g) + 1) / 256).to(BF)  # 1 + weight: nine bits, the last one set
    pages, _ = empty_cache(1, heads, 64, dim, 16)
    call = make_batch(torch.tensor([0, tokens], dtype=torch.int32), torch.tensor([tokens], dtype=torch.int32), torch.zeros(1, 1, dtype=torch.int32), [(tokens, tokens)])
    cache = paged.Cache(pages)
    got = paged.append(cache, call, *cuda(x, x, x), q_norm=weight.cuda(), k_norm=weight.cuda(), eps=0.0)
    want = R.bf16_round(torch.where(x != 0, sign * (dim / equal) ** 0.5 * (1 + weight.double()), 0.0))
    k, _ = paged.read(cache, call, tokens)
    for y in (got, k):
        assert torch.equal(y.cpu().double(), want)
