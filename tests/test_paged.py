"""The paged cache without a GPU: refusals of the C entries (made before anything touches a device) and of the Python
module, and the reference's own pieces against each other."""
import ctypes as C

import pytest
import torch

import llmcp_b200 as L
import paged_reference as R
from llmcp_b200 import paged

FAKE = 1 << 20  # an address that no refused call follows


def _kv(**changes):
    return paged._Kv(**dict(dict(pages=FAKE, scales=None, num_pages=8, page_size=16, kv_heads=2, head_dim=64), **changes))


def _batch(**changes):
    return paged._Batch(**dict(dict(q_start=FAKE, kv_len=FAKE, page_table=FAKE, sequences=2, table_width=4, table_stride=4, tokens=3,
                                    max_q=2, max_kv=64), **changes))


def _append(kv, batch, **changes):
    a = dict(q=FAKE, q_row=256, q_head=64, heads=4, k=FAKE, k_row=128, k_head=64, v=FAKE, v_row=128, v_head=64, q_norm=None, k_norm=None,
             eps=1e-6, cos=FAKE, sin=FAKE, cos_rows=64, rot=32, q_out=FAKE, status=None, stream=None)
    a.update(changes)
    return paged._library().llmcp_dev_paged_append(kv, batch, *a.values())


def _read(kv, batch, k=FAKE, v=FAKE, dtype=1):
    return paged._library().llmcp_dev_paged_read(kv, batch, k, v, dtype, None, None)


def _attention(kv, batch, **changes):
    a = dict(q=FAKE, q_row=256, q_head=64, heads=4, scale=0.125, softcap=0.0, slopes=None, prefix=None, gate=None, gate_row=0, gate_head=0,
             out=FAKE, workspace=FAKE, workspace_bytes=1 << 40, status=None, stream=None)
    a.update(changes)
    return paged._library().llmcp_dev_paged_attention(kv, batch, *a.values())


def _refused(code, word):
    assert code == 1 and word in L.last_error(), L.last_error()
    L.lib().llmcp_b200_clear_error()


@pytest.mark.parametrize("change,word", [
    (dict(pages=None), "no pages"), (dict(head_dim=96), "head_dim"), (dict(head_dim=0), "head_dim"), (dict(page_size=24), "page_size"),
    (dict(page_size=8), "page_size"), (dict(page_size=512), "page_size"), (dict(kv_heads=0), "kv_heads"), (dict(num_pages=0), "num_pages"),
    (dict(num_pages=1 << 40), "num_pages"), (dict(num_pages=-1), "num_pages"), (dict(pages=FAKE + 8), "16-byte"), (dict(scales=FAKE + 2), "16-byte")])
def test_caches_that_are_refused(change, word):
    for call in (_append, _read, _attention):
        _refused(call(_kv(**change), _batch()), word)
    assert paged._library().llmcp_dev_paged_attention_workspace(_kv(**change), _batch(), 4) == -1


@pytest.mark.parametrize("change,word", [
    (dict(sequences=-1), "sequences"), (dict(sequences=1 << 20), "sequences"), (dict(tokens=-1), "tokens"), (dict(max_q=-1), "max_q"),
    (dict(max_kv=1 << 31), "max_kv"), (dict(table_width=-1), "page table"), (dict(table_stride=3), "page table"), (dict(q_start=None), "missing"),
    (dict(kv_len=None), "missing"), (dict(page_table=None), "missing")])
def test_batches_that_are_refused(change, word):
    for call in (_append, _read, _attention):
        _refused(call(_kv(), _batch(**change)), word)


@pytest.mark.parametrize("change,word", [
    (dict(heads=-1), "heads"), (dict(rot=66), "rot"), (dict(rot=6), "rot"), (dict(rot=-8), "rot"), (dict(q=None), "q or q_out"),
    (dict(q_out=None), "q or q_out"), (dict(k=None), "k or v"), (dict(v=None), "k or v"), (dict(sin=None), "cos or sin"),
    (dict(cos_rows=-1), "cos_rows"), (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"), (dict(q_out=FAKE + 2), "q_out"), (dict(k=FAKE + 1), "boundary")])
def test_appends_that_are_refused(change, word):
    _refused(_append(_kv(), _batch(), **change), word)


@pytest.mark.parametrize("change,word", [
    (dict(heads=0), "heads"), (dict(heads=3), "heads"), (dict(heads=258), "128"), (dict(scale=float("inf")), "finite"), (dict(softcap=-1.0), "softcap"),
    (dict(softcap=float("nan")), "softcap"), (dict(q=None), "q or out"), (dict(out=None), "q or out"), (dict(q=FAKE + 2), "16-byte"),
    (dict(q_row=12), "16-byte"), (dict(q_head=3), "16-byte"), (dict(gate=FAKE, gate_row=4), "16-byte"), (dict(slopes=FAKE + 2), "slopes")])
def test_attentions_that_are_refused(change, word):
    _refused(_attention(_kv(), _batch(), **change), word)


def test_reads_that_are_refused():
    _refused(_read(_kv(), _batch(), k=None), "k_out")
    _refused(_read(_kv(), _batch(), dtype=2), "out_dtype")


@pytest.mark.parametrize("change", [dict(sequences=0), dict(tokens=0), dict(max_q=0)])
def test_calls_without_rows_do_nothing(change):
    batch = _batch(**change)
    assert _append(_kv(), batch) == 0 and _read(_kv(), batch) == 0 and _attention(_kv(), batch) == 0
    assert paged._library().llmcp_dev_paged_attention_workspace(_kv(), batch, 4) == 0


@pytest.mark.parametrize("pages,scales,word", [
    (torch.zeros(4, 2, 2, 16, 64), None, "CUDA"), (torch.zeros(4, 3, 2, 16, 64), None, "num_pages, 2"), (torch.zeros(4, 2, 16, 64), None, "num_pages, 2")])
def test_python_refuses_pages(pages, scales, word):
    with pytest.raises(L.LlmcpError, match=word):
        paged.Cache(pages, scales)


def test_python_refuses_batches_off_the_gpu():
    with pytest.raises(L.LlmcpError, match="CUDA"):
        paged.Batch(torch.zeros(2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32), torch.zeros(1, 1, dtype=torch.int32), 1, 1)


def test_reference_codes_are_nearest():
    """Every value is within half a scale of its code's value, and the largest of a block keeps its size to f16 rounding."""
    y = R.bf16_round(torch.randn(50, 64, generator=torch.Generator().manual_seed(1), dtype=torch.float64))
    codes, scale = R.quantise(y)
    back = (codes.unflatten(-1, (-1, 32)) * scale.double()[..., None]).flatten(-2)
    half = scale.double().repeat_interleave(32, -1) / 2
    assert ((back - y).abs() <= half * (1 + 2.0 ** -9)).all()
    assert codes.abs().max() == 7


def test_reference_attention_is_a_softmax():
    """Against torch's own double-precision attention on one whole sequence."""
    g = torch.Generator().manual_seed(2)
    q, total, table = torch.randn(5, 4, 64, generator=g), 37, torch.tensor([[2, 0, 1]], dtype=torch.int32)
    values = torch.randn(3, 2, 2, 16, 64, generator=g)
    out, weight, _ = R.attention(q, values, [0, 5], [total], table, 0.125)
    k, v = (R.sequence_rows(values, table, 0, which, total).double().repeat_interleave(2, 1).transpose(0, 1) for which in (0, 1))
    mask = torch.ones(5, total, dtype=torch.bool).tril(total - 5)
    want = torch.nn.functional.scaled_dot_product_attention(q.double().transpose(0, 1), k, v, attn_mask=mask, scale=0.125)
    assert torch.allclose(out, want.transpose(0, 1), rtol=1e-12, atol=1e-12) and (weight >= out.abs() - 1e-12).all()


@pytest.mark.parametrize("change", [dict(q_row=0), dict(q_head=0), dict(q_row=-256), dict(gate=FAKE, gate_row=256, gate_head=0),
                                    dict(gate=FAKE, gate_row=0, gate_head=64)])
def test_rows_of_queries_and_gates_that_overlap_are_refused(change):
    _refused(_attention(_kv(), _batch(), **change), "positive")


def test_prompts_over_4_bits_have_a_limit():
    """Their rows of 16 bits are numbered in 31 bits: refused, for the call and for its workspace, where they are more; few
    rows, and bf16 pages, have no such copy."""
    kv, long = _kv(scales=FAKE), dict(max_kv=1 << 29, table_width=1 << 25, table_stride=1 << 25)
    _refused(_attention(kv, _batch(max_q=9, **long)), "below 2^31")
    assert paged._library().llmcp_dev_paged_attention_workspace(kv, _batch(max_q=9, **long), 4) == -1
    assert "below 2^31" in L.last_error()
    L.lib().llmcp_b200_clear_error()
