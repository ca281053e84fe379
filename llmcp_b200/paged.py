"""A key/value cache in pages that many sequences share, on torch tensors: append, attention, read.

The calls of include/llmcp_b200.h (llmcp_dev_paged_*) with their checks; layouts, formulas and what ``status`` reports
are described there.  Everything is enqueued on the current stream of the tensors' device and nothing is synchronised,
so the calls can be captured into a graph; lengths and page tables may then change between replays.  Rows whose lengths or
pages do not fit (more than ``max_q`` or ``max_kv``, a page that does not exist) are left out, and results are not cleared
before: only ``status`` (one int32, raised and never cleared by the calls) tells, so pass one where that may happen.

    cache = Cache(pages, scales)                # pages bf16, or uint8 with f16 scales (4 bits)
    batch = Batch(q_start, kv_len, page_table, max_q, max_kv)
    q = append(cache, batch, q, k, v, cos, sin, q_norm=..., k_norm=...)
    out = attention(cache, batch, q, gate=...)
"""
import ctypes as C
import functools

import torch

from . import DTYPE_BF16, DTYPE_F32, LlmcpError, last_error, lib

PAGE_SIZES = (16, 32, 64, 128, 256)
HEAD_DIMS = (64, 128, 256)


class _Kv(C.Structure):
    _fields_ = [("pages", C.c_void_p), ("scales", C.c_void_p)] + [
        (n, C.c_int64) for n in ("num_pages", "page_size", "kv_heads", "head_dim")]


class _Batch(C.Structure):
    _fields_ = [(n, C.c_void_p) for n in ("q_start", "kv_len", "page_table")] + [
        (n, C.c_int64) for n in ("sequences", "table_width", "table_stride", "tokens", "max_q", "max_kv")]


_functions = None


def _library():
    global _functions
    if _functions is None:
        handle, p, i, f = lib(), C.c_void_p, C.c_int64, C.c_float
        both = [C.POINTER(_Kv), C.POINTER(_Batch)]
        handle.llmcp_dev_paged_append.argtypes = both + [p, i, i, i, p, i, i, p, i, i, p, p, f, p, p, i, i, p, p, p]
        handle.llmcp_dev_paged_read.argtypes = both + [p, p, C.c_int, p, p]
        handle.llmcp_dev_paged_attention_workspace.argtypes = both + [i]
        handle.llmcp_dev_paged_attention_workspace.restype = i
        handle.llmcp_dev_paged_attention.argtypes = both + [p, i, i, i, f, f, p, p, p, i, i, p, p, i, p, p]
        _functions = handle
    return _functions


def _refuse(what):
    raise LlmcpError("paged cache: " + what)


def _tensor(t, name, dtype, dims, device):
    """The address and strides of ``t``, which has to have that type and rank, lie on that device and be dense in its last
    dimension.  (These checks are most of a small call's time: one look at the strides, messages only where needed.)"""
    strides = t.stride()
    if t.dtype is not dtype or len(strides) != dims or t.get_device() != device.index or (strides[-1] != 1 and t.shape[-1] > 1):
        _refuse(f"{name} has to be {dtype}" if t.dtype is not dtype else
                f"{name} has to have {dims} dimensions" if len(strides) != dims else
                f"{name} has to lie on {device}" if t.get_device() != device.index else
                f"{name} has to be dense in its last dimension")
    return t.data_ptr(), strides


def _optional(t, name, dtype, dims, device):
    return None if t is None else _tensor(t, name, dtype, dims, device)[0]


class Cache:
    """One layer's pages [num_pages, 2, kv_heads, page_size, head_dim]: bf16, or uint8 [..., head_dim / 2] with
    ``scales`` [..., head_dim / 32] float16.  The tensors stay the caller's; nothing is copied."""

    def __init__(self, pages, scales=None):
        shape = pages.shape
        if len(shape) != 5 or shape[1] != 2:
            _refuse("pages has to be [num_pages, 2, kv_heads, page_size, head_dim]")
        if not pages.is_cuda:
            _refuse("pages has to lie on a CUDA device")
        if not pages.is_contiguous():
            _refuse("pages has to be contiguous")
        if pages.dtype is not (torch.bfloat16 if scales is None else torch.uint8):
            _refuse("pages has to be bfloat16, or uint8 where there are scales")
        count, _, heads, size, last = shape
        dim = last if scales is None else 2 * last
        if count < 1 or heads < 1 or size not in PAGE_SIZES or dim not in HEAD_DIMS:
            _refuse(f"page sizes are {PAGE_SIZES}, head dimensions {HEAD_DIMS}")
        self.pages, self.scales, self.device = pages, scales, pages.device
        if scales is not None and (scales.dtype is not torch.float16 or scales.shape != (count, 2, heads, size, dim // 32) or
                                   not scales.is_contiguous() or scales.device != self.device):
            _refuse("scales has to be float16 [num_pages, 2, kv_heads, page_size, head_dim / 32], contiguous, beside pages")
        self.kv_heads, self.page_size, self.head_dim = heads, size, dim
        self._c = _Kv(pages.data_ptr(), None if scales is None else scales.data_ptr(), count, size, heads, dim)


class Batch:
    """Sequence b owns rows q_start[b] to q_start[b + 1] - 1 of a call, the last ones of its kv_len[b] tokens; token j
    lies in page page_table[b, j // page_size].  int32 tensors [sequences + 1], [sequences], [sequences, width];
    ``max_q`` and ``max_kv`` bound rows and lengths of a sequence, and work is laid out for them."""

    def __init__(self, q_start, kv_len, page_table, max_q, max_kv):
        device = q_start.device
        if not q_start.is_cuda:
            _refuse("q_start has to lie on a CUDA device")
        starts, lengths = _tensor(q_start, "q_start", torch.int32, 1, device)[0], _tensor(kv_len, "kv_len", torch.int32, 1, device)[0]
        table, (stride, _) = _tensor(page_table, "page_table", torch.int32, 2, device)
        sequences, width = page_table.shape
        if q_start.shape[0] != sequences + 1 or kv_len.shape[0] != sequences:
            _refuse("q_start has one entry more than kv_len and page_table have rows")
        if sequences > 1 and stride < width:
            _refuse("rows of page_table overlap")
        self.q_start, self.kv_len, self.page_table, self.device, self.sequences = q_start, kv_len, page_table, device, sequences
        self._arguments = (starts, lengths, table, sequences, width, stride)
        self._max = (max_q, max_kv)

    def _c(self, cache, tokens):
        if self.device != cache.device:
            _refuse("cache and batch lie on different devices")
        return _Batch(*self._arguments, tokens, *self._max)


def _on_device(call):
    """The device of the call's cache is the current one while the call is made."""

    @functools.wraps(call)
    def made(cache, *arguments, **named):
        index = cache.device.index
        if torch.cuda.current_device() == index:
            return call(cache, *arguments, **named)
        with torch.cuda.device(index):
            return call(cache, *arguments, **named)
    return made


def _stream(cache):
    return torch._C._cuda_getCurrentRawStream(cache.device.index)  # torch.cuda.current_stream() without its object: 2 us less


def _checked(code):
    if code != 0:
        raise LlmcpError(last_error())


@_on_device
def append(cache, batch, q, k, v, cos=None, sin=None, q_norm=None, k_norm=None, eps=1e-6, q_out=None, status=None):
    """Normalises and rotates the rows of q [tokens, heads, head_dim] and k, stores k and v [tokens, kv_heads, head_dim]
    in their pages and returns the queries.  Rotation: the first cos.shape[1] dimensions by rows ``position`` of cos and
    sin (float32); none without them.  ``q`` may be None (keys and values only; returns None)."""
    dev, bf, dim = cache.device, torch.bfloat16, cache.head_dim
    (kp, ks), (vp, vs) = _tensor(k, "k", bf, 3, dev), _tensor(v, "v", bf, 3, dev)
    shape = k.shape
    tokens = shape[0]
    if shape[1] != cache.kv_heads or shape[2] != dim or v.shape != shape:
        _refuse("k and v have to be [tokens, kv_heads, head_dim]")
    qp, op, strides = None, None, (0, 0, 0)
    if q is not None:
        (qp, qs), shape = _tensor(q, "q", bf, 3, dev), q.shape
        if shape[0] != tokens or shape[2] != dim:
            _refuse("q has to be [tokens, heads, head_dim]")
        if q_out is None:
            q_out = torch.empty_like(q, memory_format=torch.contiguous_format)  # half of torch.empty(shape)'s time
        elif q_out.shape != shape or not q_out.is_contiguous():
            _refuse("q_out has to be [tokens, heads, head_dim], contiguous")
        op, strides = _tensor(q_out, "q_out", bf, 3, dev)[0], (qs[0], qs[1], shape[1])
    norms = _optional(q_norm, "q_norm", bf, 1, dev), _optional(k_norm, "k_norm", bf, 1, dev)
    if (q_norm is not None and q_norm.shape[0] != dim) or (k_norm is not None and k_norm.shape[0] != dim):
        _refuse("q_norm and k_norm have to have head_dim elements")
    if (cos is None) != (sin is None):
        _refuse("cos and sin come together")
    tables, rows, rot = (None, None), 0, 0
    if cos is not None:
        (cp, cs), (sp, ss) = _tensor(cos, "cos", torch.float32, 2, dev), _tensor(sin, "sin", torch.float32, 2, dev)
        rows, rot = cos.shape
        if cos.shape != sin.shape or (rows > 1 and (cs[0] != rot or ss[0] != rot)):
            _refuse("cos and sin have to be [positions, rot], contiguous")
        tables = cp, sp
    _checked(_library().llmcp_dev_paged_append(
        cache._c, batch._c(cache, tokens), qp, *strides, kp, ks[0], ks[1], vp, vs[0], vs[1], *norms, eps, *tables,
        rows, rot, op, _optional(status, "status", torch.int32, 1, dev), _stream(cache)))
    return q_out


@_on_device
def read(cache, batch, tokens, dtype=torch.bfloat16, status=None):
    """The cached keys and values of the batch's rows: two tensors [tokens, kv_heads, head_dim] of bf16 or float32.
    Rows that no sequence owns are left unset."""
    if dtype not in (torch.bfloat16, torch.float32):
        _refuse("dtype has to be bfloat16 or float32")
    k, v = torch.empty((2, tokens, cache.kv_heads, cache.head_dim), dtype=dtype, device=cache.device)
    _checked(_library().llmcp_dev_paged_read(
        cache._c, batch._c(cache, tokens), k.data_ptr(), v.data_ptr(), DTYPE_BF16 if dtype is torch.bfloat16 else DTYPE_F32,
        _optional(status, "status", torch.int32, 1, cache.device), _stream(cache)))
    return k, v


def _workspace_bytes(cache, rows, heads):
    size = _library().llmcp_dev_paged_attention_workspace(cache._c, rows, heads)
    if size < 0:
        raise LlmcpError(last_error())
    return size


@_on_device
def workspace_bytes(cache, batch, tokens, heads):
    """Bytes of working memory that ``attention`` needs for such a call."""
    return _workspace_bytes(cache, batch._c(cache, tokens), heads)


@_on_device
def attention(cache, batch, q, scale=None, softcap=0.0, slopes=None, prefix=None, gate=None, out=None, workspace=None, status=None):
    """softmax(score) v, times sigmoid(gate) where there is a gate: [tokens, heads, head_dim] bf16.  ``out`` may be q or gate
    where that is contiguous, and overlaps nothing else.  ``q`` as ``append`` returns it; ``scale`` 1 / sqrt(head_dim) by
    default; ``slopes`` float32 [heads]; ``prefix`` int32 [sequences]; ``gate`` like q.  ``workspace``: a uint8 tensor of
    workspace_bytes() that no other call uses meanwhile; taken from torch's allocator where it is not given."""
    dev, bf = cache.device, torch.bfloat16
    (qp, qs), shape = _tensor(q, "q", bf, 3, dev), q.shape
    tokens, heads, dim = shape
    if dim != cache.head_dim or heads < 1 or heads % cache.kv_heads:
        _refuse("q has to be [tokens, heads, head_dim], heads a multiple of kv_heads")
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    op, strides = _tensor(out, "out", bf, 3, dev)
    if out.shape != shape or (tokens and strides != (heads * dim, dim, 1) and not out.is_contiguous()):
        _refuse("out has to be [tokens, heads, head_dim], contiguous")
    gp, gate_strides = None, (0, 0, 1)
    if gate is not None:
        gp, gate_strides = _tensor(gate, "gate", bf, 3, dev)
        if gate.shape != shape:
            _refuse("gate has to have q's shape")
    sp, pp = _optional(slopes, "slopes", torch.float32, 1, dev), _optional(prefix, "prefix", torch.int32, 1, dev)
    if slopes is not None and slopes.shape[0] != heads:
        _refuse("slopes has to have one value per head")
    if prefix is not None and prefix.shape[0] != batch.sequences:
        _refuse("prefix has to have one value per sequence")
    rows = batch._c(cache, tokens)
    if workspace is None:
        size = _workspace_bytes(cache, rows, heads)
        workspace = torch.empty(size, dtype=torch.uint8, device=dev) if size else None
    wp = _optional(workspace, "workspace", torch.uint8, 1, dev)
    _checked(_library().llmcp_dev_paged_attention(
        cache._c, rows, qp, qs[0], qs[1], heads, dim ** -0.5 if scale is None else scale, softcap, sp, pp, gp, gate_strides[0], gate_strides[1], op,
        wp, 0 if wp is None else workspace.numel(), _optional(status, "status", torch.int32, 1, dev), _stream(cache)))
    return out
