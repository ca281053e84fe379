"""A key/value cache in pages that many sequences share, on torch tensors: append, attention, read.

The calls of include/llmcp_b200.h (llmcp_dev_paged_*) with their checks; layouts, formulas and what ``status`` reports
are described there.  Everything is enqueued on the current stream of the tensors' device and nothing is synchronised,
so the calls can be captured into a graph; lengths and page tables may then change between replays.

    cache = Cache(pages, scales)                # pages bf16, or uint8 with f16 scales (4 bits)
    batch = Batch(q_start, kv_len, page_table, max_q, max_kv)
    q = append(cache, batch, q, k, v, cos, sin, q_norm=..., k_norm=...)
    out = attention(cache, batch, q, gate=...)
"""
import ctypes as C

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


def _need(ok, what):
    if not ok:
        raise LlmcpError("paged cache: " + what)


def _tensor(t, name, dtype, dims, device):
    """The address of ``t``, which has to have that type and rank, lie on that device and be dense in its last dimension."""
    _need(t.dtype == dtype, f"{name} has to be {dtype}")
    _need(t.dim() == dims, f"{name} has to have {dims} dimensions")
    _need(t.device == device, f"{name} has to lie on {device}")
    _need(t.stride(-1) == 1 or t.shape[-1] <= 1, f"{name} has to be dense in its last dimension")
    return t.data_ptr()


class Cache:
    """One layer's pages [num_pages, 2, kv_heads, page_size, head_dim]: bf16, or uint8 [..., head_dim / 2] with
    ``scales`` [..., head_dim / 32] float16.  The tensors stay the caller's; nothing is copied."""

    def __init__(self, pages, scales=None):
        _need(pages.dim() == 5 and pages.shape[1] == 2, "pages has to be [num_pages, 2, kv_heads, page_size, head_dim]")
        _need(pages.is_cuda, "pages has to lie on a CUDA device")
        _need(pages.is_contiguous(), "pages has to be contiguous")
        _need(pages.dtype == (torch.bfloat16 if scales is None else torch.uint8), "pages has to be bfloat16, or uint8 where there are scales")
        count, _, heads, size, last = pages.shape
        dim = last if scales is None else 2 * last
        _need(count >= 1 and heads >= 1 and size in PAGE_SIZES and dim in HEAD_DIMS, f"page sizes are {PAGE_SIZES}, head dimensions {HEAD_DIMS}")
        if scales is not None:
            _need(scales.dtype == torch.float16 and tuple(scales.shape) == (count, 2, heads, size, dim // 32) and scales.is_contiguous() and
                  scales.device == pages.device, "scales has to be float16 [num_pages, 2, kv_heads, page_size, head_dim / 32], contiguous, beside pages")
        self.pages, self.scales, self.device = pages, scales, pages.device
        self.kv_heads, self.page_size, self.head_dim = heads, size, dim
        self._c = _Kv(pages.data_ptr(), None if scales is None else scales.data_ptr(), count, size, heads, dim)


class Batch:
    """Sequence b owns rows q_start[b] to q_start[b + 1] - 1 of a call, the last ones of its kv_len[b] tokens; token j
    lies in page page_table[b, j // page_size].  int32 tensors [sequences + 1], [sequences], [sequences, width];
    ``max_q`` and ``max_kv`` bound rows and lengths of a sequence."""

    def __init__(self, q_start, kv_len, page_table, max_q, max_kv):
        device = q_start.device
        _need(q_start.is_cuda, "q_start has to lie on a CUDA device")
        addresses = [_tensor(t, n, torch.int32, d, device) for t, n, d in
                     ((q_start, "q_start", 1), (kv_len, "kv_len", 1), (page_table, "page_table", 2))]
        sequences, width = page_table.shape
        _need(q_start.shape[0] == sequences + 1 and kv_len.shape[0] == sequences, "q_start has one entry more than kv_len and page_table have rows")
        _need(sequences < 2 or page_table.stride(0) >= width, "rows of page_table overlap")
        self.q_start, self.kv_len, self.page_table, self.device = q_start, kv_len, page_table, device
        self._c = _Batch(*addresses, sequences, width, page_table.stride(0), 0, max_q, max_kv)


class _Call:
    """The device of a call made current where it is not, its stream, and a batch with the call's number of rows."""

    def __init__(self, cache, batch, tokens):
        _need(batch.device == cache.device, "cache and batch lie on different devices")
        self.batch = _Batch.from_buffer_copy(batch._c)
        self.batch.tokens = tokens
        self.device = cache.device
        self.other = None

    def __enter__(self):
        if torch.cuda.current_device() != self.device.index:
            self.other = torch.cuda.device(self.device)
            self.other.__enter__()
        self.stream = torch.cuda.current_stream().cuda_stream
        return self

    def __exit__(self, *error):
        if self.other is not None:
            self.other.__exit__(*error)


def _checked(code):
    if code != 0:
        raise LlmcpError(last_error())


def _status(status, device):
    return None if status is None else _tensor(status, "status", torch.int32, 1, device)


def append(cache, batch, q, k, v, cos=None, sin=None, q_norm=None, k_norm=None, eps=1e-6, q_out=None, status=None):
    """Normalises and rotates the rows of q [tokens, heads, head_dim] and k, stores k and v [tokens, kv_heads, head_dim]
    in their pages and returns the queries.  Rotation: the first cos.shape[1] dimensions by rows ``position`` of cos and
    sin (float32); none without them.  ``q`` may be None (keys and values only; returns None)."""
    dev, bf = cache.device, torch.bfloat16
    kp, vp = _tensor(k, "k", bf, 3, dev), _tensor(v, "v", bf, 3, dev)
    tokens = k.shape[0]
    _need(tuple(k.shape[1:]) == (cache.kv_heads, cache.head_dim) and k.shape == v.shape, "k and v have to be [tokens, kv_heads, head_dim]")
    heads, qp, op = 0, None, None
    if q is not None:
        qp, heads = _tensor(q, "q", bf, 3, dev), q.shape[1]
        _need(q.shape[0] == tokens and q.shape[2] == cache.head_dim, "q has to be [tokens, heads, head_dim]")
        if q_out is None:
            q_out = torch.empty((tokens, heads, cache.head_dim), dtype=bf, device=dev)
        op = _tensor(q_out, "q_out", bf, 3, dev)
        _need(q_out.shape == q.shape and q_out.is_contiguous(), "q_out has to be [tokens, heads, head_dim], contiguous")
    norms = []
    for name, w in (("q_norm", q_norm), ("k_norm", k_norm)):
        norms.append(None if w is None else _tensor(w, name, bf, 1, dev))
        _need(w is None or w.shape[0] == cache.head_dim, f"{name} has to have head_dim elements")
    _need((cos is None) == (sin is None), "cos and sin come together")
    tables, rows, rot = [None, None], 0, 0
    if cos is not None:
        tables = [_tensor(cos, "cos", torch.float32, 2, dev), _tensor(sin, "sin", torch.float32, 2, dev)]
        _need(cos.shape == sin.shape and cos.is_contiguous() and sin.is_contiguous(), "cos and sin have to be [positions, rot], contiguous")
        rows, rot = cos.shape
    with _Call(cache, batch, tokens) as call:
        _checked(_library().llmcp_dev_paged_append(
            cache._c, call.batch, qp, q.stride(0) if heads else 0, q.stride(1) if heads else 0, heads, kp, k.stride(0), k.stride(1),
            vp, v.stride(0), v.stride(1), norms[0], norms[1], eps, tables[0], tables[1], rows, rot, op, _status(status, dev), call.stream))
    return q_out


def read(cache, batch, tokens, dtype=torch.bfloat16, status=None):
    """The cached keys and values of the batch's rows: two tensors [tokens, kv_heads, head_dim] of bf16 or float32.
    Rows that no sequence owns are left unset."""
    _need(dtype in (torch.bfloat16, torch.float32), "dtype has to be bfloat16 or float32")
    k, v = (torch.empty((tokens, cache.kv_heads, cache.head_dim), dtype=dtype, device=cache.device) for _ in range(2))
    with _Call(cache, batch, tokens) as call:
        _checked(_library().llmcp_dev_paged_read(cache._c, call.batch, k.data_ptr(), v.data_ptr(),
                                                 DTYPE_BF16 if dtype == torch.bfloat16 else DTYPE_F32, _status(status, cache.device), call.stream))
    return k, v


def workspace_bytes(cache, batch, tokens, heads):
    """Bytes of working memory that ``attention`` needs for such a call."""
    with _Call(cache, batch, tokens) as call:
        size = _library().llmcp_dev_paged_attention_workspace(cache._c, call.batch, heads)
    if size < 0:
        raise LlmcpError(last_error())
    return size


def attention(cache, batch, q, scale=None, softcap=0.0, slopes=None, prefix=None, gate=None, out=None, workspace=None, status=None):
    """softmax(score) v, times sigmoid(gate) where there is a gate: [tokens, heads, head_dim] bf16.  ``q`` as ``append``
    returns it; ``scale`` 1 / sqrt(head_dim) by default; ``slopes`` float32 [heads]; ``prefix`` int32 [sequences];
    ``gate`` like q.  ``workspace``: a uint8 tensor of workspace_bytes() that no other call uses meanwhile; taken from
    torch's allocator where it is not given."""
    dev, bf = cache.device, torch.bfloat16
    qp = _tensor(q, "q", bf, 3, dev)
    tokens, heads, dim = q.shape
    _need(dim == cache.head_dim and heads % cache.kv_heads == 0 and heads > 0, "q has to be [tokens, heads, head_dim], heads a multiple of kv_heads")
    if out is None:
        out = torch.empty((tokens, heads, dim), dtype=bf, device=dev)
    op = _tensor(out, "out", bf, 3, dev)
    _need(out.shape == q.shape and out.is_contiguous(), "out has to be [tokens, heads, head_dim], contiguous")
    gp = None
    if gate is not None:
        gp = _tensor(gate, "gate", bf, 3, dev)
        _need(gate.shape == q.shape, "gate has to have q's shape")
    sp = None if slopes is None else _tensor(slopes, "slopes", torch.float32, 1, dev)
    _need(slopes is None or slopes.shape[0] == heads, "slopes has to have one value per head")
    pp = None if prefix is None else _tensor(prefix, "prefix", torch.int32, 1, dev)
    _need(prefix is None or prefix.shape[0] == batch.kv_len.shape[0], "prefix has to have one value per sequence")
    with _Call(cache, batch, tokens) as call:
        if workspace is None:
            size = _library().llmcp_dev_paged_attention_workspace(cache._c, call.batch, heads)
            if size < 0:
                raise LlmcpError(last_error())
            workspace = torch.empty(size, dtype=torch.uint8, device=dev) if size else None
        wp = None if workspace is None else _tensor(workspace, "workspace", torch.uint8, 1, dev)
        _checked(_library().llmcp_dev_paged_attention(
            cache._c, call.batch, qp, q.stride(0), q.stride(1), heads, dim ** -0.5 if scale is None else scale, softcap, sp, pp,
            gp, gate.stride(0) if gp else 0, gate.stride(1) if gp else 0, op, wp, workspace.numel() if wp else 0,
            _status(status, dev), call.stream))
    return out
