"""Streaming attention on torch tensors: a bounded context for long rollouts and the training pass that matches it.

``sink_attention_forward`` / ``_backward`` are attention with a sliding window in which the first keys stay visible;
``paged_attention`` is attention of new tokens (one per row, or a chunk) over a paged key / value cache under the same mask;
``evict_pages`` shrinks that cache to the keys that gathered the most attention weight.  Query i sees key j when
j <= i and (window < 0 or i - j <= window or j < sinks).

The calls run on torch's current stream of the tensors' device, do not synchronise, and may be captured into a CUDA graph.
Tensors are float32 (lengths and tables int32) on one CUDA device; the channels of a head have to be contiguous.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import _lib
from ._lib import GnEvictParams, GnPagedParams, GnSinkParams, GnView, GonanoError, check


def _need(condition, message):
    if not condition:
        raise GonanoError(message)


def _same(name, tensor, dtype, device, shape):
    _need(isinstance(tensor, torch.Tensor) and tensor.dtype == dtype and tensor.device == device and tuple(tensor.shape) == tuple(shape),
          f"{name}: want a {dtype} tensor of shape {tuple(shape)} on {device}")


def _packed(name, tensor, dtype, device, shape):
    _same(name, tensor, dtype, device, shape)
    _need(tensor.is_contiguous(), f"{name}: want a contiguous tensor")


def _view4(name, t, device, shape):
    """[batch, heads, tokens, channels]"""
    _same(name, t, torch.float32, device, shape)
    sb, sh, st, sd = t.stride()
    _need(sd == 1 or t.shape[3] == 1, f"{name}: the channels of a head must be contiguous")
    return GnView(t.data_ptr(), sb, sh, st)


def _view3(name, t, device, shape):
    """[tokens, heads, channels]"""
    _same(name, t, torch.float32, device, shape)
    st, sh, sd = t.stride()
    _need(sd == 1 or t.shape[2] == 1, f"{name}: the channels of a head must be contiguous")
    return GnView(t.data_ptr(), 0, sh, st)


def _cuda(name, t, dims):
    _need(isinstance(t, torch.Tensor) and t.is_cuda and t.dtype == torch.float32 and t.dim() == dims, f"{name}: want a float32 CUDA tensor of {dims} dimensions")
    return t.device


def _workspace(nbytes, device):
    # from torch's allocator, which knows the stream and the graph that the memory is used on
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None


def _address(tensor):
    return tensor.data_ptr() if tensor is not None else None


def _sink_params(q, k, v, sinks, window, scale, lengths):
    device = _cuda("q", q, 4)
    batch, heads, seq, dim = q.shape
    _need(isinstance(k, torch.Tensor) and k.dim() == 4, "k: want a float32 CUDA tensor of 4 dimensions")
    shape = (batch, k.shape[1], seq, dim)
    p = GnSinkParams(_view4("q", q, device, q.shape), _view4("k", k, device, shape), _view4("v", v, device, shape), batch, heads, k.shape[1], seq, dim,
                     sinks, window, scale)
    if lengths is not None:
        _packed("lengths", lengths, torch.int32, device, (batch,))
        p.lengths = lengths.data_ptr()
    return p, device


def sink_attention_forward(q, k, v, sinks, window, scale=1.0, lengths=None, out=None, lse=None):
    """q [batch, heads, seq, dim], k / v [batch, kv_heads, seq, dim], any strides over contiguous channels -> out (like q), lse
    [batch, heads, seq].  ``lengths`` (int32 [batch]): tokens behind a sequence's length are padding, never read; their out is 0
    and their lse -inf.  ``window`` < 0: no window."""
    lib = _lib.load()
    p, device = _sink_params(q, k, v, sinks, window, scale, lengths)
    with torch.cuda.device(device):
        out = torch.empty(q.shape, dtype=torch.float32, device=device) if out is None else out
        lse = torch.empty(q.shape[:3], dtype=torch.float32, device=device) if lse is None else lse
        _packed("lse", lse, torch.float32, device, q.shape[:3])
        view, nbytes = _view4("out", out, device, q.shape), C.c_int64()
        check(lib.gn_attention_sink_workspace(C.byref(p), 0, C.byref(nbytes)))
        space = _workspace(nbytes.value, device)
        check(lib.gn_attention_sink_forward(C.byref(p), C.byref(view), lse.data_ptr(), _address(space), nbytes.value, torch.cuda.current_stream(device).cuda_stream))
    return out, lse


def sink_attention_backward(q, k, v, out, dout, lse, sinks, window, scale=1.0, lengths=None, dq=None, dk=None, dv=None):
    """Gradients of ``sink_attention_forward`` at ``dout`` from its ``out`` and ``lse``: dq, dk, dv, added to the tensors given
    (all three or none), else fresh.  The same call gives the same bits every time."""
    lib = _lib.load()
    p, device = _sink_params(q, k, v, sinks, window, scale, lengths)
    given = [g is not None for g in (dq, dk, dv)]
    _need(all(given) or not any(given), "sink_attention_backward: give dq, dk and dv or none of them")
    with torch.cuda.device(device):
        if not given[0]:
            dq, dk, dv = (torch.empty(x.shape, dtype=torch.float32, device=device) for x in (q, k, v))
        _packed("lse", lse, torch.float32, device, q.shape[:3])
        views = [_view4(n, t, device, like.shape) for n, t, like in (("out", out, q), ("dout", dout, q), ("dq", dq, q), ("dk", dk, k), ("dv", dv, v))]
        nbytes = C.c_int64()
        check(lib.gn_attention_sink_workspace(C.byref(p), 1, C.byref(nbytes)))
        space = _workspace(nbytes.value, device)
        check(lib.gn_attention_sink_backward(C.byref(p), C.byref(views[0]), C.byref(views[1]), lse.data_ptr(), C.byref(views[2]), C.byref(views[3]),
                                             C.byref(views[4]), int(given[0]), _address(space), nbytes.value, torch.cuda.current_stream(device).cuda_stream))
    return dq, dk, dv


def paged_attention(q, key_pages, value_pages, page_table, query_starts, context_lens, max_query, max_context=None, new_key=None, new_value=None,
                    sinks=0, window=-1, scale=1.0, mass=None, mass_out=None, out=None, lse=None):
    """Attention of the new tokens of every row over its cached keys.

    q [tokens, heads, dim] holds the rows' new tokens one row after the other: row r's are query_starts[r] .. query_starts[r + 1] - 1
    (int32 [rows + 1]), at most ``max_query`` of them.  key_pages / value_pages [pages, kv_heads, page_size, dim], contiguous; key j of
    row r is slot j % page_size of page page_table[r, j // page_size] (int32 [rows, width]).  context_lens[r] (int32 [rows]) counts the
    row's keys with its new tokens', which stand at the end; ``max_context`` is an upper bound of it (default: what the table holds).
    With new_key / new_value [tokens, kv_heads, dim] the new tokens' own keys and values are first written to the pages.
    ``mass`` [rows, kv_heads, width * page_size] is the attention weight that each key has gathered so far; ``mass_out`` (may be
    ``mass``; default: a copy) receives it with this call's added, the new tokens' own keys starting from 0.

    Returns out (like q), lse [tokens, heads] and, when mass or mass_out is given, mass_out.  Entries behind the last row's tokens
    are left as they are (0 in tensors made here)."""
    lib = _lib.load()
    device = _cuda("q", q, 3)
    tokens, heads, dim = q.shape
    _need(isinstance(key_pages, torch.Tensor) and key_pages.dim() == 4, "key_pages: want [pages, kv_heads, page_size, dim]")
    pages, kv_heads, page_size = key_pages.shape[:3]
    for name, t in (("key_pages", key_pages), ("value_pages", value_pages)):
        _packed(name, t, torch.float32, device, (pages, kv_heads, page_size, dim))
    _need(isinstance(page_table, torch.Tensor) and page_table.dim() == 2, "page_table: want [rows, width]")
    rows, width = page_table.shape
    _packed("page_table", page_table, torch.int32, device, (rows, width))
    _packed("query_starts", query_starts, torch.int32, device, (rows + 1,))
    _packed("context_lens", context_lens, torch.int32, device, (rows,))
    _need((new_key is None) == (new_value is None), "paged_attention: give new_key and new_value or neither")
    p = GnPagedParams(query=_view3("q", q, device, q.shape), key_pages=key_pages.data_ptr(), value_pages=value_pages.data_ptr(),
                      page_table=page_table.data_ptr(), query_starts=query_starts.data_ptr(), context_lens=context_lens.data_ptr(), rows=rows, tokens=tokens,
                      max_query=max_query, max_context=width * page_size if max_context is None else max_context, n_head=heads, n_kv_head=kv_heads,
                      head_dim=dim, page_size=page_size, pages=pages, table_width=width, sinks=sinks, window=window, scale=scale)
    if new_key is not None:
        p.new_key, p.new_value = (_view3(n, t, device, (tokens, kv_heads, dim)) for n, t in (("new_key", new_key), ("new_value", new_value)))
    with torch.cuda.device(device):
        if mass is not None or mass_out is not None:
            shape = (rows, kv_heads, width * page_size)
            if mass is not None:
                _packed("mass", mass, torch.float32, device, shape)
                p.mass = mass.data_ptr()
            if mass_out is None:
                mass_out = mass.clone()
            _packed("mass_out", mass_out, torch.float32, device, shape)
            p.mass_out = mass_out.data_ptr()
        out = torch.zeros(q.shape, dtype=torch.float32, device=device) if out is None else out
        lse = torch.zeros((tokens, heads), dtype=torch.float32, device=device) if lse is None else lse
        _packed("lse", lse, torch.float32, device, (tokens, heads))
        view, nbytes = _view3("out", out, device, q.shape), C.c_int64()
        check(lib.gn_attention_paged_workspace(C.byref(p), C.byref(nbytes)))
        space = _workspace(nbytes.value, device)
        check(lib.gn_attention_paged(C.byref(p), C.byref(view), lse.data_ptr(), _address(space), nbytes.value, torch.cuda.current_stream(device).cuda_stream))
    return (out, lse) if mass_out is None else (out, lse, mass_out)


def evict_pages(key_pages, value_pages, mass, page_table, context_lens, budget, sinks=0, recent=0, new_table=None, max_context=None):
    """Keeps ``budget`` keys of every (row, kv head): the first ``sinks``, the last ``recent`` and of the others those of the largest
    ``mass`` ([rows, kv_heads, n], as ``paged_attention`` gathers it; ties to the lower index), in their order, moved to the front of
    the row's pages in ``new_table`` (default: page_table itself, compaction in place - no page may then belong to two rows; else pages
    that page_table does not name, which is how a prompt shared by several rows is left whole).  Rows of at most ``budget`` keys are kept whole.

    Returns kept (int32 [rows, kv_heads, budget], the indices the keys had, -1 behind them), the new lengths (int32 [rows]) and the
    kept keys' mass [rows, kv_heads, budget]."""
    lib = _lib.load()
    device = _cuda("key_pages", key_pages, 4)
    pages, kv_heads, page_size, dim = key_pages.shape
    for name, t in (("key_pages", key_pages), ("value_pages", value_pages)):
        _packed(name, t, torch.float32, device, key_pages.shape)
    _need(isinstance(page_table, torch.Tensor) and page_table.dim() == 2, "page_table: want [rows, width]")
    rows, width = page_table.shape
    new_table = page_table if new_table is None else new_table
    _need(isinstance(new_table, torch.Tensor) and new_table.dim() == 2, "new_table: want [rows, width]")
    _packed("page_table", page_table, torch.int32, device, (rows, width))
    _packed("new_table", new_table, torch.int32, device, (rows, new_table.shape[1]))
    _packed("context_lens", context_lens, torch.int32, device, (rows,))
    _need(isinstance(mass, torch.Tensor) and mass.dim() == 3, "mass: want [rows, kv_heads, n]")
    _packed("mass", mass, torch.float32, device, (rows, kv_heads, mass.shape[2]))
    _need(budget >= 0, f"evict_pages: budget {budget} is negative")
    p = GnEvictParams(key_pages.data_ptr(), value_pages.data_ptr(), mass.data_ptr(), page_table.data_ptr(), new_table.data_ptr(), context_lens.data_ptr(), rows,
                      kv_heads, dim, page_size, pages, width, new_table.shape[1], mass.shape[2], width * page_size if max_context is None else max_context,
                      budget, sinks, recent)
    with torch.cuda.device(device):
        kept = torch.empty((rows, kv_heads, budget), dtype=torch.int32, device=device)
        lens = torch.empty((rows,), dtype=torch.int32, device=device)
        mass_out = torch.empty((rows, kv_heads, budget), dtype=torch.float32, device=device)
        check(lib.gn_cache_evict(C.byref(p), kept.data_ptr(), lens.data_ptr(), mass_out.data_ptr(), torch.cuda.current_stream(device).cuda_stream))
    return kept, lens, mass_out
