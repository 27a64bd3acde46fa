"""Streaming attention on torch tensors: a bounded context for long rollouts and the training pass that matches it.

``sink_attention_forward`` / ``_backward`` are attention with a sliding window in which the first keys stay visible;
``paged_attention`` is attention of new tokens (one per row, or a chunk) over a paged key / value cache under the same mask;
``evict_pages`` shrinks that cache to the keys that gathered the most attention weight.  Query i sees key j when
j <= i and (window < 0 or i - j <= window or j < sinks).

The calls run on torch's current stream of the tensors' device, do not synchronise, and may be captured into a CUDA graph.
Tensors are float32 (lengths and tables int32) on one CUDA device; the channels of a head have to be contiguous.

Nothing is recorded for autograd: outputs are tensors without a graph, also where inputs require gradients, which come from
``sink_attention_backward``.  Outputs may not share memory with inputs or with one another, except ``mass_out`` with ``mass``.
"""
from __future__ import annotations

import contextlib
import ctypes as C

import torch

from . import _lib
from ._lib import GnEvictParams, GnPagedParams, GnSinkParams, GnView, GonanoError, check


def _refuse(message):
    raise GonanoError(message)


_BEYOND = 2 ** 31


def _counts(**values):
    # a structure's 32-bit fields would take the low bits of larger numbers
    for name, x in values.items():
        if not -_BEYOND <= x < _BEYOND:
            _refuse(f"{name}: {x} is outside 32 bits")


def _want(name, dtype, shape, device):
    _refuse(f"{name}: want a contiguous {dtype} tensor of shape {tuple(shape)} on {device}")


def _packed(name, t, dtype, device, shape):
    if not (isinstance(t, torch.Tensor) and t.dtype is dtype and t.shape == shape and t.is_contiguous() and t.device == device):
        _want(name, dtype, shape, device)
    return t.data_ptr()


def _view4(name, t, device, shape):
    """[batch, heads, tokens, channels]"""
    if not (isinstance(t, torch.Tensor) and t.dtype is torch.float32 and t.shape == shape and t.device == device):
        _refuse(f"{name}: want a torch.float32 tensor of shape {tuple(shape)} on {device}")
    sb, sh, st, sd = t.stride()
    if sd != 1 and shape[3] > 1:
        _refuse(f"{name}: the channels of a head must be contiguous")
    return GnView(t.data_ptr(), sb, sh, st)


def _view3(name, t, device, shape):
    """[tokens, heads, channels]"""
    if not (isinstance(t, torch.Tensor) and t.dtype is torch.float32 and t.shape == shape and t.device == device):
        _refuse(f"{name}: want a torch.float32 tensor of shape {tuple(shape)} on {device}")
    st, sh, sd = t.stride()
    if sd != 1 and shape[2] > 1:
        _refuse(f"{name}: the channels of a head must be contiguous")
    return GnView(t.data_ptr(), 0, sh, st)


def _shaped(name, t, dims, what):
    if not (isinstance(t, torch.Tensor) and t.dim() == dims):
        _refuse(f"{name}: want {what}")
    return t.shape


def _cuda(name, t, dims):
    if not (isinstance(t, torch.Tensor) and t.is_cuda and t.dtype is torch.float32 and t.dim() == dims):
        _refuse(f"{name}: want a float32 CUDA tensor of {dims} dimensions")
    return t.device


def _on(device):
    """The library works on the current device: makes it the tensors' one where it is another."""
    return _HERE if torch.cuda.current_device() == device.index else torch.cuda.device(device)


_HERE = contextlib.nullcontext()
_NONE = GnView()


def _stream(device):
    return torch._C._cuda_getCurrentRawStream(device.index)   # torch.cuda.current_stream builds a Stream object, 2 us


def _workspace(nbytes, device):
    # from torch's allocator, which knows the stream and the graph that the memory is used on
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None


def _like(tensor):
    # contiguous; half the time of torch.empty with a type and a device
    return torch.empty_like(tensor, memory_format=torch.contiguous_format)


def _address(tensor):
    return tensor.data_ptr() if tensor is not None else None


def _sink_params(q, k, v, sinks, window, scale, lengths):
    _counts(sinks=sinks, window=window)
    device = _cuda("q", q, 4)
    batch, heads, seq, dim = q.shape
    kv_heads = _shaped("k", k, 4, "[batch, kv_heads, seq, dim]")[1]
    shape = (batch, kv_heads, seq, dim)
    p = GnSinkParams(_view4("q", q, device, q.shape), _view4("k", k, device, shape), _view4("v", v, device, shape), batch, heads, kv_heads, seq, dim,
                     sinks, window, scale)
    if lengths is not None:
        p.lengths = _packed("lengths", lengths, torch.int32, device, (batch,))
    return p, device


def sink_attention_forward(q, k, v, sinks, window, scale=1.0, lengths=None, out=None, lse=None):
    """q [batch, heads, seq, dim], k / v [batch, kv_heads, seq, dim], any strides over contiguous channels -> out (like q), lse
    [batch, heads, seq].  ``lengths`` (int32 [batch]): tokens behind a sequence's length are padding, never read; their out is 0
    and their lse -inf.  ``window`` < 0: no window."""
    lib = _lib.load()
    p, device = _sink_params(q, k, v, sinks, window, scale, lengths)
    with _on(device):
        out = _like(q) if out is None else out
        lse = q.new_empty(q.shape[:3]) if lse is None else lse
        _packed("lse", lse, torch.float32, device, q.shape[:3])
        view, nbytes = _view4("out", out, device, q.shape), C.c_int64()
        check(lib.gn_attention_sink_workspace(C.byref(p), 0, C.byref(nbytes)))
        space = _workspace(nbytes.value, device)
        check(lib.gn_attention_sink_forward(C.byref(p), C.byref(view), lse.data_ptr(), _address(space), nbytes.value, _stream(device)))
    return out, lse


def sink_attention_backward(q, k, v, out, dout, lse, sinks, window, scale=1.0, lengths=None, dq=None, dk=None, dv=None):
    """Gradients of ``sink_attention_forward`` at ``dout`` from its ``out`` and ``lse``: dq, dk, dv, added to the tensors given
    (all three or none), else fresh.  The same call gives the same bits every time."""
    lib = _lib.load()
    p, device = _sink_params(q, k, v, sinks, window, scale, lengths)
    given = [g is not None for g in (dq, dk, dv)]
    if any(given) and not all(given):
        _refuse("sink_attention_backward: give dq, dk and dv or none of them")
    with _on(device):
        if not given[0]:
            dq, dk, dv = _like(q), _like(k), _like(v)
        _packed("lse", lse, torch.float32, device, q.shape[:3])
        views = [_view4(n, t, device, like.shape) for n, t, like in (("out", out, q), ("dout", dout, q), ("dq", dq, q), ("dk", dk, k), ("dv", dv, v))]
        nbytes = C.c_int64()
        check(lib.gn_attention_sink_workspace(C.byref(p), 1, C.byref(nbytes)))
        space = _workspace(nbytes.value, device)
        check(lib.gn_attention_sink_backward(C.byref(p), C.byref(views[0]), C.byref(views[1]), lse.data_ptr(), C.byref(views[2]), C.byref(views[3]),
                                             C.byref(views[4]), int(given[0]), _address(space), nbytes.value, _stream(device)))
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
    if (max_query | sinks | (max_context or 0)) >> 31 or not -_BEYOND <= window < _BEYOND:   # a shortcut: the whole check takes 0.8 us
        _counts(max_query=max_query, max_context=max_context or 0, sinks=sinks, window=window)
    device = _cuda("q", q, 3)
    tokens, heads, dim = q.shape
    pages, kv_heads, page_size, _ = _shaped("key_pages", key_pages, 4, "[pages, kv_heads, page_size, dim]")
    rows, width = _shaped("page_table", page_table, 2, "[rows, width]")
    if (new_key is None) != (new_value is None):
        _refuse("paged_attention: give new_key and new_value or neither")
    store, fresh = (pages, kv_heads, page_size, dim), (tokens, kv_heads, dim)
    p = GnPagedParams(_view3("q", q, device, q.shape), _NONE if new_key is None else _view3("new_key", new_key, device, fresh),
                      _NONE if new_value is None else _view3("new_value", new_value, device, fresh), _packed("key_pages", key_pages, torch.float32, device, store),
                      _packed("value_pages", value_pages, torch.float32, device, store), _packed("page_table", page_table, torch.int32, device, (rows, width)),
                      _packed("query_starts", query_starts, torch.int32, device, (rows + 1,)), _packed("context_lens", context_lens, torch.int32, device, (rows,)),
                      None, None, rows, tokens, max_query, width * page_size if max_context is None else max_context, heads, kv_heads, dim, page_size, pages, width,
                      sinks, window, scale)
    with _on(device):
        if mass is not None or mass_out is not None:
            shape = (rows, kv_heads, width * page_size)
            if mass is not None:
                p.mass = _packed("mass", mass, torch.float32, device, shape)
            if mass_out is None:
                mass_out = mass.clone()
            p.mass_out = _packed("mass_out", mass_out, torch.float32, device, shape)
        out = torch.zeros(q.shape, dtype=torch.float32, device=device) if out is None else out
        lse = torch.zeros((tokens, heads), dtype=torch.float32, device=device) if lse is None else lse
        _packed("lse", lse, torch.float32, device, (tokens, heads))
        view, nbytes = _view3("out", out, device, q.shape), C.c_int64()
        check(lib.gn_attention_paged_workspace(C.byref(p), C.byref(nbytes)))
        space = _workspace(nbytes.value, device)
        check(lib.gn_attention_paged(C.byref(p), C.byref(view), lse.data_ptr(), _address(space), nbytes.value, _stream(device)))
    return (out, lse) if mass_out is None else (out, lse, mass_out)


def evict_pages(key_pages, value_pages, mass, page_table, context_lens, budget, sinks=0, recent=0, new_table=None, max_context=None):
    """Keeps ``budget`` keys of every (row, kv head): the first ``sinks``, the last ``recent`` and of the others those of the largest
    ``mass`` ([rows, kv_heads, n], as ``paged_attention`` gathers it; ties to the lower index), in their order, moved to the front of
    the row's pages in ``new_table`` (default: page_table itself, compaction in place).  Every page there is the row's own page of the same
    column - such a page may not belong to two rows - or one that page_table does not name, which is how a prompt shared by several rows is
    left whole; ``page_table[:, :w].contiguous()`` compacts in place too.  Rows of at most ``budget`` keys are kept whole.

    Returns kept (int32 [rows, kv_heads, budget], the indices the keys had, -1 behind them), the new lengths (int32 [rows]) and the
    kept keys' mass [rows, kv_heads, budget] (to gather further, the front of a tensor as wide as the new pages)."""
    lib = _lib.load()
    _counts(budget=budget, sinks=sinks, recent=recent, max_context=max_context or 0)
    device = _cuda("key_pages", key_pages, 4)
    pages, kv_heads, page_size, dim = store = key_pages.shape
    rows, width = _shaped("page_table", page_table, 2, "[rows, width]")
    new_table = page_table if new_table is None else new_table
    new_width = _shaped("new_table", new_table, 2, "[rows, width]")[1]
    n = _shaped("mass", mass, 3, "[rows, kv_heads, n]")[2]
    if budget < 0:
        _refuse(f"evict_pages: budget {budget} is negative")
    p = GnEvictParams(_packed("key_pages", key_pages, torch.float32, device, store), _packed("value_pages", value_pages, torch.float32, device, store),
                      _packed("mass", mass, torch.float32, device, (rows, kv_heads, n)), _packed("page_table", page_table, torch.int32, device, (rows, width)),
                      _packed("new_table", new_table, torch.int32, device, (rows, new_width)),
                      _packed("context_lens", context_lens, torch.int32, device, (rows,)), rows, kv_heads, dim, page_size, pages, width, new_width, n,
                      width * page_size if max_context is None else max_context, budget, sinks, recent)
    with _on(device):
        kept = page_table.new_empty((rows, kv_heads, budget))
        lens = torch.empty_like(context_lens)
        mass_out = mass.new_empty((rows, kv_heads, budget))
        check(lib.gn_cache_evict(C.byref(p), kept.data_ptr(), lens.data_ptr(), mass_out.data_ptr(), _stream(device)))
    return kept, lens, mass_out
