"""Paged key-value cache: its bookkeeping, the write into it and the attention that reads it.

The HBM that compressed weights free holds keys and values in pages of a
power-of-two number of tokens, which any request can use. A request with n
cached tokens holds the pages ``block_table[b, :ceil(n / page_size)]``; its
token at position p lies at slot ``block_table[b, p // page_size] * page_size
+ p % page_size`` of ``key_pages``/``value_pages`` (pages, page_size, key/value
heads, head width). The reference leaves the cache to Transformers
(neuralzip/gpu/inference.py has none).

* ``reserve_pages`` / ``release_pages``: block tables, positions and slots
  from request lengths, on the GPU;
* ``rotary_store``: query and key norms, rotary positions and the write into
  the pages, in one pass;
* ``paged_attention``: one new token a request over its pages.

Every call enqueues on torch's current stream of the tensors' device, never
synchronises, and can be captured in a CUDA graph. Between calls it keeps no
contents, addresses or results: only which layouts (types, shapes, strides,
devices, sizes) passed the checks, and the devices' limits. Tensors written by another stream need that stream waited for first,
as with any torch operator. Nothing here has a derivative: calls that would
need one, in backward or forward mode, are refused. What only the GPU can see (lengths, page ids,
positions, slots) is bounds-checked by the kernels, as each function says.
"""

from __future__ import annotations

import ctypes
import functools
import importlib.machinery
import importlib.util
import struct
from typing import NamedTuple

import torch
from torch.autograd import forward_ad

from neuralzip_b200 import _native

MAX_REQUESTS = _native.PAGED_MAX_REQUESTS
MAX_HEAD_WIDTH = _native.PAGED_MAX_DIM
_DTYPES = {torch.bfloat16: _native.PAGED_BF16, torch.float16: _native.PAGED_FP16, torch.float32: _native.PAGED_FP32}


class PageReservation(NamedTuple):
    """What ``reserve_pages`` returns; all int32."""

    positions: torch.Tensor    # (rows,) position of each row's token, 0 for a row without one
    slots: torch.Tensor        # (rows,) its slot, -1 for a row without one
    row_offsets: torch.Tensor  # (requests + 1,) first row of each request
    lengths: torch.Tensor      # (requests,) lengths with the new tokens
    used: torch.Tensor         # (1,) pages in use
    refused: torch.Tensor      # (1,) requests refused


def _tensor(name, value, dtype, dims):
    if not isinstance(value, torch.Tensor):
        raise TypeError(f"{name} must be a tensor.")
    if value.dtype is not dtype:
        raise TypeError(f"{name} must be {dtype}, not {value.dtype}.")
    if value.dim() != dims:
        raise ValueError(f"{name} must have {dims} dimensions, not {value.dim()}.")
    return value


def _vector(name, value, size=None, dtype=torch.int32):
    _tensor(name, value, dtype, 1)
    if size is not None and value.shape[0] != size:
        raise ValueError(f"{name} must have {size} elements, not {value.shape[0]}.")
    if not value.is_contiguous():
        raise ValueError(f"{name} must be contiguous.")
    return value


def _table(block_table, requests, written):
    _tensor("block_table", block_table, torch.int32, 2)
    if block_table.shape[0] != requests:
        raise ValueError(f"block_table must have {requests} rows, not {block_table.shape[0]}.")
    if not block_table.is_contiguous():
        if block_table.shape[1] > 1 and block_table.stride(1) != 1:
            raise ValueError("block_table's columns must be contiguous.")
        if written and requests > 1 and block_table.stride(0) < block_table.shape[1]:
            raise ValueError("block_table's rows must not overlap.")
    return block_table


def _rows(name, value, shape, dtype):
    """A (rows, heads, width) tensor whose last dimension is contiguous."""
    _tensor(name, value, dtype, len(shape))
    if tuple(value.shape) != tuple(shape):
        raise ValueError(f"{name} must have the shape {tuple(shape)}, not {tuple(value.shape)}.")
    if value.shape[-1] > 1 and value.stride(-1) != 1:
        raise ValueError(f"The last dimension of {name} must be contiguous.")
    return value


def _written(name, value):
    """Refuses a tensor whose elements share memory (expanded, overlapping)."""
    if value.is_contiguous():
        return
    reach = 0
    for stride, size in sorted(zip(value.stride(), value.shape)):
        if size > 1:
            if stride <= reach:
                raise ValueError(f"{name} is written and must not overlap itself.")
            reach += stride * (size - 1)


def _page_shift(page_size):
    if isinstance(page_size, bool) or not isinstance(page_size, int):
        raise TypeError("page_size must be a whole number.")
    if not 0 < page_size <= 1 << 20 or page_size & (page_size - 1):
        raise ValueError(f"page_size must be a power of two up to 2^20, not {page_size}.")
    return page_size.bit_length() - 1


def _requests(lengths):
    _vector("lengths", lengths)
    if not 0 < lengths.shape[0] <= MAX_REQUESTS:
        raise ValueError(f"There must be 1 to {MAX_REQUESTS} requests, not {lengths.shape[0]}.")
    return lengths.shape[0]


def _same_device(*tensors):
    device = tensors[0].device
    for tensor in tensors:
        if tensor is not None and tensor.device != device:
            raise ValueError(f"All tensors must be on one device, not on {device} and {tensor.device}.")
    if device.type != "cuda":
        raise ValueError(f"The tensors must be on a CUDA device, not on {device}.")
    return device


def _in_place_or_apart(name, out, source):
    """Refuses an output that covers part of the input it may replace."""
    if out is not None and 0 < abs(out.data_ptr() - source.data_ptr()) < 4 * source.shape[0]:
        raise ValueError(f"{name} overlaps its input in part.")


def _call(name, args, index):
    """One C call: `args` are the bytes of its struct."""
    with torch.cuda.device(index):
        stream = torch.cuda.current_stream(index).cuda_stream
        _native.check(getattr(_native.load(), name)(args, stream or None))


def _pack(layout, *sizes):
    try:
        return struct.pack(layout, *sizes)
    except struct.error as error:
        raise ValueError("A size or stride is out of range.") from error


def _number(name, value):
    try:
        return struct.pack("<f", value)
    except struct.error as error:
        raise TypeError(f"{name} must be a number.") from error
    except OverflowError as error:
        raise ValueError(f"{name} is out of float32's range.") from error


# The extension module that makes calls of known layouts (types, shapes,
# strides, devices and sizes; no addresses, no contents) without checking
# them again, loaded with the first call: a checked call takes 15 to 35 us of
# host time, more than most steps' kernels, one of a known layout 4.4 to 7.
# None: every call is checked. A prompt batch of a number of tokens not seen
# before is a new layout, and so checked.
_calls = None
_RESERVE, _RELEASE, _ROTARY, _ATTENTION = range(4)


@functools.cache
def _load_calls():
    global _calls
    from neuralzip_b200 import build

    try:
        loader = importlib.machinery.ExtensionFileLoader("nz_paged_torch", str(build.torch_calls()))
        module = importlib.util.module_from_spec(importlib.util.spec_from_loader("nz_paged_torch", loader))
        loader.exec_module(module)
    except ImportError:  # not built, or not against this torch
        return
    lib = _native.load()
    module.bind(*(ctypes.cast(getattr(lib, name), ctypes.c_void_p).value for name in
                  ("nz_pages_reserve", "nz_pages_release", "nz_rotary_store", "nz_paged_attention")))
    _calls = module


def _remember(operator, call, tail, workspace=0, scale=0.0):
    """Makes the layout of a call that passed its checks known."""
    _load_calls()
    if _calls is not None:
        _calls.remember(operator, call, tail, workspace, scale)


def _no_gradient(*tensors):
    if torch.is_grad_enabled() and any(getattr(t, "requires_grad", False) for t in tensors):
        raise RuntimeError("The paged cache has no backward pass; call it under torch.no_grad().")
    # Dual tensors live inside a level only; looking at each tensor takes 0.5 us.
    if getattr(forward_ad, "_current_level", 0) >= 0 and any(
            isinstance(t, torch.Tensor) and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise RuntimeError("The paged cache has no forward-mode derivatives; unpack dual tensors before the call.")


def _wrote(*tensors):
    """Tells autograd of tensors written in place, so that a backward pass that saved one is refused."""
    for tensor in tensors:
        if tensor is not None:
            torch.autograd.graph.increment_version(tensor)


def _whole(name, value, low, high):
    if isinstance(value, bool) or not isinstance(value, int):
        raise TypeError(f"{name} must be a whole number.")
    if not low <= value <= high:
        raise ValueError(f"{name} must be {low} to {high}, not {value}.")
    return value


def reserve_pages(lengths, new_tokens, block_table, free_pages, used, *, page_size, rows, row_stride=0,
                  lengths_out=None, used_out=None):
    """Reserves pages for ``new_tokens[b]`` more tokens of each request b.

    ``free_pages`` (one entry for each page of the cache) is a stack: the ids
    from ``used[0]`` on are the free pages, the entries before it are room
    for those in use. In request order, each request takes the pages it lacks
    from there; they are written into its row of ``block_table``
    (requests, most pages a request). Returns a PageReservation. Request b's
    rows begin at the number of new tokens before it (``row_stride`` 0: rows
    packed), or at ``b * row_stride``; a row without a token (behind a
    request's own, behind the last request, or of a refused request) gets
    position 0 and slot -1.

    A request is refused, keeps its length and takes no page when a count is
    negative, its tokens do not fit its rows or its row of the block table,
    or it needs pages and those needed by the requests up to it (without the
    ones refused for another reason) exceed the free ones.

    ``lengths_out`` and ``used_out`` may be ``lengths`` and ``used``, which
    updates them in place; they and ``block_table`` overlap nothing else
    that is passed. All tensors are int32."""
    call = (lengths, new_tokens, block_table, free_pages, used, page_size, rows, row_stride, lengths_out, used_out)
    if _calls is not None:
        done = _calls.reserve(*call)
        if done.__class__ is tuple:
            return PageReservation._make(done)
        if done is not None:
            _native.check(done)
    device, sizes, tail = _plan_reserve(*call)
    _in_place_or_apart("lengths_out", lengths_out, lengths)
    # One allocation: positions, slots, row offsets, refusals, lengths, pages in use.
    out = torch.empty(sum(sizes), dtype=torch.int32, device=device)
    positions, slots, row_offsets, refused, fresh_lengths, fresh_used = out.split_with_sizes(sizes)
    if lengths_out is None:
        lengths_out = fresh_lengths
    if used_out is None:
        used_out = fresh_used
    _call("nz_pages_reserve", struct.pack(
        "<11Q", lengths.data_ptr(), new_tokens.data_ptr(), block_table.data_ptr(), free_pages.data_ptr(), used.data_ptr(),
        positions.data_ptr(), slots.data_ptr(), row_offsets.data_ptr(), lengths_out.data_ptr(), used_out.data_ptr(),
        refused.data_ptr()) + tail, device.index)
    _wrote(block_table, *call[-2:])
    _remember(_RESERVE, call, tail)
    return PageReservation(positions, slots, row_offsets, lengths_out, used_out, refused)


def _plan_reserve(lengths, new_tokens, block_table, free_pages, used, page_size, rows, row_stride, lengths_out, used_out):
    requests = _requests(lengths)
    _vector("new_tokens", new_tokens, requests)
    _table(block_table, requests, True)
    _vector("free_pages", free_pages)
    _vector("used", used, 1)
    shift = _page_shift(page_size)
    _whole("rows", rows, 0, 1 << 30)
    _whole("row_stride (in rows)", row_stride, 0, 1 << 30)
    if lengths_out is not None:
        _vector("lengths_out", lengths_out, requests)
    if used_out is not None:
        _vector("used_out", used_out, 1)
    device = _same_device(lengths, new_tokens, block_table, free_pages, used, lengths_out, used_out)
    tail = _pack("<Q6I", block_table.stride(0), requests, block_table.shape[1], free_pages.shape[0], rows,
                       row_stride, shift)
    return device, (rows, rows, requests + 1, 1, requests, 1), tail


def release_pages(lengths, done, block_table, free_pages, used, *, page_size, lengths_out=None, used_out=None):
    """Gives back the pages of every request with ``done[b]`` (bool) set.

    They go under the top of the ``free_pages`` stack, in place: request
    order, each request's in table order. Returns (lengths, used) with those
    requests' lengths zero; ``lengths_out`` and ``used_out`` may be
    ``lengths`` and ``used``; they and ``free_pages`` overlap nothing else
    that is passed. The block table is left as it is (the length says how
    much of a row counts)."""
    call = (lengths, done, block_table, free_pages, used, page_size, lengths_out, used_out)
    if _calls is not None:
        released = _calls.release(*call)
        if released.__class__ is tuple:
            return released
        if released is not None:
            _native.check(released)
    device, tail = _plan_release(*call)
    _in_place_or_apart("lengths_out", lengths_out, lengths)
    if lengths_out is None:
        lengths_out = torch.empty_like(lengths)
    if used_out is None:
        used_out = torch.empty_like(used)
    _call("nz_pages_release", struct.pack(
        "<7Q", lengths.data_ptr(), done.data_ptr(), block_table.data_ptr(), free_pages.data_ptr(), used.data_ptr(),
        lengths_out.data_ptr(), used_out.data_ptr()) + tail, device.index)
    _wrote(free_pages, *call[-2:])
    _remember(_RELEASE, call, tail)
    return lengths_out, used_out


def _plan_release(lengths, done, block_table, free_pages, used, page_size, lengths_out, used_out):
    requests = _requests(lengths)
    _vector("done", done, requests, torch.bool)
    _table(block_table, requests, False)
    _vector("free_pages", free_pages)
    _vector("used", used, 1)
    shift = _page_shift(page_size)
    if lengths_out is not None:
        _vector("lengths_out", lengths_out, requests)
    if used_out is not None:
        _vector("used_out", used_out, 1)
    device = _same_device(lengths, done, block_table, free_pages, used, lengths_out, used_out)
    return device, _pack("<Q4I", block_table.stride(0), requests, block_table.shape[1], free_pages.shape[0], shift)


def _pages(key_pages, value_pages, dtype):
    """(pages, page shift, key/value heads, width) of a cache."""
    _tensor("key_pages", key_pages, dtype, 4)
    pages, page_size, kv_heads, dim = key_pages.shape
    shift = _page_shift(page_size)
    _rows("key_pages", key_pages, key_pages.shape, dtype)
    _rows("value_pages", value_pages, key_pages.shape, dtype)
    return pages, shift, kv_heads, dim


def _dtype_code(query):
    if not isinstance(query, torch.Tensor):
        raise TypeError("query must be a tensor.")
    code = _DTYPES.get(query.dtype)
    if code is None:
        raise TypeError(f"query must be bfloat16, float16 or float32, not {query.dtype}.")
    if query.dim() != 3:
        raise ValueError(f"query must have 3 dimensions, not {query.dim()}.")
    return code


def rotary_table(inv_freq, positions, scaling=1.0):
    """The (positions, 2 * len(inv_freq)) float32 table that ``rotary_store``
    takes: cosines, then sines, of position * inv_freq, times `scaling`.
    Angles are formed in 64 bits, so that far positions keep their phase."""
    angles = torch.arange(positions, dtype=torch.float64, device=inv_freq.device)[:, None] * inv_freq.double()
    return (torch.cat([angles.cos(), angles.sin()], 1) * scaling).float()


def rotary_store(query, key, value, positions, slots, rotary, key_pages, value_pages, *, interleaved=False,
                 query_norm=None, key_norm=None, eps=1e-6, query_out=None, key_out=None):
    """Norms and rotates queries and keys and writes keys and values into the
    cache, in one pass.

    ``query`` (rows, heads, width), ``key`` and ``value`` (rows, key/value
    heads, width) may be strided views (of one fused projection, say) with a
    contiguous last dimension. Each head of query and key is first
    normalised, x * w / sqrt(mean(x^2) + eps), where ``query_norm`` /
    ``key_norm`` (width,) give the weights, then its first ``rotary.shape[1]``
    elements are rotated by the row's position: pairs (i, i + half), or
    (2i, 2i + 1) with ``interleaved``. ``rotary`` (positions, rotated width)
    holds float32 cosines, then sines (``rotary_table``). All in 32 bits,
    rounded once. Returns the rotated queries (``query_out``, which may be
    ``query``); the rotated keys also go to ``key_out`` if given.

    A row whose slot lies outside the cache (-1: padding) leaves the cache as
    it is. A position outside the table gives NaN where it would rotate. Two
    rows must not name one slot (either row's elements may end there).
    ``query_out``, ``key_out`` and the cache overlap nothing else that is
    passed."""
    interleaved = bool(interleaved)
    call = (query, key, value, positions, slots, rotary, key_pages, value_pages, interleaved, query_norm, key_norm,
            query_out, key_out, eps)
    if _calls is not None:
        out = _calls.rotary(*call)
        if out.__class__ is int:
            _native.check(out)
        if out is not None:
            return out
    _no_gradient(query, key, value, rotary, query_norm, key_norm, key_pages, value_pages, query_out, key_out)
    device, tail = _plan_rotary(*call[:-1])
    eps = _number("eps", eps)
    if query_out is None:
        query_out = torch.empty_like(query, memory_format=torch.contiguous_format)
    _call("nz_rotary_store", struct.pack(
        "<12Q", query.data_ptr(), key.data_ptr(), value.data_ptr(), query_out.data_ptr(),
        0 if key_out is None else key_out.data_ptr(), key_pages.data_ptr(), value_pages.data_ptr(),
        positions.data_ptr(), slots.data_ptr(), rotary.data_ptr(), 0 if query_norm is None else query_norm.data_ptr(),
        0 if key_norm is None else key_norm.data_ptr()) + tail + eps + bytes(4), device.index)
    _wrote(key_pages, value_pages, call[11], key_out)
    _remember(_ROTARY, call, tail)
    return query_out


def _plan_rotary(query, key, value, positions, slots, rotary, key_pages, value_pages, interleaved, query_norm, key_norm,
                 query_out, key_out):
    code = _dtype_code(query)
    dtype = query.dtype
    rows, heads, dim = query.shape
    pages, shift, kv_heads, width = _pages(key_pages, value_pages, dtype)
    if width != dim:
        raise ValueError(f"The cache's head width is {width}, the query's {dim}.")
    if not 0 < dim <= MAX_HEAD_WIDTH or dim % 2:
        raise ValueError(f"The head width must be even and at most {MAX_HEAD_WIDTH}, not {dim}.")
    _rows("query", query, query.shape, dtype)
    _rows("key", key, (rows, kv_heads, dim), dtype)
    _rows("value", value, (rows, kv_heads, dim), dtype)
    _vector("positions", positions, rows)
    _vector("slots", slots, rows)
    _tensor("rotary", rotary, torch.float32, 2)
    rot = rotary.shape[1]
    if rot > dim or rot % 2:
        raise ValueError(f"The rotated width must be even and at most the head width, not {rot}.")
    if rot > 1 and rotary.stride(1) != 1:
        raise ValueError("The last dimension of rotary must be contiguous.")
    for name, weight in (("query_norm", query_norm), ("key_norm", key_norm)):
        if weight is not None:
            _vector(name, weight, dim, dtype)
    _written("key_pages", key_pages)
    _written("value_pages", value_pages)
    out_stride, key_stride = (heads * dim, dim), (0, 0)
    if query_out is not None:
        _written("query_out", _rows("query_out", query_out, (rows, heads, dim), dtype))
        out_stride = query_out.stride()[:2]
    if key_out is not None:
        _written("key_out", _rows("key_out", key_out, (rows, kv_heads, dim), dtype))
        key_stride = key_out.stride()[:2]
    device = _same_device(query, key, value, positions, slots, rotary, key_pages, value_pages, query_norm, key_norm,
                          query_out, key_out)
    tail = _pack("<17q10I", *query.stride()[:2], *key.stride()[:2], *value.stride()[:2], *out_stride, *key_stride,
                       *key_pages.stride()[:3], *value_pages.stride()[:3], rotary.stride(0), rows, heads, kv_heads, dim,
                       rot, rotary.shape[0], pages, shift, code, bool(interleaved))
    return device, tail


def paged_attention(query, key_pages, value_pages, block_table, lengths, *, scale=None, window=None, out=None,
                    return_lse=False):
    """Attention of one new token a request over its pages of the cache.

    ``query`` (requests, heads, width); heads is a multiple of the cache's
    key/value heads, query head h reading key/value head ``h // (heads //
    kv_heads)``. Request b attends to its first ``lengths[b]`` positions (its
    own token's key and value are in the cache already), or with ``window``
    to the last ``window`` of them: ``softmax(scale * q k^T) v``, statistics
    and sums in 32 bits, ``scale`` defaulting to width ** -0.5. With
    ``return_lse`` also returns the float32 (requests, heads) logarithm of
    each softmax's denominator. ``out`` overlaps no input. A request with nothing to attend to gets
    zeros and -inf.

    Positions a request does not attend to are not read, whatever they hold;
    attended queries, keys and values have to be finite. A length is held to
    what the block table's row can hold; a page id outside the cache is not
    read and its positions count as masked. The head width is a multiple of
    8 up to 256 and cache rows start on 16-byte boundaries."""
    call = (query, key_pages, value_pages, block_table, lengths, window, out, scale, return_lse)
    if _calls is not None:
        done = _calls.attention(*call)
        if done.__class__ is int:
            _native.check(done)
        if done is not None:
            return done
    _no_gradient(query, key_pages, value_pages, out)
    device, workspace_bytes, tail = _plan_attention(query, key_pages, value_pages, block_table, lengths, window, out)
    default = query.shape[2] ** -0.5
    factor = _number("scale", default if scale is None else scale)
    if out is None:
        out = torch.empty_like(query, memory_format=torch.contiguous_format)
    lse = torch.empty(query.shape[:2], dtype=torch.float32, device=device) if return_lse else None
    workspace = torch.empty(workspace_bytes, dtype=torch.uint8, device=device) if workspace_bytes else None
    _call("nz_paged_attention", struct.pack(
        "<8Q", query.data_ptr(), key_pages.data_ptr(), value_pages.data_ptr(), block_table.data_ptr(), lengths.data_ptr(),
        out.data_ptr(), 0 if lse is None else lse.data_ptr(), 0 if workspace is None else workspace.data_ptr()) + tail
        + factor, device.index)
    _wrote(call[6])
    _remember(_ATTENTION, call, tail, workspace_bytes, default)
    return (out, lse) if return_lse else out


def _plan_attention(query, key_pages, value_pages, block_table, lengths, window, out):
    code = _dtype_code(query)
    dtype = query.dtype
    requests, heads, dim = query.shape
    pages, shift, kv_heads, width = _pages(key_pages, value_pages, dtype)
    if width != dim:
        raise ValueError(f"The cache's head width is {width}, the query's {dim}.")
    if not 0 < dim <= MAX_HEAD_WIDTH or dim % 8:
        raise ValueError(f"The head width must be a multiple of 8 up to {MAX_HEAD_WIDTH}, not {dim}.")
    if not kv_heads or not heads or heads % kv_heads:
        raise ValueError(f"{heads} query heads are no multiple of {kv_heads} key/value heads.")
    if _requests(lengths) != requests:
        raise ValueError(f"lengths must have {requests} elements, not {lengths.shape[0]}.")
    _rows("query", query, query.shape, dtype)
    _table(block_table, requests, False)
    for name, cache in (("key_pages", key_pages), ("value_pages", value_pages)):
        steps = [stride for stride, size in zip(cache.stride()[:3], cache.shape) if size > 1]
        if cache.data_ptr() % 16 or any(step * cache.element_size() % 16 for step in steps):
            raise ValueError(f"The rows of {name} must start on 16-byte boundaries.")
    window = 0 if window is None else min(_whole("window", window, 1, 2 ** 63), 2 ** 31 - 1)
    out_stride = (heads * dim, dim)
    if out is not None:
        _written("out", _rows("out", out, (requests, heads, dim), dtype))
        out_stride = out.stride()[:2]
    device = _same_device(query, key_pages, value_pages, block_table, lengths, out)
    strides = (*query.stride()[:2], *out_stride, *key_pages.stride()[:3], *value_pages.stride()[:3],
               block_table.stride(0))
    tail = _pack("<11q9I", *strides, requests, heads, kv_heads, dim, pages, shift, block_table.shape[1], window,
                       code)
    need = ctypes.c_uint64()
    with torch.cuda.device(device):
        _native.check(_native.load().nz_paged_attention_workspace(bytes(64) + tail + bytes(4), ctypes.byref(need)))
    return device, need.value, tail
