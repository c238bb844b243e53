"""A paged key/value cache for serving: the plan of a step, the write of its
heads and the attention over the cache, on the kernels of ``csrc/paged_cache.hip``
and ``csrc/paged_attention.hip``. The reference keeps no cache; these stand
beside ``qwen3_block.attention``, which attends within one batch of whole
sequences.

A layer's cache is two bf16 tensors ``[pages, page_size, kv_heads, head_dim]``
of the same strides. A step appends new tokens to requests, one row each,
request behind request, with padding rows at the end. One plan serves every
layer of the step::

    plan = paged_plan(context_lens, new_lens, block_tables, page_size=16, num_pages=pages,
                      tokens=rows, free_pages=free)
    for layer in layers:
        q = paged_write(k, v, k_cache, v_cache, plan, q=q, rope_cos=cos, rope_sin=sin)
        out = paged_attention(q, k_cache, v_cache, plan)

Everything runs on torch's current stream of the tensors' device, reads no length back
to the host and can be captured in a graph, which is replayed after the lengths, the
tables and the heads changed in place.
"""

from __future__ import annotations

import ctypes
import functools
import math

import torch

from . import _lib

__all__ = ["PagedPlan", "paged_plan", "paged_write", "paged_attention", "PAGED_OK", "PAGED_BAD_LENGTH",
           "PAGED_OUT_OF_ROWS", "PAGED_OUT_OF_PAGES", "PAGED_BAD_PAGE"]

# What a plan's status says of a request.
PAGED_OK, PAGED_BAD_LENGTH, PAGED_OUT_OF_ROWS, PAGED_OUT_OF_PAGES, PAGED_BAD_PAGE = range(5)


class PagedPlan:
    """Rows, positions and slots of one step (``paged_plan``); tensors on the device.

    * ``starts`` int32 [requests + 1]: the first row of each request.
    * ``rows``, ``context`` int32 [requests]: new tokens and tokens before them, 0 for
      requests that are not admitted.
    * ``status`` int32 [requests]: ``PAGED_OK`` or why a request is not admitted.
    * ``positions`` int32 [tokens]: each row's position, -1 for rows of no admitted request.
    * ``slots`` int64 [tokens]: ``page * page_size + offset`` of each row, -1 where
      there is no page.
    * ``pages_used`` int32 [1]: how many free pages were taken, from the list's front.
    * ``pages_needed`` int32 [1]: how many the requests up to the last admitted one need together,
      admitted or not; more than the list holds once it ran out.

    It also holds the step's ``block_tables`` and sizes. One plan serves all layers of its step."""

    __slots__ = ("starts", "rows", "context", "status", "positions", "slots", "pages_used", "pages_needed",
                 "block_tables", "page_size", "num_pages", "max_new", "max_context", "requests", "tokens", "device",
                 "_positions", "_slots", "_step")

    def __repr__(self):
        return (f"PagedPlan(requests={self.requests}, tokens={self.tokens}, page_size={self.page_size}, "
                f"num_pages={self.num_pages}, max_new={self.max_new}, max_context={self.max_context})")


def _check_device(name, x, device=None):
    if not isinstance(x, torch.Tensor):
        raise TypeError(f"{name} must be a tensor, got {type(x).__name__}")
    if device is None or x.device != device:
        if not x.is_cuda:
            raise ValueError(f"the gfx950 kernel needs tensors on the HIP device (got {name} on {x.device})")
        if device is not None:
            raise ValueError(f"{name} is on {x.device}, the call on {device}")


# The stream's handle itself: torch.cuda.current_stream makes an object of it first, which takes as long as
# the launch of a decode step's kernel.
_raw_stream = torch._C._cuda_getCurrentRawStream


def _call(device, function, *args):
    """One library call on the device's current stream."""
    if torch.cuda.current_device() == device.index:
        rc = function(*args, _raw_stream(device.index))
    else:
        with torch.cuda.device(device):
            rc = function(*args, _raw_stream(device.index))
    if rc:
        _lib.check(rc)


def _int32(name, x, shape):
    if x.dtype != torch.int32 or tuple(x.shape) != shape or not x.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 tensor of shape {shape}, got {x.dtype} {tuple(x.shape)}")


def paged_plan(context_lens, new_lens, block_tables, *, page_size, num_pages, tokens, free_pages=None, max_new=None,
               max_context=None):
    """Lay out one step on the device: request ``b`` holds ``context_lens[b]``
    tokens and appends ``new_lens[b]`` (0: it sits the step out).

    ``block_tables`` int32 ``[requests, width]`` names each request's pages. With
    ``free_pages`` (int32, distinct page numbers) the requests take the pages that they
    need, ``ceil((context + new) / page_size) - ceil(context / page_size)`` each, from its front in
    request order, and their entries are written into ``block_tables``; without,
    every page must be there already. ``tokens`` is the step's number of rows
    (the new tokens and any padding behind them); ``max_new`` and ``max_context``
    bound the new tokens of a request and its tokens in all, where a program knows
    them (default: ``tokens``, and what the tables hold).

    A request whose lengths break these bounds, whose rows do not fit or whose pages ran
    out is not admitted: ``status`` says why, its table stays as it was, nothing of it is
    written and its rows of an attention are zero. Its rows keep their place. A request that
    needs no new page is admitted though others before it ran out.
    """
    _check_device("context_lens", context_lens)
    device = context_lens.device
    if context_lens.dim() != 1 or not context_lens.shape[0]:
        raise ValueError("context_lens must hold one length per request")
    requests, tokens = context_lens.shape[0], int(tokens)
    _int32("context_lens", context_lens, (requests,))
    _check_device("new_lens", new_lens, device)
    _int32("new_lens", new_lens, (requests,))
    _check_device("block_tables", block_tables, device)
    if block_tables.dtype != torch.int32 or block_tables.dim() != 2 or block_tables.shape[0] != requests \
            or not block_tables.shape[1] or block_tables.stride(1) != 1 \
            or block_tables.stride(0) < block_tables.shape[1]:
        raise ValueError(f"block_tables must be int32 [{requests}, width] with rows apart from each other, got "
                         f"{block_tables.dtype} {tuple(block_tables.shape)}")
    free_count, free = 0, None
    if free_pages is not None:
        _check_device("free_pages", free_pages, device)
        if free_pages.dim() != 1:
            raise ValueError("free_pages must be a list of page numbers")
        _int32("free_pages", free_pages, (free_pages.shape[0],))
        # an empty list too is a list: no request gets a new page
        free_count = free_pages.shape[0]
        free = free_pages.data_ptr() if free_count else new_lens.data_ptr()
    plan = PagedPlan()
    plan.block_tables, plan.page_size, plan.num_pages = block_tables, int(page_size), int(num_pages)
    plan.requests, plan.tokens, plan.device = requests, tokens, device
    width = block_tables.shape[1]
    plan.max_new = tokens if max_new is None else int(max_new)
    plan.max_context = min(width * plan.page_size, _lib.SMX_PAGED_MAX_CONTEXT) if max_context is None else int(max_context)
    # one allocation for the small tensors: slots (int64) first, then the int32 ones
    sizes = (2 * max(tokens, 1), requests + 1, requests, requests, requests, max(tokens, 1), 1, 1)
    memory = context_lens.new_empty(sum(sizes))
    (slots, plan.starts, plan.rows, plan.context, plan.status, plan.positions, plan.pages_used,
     plan.pages_needed) = memory.split_with_sizes(sizes)
    plan.slots = slots.view(torch.int64)
    at = plan._slots = memory.data_ptr()
    starts = at + 4 * sizes[0]
    rows = starts + 4 * sizes[1]
    context = rows + 4 * requests
    status = context + 4 * requests
    positions = plan._positions = status + 4 * requests
    tables, stride = block_tables.data_ptr(), block_tables.stride(0)
    _call(device, _lib.load().smx_paged_plan, requests, width, plan.page_size, plan.num_pages, tokens, plan.max_new,
          plan.max_context, context_lens.data_ptr(), new_lens.data_ptr(), tables, stride, free, free_count, starts,
          rows, context, positions, at, status, positions + 4 * sizes[5])
    plan._step = _lib.SmxPagedStep(requests, tokens, plan.max_new, tables, stride, starts, rows, context, positions)
    return plan


def _cache(k_cache, v_cache, plan):
    """The cache's description for the library; ``plan`` fixes its pages."""
    for name, x in (("k_cache", k_cache), ("v_cache", v_cache)):
        _check_device(name, x, plan.device)
        if x.dtype != torch.bfloat16 or x.dim() != 4:
            raise ValueError(f"{name} must be a bf16 tensor [pages, page_size, kv_heads, head_dim], got {x.dtype} "
                             f"{tuple(x.shape)}")
    shape = k_cache.shape
    if v_cache.shape != shape:
        raise ValueError("k_cache and v_cache must have the same shape and strides")
    strides = k_cache.stride()
    if 1 in shape:  # the stride of a dimension of one is no stride: nothing steps over it
        strides, other = (tuple(s if n > 1 else shape[3] for s, n in zip(x.stride(), shape[:3])) + x.stride()[3:]
                          for x in (k_cache, v_cache))
    else:
        other = v_cache.stride()
    if strides != other:
        raise ValueError("k_cache and v_cache must have the same shape and strides")
    pages, page_size, kv_heads, head_dim = shape
    if page_size != plan.page_size or pages != plan.num_pages:
        raise ValueError(f"the plan is of {plan.num_pages} pages of {plan.page_size} tokens, the cache of {pages} of "
                         f"{page_size}")
    if strides[3] != 1:
        raise ValueError("cache heads must be contiguous runs")
    return _lib.SmxPagedCache(k_cache.data_ptr(), v_cache.data_ptr(), strides[0], strides[1], strides[2], pages,
                              page_size, kv_heads, head_dim)


def _heads(name, x, plan, heads, head_dim, lay_out=True):
    """Head rows ``[tokens, heads, head_dim]`` for the library; rows that it cannot take as they lie
    (not 16-byte aligned runs) are laid out first, or refused."""
    _check_device(name, x, plan.device)
    shape = x.shape
    if x.dtype != torch.bfloat16 or len(shape) != 3 or shape[0] != plan.tokens or shape[2] != head_dim \
            or (heads is not None and shape[1] != heads):
        raise ValueError(f"{name} must be a bf16 tensor of shape {(plan.tokens, heads or 'heads', head_dim)}, got "
                         f"{x.dtype} {tuple(shape)}")
    token, head, unit = x.stride()
    # the stride of a dimension of one is no stride: nothing steps over it
    token, head, at = token if shape[0] > 1 else 0, head if shape[1] > 1 else 0, x.data_ptr()
    if unit != 1 or token % 8 or head % 8 or at % 16:
        if not lay_out:
            raise ValueError(f"{name} rows must be 16-byte aligned runs")
        x = x.clone(memory_format=torch.contiguous_format)
        token, head, at = shape[1] * head_dim, head_dim, x.data_ptr()
    return x, _lib.SmxHeads(at, token, head, shape[1])


def _no_gradients(*tensors):
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise ValueError("serving operators record no gradients: call them under torch.no_grad()")


def _scale(name, x, plan, head_dim):
    if x is None:
        return None
    _check_device(name, x, plan.device)
    if tuple(x.shape) != (head_dim,):
        raise ValueError(f"{name} must have shape {(head_dim,)}, got {tuple(x.shape)}")
    return _aligned(x if x.dtype in (torch.bfloat16, torch.float32) else x.float())


def _aligned(x):
    """``x``, contiguous and 16-byte aligned (laid out anew where it is not)."""
    if x.is_contiguous() and x.data_ptr() % 16 == 0:
        return x
    return x.clone(memory_format=torch.contiguous_format)


def paged_write(k, v, k_cache, v_cache, plan, *, q=None, rope_cos=None, rope_sin=None, q_scale=None, k_scale=None,
                eps=1e-6):
    """Store a step's keys and values ``[tokens, kv_heads, head_dim]`` in the cache at the
    plan's slots, and return the query heads ``q`` ready for ``paged_attention``
    (None without ``q``).

    ``q_scale`` / ``k_scale`` ``[head_dim]`` RMS-normalise the query and key heads (``eps``) and
    ``rope_cos`` / ``rope_sin`` rotate them: rows by position, at least
    ``plan.max_context`` of them, ``head_dim // 2`` values wide (or ``head_dim``, of which
    the first half is read), bf16 or float32. All of it is computed in FP32 and rounded to
    bf16 once. Heads that come normalised and rotated from the ``qk_norm_rope``
    epilogue are stored without these. Rows of no admitted request are not stored and
    zero in the result."""
    _no_gradients(k, v, q, k_cache, v_cache)
    cache = _cache(k_cache, v_cache, plan)
    head_dim = cache.head_dim
    k, k_rows = _heads("k", k, plan, cache.kv_heads, head_dim)
    v, v_rows = _heads("v", v, plan, cache.kv_heads, head_dim)
    if (rope_cos is None) != (rope_sin is None):
        raise ValueError("rope_cos= and rope_sin= go together")
    out = q_rows = None
    if q is None:
        if q_scale is not None:
            raise ValueError("q_scale= without q=")
    else:
        q, q_rows = _heads("q", q, plan, None, head_dim)
        out = q.new_empty(q.shape)
    dtypes = rope_rows = rope_stride = 0
    if rope_cos is not None:
        for name, x in (("rope_cos", rope_cos), ("rope_sin", rope_sin)):
            _check_device(name, x, plan.device)
            if x.dim() != 2 or x.shape[1] not in (head_dim // 2, head_dim) or x.shape != rope_cos.shape:
                raise ValueError(f"{name} must have rows of {head_dim // 2} or {head_dim} values, got "
                                 f"{tuple(x.shape)}")
            if x.shape[0] < plan.max_context:
                raise ValueError(f"{name} holds {x.shape[0]} positions, the plan's requests up to "
                                 f"{plan.max_context}")
        if not (rope_cos.dtype == rope_sin.dtype and rope_cos.dtype in (torch.bfloat16, torch.float32)):
            raise ValueError("RoPE tables must both be bf16 or float32")
        rope_cos, rope_sin = _aligned(rope_cos), _aligned(rope_sin)
        rope_rows, rope_stride = min(rope_cos.shape[0], 2**31 - 1), rope_cos.shape[1]
        dtypes |= _lib.SMX_PAGED_ROPE_F32 if rope_cos.dtype == torch.float32 else 0
    q_scale, k_scale = _scale("q_scale", q_scale, plan, head_dim), _scale("k_scale", k_scale, plan, head_dim)
    if q_scale is not None and q_scale.dtype == torch.float32:
        dtypes |= _lib.SMX_PAGED_Q_SCALE_F32
    if k_scale is not None and k_scale.dtype == torch.float32:
        dtypes |= _lib.SMX_PAGED_K_SCALE_F32
    _call(plan.device, _lib.load().smx_paged_write, cache, plan.tokens, plan._positions, plan._slots, q_rows,
          k_rows, v_rows, _lib.ptr(rope_cos), _lib.ptr(rope_sin), rope_rows, rope_stride, _lib.ptr(q_scale),
          _lib.ptr(k_scale), dtypes, float(eps), _lib.ptr(out))
    return out


@functools.lru_cache(maxsize=64)
def _workspace_bytes(device, head_dim):
    need = ctypes.c_int64()
    with torch.cuda.device(device):
        _lib.check(_lib.load().smx_paged_attention_workspace_bytes(head_dim, ctypes.byref(need)))
    return need.value


def paged_attention(q, k_cache, v_cache, plan, *, scale=None, window=None, out=None):
    """Causal grouped-query attention of a step's new tokens ``q`` ``[tokens, heads, head_dim]``
    over the cache, the step's own keys and values (``paged_write``) among it: the row at
    position p of its request sees that request's positions 0 .. p, with ``window``
    only the last ``window`` of them. ``scale`` defaults to ``head_dim ** -0.5``.

    Softmax in FP32; its weights are rounded to bf16 for the product with the values, and
    the result once. Keys of table entries that are no page of the cache are not seen; a row
    that sees none is zero. A request's values must be finite up to its last token: one that is
    not spoils rows of the step that do not see it, too. (Nothing behind that token is
    read.) Rows of no admitted request are zero in a new result, and left as they
    were in ``out`` (bf16 ``[tokens, heads, head_dim]``, rows 16-byte aligned)."""
    _no_gradients(q, k_cache, v_cache, out)
    cache = _cache(k_cache, v_cache, plan)
    head_dim = cache.head_dim
    q, q_rows = _heads("q", q, plan, None, head_dim)
    if scale is None:
        scale = head_dim ** -0.5
    if not (math.isfinite(scale) and scale > 0):
        raise ValueError(f"scale must be positive and finite, got {scale}")
    if window is None:
        window = 0
    elif not isinstance(window, int) or not 0 < window < 2**31:
        raise ValueError(f"window must be a positive number of tokens, got {window!r}")
    zero_rows = out is None
    if zero_rows:
        out = q.new_empty(q.shape)
    _, out_rows = _heads("out", out, plan, q.shape[1], head_dim, lay_out=False)
    need = _workspace_bytes(plan.device, head_dim)
    workspace = torch.empty(need, dtype=torch.uint8, device=plan.device)
    _call(plan.device, _lib.load().smx_paged_attention, cache, plan._step, q_rows, out_rows, float(scale), window,
          zero_rows, workspace.data_ptr(), need)
    return out
