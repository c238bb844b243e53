"""A paged key/value cache for serving: the plan of a step, the write of its
heads, the attention over the cache, the weight that keys receive in it and the eviction by that weight, on the
kernels of ``csrc/paged_cache.hip``, ``csrc/paged_attention.hip``, ``csrc/paged_weights.hip`` and
``csrc/paged_evict.hip``. The reference keeps no cache; these stand
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

from . import _lib

__all__ = ["PagedPlan", "paged_plan", "paged_write", "paged_attention", "paged_key_weights", "paged_evict", "PAGED_OK", "PAGED_BAD_LENGTH",
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
    * ``slots`` int64 [tokens]: ``page * page_size + offset`` of each row, -1 for rows of no admitted
      request, and where the free list gave a number that is no page of the cache.
    * ``pages_used`` int32 [1]: how many free pages were taken, from the list's front.
    * ``pages_needed`` int32 [1]: how many the requests up to the last admitted one need together,
      admitted or not; more than the list holds once it ran out.

    It also holds the step's ``block_tables`` and sizes. One plan serves all layers of its step."""

    __slots__ = ("starts", "rows", "context", "status", "positions", "slots", "pages_used", "pages_needed",
                 "block_tables", "page_size", "num_pages", "max_new", "max_context", "requests", "tokens", "_native")

    def __repr__(self):
        return (f"PagedPlan(requests={self.requests}, tokens={self.tokens}, page_size={self.page_size}, "
                f"num_pages={self.num_pages}, max_new={self.max_new}, max_context={self.max_context})")


def paged_plan(context_lens, new_lens, block_tables, *, page_size, num_pages, tokens, free_pages=None, max_new=None,
               max_context=None):
    """Lay out one step on the device: request ``b`` holds ``context_lens[b]``
    tokens and appends ``new_lens[b]`` (0: it sits the step out).

    ``block_tables`` int32 ``[requests, width]`` names each request's pages. With
    ``free_pages`` (int32, distinct numbers of the cache's pages) the requests take the pages that they
    need, ``ceil((context + new) / page_size) - ceil(context / page_size)`` each, from its front in
    request order, and their entries are written into ``block_tables`` (which shares no memory
    with the other arguments); without, every page must be there already. ``tokens`` is the step's number of rows
    (the new tokens and any padding behind them); ``max_new`` and ``max_context``
    bound the new tokens of a request and its tokens in all, where a program knows
    them (default: ``tokens``, and what the tables hold). ``paged_attention`` picks its kernel by ``max_new``:
    say 1 of a decode step, which else runs in the tiles of a prompt (64 requests: 248 us, not 205).

    A request whose lengths break these bounds, whose rows do not fit, whose pages ran
    out, or whose table does not name the page that its context ends in (without ``free_pages``: any
    page that its new tokens go to) is not admitted: ``status`` says why, its table stays as it was, nothing of it is
    written and its rows of an attention are zero. Its rows keep their place. A request that
    needs no new page is admitted though others before it ran out.
    """
    plan = PagedPlan()
    (plan._native, plan.requests, plan.max_new, plan.max_context, plan.starts, plan.rows, plan.context, plan.status,
     plan.positions, plan.slots, plan.pages_used, plan.pages_needed) = _lib.host().plan(
         context_lens, new_lens, block_tables, page_size, num_pages, tokens, free_pages, max_new, max_context)
    plan.block_tables, plan.page_size, plan.num_pages, plan.tokens = block_tables, page_size, num_pages, tokens
    return plan


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
    zero in the result. The heads share no memory with the cache, nor the cache's keys and values with each
    other."""
    return _lib.host().write(k, v, k_cache, v_cache, plan._native, q, rope_cos, rope_sin, q_scale, k_scale, eps)


def paged_attention(q, k_cache, v_cache, plan, *, scale=None, window=None, out=None, lse=None):
    """Causal grouped-query attention of a step's new tokens ``q`` ``[tokens, heads, head_dim]``
    over the cache, the step's own keys and values (``paged_write``) among it: the row at
    position p of its request sees that request's positions 0 .. p, with ``window``
    only the last ``window`` of them. ``scale`` defaults to ``head_dim ** -0.5``.

    Softmax in FP32; its weights are rounded to bf16 for the product with the values, and
    the result once. Keys of table entries that are no page of the cache are not seen; a row
    that sees none is zero (one all of whose scores are -inf is NaN). Infinities and NaN in the cache
    reach the rows that see them and no others. Rows of no admitted request are zero in a new result, and left as they
    were in ``out`` (bf16 ``[tokens, heads, head_dim]``, rows 16-byte aligned). ``out`` may be ``q``; else its rows
    share memory neither with each other nor with ``q`` or the cache.

    ``lse`` float32 ``[tokens, heads]``, contiguous and of memory of its own, receives the logarithm of each row's
    sum of exponentials, for ``paged_key_weights``: -inf for a row that sees no key or whose scores are all
    -inf. Rows of no admitted request are left as they were."""
    return _lib.host().attention(q, k_cache, v_cache, plan._native, scale, window, out, lse)


def paged_key_weights(q, k_cache, key_weights, plan, lse, *, scale=None, window=None):
    """Add the attention weight that each cached key receives in a step to ``key_weights``
    float32 ``[pages, kv_heads, page_size]`` (contiguous), in place::

        out = paged_attention(q, k_cache, v_cache, plan, lse=lse)
        paged_key_weights(q, k_cache, key_weights, plan, lse)

    A key receives ``exp(scale q . k - lse)``, its softmax weight, from every row that sees it and
    every query head of its key/value head. The step's own keys start from zero, so that slots of
    reused pages need no clearing, as long as every step that writes keys is followed by this call. ``q``, ``scale``
    and ``window`` are those of the attention that gave ``lse``. Scores and sums in FP32, in an order that depends on the
    lengths alone. Slots that hold no key of an admitted request stay as they were, as do those of table entries that
    are no page of the cache. Requests must not share pages. ``key_weights`` shares no memory with the other tensors."""
    _lib.host().key_weights(q, k_cache, key_weights, plan._native, lse, scale, window)


def paged_evict(k_cache, v_cache, key_weights, context_lens, block_tables, keep, *, recent=0, max_context=None):
    """Cut requests of more than ``keep`` cached tokens (``context_lens`` int32 ``[requests]``) down to
    ``keep``, a number or an int32 tensor of one for each request, in place, and return the
    lengths that the cache then holds (int32 ``[requests]``).

    Each key/value head keeps the last ``min(recent, keep)`` tokens and, of those before, the ones
    with the largest ``key_weights`` (``paged_key_weights``; equal ones: the lowest index, NaN counts as
    the largest). Keys, values and weights then lie at the request's indices 0 .. keep - 1, those
    kept for their weight first, the recent ones behind them in their order: a survivor whose index is below ``keep -
    min(recent, keep)`` stays, the j-th place that became free below it takes the j-th survivor from behind. So heads hold
    different tokens at an index, and the index no longer says a token's position: rotate new heads by
    positions of your own (``rotary``), and attend without a window. Every layer's cache is cut by a call of its
    own, with the same ``block_tables`` and lengths.

    A request is left as it was, and its length returned, if it holds ``keep`` tokens or fewer, if a
    length is negative or above ``max_context`` (default: what the tables hold), or if a table entry of its tokens is no page of
    the cache. ``max_context`` sizes the call's workspace, about 5 bytes a token and head, and picks its kernels: where tables
    hold far more than the requests do, a bound near their lengths is faster (eight requests cut from 1040 tokens to 1024: 11 us
    by a bound of 1040, 23 by that of tables for 131,072). ``block_tables`` is not
    changed: pages behind the last kept token stay the request's, for its next tokens or for the program to
    take back. Requests must not share pages."""
    return _lib.host().evict(k_cache, v_cache, key_weights, context_lens, block_tables, keep, recent, max_context)
