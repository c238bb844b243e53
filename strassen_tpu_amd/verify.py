"""Verification of drafted tokens in a serving step, on the kernels of ``csrc/verify.hip``.

A request with drafts appends its last token and the drafts as the new tokens of one step (``paged_plan``); the
model's probabilities of the tokens behind them say which drafts stay."""

from __future__ import annotations

from . import _lib

__all__ = ["verify_drafts"]


def verify_drafts(target, tokens, plan, accept, sample, *, draft=None):
    """Accept or replace the drafts of a step, so that what a request emits is distributed as if drawn from ``target``::

        plan = paged_plan(context_lens, drafts + 1, block_tables, ...)
        ...                                     # the model's step
        emitted, counts = verify_drafts(probabilities, tokens, plan, accept, sample, draft=draft)
        context_lens += counts                  # the refused drafts' keys are overwritten by the next step

    ``tokens [plan.tokens]`` (int32 or int64) are the rows' tokens. Row ``i`` of ``target [plan.tokens, vocab]``
    (float32 or bf16) holds the model's probabilities of the token behind row ``i``, row ``i`` of ``draft`` (like ``target``)
    those that the draft behind row ``i`` was drawn from; the last row of a request in ``draft`` is not read. Without ``draft``
    the drafts were not drawn (looked up, or a smaller model's best): their own probability counts as 1.

    ``accept [plan.tokens]`` and ``sample [requests]`` (float32) are independent random numbers, uniform in [0, 1). The draft
    ``x`` behind row ``i`` is accepted if ``accept[i] * draft[i, x] < target[i, x]`` and those before it were. The next token
    is drawn from ``max(target - draft, 0)`` of the row whose draft was refused (from ``target`` where that is zero everywhere),
    or from ``target`` of the last row: the first token whose running sum exceeds ``sample`` times the whole. Products and sums
    are in 64 bits: the same call gives the same tokens, and a request in calls of other sizes (whose sums go in another
    order) the same but for numbers within the rounding of such sums, 2^-50 or so of the whole, of a border between two
    tokens. Probabilities need not add up to 1, and such as are no positive finite numbers count as zero (a draft outside the
    vocabulary too).

    Returns ``emitted [plan.tokens]`` (as ``tokens``) with each request's accepted drafts and its next token from its first
    row on, -1 behind them and in rows of no admitted request, and ``counts`` int32 ``[requests]``: how
    many were emitted, 0 for requests without rows. A row without any probability emits -1."""
    return _lib.host().verify(target, tokens, plan._native, accept, sample, draft)
