"""Generation from a paged key-value cache: the tokens of many sequences in pages that are given out and taken back.

The reference computes attention over whole key and value arrays (ring.py:246-325); a program that generates with such a
model keeps them for many sequences of different lengths, which come, grow by a token a step and end.  Here they lie in a pool
``[pages, page_size, kv_heads, d]`` for keys and one for values (any strides with the last dimension contiguous), and row b of
``block_table`` names the pages of sequence b in order.  A step of a model is

    slots, starts, lengths, free_state = page_slots(block_table, lengths, new_lengths, free_pages, free_state, page_size, num_tokens)
    ...                                                                             # in each layer:
    write_pages(k, v, k_pages, v_pages, slots)                                      # k, v: [num_tokens, kv_heads, d]
    out = paged_attention(q, k_pages, v_pages, block_table, lengths)                # q: [sequences, heads, d], a token each

(a prompt's own attention is ``ring_attention``'s), and with a cache that is too long to be read whole

    page_means(k_pages, block_table, lengths_before, lengths, means)
    pages = select_pages(q, means, block_table, lengths, page_size, count)
    out = paged_attention(q, k_pages, v_pages, block_table, lengths, pages=pages)

Lengths, tables and the pool's state live on the GPU, nothing here waits for it, and every call can be captured into a graph: what the arrays on
the device hold when it is replayed counts.  None of them has a gradient.  What is on the device is not trusted: lengths are cut to what a row of the
table can name, and pages and slots that are not in the pool take no part.  ``page_size`` is a power of two from 16 on, ``d`` 32, 64,
96 or 128, up to 4096 sequences take part in a call.  Everything runs through ``libringattn_hip.so``.
"""
from __future__ import annotations

import math
from typing import Optional

import torch

from . import _lib
from .bias import BiasFn


def page_slots(block_table, lengths, new_lengths, free_pages, free_state, page_size: int, num_tokens: int):
    """Gives pages to the sequences that grow from ``lengths`` to ``new_lengths`` tokens, takes them back from those that shrink or end (0), and
    says where the new tokens go.

    Args:
        block_table: int32 ``[sequences, width]``, rows contiguous; entries of new pages are written, others left.  A page belongs to one row here:
            of rows that name the same page (which attention allows) one at most may end or shrink below it, or it is given back twice.
        lengths, new_lengths: int32 ``[sequences]``.  (A row that ends and takes a new sequence at once goes through 0 in a call of its own.)
        free_pages: int32 ``[pages]``, a ring: from place ``free_state[0]`` on, around its end, ``free_state[1]`` pages are free.  To
            begin with ``arange(pages)`` and ``(0, pages)``.  Pages given back are written behind the free ones.
        free_state: int32 ``[2]``.
        num_tokens: the length of ``slots``; a captured step has one that is large enough for every replay.
    Returns:
        ``slots`` int64 ``[num_tokens]``, ``page * page_size + place`` of each new token, sequence after sequence: -1 for one that has no
        page and behind the last;
        ``starts`` int32 ``[sequences + 1]``, where the tokens of each sequence begin in it;
        ``lengths`` int32 ``[sequences]`` to go on with: the new ones, cut to what there were pages for (pages go out in the order of the
        sequences; those given back by a call are there for the next one);
        ``free_state`` to go on with.
    """
    return _lib.host().page_slots(block_table, lengths, new_lengths, free_pages, free_state, page_size, num_tokens)


def write_pages(k, v, k_pages, v_pages, slots) -> None:
    """Writes keys and values ``[tokens, kv_heads, d]`` (bfloat16, float16 or float32, any strides) to their ``slots`` (int64) of the
    pools, rounded to the pools' type.  A token with a slot outside of the pools is left out.  A slot may occur once: of two tokens
    with the same one either may be what remains."""
    _lib.host().write_pages(k, v, k_pages, v_pages, slots)


def page_means(k_pages, block_table, lengths, new_lengths, means) -> None:
    """Makes ``means`` ``[pages, kv_heads, d]`` (of the pool's type) again for the pages whose tokens changed as the sequences went from
    ``lengths`` to ``new_lengths``: the mean of the keys that a page holds, summed in 32 bits and rounded once.  After ``write_pages``."""
    _lib.host().page_means(k_pages, block_table, lengths, new_lengths, means)


def select_pages(q, means, block_table, lengths, page_size: int, count: int, first: int = 1, last: int = 1) -> torch.Tensor:
    """The pages that a token is to attend to, by a score that reads one vector a page.

    The query heads that share a head of the cache share its pages too: a page's score is the sum of their queries times the page's
    mean key, in 64 bits.  Of each sequence the ``first`` and the ``last`` pages and, of the others, those with the largest scores are chosen
    (of equal ones the lowest), ``count`` in all.  A mean that is not a number ranks before all numbers, and a page that is not in
    the pool behind all pages that are.

    Returns int32 ``[sequences, kv_heads, count]``, numbers of pages within their sequence, in order; a sequence of fewer pages has all
    of them, and -1 behind."""
    return _lib.host().select_pages(q, means, block_table, lengths, page_size, count, first, last)


def paged_attention_with_lse(q, k_pages, v_pages, block_table, lengths, bias_fn: Optional[BiasFn] = None, sm_scale: Optional[float] = None,
                             pages: Optional[torch.Tensor] = None):
    """``paged_attention`` that also returns the logsumexp ``[sequences, heads]``, float32."""
    window, slopes = 0, None
    if bias_fn is not None:
        if not isinstance(bias_fn, BiasFn) or bias_fn.segments or bias_fn.prefix or bias_fn.relative is not None:
            raise ValueError("attention over a paged cache takes causal, sliding-window and ALiBi terms only (a ring_attention.BiasFn of them)")
        window, slopes = bias_fn.window or 0, bias_fn.alibi_slopes
        window = min(window, 1 << 30)  # (wider than any sequence)
        if slopes is not None and slopes.is_cuda and slopes.device != q.device:
            slopes = slopes.to(q.device)
    return _lib.host().paged_attention(q, k_pages, v_pages, block_table, lengths, pages, slopes, window,
                                       1.0 / math.sqrt(q.shape[-1]) if sm_scale is None else sm_scale)


def paged_attention(q, k_pages, v_pages, block_table, lengths, bias_fn: Optional[BiasFn] = None, sm_scale: Optional[float] = None,
                    pages: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of one token per sequence, its last one, over the sequence's tokens in the pool, its own among them.

    Args:
        q: ``[sequences, heads, d]`` of the pools' type; ``heads`` is a multiple of ``kv_heads``, and heads ``h * heads / kv_heads`` up
            to the next share head h of the cache.
        k_pages, v_pages: ``[pages, page_size, kv_heads, d]``, bfloat16 or float16.
        block_table, lengths: int32 ``[sequences, width]`` and ``[sequences]``.  A row of length 0 has an output of zeros and a logsumexp
            of -inf.  Several tokens of one sequence are several rows with the same pages, each with its own length.
        bias_fn: ``sliding_window_bias(w)`` (pages outside of it are not read), ``alibi_bias(slopes)``, their sum, ``causal_bias()``.  Slopes on the
            host (``alibi_slopes``) go along with a small kernel of each call, without waiting, and are what they are when the call is made or
            captured; slopes on the device save that kernel, and slopes on another device are copied, which cannot be captured.
        sm_scale: softmax scale, 1/sqrt(d) if unspecified.
        pages: int32 ``[sequences, kv_heads, count]``, the pages of each sequence that are read (``select_pages``), each at most once. Of a
            sequence of n pages the first n entries count; numbers that are no pages are left out.
    Returns:
        ``[sequences, heads, d]`` of q's type.
    """
    return paged_attention_with_lse(q, k_pages, v_pages, block_table, lengths, bias_fn, sm_scale, pages)[0]
