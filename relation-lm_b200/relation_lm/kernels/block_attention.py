"""Attention over the blocks that the router chooses (extension): a layer that attends where the selectors of this library
pick single rows.

Three operators, used one after another; the block statistics in between are those of ``router_cache_update``:

* ``rotary_append``: rotary positions of queries and keys, keys and values into the caches;
* ``route_blocks``: the best remote blocks of every row by the router's score (the anchor stream's of
  ``relation_select_packed``);
* ``block_attention``: softmax attention over those blocks and the row's local window.

Each comes in the forms of the selectors: for one decode position (``position``, a 0-d int64 device tensor, one row for each
sequence), for rows with a sequence and a position of their own (``*_rows``; int32 ``row_batch`` and ``row_position``, a
negative position marks a row of padding) and for whole sequences (``*_prefill``; row ``b * query_length + t``).  Rows of
padding and rows outside the caches give zeros (index -1, score and lse -inf) and write nothing; the latter also set the
status word.  ``route_blocks`` knows no cache: only sequences outside its statistics count there, and a position beyond them
has all their blocks behind it.  Nothing here has a derivative.
"""
from __future__ import annotations

import math

import torch
from torch import Tensor

from relation_lm.kernels import _abi

# The operators themselves are registered by csrc/torch_ops.cpp; the functions below document them.
_rotary_append = _abi.operator("rotary_append")
_rotary_append_rows = _abi.operator("rotary_append_rows")
_rotary_append_prefill = _abi.operator("rotary_append_prefill")
_route_blocks = _abi.operator("route_blocks")
_route_blocks_rows = _abi.operator("route_blocks_rows")
_route_blocks_prefill = _abi.operator("route_blocks_prefill")
_block_attention = _abi.operator("block_attention")
_block_attention_rows = _abi.operator("block_attention_rows")
_block_attention_prefill = _abi.operator("block_attention_prefill")


def rotary_frequencies(rotary: int, base: float = 10000.0, *, scaling: str | None = None, factor: float = 1.0,
                       trained_context: int = 0, fast: float = 32.0, slow: float = 1.0,
                       device: torch.device | str | None = None) -> tuple[Tensor, float]:
    """``(frequencies, magnitude)`` for ``rotary_append``: ``base ** (-2 i / rotary)`` for ``i < rotary / 2``, fp64, and 1.

    ``scaling`` stretches them for contexts ``factor`` times the trained one: ``"linear"`` divides them by ``factor``;
    ``"base"`` raises the base so that the slowest is divided by ``factor`` and the fastest stays; ``"by_parts"`` (Peng et
    al., YaRN, 2023) divides those that turn fewer than ``slow`` times in ``trained_context`` positions, leaves those that
    turn more than ``fast`` times, blends in between, and returns the magnitude ``1 + 0.1 log(factor)``.  The blend is linear
    in the number of turns, as published; models trained with one that is linear in the component's index ``i`` need their own
    frequencies, which ``rotary_append`` takes as they are.
    """
    if rotary < 0 or rotary % 2 != 0:
        raise ValueError("the rotary width must be even")
    if not base > 1.0 or not factor >= 1.0:
        raise ValueError("base must be above 1 and factor at least 1")
    if scaling not in (None, "linear", "base", "by_parts"):
        raise ValueError(f"unknown scaling {scaling!r}; use 'linear', 'base' or 'by_parts'")
    if scaling == "base" and rotary > 2:
        base = base * factor ** (rotary / (rotary - 2))
    step = torch.arange(rotary // 2, dtype=torch.float64)
    frequencies, magnitude = base ** (-2.0 * step / max(rotary, 1)), 1.0
    if scaling == "linear":
        frequencies = frequencies / factor
    elif scaling == "by_parts":
        if trained_context < 1 or not fast > slow:
            raise ValueError("by_parts needs the trained context and fast > slow")
        turns = trained_context * frequencies / (2.0 * math.pi)
        keep = ((turns - slow) / (fast - slow)).clamp(0.0, 1.0)
        frequencies = frequencies * (keep + (1.0 - keep) / factor)
        magnitude = 1.0 + 0.1 * math.log(factor)
    return frequencies.to(device), magnitude


def rotary_append(query: Tensor, key: Tensor, value: Tensor, key_cache: Tensor, value_cache: Tensor, frequencies: Tensor,
                  position: Tensor, interleaved: bool = False, magnitude: float = 1.0) -> Tensor:
    """Turn queries and keys by their position, write keys and values into the caches; returns the turned queries.

    ``query [N, heads, width]``, ``key``, ``value [N, kv_heads, width]`` (any row and head strides), caches
    ``[B, T, kv_heads, width]`` (any strides but the innermost), all of one dtype.  ``frequencies`` (fp32 or fp64,
    ``[rotary / 2]``, ``rotary <= width``): component pairs ``(2i, 2i + 1)`` (``interleaved``) or ``(i, i + rotary / 2)`` turn
    by ``position * frequencies[i]`` (worked out in 64 bits) and are multiplied by ``magnitude``; the rest is copied.  A
    position of a sequence must not occur twice in a call; the inputs must not lie in the caches, nor may the caches have an
    element in common (views of one buffer that lie between one another are fine).
    """
    return _rotary_append(query, key, value, key_cache, value_cache, frequencies, position, interleaved, magnitude)


@torch.library.register_fake("relation_lm::rotary_append")
def _(query, key, value, key_cache, value_cache, frequencies, position, interleaved, magnitude):
    return query.new_empty(query.shape)


def rotary_append_rows(query: Tensor, key: Tensor, value: Tensor, key_cache: Tensor, value_cache: Tensor, frequencies: Tensor,
                       row_batch: Tensor, row_position: Tensor, interleaved: bool = False, magnitude: float = 1.0) -> Tensor:
    """``rotary_append`` for rows with a sequence and a position of their own."""
    return _rotary_append_rows(query, key, value, key_cache, value_cache, frequencies, row_batch, row_position, interleaved,
                               magnitude)


@torch.library.register_fake("relation_lm::rotary_append_rows")
def _(query, key, value, key_cache, value_cache, frequencies, row_batch, row_position, interleaved, magnitude):
    return query.new_empty(query.shape)


def rotary_append_prefill(query: Tensor, key: Tensor, value: Tensor, key_cache: Tensor, value_cache: Tensor,
                          frequencies: Tensor, query_length: int, interleaved: bool = False, magnitude: float = 1.0) -> Tensor:
    """``rotary_append`` for positions ``0 .. query_length - 1`` of every sequence."""
    return _rotary_append_prefill(query, key, value, key_cache, value_cache, frequencies, query_length, interleaved, magnitude)


@torch.library.register_fake("relation_lm::rotary_append_prefill")
def _(query, key, value, key_cache, value_cache, frequencies, query_length, interleaved, magnitude):
    return query.new_empty(query.shape)


def route_blocks(router_query: Tensor, block_mean: Tensor, block_std: Tensor, gamma: Tensor, bias: Tensor, position: Tensor,
                 block_size: int, local_window: int, top_blocks: int, strict_valid: bool) -> tuple[Tensor, Tensor]:
    """The ``top_blocks`` best blocks of every row: indices (int32) and scores (fp32) ``[N, top_blocks]``, best first.

    ``router_query [N, 64]``, statistics ``[B, blocks, 4, 16]``, ``gamma [4]``, ``bias [4, buckets]``.  Blocks that are complete
    at the row's position take part, with ``strict_valid`` only those that end before its local window.  Ties go to the
    lowest block; places without a block hold -1 and -inf.  Scores are compared in 64 bits, so the choice does not depend
    on the form of the call.  (``relation_select_packed`` compares the same scores in 32 bits and takes those above -1e30
    only: where two are as near as 32 bits tell apart, it may look into another block.)
    """
    return _route_blocks(router_query, block_mean, block_std, gamma, bias, position, block_size, local_window, top_blocks,
                         strict_valid)


def _route_fake(router_query, top_blocks):
    rows = router_query.size(0)
    return (router_query.new_empty((rows, top_blocks), dtype=torch.int32),
            router_query.new_empty((rows, top_blocks), dtype=torch.float32))


@torch.library.register_fake("relation_lm::route_blocks")
def _(router_query, block_mean, block_std, gamma, bias, position, block_size, local_window, top_blocks, strict_valid):
    return _route_fake(router_query, top_blocks)


def route_blocks_rows(router_query: Tensor, block_mean: Tensor, block_std: Tensor, gamma: Tensor, bias: Tensor,
                      row_batch: Tensor, row_position: Tensor, block_size: int, local_window: int, top_blocks: int,
                      strict_valid: bool) -> tuple[Tensor, Tensor]:
    """``route_blocks`` for rows with a sequence and a position of their own."""
    return _route_blocks_rows(router_query, block_mean, block_std, gamma, bias, row_batch, row_position, block_size,
                              local_window, top_blocks, strict_valid)


@torch.library.register_fake("relation_lm::route_blocks_rows")
def _(router_query, block_mean, block_std, gamma, bias, row_batch, row_position, block_size, local_window, top_blocks,
      strict_valid):
    return _route_fake(router_query, top_blocks)


def route_blocks_prefill(router_query: Tensor, block_mean: Tensor, block_std: Tensor, gamma: Tensor, bias: Tensor,
                         query_length: int, block_size: int, local_window: int, top_blocks: int,
                         strict_valid: bool) -> tuple[Tensor, Tensor]:
    """``route_blocks`` for positions ``0 .. query_length - 1`` of every sequence."""
    return _route_blocks_prefill(router_query, block_mean, block_std, gamma, bias, query_length, block_size, local_window,
                                 top_blocks, strict_valid)


@torch.library.register_fake("relation_lm::route_blocks_prefill")
def _(router_query, block_mean, block_std, gamma, bias, query_length, block_size, local_window, top_blocks, strict_valid):
    return _route_fake(router_query, top_blocks)


def block_attention(query: Tensor, key_cache: Tensor, value_cache: Tensor, block_index: Tensor, position: Tensor,
                    block_size: int, local_window: int, scale: float) -> tuple[Tensor, Tensor]:
    """Softmax attention over each row's local window and its chosen blocks: ``(out [N, heads, width], lse [N, heads])``.

    With ``ls = max(0, t - local_window + 1)`` a row at position ``t`` sees ``[ls, t]`` and of every block ``n`` among its
    indices the rows ``[n * block_size, min((n + 1) * block_size, ls))``.  ``block_index`` (int32) is ``[N, blocks]``, one choice
    for all heads, or ``[N, kv_heads, blocks]``; negative and repeated indices count for nothing, at most 128 are given.
    Query head ``h`` reads key head ``h // (heads / kv_heads)`` of the caches ``[B, T, kv_heads, width]`` (any strides but the
    innermost; widths 32, 64, 96, 128; rows on 16-byte boundaries).  ``lse`` (fp32) is the logarithm of the softmax denominator; a row that sees
    nothing is zero with -inf.  Sums are fp32, 16-bit operands' softmax weights are rounded to 16 bits (half a step of each weight;
    in fp16 all bits down to 2^-29 of the row's largest).  A block may be longer than the cache.
    """
    return _block_attention(query, key_cache, value_cache, block_index, position, block_size, local_window, scale)


def _attention_fake(query):
    return query.new_empty(query.shape), query.new_empty(query.shape[:2], dtype=torch.float32)


@torch.library.register_fake("relation_lm::block_attention")
def _(query, key_cache, value_cache, block_index, position, block_size, local_window, scale):
    return _attention_fake(query)


def block_attention_rows(query: Tensor, key_cache: Tensor, value_cache: Tensor, block_index: Tensor, row_batch: Tensor,
                         row_position: Tensor, block_size: int, local_window: int, scale: float) -> tuple[Tensor, Tensor]:
    """``block_attention`` for rows with a sequence and a position of their own."""
    return _block_attention_rows(query, key_cache, value_cache, block_index, row_batch, row_position, block_size, local_window,
                                 scale)


@torch.library.register_fake("relation_lm::block_attention_rows")
def _(query, key_cache, value_cache, block_index, row_batch, row_position, block_size, local_window, scale):
    return _attention_fake(query)


def block_attention_prefill(query: Tensor, key_cache: Tensor, value_cache: Tensor, block_index: Tensor, query_length: int,
                            block_size: int, local_window: int, scale: float) -> tuple[Tensor, Tensor]:
    """``block_attention`` for positions ``0 .. query_length - 1`` of every sequence.

    In 16 bits and from about a thousand (row, key head) pairs on it allocates a workspace for the duration of the call: about
    ``4 * heads * blocks * (width + 2)`` bytes a row, up to some 512 MB (at least one part of a sequence), whatever the batch.
    """
    return _block_attention_prefill(query, key_cache, value_cache, block_index, query_length, block_size, local_window, scale)


@torch.library.register_fake("relation_lm::block_attention_prefill")
def _(query, key_cache, value_cache, block_index, query_length, block_size, local_window, scale):
    return _attention_fake(query)
