"""Attention over router-chosen blocks without a GPU: what the entry points take at the borders of their checks."""
from __future__ import annotations

import ctypes

import pytest

from relation_lm.kernels import _abi
from test_block_attention_cpu import ATTENTION, ROUTE, refused, strides


def accepted(**changes):
    assert _abi.LIB.rlm_block_attention(*{**ATTENTION, **changes}.values()) == 0, (changes, _abi.LIB.rlm_last_error())


@pytest.mark.parametrize("which,ones", [(1, dict(heads=1, kv_heads=1)), (2, dict(n_seq=1)), (3, dict(max_t=1)), (4, dict(kv_heads=1)),
                                        (5, dict(n_seq=1)), (6, dict(max_t=1)), (7, dict(kv_heads=1))])
def test_the_step_of_a_single_one_is_of_no_account(which, ones):
    # a stride that is no multiple of 16 bytes is refused only where it leads somewhere; calls without rows launch nothing
    steps = [512, 64, 8192, 128, 64, 8192, 128, 64, 4, 0]
    steps[which] += 1
    none = dict(n_rows=0, position=None, row_batch=1 << 20, row_position=1 << 20, strides=strides(*steps))
    refused("rlm_block_attention", ATTENTION, -4, **none)
    accepted(**none, **ones)


def test_more_rows_than_a_launch_holds_are_refused():
    # rows whose blocks need a cluster of eight CTAs each: the number of CTAs passes 32 bits
    many = dict(position=None, row_batch=1 << 20, row_position=1 << 20, n_rows=0x7fffffff, n_blocks=40000, block=1)
    refused("rlm_block_route", ROUTE, -2, **many)
    refused("rlm_block_attention", ATTENTION, -2, position=None, row_batch=1 << 20, row_position=1 << 20, n_rows=0x7fffffff)
