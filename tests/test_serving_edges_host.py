"""What the serving-step operators refuse at the edges of their ranges, without a GPU (every status is decided before any
launch), and the host side of their Python functions."""
import ctypes as C

import pytest
import torch

import tinystrata_b200 as T

from .test_serving_host import ALIGN, ARG, CUDA, UNSUP, WS, attend, built, cache, desc, rule, tables  # noqa: F401


@pytest.mark.parametrize("block", [16, 32, 64])
def test_attention_lengths_near_the_end_of_32_bits(block):
    """A request's positions, and those of the tiles read ahead of its last one, stay below 2^31."""
    c = cache(block_size=block)
    for over in (-1, 64, 512):
        width = (2 ** 31 - over) // block
        assert attend(c, table_width=width, table_stride=width) == UNSUP
        d = desc(table_width=width, table_stride=width)
        assert T.lib().tsb_kv8_attention_workspace_bytes(C.byref(c), C.byref(d)) == 0
