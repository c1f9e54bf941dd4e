"""The attention layer of kv4_layer.py: projections, cache and attention together, prompts and steps from a graph.

Tolerance, of the largest output: attention's own (2^-11 for the type, 2^-10 of sum p |v| / sum p), the values that the fp32
side reads as fp16 (2^-11 of keys and of values; the keys' part of a score comes with random signs, 2^-11 of about one), and
the output projection's rounding, 2^-11: together under 2^-8.
"""
from __future__ import annotations

import pytest
import torch

from tests._helpers import torch_cuda


def layer():
    import kv4_layer
    return kv4_layer


def test_slots_follow_the_block_table():
    pages = layer().Pages(torch, 3, 70, 16, "cpu")
    assert pages.table.shape == (3, 5) and pages.count == 15 and sorted(pages.table.flatten().tolist()) == list(range(15))
    got = pages.slots(torch.tensor([0, 2, 2]), torch.tensor([0, 17, 69]))
    assert got.tolist() == [int(pages.table[0, 0]) * 16, int(pages.table[2, 1]) * 16 + 1, int(pages.table[2, 4]) * 16 + 5]


@pytest.mark.gpu
@pytest.mark.parametrize("head_dim,group,page,window,heads,kv_heads,prompts", [
    (128, 128, 64, 0, 8, 2, (200, 0, 333, 64)), (128, 64, 16, 0, 8, 8, (1, 0, 90)), (64, 64, 32, 100, 8, 1, (150, 0, 17, 301, 2))])
def test_layer_serves_prompts_and_steps(head_dim, group, page, window, heads, kv_heads, prompts):
    torch_cuda()
    for error in layer().serve(torch, 1024, heads, kv_heads, head_dim, group, page, 5, prompts, window):
        assert error <= 2.0**-8
