"""Shared-prefix decode: lengths that do not fit the C entry point's 32 bits are refused, not cut."""
from __future__ import annotations

import pytest
import torch

import nvattn
from nvattn import ops

pytestmark = pytest.mark.gpu
dev = torch.device("cuda")


@pytest.mark.parametrize("shared", [2 ** 32, 2 ** 32 + 256, 2 ** 33 - 2 ** 32, -2 ** 32, 2 ** 64 + 128, 2 ** 31])
def test_lengths_past_32_bits(shared):
    q = torch.zeros(2, 4, 128, dtype=torch.bfloat16, device=dev)
    c = torch.zeros(4, 128, 2, 128, dtype=torch.bfloat16, device=dev)
    lens = torch.full((2,), 300, dtype=torch.int32, device=dev)
    bt = torch.tensor([[0, 1, 2], [0, 1, 3]], dtype=torch.int32, device=dev)
    ops.shared_prefix_decode(q, c, c, lens, bt, 256)
    with pytest.raises((ValueError, nvattn._lib.NvattnError), match="whole blocks"):
        ops.shared_prefix_decode(q, c, c, lens, bt, shared)


def test_an_empty_batch_is_taken_at_any_length():
    q = torch.zeros(0, 4, 128, dtype=torch.bfloat16, device=dev)
    c = torch.zeros(4, 128, 2, 128, dtype=torch.bfloat16, device=dev)
    none = torch.zeros(0, dtype=torch.int32, device=dev)
    assert ops.shared_prefix_decode(q, c, c, none, none.view(0, 1), 512).shape == (0, 4, 128)
