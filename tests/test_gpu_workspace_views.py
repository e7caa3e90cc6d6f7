"""Decode operators: a workspace that is not one run of bytes is refused (a view with gaps or of one
repeated byte has fewer bytes behind its pointer than it has elements)."""
from __future__ import annotations

import pytest
import torch

from nvattn import ops

pytestmark = pytest.mark.gpu
dev = torch.device("cuda")


def _args(fp8):
    q = torch.zeros(40, 8, 128, dtype=torch.bfloat16, device=dev)
    c = torch.zeros(4, 256, 2, 128, dtype=torch.bfloat16, device=dev)
    lens = torch.full((40,), 700, dtype=torch.int32, device=dev)
    bt = torch.tensor([[0, 1, 2] + [3] * 13] * 40, dtype=torch.int32, device=dev)
    if not fp8:
        return q, c, c, lens, bt
    s = torch.full((4, 2, 256), 127, dtype=torch.uint8, device=dev)
    return q, c.to(torch.float8_e4m3fn), c.to(torch.float8_e4m3fn), s, s, lens, bt


@pytest.mark.parametrize("fp8", [False, True])
def test_views_are_refused(fp8):
    args = _args(fp8)
    if fp8:
        def call(ws):
            return ops.paged_decode_fp8(*args, workspace=ws)
        need = ops.decode_fp8_workspace_bytes(40, 8, 2, 16, 256)
    else:
        def call(ws):
            return ops.shared_prefix_decode(*args, 256, workspace=ws)
        need = ops.shared_prefix_workspace_bytes(40, 8, 2, 16, 256, 256)
    assert need > 0
    whole = torch.empty(2 * need, dtype=torch.uint8, device=dev)
    assert torch.equal(call(whole[:need]), call(None))
    for ws in (whole[::2], whole.view(2, need).t(), whole[:1].expand(need)):
        with pytest.raises(ValueError, match="contiguous"):
            call(ws)
