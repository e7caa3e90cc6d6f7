"""Draft verification with a NaN temperature: not above zero, so greedy, as the sampler takes it."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import reference_math as R

from nvattn import ops

pytestmark = pytest.mark.gpu
dev = torch.device("cuda")


@pytest.mark.parametrize("form", ["chain", "draft", "tree"])
def test_nan_is_greedy(form):
    B, n, V = 6, 4, 701
    g = torch.Generator().manual_seed(1)
    x = torch.randn(B, n, V, generator=g).to(torch.bfloat16)
    tok = x[:, :n - 1].float().argmax(-1)
    tok[::2, 1] = 5
    u, pick = torch.rand(B, n - 1, generator=g), torch.rand(B, generator=g)
    temps = torch.tensor([float("nan"), 1.0, float("nan"), 0.0, -1.0, float("nan")])
    kw = {}
    if form == "draft":
        kw["draft_logits"] = torch.randn(B, n - 1, V, generator=g).to(torch.bfloat16)
    if form == "tree":
        kw["parents"] = torch.tensor([[-1, 0, 0, 1]] * B, dtype=torch.int32)
    got = ops.verify_draft(x.to(dev), tok.to(dev), u.to(dev), pick.to(dev), temps.to(dev),
                           **{k: v.to(dev) for k, v in kw.items()})
    want = R.verify_draft(x, tok.numpy(), u.numpy(), pick.numpy(), temperatures=temps, **kw)
    for name, a, b in zip(("tokens", "path", "accepted"), got, want):
        assert np.array_equal(a.cpu().numpy(), b), name
    assert torch.equal(ops.sample(x[:, 0].to(dev), temps.to(dev))[[0, 2, 5]].cpu(),
                       x[[0, 2, 5], 0].float().argmax(-1))
