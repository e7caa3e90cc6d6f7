"""Draft verification over rows whose largest logit is the lowest finite bf16, a common mask value:
the columns that hold it share the probability, and nothing else is ever drawn."""
from __future__ import annotations

from fractions import Fraction

import numpy as np
import pytest
import torch

from oracle import reference_math as R

from nvattn import ops

pytestmark = pytest.mark.gpu
dev = torch.device("cuda")
LOWEST = torch.finfo(torch.bfloat16).min
PICKS = (0.0, 2.0 ** -24, 0.31, 0.5, 0.97, 1.0 - 2.0 ** -24)


def _flat_walk(x, tok, u, pick, temperatures, draft_logits=None, parents=None):
    """The walk over rows whose live columns all hold the lowest value, in exact arithmetic: a random
    number may lie on a border here (half of six equal columns), where sums of 1/7 in fp64 round. Draft
    rows are flat too at the ends of the temperatures: over the columns of their top, or over all."""
    B, n, V = x.shape
    tokens, path = np.full((B, n), -1, np.int64), np.full((B, n), -1, np.int32)
    num = np.zeros(B, np.int32)
    for b in range(B):
        up = [-1] + list(range(n - 1)) if parents is None else parents[b].tolist()
        T = float(temperatures[b])
        node, path[b, 0] = 0, 0
        while True:
            live = (x[b, node] == LOWEST).nonzero().flatten().tolist()
            rest, found, drawn, r = list(live), None, None, Fraction(float(pick[b]))
            for c in range(node + 1, n):
                t, uu = int(tok[b, c - 1]), Fraction(float(u[b, c - 1]))
                if up[c] != node:
                    continue
                if draft_logits is not None:
                    d = draft_logits[b, node].float()
                    q = torch.from_numpy(R.verify_law(d, T))
                    if t in live and uu * Fraction(float(q[t])) * len(live) < 1:
                        found = c
                    elif T < 1e-20:  # q is the draft's top alone
                        top = (d == d.max()).nonzero().flatten().tolist()
                        assert len(top) == 1 or len(top) < len(live)
                        rest = [i for i in live if i not in top] or live
                    elif T < 1e20:   # (at 1e30 q is flat: the live columns keep equal weights)
                        p = (x[b, node] == LOWEST).double()
                        drawn = R.verify_draw((p / p.sum() - q).clamp_min(0).numpy(), float(pick[b]))
                    break
                if t not in rest:
                    continue
                if uu * len(rest) < 1:
                    found = c
                    break
                rest.remove(t)
            if found is None:
                break
            tokens[b, num[b]] = int(tok[b, found - 1])
            node, num[b] = found, num[b] + 1
            path[b, num[b]] = node
        rest = rest or live
        tokens[b, num[b]] = rest[int(r * len(rest))] if drawn is None else drawn
    return tokens, path, num


def _check(x, tok, u, pick, view=None, flat=True, **kw):
    """The kernels' answer on x (or on an equal view of it on the GPU) is the exact walk's, or where the
    target's rows are not flat the oracle's, and every token is a column."""
    gpu = {k: v.to(dev) for k, v in kw.items()}
    got = ops.verify_draft(x.to(dev) if view is None else view, tok.to(dev), u.to(dev), pick.to(dev), **gpu)
    t, path, num = [g.cpu().numpy() for g in got]
    for b in range(len(num)):
        assert (t[b, :num[b] + 1] >= 0).all() and (t[b, :num[b] + 1] < x.shape[2]).all(), t[b]
    if flat:
        want = _flat_walk(x, tok, u, pick, **kw)
    else:
        want = R.verify_draft(x, tok.numpy(), u.numpy(), pick.numpy(), **kw)
    for name, a, b in zip(("tokens", "path", "accepted"), (t, path, num), want):
        assert np.array_equal(a, b), (name, a, b)


def _rows(V, B, n, live, g):
    """Rows of -inf (every third NaN) but for `live` columns of the lowest finite value (all: None)."""
    if live is None:
        return torch.full((B, n, V), LOWEST).to(torch.bfloat16)
    x = torch.full((B, n, V), float("-inf"))
    x[:, :, ::3] = float("nan")
    x.scatter_(2, torch.randint(0, V, (B, n, live), generator=g), LOWEST)
    return x.to(torch.bfloat16)


@pytest.mark.parametrize("form", ["chain", "draft", "tree"])
@pytest.mark.parametrize("live", [None, 3])
@pytest.mark.parametrize("V", [1, 7, 130, 997, 151936])
def test_target_rows(V, live, form):
    B, n = len(PICKS) * 2, 4
    g = torch.Generator().manual_seed(V)
    x = _rows(V, B, n, live, g)
    tok = torch.randint(0, V, (B, n - 1), generator=g)
    kw = dict(temperatures=torch.tensor([0.7, 1e-30, 1e30, 3.0] * (B // 4)))
    if form == "draft":
        kw["draft_logits"] = torch.randn(B, n - 1, V, generator=g).to(torch.bfloat16)
    if form == "tree":
        kw["parents"] = torch.tensor([[-1, 0, 0, 0]] * B, dtype=torch.int32)
    for u in (0.0, 1.0 - 2.0 ** -24):
        _check(x, tok, torch.full((B, n - 1), u), torch.tensor(PICKS * 2), **kw)


@pytest.mark.parametrize("V", [130, 997])
def test_rows_at_odd_addresses(V):
    B, n = len(PICKS), 2
    g = torch.Generator().manual_seed(V)
    x = _rows(V, B, n, None, g)
    for at in (1, 3, 7):
        wide = torch.full((B, n, V + 13), 5.0, dtype=torch.bfloat16, device=dev)
        wide[:, :, at:at + V] = x.to(dev)
        _check(x, torch.randint(0, V, (B, 1), generator=g), torch.full((B, 1), 0.999), torch.tensor(PICKS),
               view=wide[:, :, at:at + V], temperatures=torch.full((B,), 0.7))


@pytest.mark.parametrize("live", [None, 5])
def test_draft_rows(live):
    """An ordinary target against draft rows of the lowest value: a flat law over the live columns."""
    V, B, n = 997, len(PICKS) * 2, 3
    g = torch.Generator().manual_seed(5)
    x = torch.randn(B, n, V, generator=g).to(torch.bfloat16)
    d = _rows(V, B, n - 1, live, g)
    tok = d.float().nan_to_num(nan=-torch.inf).argmax(-1)  # one that the draft can give
    for u in (0.0, 0.5, 1.0 - 2.0 ** -24):
        _check(x, tok, torch.full((B, n - 1), u), torch.tensor(PICKS * 2), flat=False,
               draft_logits=d, temperatures=torch.full((B,), 0.8))
