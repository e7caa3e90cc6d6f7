"""Draft verification, the draw from max(p - q, 0): columns whose p and q differ by less than fp32 sums of
the rows can tell are on the side that 64-bit sums put them."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import reference_math as R

from nvattn import ops

pytestmark = pytest.mark.gpu
dev = torch.device("cuda")
INF = float("inf")


def _at_border(x, d, T, u, token):
    """Whether 64-bit sums leave open if u draws `token` from max(p - q, 0): p = w / a and q = v / d,
    a sum of V terms added up in a chain of up to V / 512 and a tree of 40 more (the fewest threads that
    share a row are 512) is off by (V / 512 + 48) * 2^-53 of itself with its exponentials' own 2^-50, and
    so is every w / a, all together by that of sum p = 1; the same holds for q. Here in 64 bits of
    mantissa."""
    w, v = [np.exp((r.double().numpy() - r.double().max().item()).astype(np.longdouble)
                   / np.longdouble(np.float32(T))) for r in (x, d)]
    c = np.cumsum(np.maximum(w / w.sum() - v / v.sum(), 0))
    delta = 2 * (x.numel() / 512 + 48) * 2.0 ** -53
    want = np.longdouble(np.float32(u)) * c[-1]
    return c[token] + delta > want and (token == 0 or c[token - 1] - delta <= want)


def _check(x, tok, u, pick, **kw):
    got = [t.cpu().numpy() for t in
           ops.verify_draft(x.to(dev), tok.to(dev), u.to(dev), pick.to(dev),
                            **{k: v.to(dev) for k, v in kw.items()})]
    want = R.verify_draft(x, tok.numpy(), u.numpy(), pick.numpy(), **kw)
    for name, a, b in zip(("path", "accepted"), got[1:], want[1:]):
        assert np.array_equal(a, b), name
    for b in np.nonzero((got[0] != want[0]).any(1))[0]:
        assert want[2][b] == 0 and _at_border(x[b, 0], kw["draft_logits"][b, 0], kw["temperatures"][b],
                                              pick[b], got[0][b, 0]), (b, got[0][b], want[0][b])
    return got


def test_four_columns():
    """Both fp32 sums are 1.0014648; the true quotient is 1 - 1.5e-8, and column 1 has that much."""
    x = torch.tensor([[[-10.0, 0.0, -11.0, -INF], [0.0] * 4]]).to(torch.bfloat16)
    d = torch.tensor([[[-11.0, 0.0, -10.0, -26.0]]]).to(torch.bfloat16)
    for pick, token in ((0.5, 0), (1 - 2.0 ** -16, 1), (1 - 2.0 ** -24, 1)):
        t, _, _ = _check(x, torch.tensor([[3]]), torch.tensor([[0.5]]), torch.tensor([pick]),
                         temperatures=torch.tensor([1.4426950408889634]), draft_logits=d)
        assert t[0, 0] == token


@pytest.mark.parametrize("V", [6, 40, 3001, 151936])
@pytest.mark.parametrize("less", [False, True])
def test_rows_that_differ_in_a_few_columns(V, less):
    """All columns but four hold the same logits: their common quotient is 1 within 1e-6 down to 1e-9,
    on either side, and the residual is far larger. The first column of the residual is drawn, or its
    last, where the many come in."""
    B = 64
    g = torch.Generator().manual_seed(V + less)
    x = torch.randn(B, 2, V, generator=g)
    x[:, :, 2] = (x.amax((1, 2)) + 2 + torch.rand(B, generator=g))[:, None]
    d = x[:, :1].clone()
    top = x[:, 0, 2]
    x[:, 0, 0], x[:, 0, 1] = top - 5, top - 7       # swapped: the sums stay the same
    d[:, 0, 0], d[:, 0, 1] = top - 7, top - 5
    tail = top - 13 - 8 * torch.rand(B, generator=g)  # one column's weight that only one row has
    x[:, 0, 3], d[:, 0, 3] = (tail, tail - 30) if less else (tail - 30, tail)
    x, d = x.to(torch.bfloat16), d.to(torch.bfloat16)
    x[:, 0, 0], x[:, 0, 1] = d[:, 0, 1], d[:, 0, 0]
    tok = torch.full((B, 1), 1)                       # q has more of it: rejected for most u
    for pick in (0.0, 1.0 - 2.0 ** -24, 1.0 - 2.0 ** -16, 0.5):
        w = _check(x, tok, torch.full((B, 1), 1.0 - 2.0 ** -24), torch.full((B,), pick),
                   temperatures=torch.full((B,), 0.9) + 0.2 * torch.rand(B, generator=g), draft_logits=d)
        assert (w[2] == 0).all()


def _balance(x, d, up=True):
    """The fp32 temperature at which both rows' sums of exp((l - top) / T) are closest to equal from
    one side, or None."""
    def f(T):
        return np.exp((x - x.max()) / T).sum() - np.exp((d - d.max()) / T).sum()
    lo, hi = np.float32(0.3), np.float32(3.0)
    if f(lo) * f(hi) > 0:
        return None
    while np.nextafter(lo, hi) < hi:
        mid = np.float32((np.float64(lo) + np.float64(hi)) / 2)
        lo, hi = (mid, hi) if f(mid) * f(lo) > 0 else (lo, mid)
    return lo if (f(lo) > 0) == up else hi


@pytest.mark.parametrize("equal", [0, 1, 40])
@pytest.mark.parametrize("up", [False, True])
@pytest.mark.parametrize("V", [50, 2000])
def test_one_column_at_the_common_quotient(V, up, equal):
    """Independent rows with the same largest logit, in column 0, at the temperature where their sums
    agree: column 0 (and `equal` others) lies within 1e-8 of the border between the sides, every other
    column far from it. Column 0 is drawn by the smallest random numbers, if it is in the residual."""
    g = torch.Generator().manual_seed(V + 2 * equal + up)
    rows, temps = [], []
    while len(rows) < 24:
        r = torch.randn(2, V, generator=g)
        r[:, 0] = 5.0
        r[1, V - equal:] = r[0, V - equal:]
        r = r.to(torch.bfloat16)
        T = _balance(r[0].double().numpy(), r[1].double().numpy(), up)
        if T is not None:
            rows.append(r)
            temps.append(float(T))
    r = torch.stack(rows)
    B = len(rows)
    x = torch.stack([r[:, 0], r[:, 0]], 1)
    d = r[:, 1:]
    tok = (d[:, 0].float() - x[:, 0].float()).argmax(-1, keepdim=True)  # most of it the draft's alone
    first = []
    for pick in (0.0, 1e-12, 1e-10, 3e-9, 0.7, 1.0 - 2.0 ** -24):
        w = _check(x, tok, torch.full((B, 1), 1.0 - 2.0 ** -24), torch.full((B,), pick),
                   temperatures=torch.tensor(temps), draft_logits=d.contiguous())
        assert (w[2] == 0).all()
        first.append((w[0][:, 0] == 0).mean())
    assert (first[0] == 0) if up else (first[0] > 0.9)
