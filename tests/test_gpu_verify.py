"""Draft verification on the GPU: tokens, paths and counts equal to the oracle's
64-bit walk, at the sizes, masks and random numbers where they could differ."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import reference_math as R

from nvattn import ops, tree

pytestmark = pytest.mark.gpu
dev = torch.device("cuda")


def _inputs(B, n, V, seed, form="chain", noise=1.0, hot=8):
    g = torch.Generator().manual_seed(seed)
    x = 2 * torch.randn(B, n, V, generator=g)
    x.scatter_add_(2, torch.randint(0, V, (B, n, hot), generator=g),
                   4 + 6 * torch.rand(B, n, hot, generator=g))
    d = x + noise * torch.randn(B, n, V, generator=g)
    x, d = x.to(torch.bfloat16), d.to(torch.bfloat16)
    temps = 0.5 + torch.rand(B, generator=g)
    temps[2::5] = 0.0
    kw = dict(temperatures=temps)
    if form == "tree":
        par, _ = tree.build_draft_tree((4, 3, 2, 1, 1, 1), n)
        rank = [int((par[1:j] == par[j]).sum()) for j in range(1, n)]
        top = d.float().topk(min(4, V), -1).indices
        tok = top[:, torch.from_numpy(par[1:].astype(np.int64)), torch.tensor(rank, dtype=torch.int64) % min(4, V)]
        kw["parents"] = torch.from_numpy(par)[None].expand(B, n)
    else:
        tok = d[:, :n - 1].float().argmax(-1)
        if form == "draft":
            kw["draft_logits"] = d[:, :n - 1].contiguous()
            e = torch.empty(B, n - 1, V).exponential_(generator=g)
            t = temps.clamp_min(0.5)[:, None, None]
            tok = (kw["draft_logits"].float() / t - e.log()).argmax(-1)
    return x, tok.contiguous(), torch.rand(B, n - 1, generator=g), torch.rand(B, generator=g), kw


def _run(x, tok, u, pick, kw):
    out = ops.verify_draft(x.to(dev), tok.to(dev), u.to(dev), pick.to(dev),
                           **{k: v.to(dev) if torch.is_tensor(v) else v for k, v in kw.items()})
    return [t.cpu().numpy() for t in out]


def _check(x, tok, u, pick, kw):
    got = _run(x, tok, u, pick, kw)
    want = R.verify_draft(x, tok.numpy(), u.numpy(), pick.numpy(), **kw)
    for name, a, b in zip(("tokens", "path", "accepted"), got, want):
        assert np.array_equal(a, b), (name, a, b)
    return want


@pytest.mark.parametrize("form", ["chain", "draft", "tree"])
@pytest.mark.parametrize("B,n,V", [(1, 1, 1000), (3, 2, 7), (40, 5, 1000), (7, 9, 33001),
                                   (2, 4, 151936), (5, 64, 2049), (300, 3, 64)])
def test_equals_the_walk(form, B, n, V):
    for seed in (0, 1):
        w = _check(*_inputs(B, n, V, seed + V, form))
    if B >= 40 and n > 2:
        assert 0 < w[2].mean() < n - 1  # some drafts stand, some fall


@pytest.mark.parametrize("form", ["chain", "draft", "tree"])
def test_flat_rows_whose_borders_lie_close(form):
    """151,936 nearly equal weights: a border every 6.6e-6, drawn 200 times."""
    x, tok, u, pick, kw = _inputs(100, 2, 151936, 3, form, hot=1)
    x = (x.float() * 0.05).to(torch.bfloat16)
    kw["temperatures"] = torch.full((100,), 0.9)
    if form == "draft":
        kw["draft_logits"] = (kw["draft_logits"].float() * 0.05).to(torch.bfloat16)
    for seed in range(2):
        pick = torch.rand(100, generator=torch.Generator().manual_seed(seed))
        _check(x, tok, u, pick, kw)


def test_ragged_and_padding_rows():
    for form in ("chain", "draft", "tree"):
        x, tok, u, pick, kw = _inputs(9, 6, 501, 5, form)
        kw["num_nodes"] = torch.tensor([0, 1, 2, 3, 6, 9, -4, 5, 1], dtype=torch.int32)
        t, p, a = _check(x, tok, u, pick, kw)
        assert (t[0] == -1).all() and a[0] == 0 and (p[6] == -1).all()


def test_random_numbers_at_their_ends():
    for form in ("chain", "draft", "tree"):
        x, tok, _, _, kw = _inputs(8, 4, 300, 8, form)
        for uv in (0.0, 1.0 - 2.0 ** -24):
            for pv in (0.0, 2.0 ** -149, 1.0 - 2.0 ** -24):
                _check(x, tok, torch.full((8, 3), uv), torch.full((8,), pv), kw)


def test_masked_and_infinite_logits():
    V = 130
    x, tok, u, pick, kw = _inputs(10, 3, V, 11)
    kw["temperatures"] = torch.full((10,), 0.7)
    kw["temperatures"][5:] = 0.0
    inf = float("inf")
    for o in (0, 5):
        x[o + 0, 0, 20:] = -inf              # a constrained vocabulary
        x[o + 1, :] = -inf                   # nothing left: column 0
        x[o + 2, 0, 7] = inf                 # all of the probability
        x[o + 2, 0, 99] = inf                # shared by two
        x[o + 3, :, ::2] = float("nan")
        x[o + 4, 0] = torch.finfo(torch.bfloat16).min
        x[o + 4, 0, 55] = -3e38
    tok[2, 0] = 99
    t, _, _ = _check(x, tok, u, pick, kw)
    assert t[1, 0] == 0 and t[6, 0] == 0 and t[7, 0] in (7, 99)
    # the draft's rows masked too: a token the draft could not have proposed stands
    x, tok, u, pick, kw = _inputs(6, 3, V, 12, "draft")
    kw["draft_logits"][0] = -inf
    kw["draft_logits"][1, :, 50:] = -inf
    kw["draft_logits"][2, 0, 3] = inf
    kw["draft_logits"][3, 0, ::3] = float("nan")
    _check(x, tok, u, pick, kw)


def test_ties_take_the_lowest_column():
    x = torch.zeros(2, 3, 5000, dtype=torch.bfloat16)
    x[:, :, [4000, 77, 2500]] = 3.0
    tok = torch.tensor([[77, 2500], [2500, 77]])
    t, p, a = _check(x, tok, torch.zeros(2, 2), torch.zeros(2), dict(temperatures=None))
    assert t[0].tolist() == [77, 77, -1] and t[1].tolist() == [77, -1, -1]
    x[:, :, 0] = -0.0  # equal to +0
    x[:, :, [4000, 77, 2500]] = -1.0
    t, _, _ = _check(x, tok, torch.zeros(2, 2), torch.zeros(2), dict(temperatures=None))
    assert (t[:, 0] == 0).all()


def test_drafts_that_are_the_target_all_stand():
    """p = q: u * q < p for every u < 1; with sums off in the last bits some would fall."""
    x, _, _, pick, kw = _inputs(64, 6, 40001, 13, "draft", noise=0.0)
    kw["draft_logits"] = x[:, :5].contiguous()
    kw["temperatures"] = torch.full((64,), 1.0)
    tok = x[:, :5].float().argmax(-1)
    u = torch.full((64, 5), 1.0 - 2.0 ** -24)
    _, _, a = _check(x, tok, u, pick, kw)
    assert (a == 5).all()


def test_rejected_siblings_take_all_but_one_token():
    """Two columns hold everything; the children are tried, twice the same one, until nothing is left."""
    x = torch.full((4, 4, 64), -200.0)
    x[:, :, 5], x[:, :, 9] = 1.0, 0.0
    x = x.to(torch.bfloat16)
    tok = torch.tensor([[5, 5, 9]] * 3 + [[9, 9, 9]])
    par = torch.tensor([[-1, 0, 0, 0]] * 4, dtype=torch.int32)
    u = torch.tensor([[0.99, 0.0, 0.999], [0.99, 0.99, 1 - 2.0 ** -24], [0.1, 0.1, 0.1],
                      [0.9, 0.0, 0.0]])
    _check(x, tok, u, torch.rand(4, generator=torch.Generator().manual_seed(1)),
           dict(temperatures=torch.ones(4), parents=par))


def test_tokens_and_parents_out_of_range_are_rejected():
    x, tok, u, pick, kw = _inputs(5, 4, 100, 15)
    tok[0, 0], tok[1, 0], tok[2, 1] = -1, 100, 2 ** 40
    _check(x, tok, torch.zeros_like(u), pick, kw)
    par = torch.tensor([[-1, 0, 9, 1], [-1, 1, 2, 3], [7, -5, 0, 0], [-1, 0, 0, 2], [-1, 3, 3, 0]],
                       dtype=torch.int32)
    tok = tok.clamp(0, 99)
    _check(x, tok, u, pick, dict(kw, parents=par))


def test_strided_and_unaligned_rows():
    """Logits as slices of a wider buffer at odd offsets and strides; a tree row shared by expand."""
    for form in ("draft", "tree"):
        x, tok, u, pick, kw = _inputs(3, 5, 997, 17, form)
        wide = torch.full((3, 7, 1003), 9.0, dtype=torch.bfloat16)
        wide[:, 1:6, 3:1000] = x
        got = {k: v.to(dev) for k, v in kw.items()}
        if form == "draft":
            dw = torch.full((3, 9, 1001), 9.0, dtype=torch.bfloat16)
            dw[:, ::2][:, :4, 1:998] = kw["draft_logits"]
            got["draft_logits"] = dw.to(dev)[:, ::2][:, :4, 1:998]
        out = ops.verify_draft(wide.to(dev)[:, 1:6, 3:1000], tok.to(dev), u.to(dev), pick.to(dev), **got)
        want = R.verify_draft(x, tok.numpy(), u.numpy(), pick.numpy(), **kw)
        for a, b in zip(out, want):
            assert np.array_equal(a.cpu().numpy(), b)


def test_largest_vocabulary_and_one_column():
    for form in ("chain", "draft"):
        _check(*_inputs(2, 3, 1 << 20, 18, form))
        x, tok, u, pick, kw = _inputs(2, 3, 1, 19, form, hot=1)
        _check(x, tok, u, pick, kw)


def test_argument_checks():
    x, tok, u, pick, kw = _inputs(2, 3, 16, 20)
    d = [t.to(dev) for t in (x, tok, u, pick)]
    with pytest.raises(ValueError, match="draft_tokens"):
        ops.verify_draft(d[0], d[1].int(), *d[2:])
    with pytest.raises(ValueError, match="u_accept"):
        ops.verify_draft(d[0], d[1], d[2][:, :1], d[3])
    with pytest.raises(TypeError, match="bfloat16"):
        ops.verify_draft(d[0].float(), *d[1:])
    with pytest.raises(ValueError, match="chain"):
        ops.verify_draft(*d, draft_logits=d[0][:, :2].contiguous(),
                         parents=torch.zeros(2, 3, dtype=torch.int32, device=dev))
    with pytest.raises(ValueError, match="parents"):
        ops.verify_draft(*d, parents=torch.zeros(3, dtype=torch.int32, device=dev))
    t, p, a = ops.verify_draft(d[0][:0], d[1][:0], d[2][:0], d[3][:0])
    assert t.shape == (0, 3) and a.numel() == 0


def test_graph_replay_and_two_streams():
    x, tok, u, pick, kw = _inputs(6, 5, 3001, 21, "draft")
    s = [t.to(dev) for t in (x, tok, u, pick)]
    k = {n: t.to(dev) for n, t in kw.items()}
    ops.verify_draft(*s, **k)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.verify_draft(*s, **k)
    for seed in (30, 31):
        y = _inputs(6, 5, 3001, seed, "draft")
        for dst, src in zip(s, y[:4]):
            dst.copy_(src)
        for n in k:
            k[n].copy_(y[4][n])
        graph.replay()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            beside = ops.verify_draft(*s, **k)
        torch.cuda.synchronize()
        want = R.verify_draft(y[0], y[1].numpy(), y[2].numpy(), y[3].numpy(), **y[4])
        for a, c, b in zip(out, beside, want):
            assert np.array_equal(a.cpu().numpy(), b) and np.array_equal(c.cpu().numpy(), b)


def test_extreme_temperatures():
    """From almost greedy (only ties of the top share) to flat, with masked columns: they are never drawn."""
    for form in ("chain", "draft", "tree"):
        x, tok, u, pick, kw = _inputs(12, 4, 777, 22, form)
        x[:, :, 100:] = float("-inf")
        x[3:6] = (x[3:6].float() * 1e-3).to(torch.bfloat16)
        x[6, :, 5:9] = 1.0
        tok = tok % 100
        kw["temperatures"] = torch.tensor([1e-38, 1e-30, 1e-6, 1e-20, 1e-4, 3e-3, 1e-7, 1e3, 1e8, 1e30,
                                           1e-45, 2e-4])
        for pv in (0.0, 0.37, 1.0 - 2.0 ** -24):
            _check(x, tok, u, torch.full((12,), pv), kw)


@pytest.mark.parametrize("V", [9, 255, 5000])
@pytest.mark.parametrize("gap", [3.0, 8.0, 16.0, 24.0])
def test_draft_rows_that_almost_agree(V, gap):
    """Peaked rows whose residual max(p - q, 0) is small (down to about 1e-10, still far above what 64-bit
    sums of p and q round off): drafts that q never gives are rejected and the residual drawn from."""
    g = torch.Generator().manual_seed(int(V + gap))
    B, n = 48, 4
    x = torch.randn(B, n, V, generator=g)
    x.scatter_(2, torch.randint(0, V, (B, n, 1), generator=g), gap)
    d = x[:, :n - 1].clone()
    other = torch.randint(0, V, (B, n - 1, 3), generator=g)
    d.scatter_(2, other, d.gather(2, other) - 1.0)  # the residual: columns that the draft has less of
    d.scatter_add_(2, other[..., :1].roll(1, 1), torch.full((B, n - 1, 1), 0.5))
    x, d = x.to(torch.bfloat16), d.to(torch.bfloat16)
    tok = x[:, :n - 1].float().argmin(-1)
    tok[:, 0] = x[:, 0].float().argmax(-1)
    u = torch.full((B, n - 1), 1.0 - 2.0 ** -24)
    u[:, 0] = 0.5
    _check(x, tok, u, torch.rand(B, generator=g), dict(temperatures=0.6 + torch.rand(B, generator=g),
                                                       draft_logits=d))


def test_draft_rows_that_agree_but_for_the_deep_tail():
    """Almost greedy rows with the same largest logit in both: the residual is a single column's weight,
    100 and more decimal orders below one."""
    g = torch.Generator().manual_seed(77)
    B, n, V = 24, 3, 255
    x = torch.randn(B, n, V, generator=g)
    d = x[:, :n - 1] + 0.1 * torch.randn(B, n - 1, V, generator=g)
    top = torch.randint(0, V, (B, 1, 1), generator=g)
    x.scatter_(2, top.expand(B, n, 1), 4.0 + torch.rand(B, n, 1, generator=g))
    d.scatter_(2, top.expand(B, n - 1, 1), 4.0 + torch.rand(B, n - 1, 1, generator=g))
    tok = x[:, :n - 1].float().argmin(-1)
    _check(x.to(torch.bfloat16), tok, torch.full((B, n - 1), 0.5), torch.rand(B, generator=g),
           dict(temperatures=torch.full((B,), 4e-3) + 4e-3 * torch.rand(B, generator=g),
                draft_logits=d.to(torch.bfloat16)))
