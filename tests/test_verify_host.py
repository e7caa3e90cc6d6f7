"""Draft verification, host side: the oracle's walk keeps the target's law, and
every refusal of the C entry point and the operator (no GPU needed)."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from oracle import reference_math as R

from nvattn import _lib, ops

FAKE = ctypes.c_void_p(0x10000)


def _first_tokens(N, V, make):
    """Empirical law of the first emitted token over N draws, against the target's."""
    rng = np.random.default_rng(0)
    counts, p = np.zeros(V), None
    for _ in range(N):
        args, p = make(rng)
        t, _, _ = R.verify_draft(*args[0], **args[1])
        counts[t[0, 0]] += 1
    # each count is binomial: six standard deviations over V columns
    sd = np.sqrt(N * p * (1 - p)) + 1
    assert (np.abs(counts - N * p) < 6 * sd).all()


def test_oracle_keeps_the_targets_law_with_draft_logits():
    V = 6
    t = torch.tensor([[[1.0, 0.2, -1.0, 0.5, 2.0, -3.0], [0.0] * V]]).to(torch.bfloat16)
    d = torch.tensor([[[0.1, 1.5, -1.0, 0.0, 1.0, 0.3]]]).to(torch.bfloat16)
    q = R.verify_law(d[0, 0], 0.8)

    def make(rng):
        x = np.array([[rng.choice(V, p=q)]])
        u = rng.random((1, 1)), rng.random(1)
        return ((t, x, *u), dict(temperatures=[0.8], draft_logits=d)), R.verify_law(t[0, 0], 0.8)
    _first_tokens(6000, V, make)


def test_oracle_keeps_the_targets_law_for_trees():
    V = 5
    t = torch.tensor([[[1.0, 0.2, -1.0, 0.5, 2.0]] * 4]).to(torch.bfloat16)
    tok = np.array([[4, 0, 4]])  # three children of the root, one of them twice

    def make(rng):
        return (((t, tok, rng.random((1, 3)), rng.random(1)),
                 dict(temperatures=[1.0], parents=np.array([[-1, 0, 0, 0]]))),
                R.verify_law(t[0, 0], 1.0))
    _first_tokens(6000, V, make)


def test_oracle_greedy_walk_equals_the_host_helper():
    from nvattn import tree
    rng = np.random.default_rng(1)
    par, _ = tree.build_draft_tree((3, 2, 1), 10)
    for seed in range(20):
        logits = torch.from_numpy(rng.standard_normal((1, 10, 4))).to(torch.bfloat16)
        tok = rng.integers(0, 4, (1, 9))
        t, path, num = R.verify_draft(logits, tok, np.zeros((1, 9)), np.zeros(1),
                                      parents=par[None])
        want = tree.greedy_accept(par, np.concatenate([[0], tok[0]]),
                                  logits[0].float().argmax(-1).numpy())
        assert path[0, :num[0] + 1].tolist() == want


def _call(batch=2, nodes=4, vocab=100, logits=FAKE, draft=None, parents=None, stride=1, tok=FAKE):
    return _lib.load().nvattn_verify_draft(logits, 400, 100 * stride, draft, 300, 100, tok, parents, 0,
                                           FAKE, FAKE, None, None, batch, nodes, vocab, FAKE, FAKE,
                                           FAKE, None)


def test_c_refusals():
    lib = _lib.load()
    assert _call(batch=0, logits=None) == _lib.OK and _call(nodes=0, logits=None) == _lib.OK
    for kw, code, text in ((dict(batch=-1), _lib.ERR_INVALID, b"negative size"),
                           (dict(logits=None), _lib.ERR_INVALID, b"NULL"),
                           (dict(tok=None), _lib.ERR_INVALID, b"NULL"),
                           (dict(nodes=65), _lib.ERR_UNSUPPORTED, b"64 nodes"),
                           (dict(vocab=0), _lib.ERR_INVALID, b"vocab"),
                           (dict(vocab=2 ** 20 + 1), _lib.ERR_UNSUPPORTED, b"2^20"),
                           (dict(draft=FAKE, parents=FAKE), _lib.ERR_UNSUPPORTED, b"chain"),
                           (dict(stride=-1), _lib.ERR_INVALID, b"negative stride"),
                           (dict(logits=ctypes.c_void_p(0x10001)), _lib.ERR_INVALID, b"2-byte"),
                           (dict(batch=2 ** 30), _lib.ERR_INVALID, b"batch too large")):
        assert _call(**kw) == code and text in lib.nvattn_last_error(), (kw, lib.nvattn_last_error())


def test_operator_refuses_cpu_tensors():
    x = torch.zeros(1, 2, 8, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        ops.verify_draft(x, torch.zeros(1, 1, dtype=torch.int64), torch.zeros(1, 1), torch.zeros(1))
