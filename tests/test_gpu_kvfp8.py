"""fp8 KV cache on the GPU: quantised scatter and read-back bit for bit against
the oracle, decode attention against 64 bits with a derived bound."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from helpers import cu, paged_layout
from oracle import reference_math as R

import nvattn
from nvattn import context as ctxmod
from nvattn import ops

pytestmark = pytest.mark.gpu
dev = torch.device("cuda")
SCALE = 128 ** -0.5


def u8(t):
    return t.view(torch.uint8)


def empty_cache(blocks, bs, kvh, byte=0x7F):
    """Pages of e4m3 NaN (stale bytes) with exponent bytes of 255."""
    c = torch.full((blocks, bs, kvh, 128), byte, dtype=torch.uint8, device=dev)
    s = torch.full((blocks, kvh, bs), 255, dtype=torch.uint8, device=dev)
    return c.view(torch.float8_e4m3fn), s


def filled_cache(blocks, bs, kvh, g, spread=0.0):
    """A random cache on the CPU: rows of magnitudes 2^(+-spread)."""
    x = torch.randn(blocks, bs, kvh, 128, generator=g)
    if spread:
        x = x * torch.exp2((2 * torch.rand(blocks, bs, kvh, 1, generator=g) - 1) * spread)
    q, e = R.quantise_rows_fp8(x.to(torch.bfloat16))
    return q, e.transpose(1, 2).contiguous()


def bound(ref, mag, cache_v_exp_max=None):
    """How far the kernel may be from fp64 (per element).

    Elements of K and V and their exponents are exact; q is off by 2^-25 of
    its row's largest element, S sums 128 products in fp32 (each partial sum
    off by 2^-24 of the magnitudes' total, and exp2's argument by two more
    roundings), so a score moves by at most 2 * 136 * 2^-24 * dot and a
    weight, and the sum of weights, by that relative amount each; ex2.approx
    adds 2^-22 and the f16 weight 2^-12, weights below 2^-14 of the largest
    2^-25 of it: sum_j 2^-25 |v8_j| 2^kv, at most n * 2^-25 * 448 * 2 times the
    largest mixed value an element can have; the O sum over n / 16 MMA steps
    2^-24 each; the output is rounded once to bf16, 2^-8."""
    score = 2 * 136 * 2.0 ** -24 * mag["dot"] + 2.0 ** -21
    rel = 2 * score + 2.0 ** -12 + (mag["n"] / 16 + 64) * 2.0 ** -24
    row = mag["mix"].amax(-1) + 2.0 ** -60
    return (2.0 ** -8 * ref.abs() + rel[..., None] * mag["mix"]
            + (mag["n"] * 2.0 ** -25 * 4 * row)[..., None])


def check(out, ref, mag, what=""):
    out = out.double().cpu()
    tol = bound(ref, mag)
    over = ((out - ref).abs() - tol).max().item()
    print(f"[fp8 decode] {what}: max-abs {(out - ref).abs().max():.3e}, margin {-over:.3e}")
    assert not torch.isnan(out).any() and over <= 0, f"{what}: beyond the bound by {over:.3g}"


# ------------------------------------------------------------------------ store

@pytest.mark.parametrize("N,kvh,bs", [(1, 1, 64), (3, 8, 256), (130, 2, 64), (1000, 5, 128)])
def test_store_matches_the_oracle_bit_for_bit(N, kvh, bs):
    g = torch.Generator().manual_seed(N)
    blocks = (N + bs - 1) // bs + 2
    # V as the strided view of a fused projection, K contiguous; magnitudes from 2^-40 to 2^40
    k = torch.randn(N, kvh, 128, generator=g) * torch.exp2(80 * torch.rand(N, kvh, 1, generator=g) - 40)
    qkv = torch.randn(N, 3 * kvh * 128, generator=g)
    k, qkv = k.to(torch.bfloat16), qkv.to(torch.bfloat16)
    v = qkv[:, 2 * kvh * 128:].view(N, kvh, 128)
    slots = torch.randperm(blocks * bs, generator=g)[:N].to(torch.int32)
    slots[::7] = -1
    kc, ks = empty_cache(blocks, bs, kvh, 0x11)
    vc, vs = empty_cache(blocks, bs, kvh, 0x22)
    want = [t.cpu().clone() for t in (u8(kc), u8(vc), ks, vs)]
    ops.store_kvcache_fp8(k.to(dev), qkv.to(dev)[:, 2 * kvh * 128:].view(N, kvh, 128), kc, vc, ks, vs,
                          slots.to(dev))
    for x, c, s in ((k, want[0], want[2]), (v, want[1], want[3])):
        q, e = R.quantise_rows_fp8(x)
        for i, slot in enumerate(slots.tolist()):
            if slot >= 0:
                c[slot // bs, slot % bs] = u8(q)[i]
                s[slot // bs, :, slot % bs] = e[i]
    for got, w in zip((u8(kc), u8(vc), ks, vs), want):
        assert torch.equal(got.cpu(), w)
    assert ops.read_status() == 0


def test_store_edge_rows_and_unaligned_views():
    """Zero, subnormal, largest, infinite and NaN rows; token strides that are not 16-byte multiples."""
    rows = torch.zeros(8, 1, 128)
    rows[1, 0, 3] = 448.0
    rows[2, 0, 3] = 450.0
    rows[3, 0, 127] = float("-inf")
    rows[4, 0, 0] = float("nan")
    rows[5, 0] = 2.0 ** -133
    rows[6, 0] = torch.linspace(-3.3e38, 3.3e38, 128)
    rows[7, 0] = torch.arange(128) / 64.0
    buf = torch.zeros(8, 131).to(torch.bfloat16)
    buf[:, 1:129] = rows.view(8, 128).to(torch.bfloat16)
    x = buf.to(dev)[:, 1:129].unflatten(1, (1, 128))
    kc, ks = empty_cache(1, 64, 1)
    vc, vs = empty_cache(1, 64, 1)
    ops.store_kvcache_fp8(x, x, kc, vc, ks, vs, torch.arange(8, dtype=torch.int32, device=dev))
    q, e = R.quantise_rows_fp8(rows.to(torch.bfloat16))
    assert torch.equal(u8(kc).cpu()[0, :8], u8(q)) and torch.equal(ks.cpu()[0, :, :8], e.T)
    assert torch.equal(u8(vc).cpu(), u8(kc).cpu()) and torch.equal(vs, ks)


def test_store_skips_and_flags_bad_slots():
    x = torch.ones(4, 2, 128, dtype=torch.bfloat16, device=dev)
    kc, ks = empty_cache(2, 64, 2)
    vc, vs = empty_cache(2, 64, 2)
    before = u8(kc).clone()
    ops.read_status()
    ops.store_kvcache_fp8(x, x, kc, vc, ks, vs,
                          torch.tensor([-1, 128, -7, 2 ** 30], dtype=torch.int32, device=dev))
    assert torch.equal(u8(kc), before) and (ks == 255).all()
    assert ops.read_status() == nvattn._lib.STATUS_BAD_SLOT
    ops.store_kvcache_fp8(x[:0], x[:0], kc, vc, ks, vs, torch.empty(0, dtype=torch.int32, device=dev))
    assert ops.read_status() == 0


# ------------------------------------------------------------------------- load

@pytest.mark.parametrize("lens,kvh,bs", [([1], 1, 64), ([0, 5, 0, 0, 700, 1], 2, 256),
                                         ([63, 64, 65, 129], 8, 64), ([1000, 0], 5, 512)])
def test_load_is_exact(lens, kvh, bs):
    g = torch.Generator().manual_seed(len(lens))
    blocks, bt = paged_layout(lens, bs, seed=3)
    kc, ks = filled_cache(blocks, bs, kvh, g, spread=30)
    vc, vs = filled_cache(blocks, bs, kvh, g)
    total = sum(lens) + 9  # rows behind the last sequence stay
    k_out = torch.full((total, kvh, 128), 7.0, dtype=torch.bfloat16, device=dev)
    v_out = k_out.clone()
    ops.read_status()
    got = ops.load_kvcache_fp8(kc.to(dev), vc.to(dev), ks.to(dev), vs.to(dev), cu(lens).to(dev),
                               bt.to(dev), total, k_out, v_out)
    assert got[0] is k_out and got[1] is v_out and ops.read_status() == 0
    for out, c, s in ((k_out, kc, ks), (v_out, vc, vs)):
        val = R.expand_cache_fp8(c, s)
        at = 0
        for b, n in enumerate(lens):
            want = R.gather_paged(val, bt[b].numpy(), n)
            assert torch.equal(out[at:at + n].cpu().double(), want)
            at += n
        assert (out[at:] == 7.0).all()


def test_load_zeroes_the_rest_of_new_outputs():
    """A dense prefill over the rows reads a little past each sequence: what is there must be finite."""
    g = torch.Generator().manual_seed(6)
    kc, ks = filled_cache(2, 64, 2, g)
    args = [t.to(dev) for t in (kc, kc, ks, ks)]
    bt = torch.tensor([[0, 1]], dtype=torch.int32, device=dev)
    for _ in range(4):  # the allocator hands these blocks out again
        poison = [torch.full((300, 2, 128), float("nan"), dtype=torch.bfloat16, device=dev)
                  for _ in range(3)]
        del poison
        k, v = ops.load_kvcache_fp8(*args, cu([100]).to(dev), bt, 300)
        assert (k[100:] == 0).all() and (v[100:] == 0).all()
        assert torch.isfinite(k.float()).all() and torch.isfinite(v.float()).all()


def test_load_bad_pages_give_zeros_and_a_flag():
    g = torch.Generator().manual_seed(1)
    kc, ks = filled_cache(3, 64, 2, g)
    bt = torch.tensor([[1, 99], [0, 2]], dtype=torch.int32)
    lens = [100, 200]  # the first has a page outside, the second runs past its table
    ops.read_status()
    k, v = ops.load_kvcache_fp8(kc.to(dev), kc.to(dev), ks.to(dev), ks.to(dev), cu(lens).to(dev),
                                bt.to(dev), 300)
    assert ops.read_status() == nvattn._lib.STATUS_BAD_BLOCK
    val = R.expand_cache_fp8(kc, ks)
    assert torch.equal(k[:64].cpu().double(), val[1]) and (k[64:100] == 0).all()
    assert torch.equal(v[100:228].cpu().double(), torch.cat([val[0], val[2]])) and (v[228:] == 0).all()


# ----------------------------------------------------------------------- decode

def _decode(lens, H, kvh, bs=256, seed=0, spread=0.0, stale=0x7F, pad_width=0, qmul=1.0):
    g = torch.Generator().manual_seed(seed)
    blocks, bt = paged_layout(lens, bs, seed=seed)
    if pad_width:
        bt = torch.cat([bt, torch.full((len(lens), pad_width), -1, dtype=torch.int32)], 1)
    kc, ks = filled_cache(blocks, bs, kvh, g, spread=min(spread, 2.0))
    vc, vs = filled_cache(blocks, bs, kvh, g, spread=spread)
    for b, n in enumerate(lens):  # stale bytes past each end: NaN elements, NaN exponents
        for j in range(n, -(-n // bs) * bs):
            blk, off = int(bt[b, j // bs]), j % bs
            for c, s in ((kc, ks), (vc, vs)):
                u8(c)[blk, off] = stale
                s[blk, :, off] = 255
    q = (torch.randn(len(lens), H, 128, generator=g) * qmul).to(torch.bfloat16)
    sl = torch.tensor(lens, dtype=torch.int32)
    ops.read_status()
    out = ops.paged_decode_fp8(q.to(dev), kc.to(dev), vc.to(dev), ks.to(dev), vs.to(dev), sl.to(dev),
                               bt.to(dev), softmax_scale=SCALE)
    assert ops.read_status() == 0
    val = [torch.nan_to_num(R.expand_cache_fp8(c, s)) for c, s in ((kc, ks), (vc, vs))]
    ref, mag = R.decode_attention_f64(q, *val, lens, bt.clamp_min(0), SCALE)
    return out, ref, mag


@pytest.mark.parametrize("H,kvh", [(16, 8), (8, 8), (32, 8), (5, 1), (16, 1), (24, 2)])
def test_decode_groups(H, kvh):
    lens = np.random.default_rng(H).integers(1, 900, size=5).tolist()
    check(*_decode(lens, H, kvh, seed=H), what=f"{H}/{kvh}")


@pytest.mark.parametrize("bs", [64, 128, 256, 512])
def test_decode_lengths_around_tiles_and_pages(bs):
    lens = [1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 255, 256, 257, 511, 512, 513, 700]
    check(*_decode(lens, 4, 2, bs=bs, seed=bs), what=f"block {bs}")


def test_decode_empty_rows_give_zeros():
    out, ref, mag = _decode([0, 300, 0, 1], 8, 4, seed=2)
    assert (out[0] == 0).all() and (out[2] == 0).all()
    check(out, ref, mag)
    # one split covers the table: the kernel itself writes the zeros
    lens = [0, 200] * 300
    assert ops.decode_fp8_workspace_bytes(600, 4, 2, 1, 256) == 0
    out, ref, mag = _decode(lens, 4, 2, seed=3)
    assert (out[::2] == 0).all()
    check(out, ref, mag)


def test_decode_values_of_very_different_magnitudes():
    """V rows from 2^-50 to 2^50 and steep scores: the weights' reference follows score and exponent."""
    check(*_decode([700, 64, 333], 8, 2, seed=4, spread=50, qmul=4.0), what="spread 2^50")


def test_decode_all_zero_values_and_far_scores():
    """V rows of zeros carry the smallest exponent; rows next to them keep their weight."""
    g = torch.Generator().manual_seed(9)
    k = torch.randn(1, 64, 1, 128, generator=g).to(torch.bfloat16)
    v = torch.zeros(1, 64, 1, 128, dtype=torch.bfloat16)
    v[0, 1::2] = torch.randn(32, 1, 128, generator=g).to(torch.bfloat16) * 2.0 ** 40
    (kc, ks), (vc, vs) = R.quantise_rows_fp8(k), R.quantise_rows_fp8(v)
    ks, vs = ks.transpose(1, 2).contiguous(), vs.transpose(1, 2).contiguous()
    q = torch.randn(1, 4, 128, generator=g).to(torch.bfloat16)
    bt = torch.zeros(1, 1, dtype=torch.int32)
    for n in (1, 2, 64):
        out = ops.paged_decode_fp8(q.to(dev), kc.to(dev), vc.to(dev), ks.to(dev), vs.to(dev),
                                   torch.tensor([n], dtype=torch.int32, device=dev), bt.to(dev))
        ref, mag = R.decode_attention_f64(q, R.expand_cache_fp8(kc, ks), R.expand_cache_fp8(vc, vs),
                                          [n], bt, SCALE)
        check(out, ref, mag, f"{n} keys")


def test_decode_extreme_queries():
    """q rows of 2^-100 and 2^60 next to ordinary ones (with a scale that brings them back)."""
    g = torch.Generator().manual_seed(11)
    kc, ks = filled_cache(2, 64, 1, g)
    vc, vs = filled_cache(2, 64, 1, g)
    q = torch.randn(1, 3, 128, generator=g)
    q[0, 1] *= 2.0 ** -100
    q[0, 2] = 0
    q = q.to(torch.bfloat16)
    bt = torch.tensor([[1, 0]], dtype=torch.int32)
    for mul, scale in ((1.0, SCALE), (2.0 ** 60, SCALE * 2.0 ** -60)):
        qq = (q.float() * mul).to(torch.bfloat16)
        out = ops.paged_decode_fp8(qq.to(dev), kc.to(dev), vc.to(dev), ks.to(dev), vs.to(dev),
                                   torch.tensor([100], dtype=torch.int32, device=dev), bt.to(dev),
                                   softmax_scale=scale)
        ref, mag = R.decode_attention_f64(qq, R.expand_cache_fp8(kc, ks), R.expand_cache_fp8(vc, vs),
                                          [100], bt, scale)
        check(out, ref, mag, f"q x {mul}")


def test_decode_nan_rows_reach_only_their_sequence():
    g = torch.Generator().manual_seed(12)
    kc, ks = filled_cache(2, 64, 1, g)
    vc, vs = filled_cache(2, 64, 1, g)
    u8(kc)[0, 10], ks[0, 0, 10] = 0x7F, 255
    q = torch.randn(2, 2, 128, generator=g).to(torch.bfloat16)
    out = ops.paged_decode_fp8(q.to(dev), kc.to(dev), vc.to(dev), ks.to(dev), vs.to(dev),
                               torch.tensor([20, 64], dtype=torch.int32, device=dev),
                               torch.tensor([[0], [1]], dtype=torch.int32, device=dev))
    assert torch.isnan(out[0].float()).all() and not torch.isnan(out[1].float()).any()


def test_decode_long_and_wide_tables():
    check(*_decode([20000], 16, 1, seed=21), what="20000 keys, 16 heads")
    lens = np.random.default_rng(24).integers(1, 2000, size=24).tolist()
    check(*_decode(lens, 4, 2, seed=24, pad_width=56), what="wide table")


def test_decode_strided_inputs_and_bad_pages():
    """q and out as slices, the table as a slice of a wider one; bad block ids and lengths past the
    table are flagged."""
    g = torch.Generator().manual_seed(31)
    kc, ks = filled_cache(4, 64, 2, g)
    vc, vs = filled_cache(4, 64, 2, g)
    qkv = torch.randn(2, 8 * 128, generator=g).to(torch.bfloat16)
    q = qkv.to(dev)[:, :512].view(2, 4, 128)
    wide = torch.tensor([[9, 0, 1, 9], [9, 3, 2, 9]], dtype=torch.int32)
    buf = torch.full((2, 4, 256), 5.0, dtype=torch.bfloat16, device=dev)
    sl = torch.tensor([100, 128], dtype=torch.int32)
    args = [t.to(dev) for t in (kc, vc, ks, vs)]
    out = ops.paged_decode_fp8(q, *args, sl.to(dev), wide.to(dev)[:, 1:3], out=buf[:, :, :128])
    ref, mag = R.decode_attention_f64(qkv[:, :512].view(2, 4, 128), R.expand_cache_fp8(kc, ks),
                                      R.expand_cache_fp8(vc, vs), sl, wide[:, 1:3], SCALE)
    check(out, ref, mag)
    assert (buf[:, :, 128:] == 5.0).all() and ops.read_status() == 0
    ops.paged_decode_fp8(q, *args, sl.to(dev), wide.to(dev)[:, :2].contiguous())
    assert ops.read_status() == nvattn._lib.STATUS_BAD_BLOCK
    ops.paged_decode_fp8(q, *args, torch.tensor([100, 129], dtype=torch.int32, device=dev),
                         wide.to(dev)[:, 1:3])
    assert ops.read_status() == nvattn._lib.STATUS_BAD_BLOCK


def test_decode_graph_and_other_stream():
    g = torch.Generator().manual_seed(13)
    B, H, kvh, bs, width = 6, 8, 2, 128, 10
    blocks = B * width
    kc, ks = filled_cache(blocks, bs, kvh, g)
    vc, vs = filled_cache(blocks, bs, kvh, g)
    args = [t.to(dev) for t in (kc, vc, ks, vs)]
    val = [R.expand_cache_fp8(kc, ks), R.expand_cache_fp8(vc, vs)]
    q = torch.zeros(B, H, 128, dtype=torch.bfloat16, device=dev)
    lens = torch.zeros(B, dtype=torch.int32, device=dev)
    bt = torch.zeros(B, width, dtype=torch.int32, device=dev)
    ops.status_tensor()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.paged_decode_fp8(q, *args, lens, bt)
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):  # two graphs, each with its own workspace from its pool
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = ops.paged_decode_fp8(q, *args, lens, bt)
        graphs.append((graph, out))
    for trial in range(2):
        rng = np.random.default_rng(trial)
        new = rng.integers(0, width * bs, size=B).astype(np.int32)
        perm = torch.from_numpy(rng.permutation(blocks).reshape(B, width).astype(np.int32))
        qn = torch.randn(B, H, 128, generator=g).to(torch.bfloat16)
        q.copy_(qn), lens.copy_(torch.from_numpy(new)), bt.copy_(perm)
        for graph, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        ref, mag = R.decode_attention_f64(qn, *val, new, perm, SCALE)
        for _, out in graphs:
            check(out, ref, mag, "replay")


# ------------------------------------------------------------------ the operators together

def test_attention_module_with_an_fp8_cache():
    """Prefill, prefix-cache prefill and decode steps through nvattn.Attention bound to an fp8 cache,
    against 64 bits over the values that the cache stands for."""
    H, KVH, bs = 8, 2, 256
    g = torch.Generator().manual_seed(5)
    attn = nvattn.Attention(H, 128, SCALE, KVH)
    attn.k_cache, attn.k_scale = empty_cache(6, bs, KVH)
    attn.v_cache, attn.v_scale = empty_cache(6, bs, KVH)
    lens, bt = [300, 70], torch.tensor([[4, 1], [2, 5]], dtype=torch.int32)

    def rows(b, lo, hi):
        return [int(bt[b, p // bs]) * bs + p % bs for p in range(lo, hi)]

    def values():
        return [torch.nan_to_num(R.expand_cache_fp8(c.cpu(), s.cpu()))
                for c, s in ((attn.k_cache, attn.k_scale), (attn.v_cache, attn.v_scale))]

    def step(n):
        return [torch.randn(n, h, 128, generator=g).to(torch.bfloat16) for h in (H, KVH, KVH)]

    ops.read_status()
    # fresh prompts: dense prefill over the projections themselves
    q, k, v = step(sum(lens))
    slots = torch.tensor(rows(0, 0, 300) + rows(1, 0, 70), dtype=torch.int32, device=dev)
    c = cu(lens).to(dev)
    ctxmod.set_context(True, c, c, 300, 300, slots)
    o = attn(q.to(dev), k.to(dev), v.to(dev))
    ref = R.varlen_attention(q, k, v, c.cpu().numpy(), c.cpu().numpy(), SCALE, True)
    assert (o.float().cpu() - ref).abs().max() <= 1e-2 + 2.0 ** -8 * ref.abs().max()
    # continuation chunks over the cache
    add = [40, 3]
    q, k, v = step(sum(add))
    tot = [n + a for n, a in zip(lens, add)]
    slots = torch.tensor(rows(0, 300, 340) + rows(1, 70, 73), dtype=torch.int32, device=dev)
    cq, ck = cu(add), cu(tot)
    ctxmod.set_context(True, cq.to(dev), ck.to(dev), 40, 340, slots, None, bt.to(dev))
    o = attn(q.to(dev), k.to(dev), v.to(dev))
    kv = [torch.cat([R.gather_paged(x, bt[b].numpy(), n) for b, n in enumerate(tot)]).to(torch.bfloat16)
          for x in values()]
    ref = R.varlen_attention(q, *kv, cq.numpy(), ck.numpy(), SCALE, True)
    assert (o.float().cpu() - ref).abs().max() <= 1e-2 + 2.0 ** -8 * ref.abs().max()
    # decode steps
    for _ in range(3):
        tot = [n + 1 for n in tot]
        q, k, v = step(2)
        slots = torch.tensor([rows(b, n - 1, n)[0] for b, n in enumerate(tot)], dtype=torch.int32)
        ctxmod.set_context(False, slot_mapping=slots.to(dev),
                           context_lens=torch.tensor(tot, dtype=torch.int32, device=dev),
                           block_tables=bt.to(dev))
        o = attn(q.to(dev), k.to(dev), v.to(dev))
        assert o.shape == (2, 1, H, 128)
        ref, mag = R.decode_attention_f64(q, *values(), tot, bt, SCALE)
        check(o[:, 0], ref, mag, "module step")
    ctxmod.reset_context()
    assert ops.read_status() == 0


@pytest.mark.parametrize("keys", [1, 700, 1 << 18])
def test_module_prefill_reads_back_in_groups(monkeypatch, keys):
    """A ragged prefix-cache prefill over an fp8 cache, read back one sequence at a time, two at a
    time and all together (one sequence has no new tokens)."""
    from nvattn import attention as attention_module
    monkeypatch.setattr(attention_module, "READ_BACK_KEYS", keys)
    H, KVH, bs = 4, 2, 64
    g = torch.Generator().manual_seed(77)
    tot, add = [300, 1, 130, 64, 257], [7, 1, 0, 64, 33]
    attn = nvattn.Attention(H, 128, SCALE, KVH)
    caches, bt = [], torch.arange(30, dtype=torch.int32).flip(0).view(5, 6)[:, :5].contiguous()
    for name in "kv":
        q, e = filled_cache(30, bs, KVH, g)
        caches.append(R.expand_cache_fp8(q, e))
        setattr(attn, f"{name}_cache", q.to(dev))
        setattr(attn, f"{name}_scale", e.to(dev))
    n = sum(add)
    q, k, v = [torch.randn(n, h, 128, generator=g).to(torch.bfloat16) for h in (H, KVH, KVH)]
    cq, ck = cu(add), cu(tot)
    skip = torch.full((n,), -1, dtype=torch.int32, device=dev)  # the keys are there already
    ctxmod.set_context(True, cq.to(dev), ck.to(dev), max(add), max(tot), skip, None, bt.to(dev))
    ops.read_status()
    o = attn(q.to(dev), k.to(dev), v.to(dev))
    ctxmod.reset_context()
    kv = [torch.cat([R.gather_paged(c, bt[b].numpy(), m) for b, m in enumerate(tot)]).to(torch.bfloat16)
          for c in caches]
    ref = R.varlen_attention(q, *kv, cq.numpy(), ck.numpy(), SCALE, True)
    assert (o.float().cpu() - ref).abs().max() <= 1e-2 + 2.0 ** -8 * ref.abs().max()
    assert ops.read_status() == 0


def test_module_fused_step_equals_the_separate_one():
    """forward_fused bound to an fp8 cache: its cache bytes and outputs are those of forward on the
    normalised, rotated q and k."""
    H, KVH, bs, n = 8, 2, 64, 3
    g = torch.Generator().manual_seed(78)
    qkv = torch.randn(n, (H + 2 * KVH) * 128, generator=g).to(torch.bfloat16).to(dev)
    q, k, v = [t.view(n, -1, 128) for t in qkv.split([H * 128, KVH * 128, KVH * 128], -1)]
    w = torch.randn(2, 128, generator=g).to(torch.bfloat16).to(dev)
    angles = torch.rand(100, 1, 64, generator=g)
    table = torch.cat([angles.cos(), angles.sin()], -1).to(dev)
    pos = torch.tensor([0, 70, 33], device=dev)
    bt = torch.tensor([[5, 0], [1, 4], [3, 2]], dtype=torch.int32, device=dev)
    slots = torch.tensor([5 * bs, 4 * bs + 6, 3 * bs + 33], dtype=torch.int32, device=dev)
    lens = torch.tensor([1, 71, 34], dtype=torch.int32, device=dev)
    start = [filled_cache(6, bs, KVH, g) for _ in "kv"]
    results = []
    for fused in (True, False):
        attn = nvattn.Attention(H, 128, SCALE, KVH)
        (attn.k_cache, attn.k_scale), (attn.v_cache, attn.v_scale) = [
            (c.to(dev), s.to(dev)) for c, s in start]
        ctxmod.set_context(False, slot_mapping=slots, context_lens=lens, block_tables=bt)
        if fused:
            o = attn.forward_fused(pos, q, k, v, w[0], w[1], table, 1e-6)
        else:
            o = attn(*ops.qk_norm_rope_store(pos, q, k, v, w[0], w[1], table, 1e-6), v)
        results.append([o, u8(attn.k_cache), u8(attn.v_cache), attn.k_scale, attn.v_scale])
    ctxmod.reset_context()
    for a, b in zip(*results):
        assert torch.equal(a, b)
    changed = (results[0][1] != u8(start[0][0]).to(dev)).flatten(2).any(-1).view(-1).nonzero()
    assert set(changed.flatten().tolist()) <= set(slots.tolist()) and len(changed)


def test_load_of_no_sequences_gives_zeros():
    kc, ks = empty_cache(2, 64, 3)
    none = torch.zeros(1, dtype=torch.int32, device=dev)
    k, v = ops.load_kvcache_fp8(kc, kc, ks, ks, none, none.new_empty(0, 4), 5)
    assert k.shape == (5, 3, 128) and not k.any() and not v.any()


def test_single_rows_whose_strides_are_arbitrary():
    """One sequence: torch leaves the stride of a dimension of size one at any value."""
    H, kvh, bs, n = 4, 2, 128, 300
    g = torch.Generator().manual_seed(91)
    (kc, ks), (vc, vs) = [filled_cache(4, bs, kvh, g) for _ in "kv"]
    q = torch.randn(1, H, 128, generator=g).to(torch.bfloat16)
    bt = torch.tensor([[3, 1, 0]], dtype=torch.int32)
    ref, mag = R.decode_attention_f64(q, R.expand_cache_fp8(kc, ks), R.expand_cache_fp8(vc, vs), [n], bt,
                                      SCALE)
    odd_q = torch.as_strided(q.to(dev), (1, H, 128), (3, 128, 1))
    odd_bt = torch.as_strided(bt.to(dev), (1, 3), (1, 1))
    c = [t.to(dev) for t in (kc, vc, ks, vs)]
    lens = torch.tensor([n], dtype=torch.int32, device=dev)
    check(ops.paged_decode_fp8(odd_q, *c, lens, odd_bt, softmax_scale=SCALE), ref, mag, "one row")
    out = ops.shared_prefix_decode(odd_q, c[0], c[1], lens, odd_bt, bs, SCALE, c[2], c[3])
    assert (out.double().cpu() - ref).abs().max() <= 1e-2 + 2.0 ** -8 * ref.abs().max()
    k, _ = ops.load_kvcache_fp8(*c, cu([n]).to(dev), odd_bt, n)
    assert torch.equal(k[:bs].double().cpu(), R.expand_cache_fp8(kc, ks)[3])
