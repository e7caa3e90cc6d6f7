"""Decode over a shared prefix on the GPU against 64 bits, bf16 and fp8 caches, and
the serving-step operators run together."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import reference_math as R

import nvattn
from nvattn import ops, tree

pytestmark = pytest.mark.gpu
dev = torch.device("cuda")
SCALE = 128 ** -0.5


def bound(ref, mag):
    """How far the kernels may be from fp64 (per element). Scores sum 128 bf16 or
    e4m3 products in fp32 and exp2's argument is rounded twice more: 2 * 136 *
    2^-24 * dot; exp2 is the MUFU's (2^-22) or the prefix kernel's polynomial
    (7.5e-5), in the weight and in the sum; weights go to the tensor cores as
    bf16 (2^-8); sums over n keys in fp32, 2^-24 each of n / 16 steps, rescales
    and merges a few more; one rounding of the output to bf16, 2^-8."""
    rel = 2 * (2 * 136 * 2.0 ** -24 * mag["dot"] + 7.5e-5) + 2.0 ** -8 \
        + (mag["n"] / 16 + 256) * 2.0 ** -24
    return 2.0 ** -8 * ref.abs() + rel[..., None] * mag["mix"]


def check(out, ref, mag, what=""):
    out = out.double().cpu()
    over = ((out - ref).abs() - bound(ref, mag)).max().item()
    print(f"[shared prefix] {what}: max-abs {(out - ref).abs().max():.3e}, margin {-over:.3e}")
    assert not torch.isnan(out).any() and over <= 0, f"{what}: beyond the bound by {over:.3g}"


def build(B, kvh, bs, shared, lens, fp8, seed, width=0, stale=True):
    """Caches on the CPU, block tables with the shared pages first in every row with that many
    keys, all other pages distinct; bytes past each end are NaN."""
    g = torch.Generator().manual_seed(seed)
    ns = shared // bs
    need = [max(0, -(-n // bs) - (ns if n >= shared else 0)) for n in lens]
    pages = ns + sum(need) + 1
    ids = torch.randperm(pages, generator=g).to(torch.int32)
    w = max([ns] + [d + (ns if n >= shared else 0) for d, n in zip(need, lens)] + [1, width])
    bt = torch.full((B, w), -1, dtype=torch.int32)
    bt[0, :ns] = ids[:ns]
    at = ns
    for b, n in enumerate(lens):
        start = 0
        if n >= shared:
            bt[b, :ns] = ids[:ns]
            start = ns
        bt[b, start:start + need[b]] = ids[at:at + need[b]]
        at += need[b]
    vals = []
    for _ in range(2):
        x = torch.randn(pages, bs, kvh, 128, generator=g).to(torch.bfloat16)
        vals.append(x)
    if fp8:
        caches, scales = [], []
        for x in vals:
            q, e = R.quantise_rows_fp8(x)
            caches.append(q)
            scales.append(e.transpose(1, 2).contiguous())
        vals = [R.expand_cache_fp8(c, s) for c, s in zip(caches, scales)]
    else:
        caches, scales = [x.clone() for x in vals], [None, None]
    for b, n in enumerate(lens):
        if not stale or n == 0 or n % bs == 0:
            continue
        blk = int(bt[b, n // bs])
        for c, s in zip(caches, scales):
            if fp8:
                c.view(torch.uint8)[blk, n % bs:] = 0x7F
                s[blk, :, n % bs:] = 255
            else:
                c[blk, n % bs:] = float("nan")
    return caches, scales, vals, bt


def run(q, caches, scales, lens, bt, shared, **kw):
    to = lambda t: None if t is None else t.to(dev)  # noqa: E731
    return ops.shared_prefix_decode(to(q), *map(to, caches), torch.tensor(lens, dtype=torch.int32).to(dev),
                                    to(bt), shared, softmax_scale=SCALE, k_scale=to(scales[0]),
                                    v_scale=to(scales[1]), **kw)


def apart(lens, kvh, shared, fp8):
    """Padding rows that bring a batch past the size from which the prefix is attended apart from
    the own keys: 32 MB of K and V read once a row (64 MB in fp8)."""
    need = (64 << 20) // (258 * kvh * shared) if fp8 else (32 << 20) // (512 * kvh * shared)
    return list(lens) + [0] * max(0, need + 1 - len(lens))


def case(B, H, kvh, bs, shared, lens, fp8, seed=0, **kw):
    caches, scales, vals, bt = build(B, kvh, bs, shared, lens, fp8, seed, **kw)
    q = torch.randn(B, H, 128, generator=torch.Generator().manual_seed(seed + 1)).to(torch.bfloat16)
    ops.read_status()
    out = run(q, caches, scales, lens, bt, shared)
    assert ops.read_status() == 0
    ref, mag = R.decode_attention_f64(q, *vals, lens, bt.clamp_min(0), SCALE)
    check(out, ref, mag, f"B{B} {H}/{kvh} block {bs} prefix {shared}{' fp8' if fp8 else ''}")
    return out


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("B,H,kvh,bs,shared", [(1, 8, 8, 128, 128), (3, 16, 8, 256, 512),
                                               (5, 5, 1, 128, 384), (20, 16, 1, 256, 256),
                                               (70, 8, 2, 128, 1280), (9, 24, 2, 512, 1024)])
def test_equals_64_bits(B, H, kvh, bs, shared, fp8):
    own = np.random.default_rng(B).integers(1, 400, size=B)
    lens = (shared + own).tolist()
    case(B, H, kvh, bs, shared, lens, fp8, seed=B)
    lens = apart(lens, kvh, shared, fp8)
    case(len(lens), H, kvh, bs, shared, lens, fp8, seed=B)


@pytest.mark.parametrize("fp8", [False, True])
def test_own_lengths_around_tiles_and_short_rows(fp8):
    """No own key, one, tile edges; padding rows; rows with fewer keys than the prefix."""
    shared = 512
    lens = [shared + n for n in (1, 0, 63, 64, 65, 127, 128, 129, 300)] + [0, 1, 64, 511, 0, 200]
    for lens in (lens, apart(lens, 2, shared, fp8)):
        out = case(len(lens), 8, 2, 128, shared, lens, fp8, seed=7)
        assert (out[9] == 0).all() and (out[13] == 0).all() and (out[15:] == 0).all()


@pytest.mark.parametrize("fp8", [False, True])
def test_no_row_has_own_keys_or_none_reaches_the_prefix(fp8):
    for pad in (lambda lens, *_: lens, apart):
        lens = pad([256] * 4, 2, 256, fp8)
        case(len(lens), 4, 2, 128, 256, lens, fp8, seed=8)     # the table ends with the prefix
        lens = pad([5, 700, 0], 2, 1024, fp8)
        case(len(lens), 4, 2, 128, 1024, lens, fp8, seed=9)    # all shorter
        lens = pad([0, 0, 0], 2, 256, fp8)
        out = case(len(lens), 4, 2, 128, 256, lens, fp8, seed=10)
        assert (out == 0).all()


@pytest.mark.parametrize("fp8", [False, True])
def test_nothing_shared(fp8):
    case(6, 8, 2, 128, 0, [1, 300, 0, 128, 77, 513], fp8, seed=11)


def test_wide_table_and_long_prefix():
    """A static table far wider than the rows; a prefix of many splits."""
    case(12, 8, 1, 256, 16384, (16384 + np.arange(12) * 37).tolist(), False, seed=12, width=80)
    case(150, 2, 2, 128, 2048, (2048 + np.arange(150)).tolist(), False, seed=13)


def test_growing_maxima_in_the_prefix():
    """Keys scaled up deep in the prefix: every row's maximum grows far past the rescale threshold."""
    B, H, kvh, bs, shared = 80, 4, 1, 128, 1024  # attended apart
    lens = [shared + 50] * B
    caches, scales, vals, bt = build(B, kvh, bs, shared, lens, False, 14)
    for page, mul in ((int(bt[0, 3]), 6.0), (int(bt[0, 6]), 14.0)):
        caches[0][page, 40:] = (caches[0][page, 40:].float() * mul).to(torch.bfloat16)
        vals[0][page] = caches[0][page]
    q = torch.randn(B, H, 128, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16)
    out = run(q, caches, scales, lens, bt, shared)
    ref, mag = R.decode_attention_f64(q, *vals, lens, bt.clamp_min(0), SCALE)
    check(out, ref, mag, "growing maxima")


@pytest.mark.parametrize("pad", [False, True])
def test_agrees_with_paged_decode(pad):
    for fp8 in (False, True):
        lens = [600, 513, 900, 0, 512]
        if pad:
            lens = apart(lens, 2, 512, fp8)
        caches, scales, _, bt = build(len(lens), 2, 128, 512, lens, fp8, 15)
        q = torch.randn(len(lens), 8, 128, generator=torch.Generator().manual_seed(4)).to(torch.bfloat16)
        a = run(q, caches, scales, lens, bt, 512)
        sl = torch.tensor(lens, dtype=torch.int32, device=dev)
        if fp8:
            b = ops.paged_decode_fp8(q.to(dev), *(t.to(dev) for t in (*caches, *scales)), sl, bt.to(dev))
        else:
            b = ops.paged_decode(q.to(dev), *(t.to(dev) for t in caches), sl, bt.to(dev))
        # two kernels, each within 2 roundings of the same values
        assert (a.float() - b.float()).abs().max() < 4 * 2.0 ** -8 * 3


@pytest.mark.parametrize("pad", [False, True])
def test_bad_pages_and_lengths_are_flagged(pad):
    lens = apart([300, 300], 1, 256, False) if pad else [300, 300]
    caches, scales, _, bt = build(len(lens), 1, 128, 256, lens, False, 16)
    q = torch.randn(len(lens), 2, 128).to(torch.bfloat16)
    for where, value in (((0, 1), 1000), ((0, 1), -5), ((1, 2), 77)):
        bad = bt.clone()
        bad[where] = value
        ops.read_status()
        run(q, caches, scales, lens, bad, 256)
        assert ops.read_status() == nvattn._lib.STATUS_BAD_BLOCK
    run(q, caches, scales, [300, 128 * bt.shape[1] + 1] + lens[2:], bt, 256)
    assert ops.read_status() == nvattn._lib.STATUS_BAD_BLOCK


def test_strided_q_and_out_and_checks():
    lens = [300, 260]
    caches, scales, vals, bt = build(2, 2, 128, 256, lens, False, 17)
    qkv = torch.randn(2, 8 * 128, generator=torch.Generator().manual_seed(5)).to(torch.bfloat16)
    buf = torch.full((2, 4, 200), 3.0, dtype=torch.bfloat16, device=dev)
    out = ops.shared_prefix_decode(qkv.to(dev)[:, 128:640].view(2, 4, 128), *(t.to(dev) for t in caches),
                                   torch.tensor(lens, dtype=torch.int32, device=dev), bt.to(dev), 256,
                                   out=buf[:, :, 10:138])
    ref, mag = R.decode_attention_f64(qkv[:, 128:640].view(2, 4, 128), *vals, lens, bt, SCALE)
    check(out, ref, mag, "strided")
    assert (buf[:, :, :10] == 3).all() and (buf[:, :, 138:] == 3).all()
    with pytest.raises(ValueError, match="both"):
        run(qkv[:, :512].view(2, 4, 128), caches, [torch.zeros(1, dtype=torch.uint8), None], lens, bt, 256)
    with pytest.raises(nvattn._lib.NvattnError, match="whole blocks"):
        run(qkv[:, :512].view(2, 4, 128), caches, scales, lens, bt, 200)


def test_only_row_0_of_the_table_holds_the_prefix():
    """The other rows' entries for it are not read, unless the row is shorter than the prefix."""
    for fp8 in (False, True):
        for pad in (False, True):
            lens = [600, 700, 300, 512, 1]
            if pad:
                lens = apart(lens, 2, 512, fp8)
            caches, scales, vals, bt = build(len(lens), 2, 128, 512, lens, fp8, 19)
            q = torch.randn(len(lens), 8, 128, generator=torch.Generator().manual_seed(9)).to(torch.bfloat16)
            ref, mag = R.decode_attention_f64(q, *vals, lens, bt.clamp_min(0), SCALE)
            bt[1, :4] = bt[3, :4] = -1
            ops.read_status()
            check(run(q, caches, scales, lens, bt, 512), ref, mag, "row 0")
            assert ops.read_status() == 0


@pytest.mark.parametrize("B", [10, 260])
@pytest.mark.parametrize("fp8", [False, True])
def test_graphs_and_streams(fp8, B):
    """Two captured graphs with pools of their own and eager calls on two streams at once, of a
    batch that reads the prefix with its own keys and of one (mostly padding) that does not."""
    H, kvh, bs, shared, width = 8, 2, 128, 512, 8
    lens = [900] * 10 + [0] * (B - 10)
    caches, scales, vals, bt = build(B, kvh, bs, shared, lens, fp8, 18, width=width, stale=False)
    args = [t.to(dev) for t in caches]
    sc = dict(k_scale=None, v_scale=None)
    if fp8:
        sc = dict(zip(("k_scale", "v_scale"), (t.to(dev) for t in scales)))
    q = torch.zeros(B, H, 128, dtype=torch.bfloat16, device=dev)
    sl = torch.zeros(B, dtype=torch.int32, device=dev)
    btd = bt.to(dev)

    def call():
        return ops.shared_prefix_decode(q, *args, sl, btd, shared, softmax_scale=SCALE, **sc)
    call()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call()
        graphs.append((graph, out))
    g = torch.Generator().manual_seed(6)
    for trial in range(2):
        new = np.random.default_rng(trial).integers(shared, 900, size=B)
        new[-2:] = 0
        new[10:] = 0
        qn = torch.randn(B, H, 128, generator=g).to(torch.bfloat16)
        q.copy_(qn), sl.copy_(torch.from_numpy(new.astype(np.int32)))
        for graph, _ in graphs:
            graph.replay()
        side = [torch.cuda.Stream() for _ in range(2)]
        beside = []
        for s in side:
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                beside.append(call())
        torch.cuda.synchronize()
        ref, mag = R.decode_attention_f64(qn, *vals, new, bt.clamp_min(0), SCALE)
        for out in [o for _, o in graphs] + beside:
            check(out, ref, mag, "replay")


# ------------------------------------------------------------- a serving step together

def test_speculative_step_over_an_fp8_cache_with_a_shared_prefix():
    """One step as a server runs it: the new tokens' rows go into the fp8 cache, attention reads the
    shared prompt once, a toy head makes logits of it, drafts are verified, and the accepted
    path's length is what the next step continues from; a second step follows."""
    B, H, kvh, bs, shared, V, n = 6, 8, 2, 128, 256, 500, 4
    g = torch.Generator().manual_seed(19)
    lens = [shared + int(x) for x in np.random.default_rng(2).integers(1, 100, size=B)]
    caches, scales, vals, bt = build(B, kvh, bs, shared, [x + 60 for x in lens], True, 20, stale=False)
    kc, vc, ks, vs = (t.to(dev) for t in (*caches, *scales))
    host = [t.clone() for t in (*caches, *scales)]
    head = torch.randn(H * 128, V, generator=g)
    for step in range(2):
        q, k, v = (torch.randn(B, h, 128, generator=g).to(torch.bfloat16) for h in (H, kvh, kvh))
        slots = torch.tensor([int(bt[b, m // bs]) * bs + m % bs for b, m in enumerate(lens)],
                             dtype=torch.int32)
        lens = [m + 1 for m in lens]
        ops.store_kvcache_fp8(k.to(dev), v.to(dev), kc, vc, ks, vs, slots.to(dev))
        o = ops.shared_prefix_decode(q.to(dev), kc, vc, torch.tensor(lens, dtype=torch.int32, device=dev),
                                     bt.to(dev), shared, softmax_scale=SCALE, k_scale=ks, v_scale=vs)
        # the same step on the host, from the values that the cache stands for
        for x, c, s in ((k, host[0], host[2]), (v, host[1], host[3])):
            qq, e = R.quantise_rows_fp8(x)
            for b, slot in enumerate(slots.tolist()):
                c.view(torch.uint8)[slot // bs, slot % bs] = qq[b].view(torch.uint8)
                s[slot // bs, :, slot % bs] = e[b]
        for a, b_ in zip((kc, vc, ks, vs), host):
            assert torch.equal(a.cpu().view(torch.uint8), b_.view(torch.uint8))
        ref, mag = R.decode_attention_f64(q, R.expand_cache_fp8(host[0], host[2]),
                                          R.expand_cache_fp8(host[1], host[3]), lens, bt.clamp_min(0), SCALE)
        check(o, ref, mag, f"step {step}")
        # drafts: the row's own logits and noisy rows after them stand for a tree's answers
        base = (o.float().cpu().reshape(B, -1) @ head)[:, None] + 3 * torch.randn(B, n, V, generator=g)
        logits = base.to(torch.bfloat16)
        tok = (base[:, :n - 1] + torch.randn(B, n - 1, V, generator=g)).argmax(-1)
        par = torch.tensor([-1, 0, 0, 1], dtype=torch.int32)
        u, pick = torch.rand(B, n - 1, generator=g), torch.rand(B, generator=g)
        temps = torch.full((B,), 0.8)
        got = ops.verify_draft(logits.to(dev), tok.to(dev), u.to(dev), pick.to(dev), temps.to(dev),
                               parents=par.to(dev).expand(B, n))
        want = R.verify_draft(logits, tok.numpy(), u.numpy(), pick.numpy(), temps,
                              parents=par.expand(B, n))
        for a, b_ in zip(got, want):
            assert np.array_equal(a.cpu().numpy(), b_)
        path, acc = got[1].cpu(), got[2].cpu()
        for b in range(B):  # the path is one that the compaction helper takes
            nodes = path[b, :acc[b] + 1].tolist()
            src, dst = tree.compaction_moves(lens[b], nodes, bt[b].tolist(), bs)
            assert len(src) == len(dst)
    assert ops.read_status() == 0


def test_pages_whose_offsets_pass_32_bits():
    """Caches of more than 2^32 bytes: pages at their far end give what the same rows in a small
    cache give, bit for bit, in every operator over them."""
    bs, kvh, H, d = 256, 8, 16, 128
    far = 2 ** 33 // (bs * kvh * d) + 7  # bytes of an fp8 cache; a bf16 one has twice as many
    lens = torch.tensor([700, 300, 513], dtype=torch.int32, device=dev)
    small = torch.tensor([[2, 0, 5], [2, 3, -1], [2, 1, 4]], dtype=torch.int32, device=dev)
    moved = torch.where(small >= 0, far - 1 - small, small)
    g = torch.Generator().manual_seed(90)
    n = 6 * bs
    k, v = [torch.randn(n, kvh, d, generator=g).to(torch.bfloat16).to(dev) for _ in "kv"]
    q = torch.randn(3, H, d, generator=g).to(torch.bfloat16).to(dev)
    slots = torch.arange(n, dtype=torch.int32, device=dev)
    results = []
    ops.read_status()
    for blocks, table in ((6, small), (far, moved)):
        rows = slots if blocks == 6 else (far - 1 - slots // bs) * bs + slots % bs
        kc, vc = [torch.empty(blocks, bs, kvh, d, dtype=torch.float8_e4m3fn, device=dev) for _ in "kv"]
        ks, vs = [torch.empty(blocks, kvh, bs, dtype=torch.uint8, device=dev) for _ in "kv"]
        ops.store_kvcache_fp8(k, v, kc, vc, ks, vs, rows.int())
        cu_k = torch.tensor([0, 700, 1000, 1513], dtype=torch.int32, device=dev)
        out = list(ops.load_kvcache_fp8(kc, vc, ks, vs, cu_k, table, 1513))
        out.append(ops.paged_decode_fp8(q, kc, vc, ks, vs, lens, table))
        out.append(ops.shared_prefix_decode(q, kc, vc, lens, table, bs, k_scale=ks, v_scale=vs))
        del kc, vc, ks, vs
        kc, vc = [torch.empty(blocks, bs, kvh, d, dtype=torch.bfloat16, device=dev) for _ in "kv"]
        ops.store_kvcache(k, v, kc, vc, rows.int())
        out.append(ops.shared_prefix_decode(q, kc, vc, lens, table, bs))
        results.append(out)
        del kc, vc
    assert ops.read_status() == 0
    for a, b in zip(*results):
        assert torch.equal(a, b)
    torch.cuda.empty_cache()
