"""fp8 decode over V rows of very different magnitudes: what a large value in one channel leaves of the
others, and rows near the ends of the exponent's range."""
from __future__ import annotations

import pytest
import torch

from oracle import reference_math as R

from nvattn import ops

pytestmark = pytest.mark.gpu
dev = torch.device("cuda")
SCALE = 128 ** -0.5
H = 4


def _run(k, v, q, n):
    """One sequence over one page of KVH 1; the reference and its magnitudes over the stored values."""
    (kc, ks), (vc, vs) = R.quantise_rows_fp8(k), R.quantise_rows_fp8(v)
    ks, vs = [s.transpose(1, 2).contiguous() for s in (ks, vs)]
    bt = torch.arange(k.shape[0], dtype=torch.int32)[None]
    out = ops.paged_decode_fp8(q.to(dev), *(t.to(dev) for t in (kc, vc, ks, vs)),
                               torch.tensor([n], dtype=torch.int32, device=dev), bt.to(dev))
    ref, mag = R.decode_attention_f64(q, R.expand_cache_fp8(kc, ks), R.expand_cache_fp8(vc, vs), [n], bt, SCALE)
    return out.double().cpu(), ref, mag


def _bound(ref, mag):
    """Per element and channel: a score is off by 136 * 2^-24 of the products' magnitudes and exp2's
    argument and result add 2^-21, in the weight and in the sum; the weights take one rounding to f16,
    2^-12, where they lie within 2^-28 of their warp's largest (that holds for the inputs below); sums in
    fp32; the output is rounded once to bf16, 2^-8."""
    rel = 2 * (2 * 136 * 2.0 ** -24 * mag["dot"] + 2.0 ** -21) + 2.0 ** -12 + (mag["n"] / 16 + 64) * 2.0 ** -24
    return 2.0 ** -8 * ref.abs() + rel[..., None] * mag["mix"]


@pytest.mark.parametrize("log2", [8, 16, 18, 22, 26])
@pytest.mark.parametrize("n", [64, 300])
def test_a_large_channel_costs_the_others_nothing(n, log2):
    """One key of 2^log2 in channel 0 and nothing elsewhere; the others' values are normal."""
    g = torch.Generator().manual_seed(n + log2)
    k = 0.2 * torch.randn(3, 128, 1, 128, generator=g)
    v = torch.randn(3, 128, 1, 128, generator=g)
    v[0, 7] = 0
    v[0, 7, 0, 0] = 2.0 ** log2
    q = torch.randn(1, H, 128, generator=g).to(torch.bfloat16)
    out, ref, mag = _run(k.to(torch.bfloat16), v.to(torch.bfloat16), q, n)
    over = ((out - ref).abs() - _bound(ref, mag)).amax((0, 1))
    print(f"[max-abs] fp8 channel of 2^{log2}: {(out - ref).abs()[..., 1:].max():.3e}")
    assert (over <= 0).all(), over.max()


def test_values_near_the_largest_bf16():
    """A key of 3e38 whose score is highest, beside keys of 2^-6 to 2^-12 of its weight each with
    ordinary values: together they take a third of the softmax's sum."""
    g = torch.Generator().manual_seed(3)
    k = torch.zeros(1, 64, 1, 128)
    k[0, 0, 0, 0] = 1.0
    k[0, :, 0, 1] = 0.25 * torch.rand(64, generator=g)
    v = torch.randn(1, 64, 1, 128, generator=g)
    v[0, 0] = 3e38 * torch.sign(v[0, 0])
    q = torch.zeros(1, H, 128)
    q[0, :, 0] = torch.tensor([4.5, 5.5, 6.5, 7.5]) / SCALE
    q[0, :, 1] = 1.0 / SCALE
    out, ref, mag = _run(k.to(torch.bfloat16), v.to(torch.bfloat16), q.to(torch.bfloat16), 64)
    over = (out - ref).abs() - _bound(ref, mag)
    assert torch.isfinite(out).all() and (over <= 0).all(), (out / ref)[0, :, 0]


def test_all_values_zero_or_tiny():
    """Rows of zeros and of the smallest exponents next to ordinary ones, with scores far apart."""
    g = torch.Generator().manual_seed(4)
    k = 4 * torch.randn(24, 128, 1, 128, generator=g)
    q = torch.randn(1, H, 128, generator=g).to(torch.bfloat16)
    for fill in (0.0, 2.0 ** -95, 2.0 ** -60):
        v = torch.randn(24, 128, 1, 128, generator=g)
        v[:, ::2] = fill * v[:, ::2]
        v[8:16] = fill * v[8:16]
        out, ref, mag = _run(k.to(torch.bfloat16), v.to(torch.bfloat16), q, 3000)
        over = (out - ref).abs() - _bound(ref, mag)
        assert (over <= 0).all(), (fill, over.max())
        tiny = fill * torch.randn(24, 128, 1, 128, generator=g)
        out, ref, mag = _run(k.to(torch.bfloat16), tiny.to(torch.bfloat16), q, 3000)
        # stored rows below 2^-100 * 2^-9 are zeros; every element is at most one subnormal step off
        over = (out - ref).abs() - _bound(ref, mag)
        assert (over <= 0).all(), (fill, over.max())
