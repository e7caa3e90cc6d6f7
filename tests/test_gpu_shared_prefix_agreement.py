"""Shared-prefix decode and paged decode of the same batch, element by element within what the two
kernels' roundings allow."""
from __future__ import annotations

import pytest
import torch

from oracle import reference_math as R

from nvattn import ops
from test_gpu_shared_prefix import apart, bound, build, run

pytestmark = pytest.mark.gpu
dev = torch.device("cuda")
SCALE = 128 ** -0.5


@pytest.mark.parametrize("pad", [False, True])
@pytest.mark.parametrize("fp8", [False, True])
def test_every_element(fp8, pad):
    """Each kernel lies within `bound` of 64 bits (its terms hold for all of them), so the two differ by
    twice that at most: about 0.007 (the weights' rounding to bf16, 2^-8 of sum p |v|) where outputs are
    about 0.05 and keys that went missing, 60 of 600 say, move some of them by 0.02."""
    lens = [600, 513, 900, 0, 512, 777]
    if pad:
        lens = apart(lens, 2, 512, fp8)
    caches, scales, vals, bt = build(len(lens), 2, 128, 512, lens, fp8, 25)
    q = torch.randn(len(lens), 8, 128, generator=torch.Generator().manual_seed(4)).to(torch.bfloat16)
    a = run(q, caches, scales, lens, bt, 512)
    sl = torch.tensor(lens, dtype=torch.int32, device=dev)
    if fp8:
        b = ops.paged_decode_fp8(q.to(dev), *(t.to(dev) for t in (*caches, *scales)), sl, bt.to(dev))
    else:
        b = ops.paged_decode(q.to(dev), *(t.to(dev) for t in caches), sl, bt.to(dev))
    ref, mag = R.decode_attention_f64(q, *vals, lens, bt.clamp_min(0), SCALE)
    diff, tol = (a.double() - b.double()).abs().cpu(), 2 * bound(ref, mag)
    print(f"[max-abs] shared prefix against paged decode: {diff.max():.3e}, margin {(tol - diff).min():.3e}")
    assert (diff <= tol).all()
