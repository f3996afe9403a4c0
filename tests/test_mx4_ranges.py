"""MXFP4 operators at the ends of their ranges, against 64 bits: block scales near the ends of the exponent range. The
tolerances are those that ``test_mx4`` derives."""
import pytest
import torch

from test_mx4 import close, linear_ref, op64, rnd

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------ block scales
# (x is about 2^p, w about 2^q): each scale, and the product of a sum with either one, may leave fp32's range while the
# result does not. A term below 2^-149 may be lost: less than the half subnormal of bf16 that the bound has.
@pytest.mark.parametrize("p,q", [(121, -20), (124, -30), (124, -120), (-125, 100), (100, -125), (-40, 124), (60, 58)])
@pytest.mark.parametrize("M,N,act", [(1, 64, 0), (2, 40, 0), (8, 64, 2), (130, 64, 0)])
def test_linear_scales_near_the_ends(sdg, cuda, M, N, act, p, q):
    K = 96
    if act == 2:        # the product of value and GELU(gate) has to stay finite as well
        p, q = (p, q) if p + q < 60 else (p, q - 60)
    x = (rnd(M, K, seed=1) * 2.0 ** p).bfloat16()
    w = (rnd(N, K, seed=2).double() * 2.0 ** q).float()
    wc, ws = sdg.quantize_mx4(w)
    xq = sdg.quantize_mx4(x)
    ref, d = linear_ref(op64(*xq, K), op64(wc, ws, K), None, None, act)
    assert bool((ref.abs() < 2.0 ** 127).all())
    for y in (sdg.linear_mx4(x, wc, ws, act=act),
              sdg.linear_mx4(xq[0], wc, ws, act=act, xscale=xq[1], dtype=torch.bfloat16)):
        assert bool(torch.isfinite(y).all())
        close(y, ref, d)


@pytest.mark.parametrize("M", [1, 5])
def test_linear_zero_products_of_large_scales(sdg, cuda, M):
    """Blocks whose scales' product is past fp32 but whose values meet only zeros add nothing."""
    x = torch.zeros(M, 64, dtype=torch.bfloat16, device=cuda)
    w = torch.zeros(8, 64, device=cuda)
    x[:, 0], w[:, 1] = 2.0 ** 124, 2.0 ** 100
    x[:, 40], w[:, 40] = 1.5, 2.0
    y = sdg.linear_mx4(x, *sdg.quantize_mx4(w))
    assert bool((y == 3.0).all())
