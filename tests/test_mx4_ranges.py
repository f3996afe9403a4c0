"""MXFP4 operators at the ends of their ranges, against 64 bits: block scales near the ends of the exponent range, very many
pixels. The tolerances are those that ``test_mx4`` derives, unless a test says otherwise."""
import numpy as np
import pytest
import torch

from test_mx4 import check_groupnorm, close, groupnorm_ref, linear_ref, op64, rnd

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


# ------------------------------------------------------------------ GroupNorm of very many pixels
def test_groupnorm_statistics_of_many_pixels(sdg, cuda):
    """2^26 pixels: a thread has 1024 of them, and its first four are unlike the rest, which are all alike. Sums of squares
    about those four's mean would lose 2^8 to cancellation, and roundings of equal terms all go one way: 0.4 % of the variance.

    Bound: a run of 32 pixels is summed with at most 40 roundings, times 9 for the cancellation; 32 runs, 256 rows x 8
    channels over 8 lanes and 256 chunks over 8 lanes merge with at most 4 roundings a run and one a term, 64 for the rest."""
    HW, C, part = 1 << 26, 8, 1 << 18
    x = torch.full((1, HW, C), 2.125, dtype=torch.float16, device=cuda)
    x.view(HW // part, part, C)[:, :1024] = 250.0
    tail = 4096
    g = torch.Generator(device=cuda).manual_seed(1)
    x[0, -tail:] = (torch.rand(tail, C, generator=g, device=cuda) * 500 - 250).half()
    pieces = x.view(64, -1)
    mu = sum(p.double().sum() for p in pieces) / (HW * C)
    var = sum((p.double() - mu).square().sum() for p in pieces) / (HW * C)
    mag = sum(p.double().abs().sum() for p in pieces) / (HW * C)
    got = sdg.groupnorm_mx4(x, torch.ones(C, device=cuda), torch.zeros(C, device=cuda), 1e-5, False, groups=1)
    rs = torch.rsqrt(var + 1e-5)
    t = x[0, -tail:].double()
    y = (t - mu) * rs
    e_mu = (40 + 4 * 32 + 256 + 32 + 64) * 2.0 ** -24 * mag
    rel = (9 * 40 + 4 * 32 + 256 + 32 + 64) * 2.0 ** -24 + 2.0 ** -20 + (e_mu * rs) ** 2
    delta = rs * e_mu + y.abs() * rel + rs * 2.0 ** -23 * (t.abs() + mu.abs()) + 2.0 ** -22 * y.abs()
    check_groupnorm((got[0][-tail:], got[1][-tail // 128:]), y.cpu().numpy(), delta.cpu().numpy())


# ------------------------------------------------------------------ offsets past 32 bits
def test_element_offsets_past_32_bits(sdg, cuda):
    """4.4e9 elements: the rows behind element 2^32 of every operator's input and output."""
    if torch.cuda.mem_get_info()[0] < 48 << 30:
        pytest.skip("needs 48 GB of device memory")
    R, K = (1 << 22) + 77, 1056
    x = torch.randn(R, K, dtype=torch.float16, device=cuda, generator=torch.Generator(device=cuda).manual_seed(1))
    t0 = R // 128 * 128 - 256          # (whole row tiles)
    assert t0 * K > 1 << 32
    tail = x[t0:].clone()
    want = sdg.quantize_mx4(tail)
    q = sdg.quantize_mx4(x)
    assert torch.equal(q[0][t0:], want[0]) and torch.equal(q[1][t0 // 128:], want[1])
    v = sdg.dequantize_mx4(*q)
    assert torch.equal(v[t0:], sdg.dequantize_mx4(*want))
    del v
    wc, ws = sdg.quantize_mx4(rnd(K, K, seed=2) / K ** 0.5)
    ref, d = linear_ref(op64(*want, K), op64(wc, ws, K), None, tail, 0)
    y = sdg.linear_mx4(x, wc, ws, residual=x)
    close(y[t0:], ref, d)
    torch.cuda.synchronize()
    y.zero_()
    close(sdg.linear_mx4(q[0], wc, ws, residual=x, xscale=q[1], out=y)[t0:], ref, d)
    del y, q
    g = x[:1 << 22].view(4, 1 << 20, K)
    gamma, beta = 1 + 0.2 * rnd(K, seed=3), 0.2 * rnd(K, seed=4)
    a = sdg.groupnorm_mx4(g, gamma, beta, 1e-5, True)
    b = sdg.groupnorm_mx4(g[3:].clone(), gamma, beta, 1e-5, True)
    assert torch.equal(a[0][3 << 20:], b[0]) and torch.equal(a[1][(3 << 20) // 128:], b[1])


# ------------------------------------------------------------------ SiLU far below zero
@pytest.mark.parametrize("HW", [8, 512])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_groupnorm_silu_of_very_negative_blocks(sdg, cuda, HW, dtype):
    """Blocks whose values are all SiLU of -20 to -84: tiny, but an operand's exponent follows them.

    There SiLU is y exp(y) but for 2^-28, its relative slope 1 + 1 / y: an error d of y counts 1.1 d, the exponent's rounding
    |y| 2^-24 and the function 2^-21, each relative."""
    C = 320
    x = rnd(2, HW, C, seed=6, dtype=dtype)
    gamma = 1 + 0.2 * rnd(C, seed=1)
    beta = -24.0 - 56.0 * (torch.arange(C, device=cuda) // 32) / 9
    y, d = groupnorm_ref(x, gamma, beta, 1e-5, False, 32)
    assert y.max() < -16 and y.min() > -87
    ref = y / (1 + np.exp(-y))
    delta = np.abs(ref) * (1.1 * d + np.abs(y) * 2.0 ** -23 + 2.0 ** -21)
    check_groupnorm(sdg.groupnorm_mx4(x, gamma, beta, 1e-5, True), ref, delta)
