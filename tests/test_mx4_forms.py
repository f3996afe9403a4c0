"""MXFP4 operators: every kernel form that a size can lead to, against 64 bits, with the tolerances that ``test_mx4`` derives."""
import numpy as np
import pytest
import torch

from oracle import mx4 as O
from test_mx4 import DT, check_groupnorm, close, groupnorm_ref, linear_ref, op64, rnd, weight

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------ linear
# pairs with GEGLU (a w tile of which the odd CTA has rows, and one of which it has none); pairs with one 8-wide column tile;
# few rows too long for the few-rows kernel and the longest that it takes; rows shorter than a block
LINEAR = [(20001, 224, 1824), (9985, 544, 2560), (9985, 576, 2560), (38000, 8, 1800), (3, 64, 10016), (8, 96, 9856),
          (8, 64, 9824), (40, 32, 1), (300, 64, 8), (33, 8, 5), (20000, 32, 31), (700, 352, 640), (20001, 160, 1100)]


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("M,N,K", LINEAR)
def test_linear_forms(sdg, cuda, M, N, K, dtype):
    t = DT[dtype]
    wc, ws = weight(sdg, N, K, 1)
    x = rnd(M, K, seed=M + N + K, dtype=t, spread=1.0)
    xq = sdg.quantize_mx4(x)
    xv, wv = op64(*xq, K), op64(wc, ws, K)
    bias, res = 0.1 * rnd(N, seed=5), rnd(M, N, seed=6, dtype=t)
    for b, r, act in ((bias, res, 1), (bias, None, 2), (None, None, 2)):
        if act == 2 and N % 32:
            continue
        ref, d = linear_ref(xv, wv, b, r, act)
        y = sdg.linear_mx4(x, wc, ws, b, residual=r, act=act)
        assert y.shape == ref.shape and y.dtype == t
        close(y, ref, d)
        assert torch.equal(sdg.linear_mx4(xq[0], wc, ws, b, residual=r, act=act, xscale=xq[1], dtype=t), y)
        assert torch.equal(sdg.linear_mx4(x, wc, ws, b, residual=r, act=act), y)


@pytest.mark.parametrize("K", [3, 5, 12, 33])
def test_linear_reads_only_its_columns(sdg, cuda, K):
    """Rows of K columns in a wider matrix whose other columns are NaN, through the form that brings x in by TMA."""
    wide = torch.full((300, 40), torch.nan, dtype=torch.float16, device=cuda)
    wide[:, :K] = rnd(300, K, seed=K, dtype=torch.float16)
    x = wide[:, :K]
    wc, ws = weight(sdg, 64, K, 2)
    ref, d = linear_ref(op64(*sdg.quantize_mx4(x), K), op64(wc, ws, K), None, None, 0)
    close(sdg.linear_mx4(x, wc, ws), ref, d)


@pytest.mark.parametrize("M,N,K", [(100, 64, 1536), (130, 64, 4096), (20001, 160, 1536), (20001, 160, 4096)])
def test_linear_keeps_terms_below_half_a_16_bit_step(sdg, cuda, M, N, K):
    """16384, then one 1 a block, then -16384: a sum held in 16 bits anywhere (steps of 16 there) would end at 0."""
    x = torch.zeros(M, K, dtype=torch.float16, device=cuda)
    w = torch.zeros(N, K, device=cuda)
    x[:, :32], w[:, :32] = 1.0, 512.0
    x[:, 32::32], w[:, 32::32] = 1.0, 1.0
    x[:, -32:], w[:, -32:] = 1.0, -512.0
    y = sdg.linear_mx4(x, *sdg.quantize_mx4(w))
    assert bool((y == K // 32 - 2).all())


# ------------------------------------------------------------------ GroupNorm
# up to 16 pixels an image, on several row tiles and more images than a tile of the other form may touch; several row tiles a
# block with image boundaries inside; chunks of several runs; up to 4096 channels; one group, and a group per channel
GN = [(64, 1, 320, 32), (40, 16, 640, 32), (300, 5, 64, 8), (700, 1, 72, 9), (2000, 16, 320, 32), (15, 17, 320, 32),
      (40, 1000, 640, 32), (64, 300, 1280, 32), (333, 129, 320, 32), (1, 16384, 2560, 32), (2, 50001, 320, 32),
      (1, 70000, 40, 5), (2, 100, 4096, 32), (1, 17, 2568, 3), (3, 1000, 4096, 64), (1, 300, 3000, 8), (2, 64, 64, 64),
      (3, 130, 320, 1), (1, 4096, 4096, 4096), (65535, 1, 8, 1)]


def check_tiles(got, y, delta):
    """check_groupnorm on the first, the last and some row tiles between them."""
    R, tiles = y.shape[0], -(-y.shape[0] // 128)
    pick = sorted({0, 1, tiles // 3, tiles // 2, tiles - 2, tiles - 1} & set(range(tiles)))
    off = []
    for t in pick:
        rows = slice(128 * t, min(R, 128 * t + 128))
        off.append(check_groupnorm((got[0][rows], got[1][t:t + 1]), y[rows], delta[rows]))
    return float(np.mean(off))


@pytest.mark.parametrize("dtype,silu", [("fp16", False), ("bf16", True)])
@pytest.mark.parametrize("B,HW,C,groups", GN)
def test_groupnorm_forms(sdg, cuda, B, HW, C, groups, silu, dtype):
    x = (1.5 * rnd(B, HW, C, seed=B + HW + C) + rnd(B, 1, C, seed=9) + rnd(B, 1, 1, seed=10)).to(DT[dtype])
    gamma, beta = 1 + 0.2 * rnd(C, seed=1), 0.2 * rnd(C, seed=2)
    got = sdg.groupnorm_mx4(x, gamma, beta, 1e-5, silu, groups=groups)
    assert check_tiles(got, *groupnorm_ref(x, gamma, beta, 1e-5, silu, groups)) < 1e-3
    again = sdg.groupnorm_mx4(x, gamma, beta, 1e-5, silu, groups=groups)
    assert torch.equal(got[0], again[0]) and torch.equal(got[1], again[1])


@pytest.mark.parametrize("value", [3.0, -1000.0, 0.0])
@pytest.mark.parametrize("HW", [5, 100, 4096])
def test_groupnorm_constant_group_is_beta(sdg, cuda, HW, value):
    """A group without variance: eps carries it, and its values are beta within the bound."""
    x = rnd(2, HW, 64, seed=1).half()
    x[0, :, 0:8] = value
    gamma, beta = 1 + 0.2 * rnd(64, seed=2), 0.25 + 0.5 * rnd(64, seed=3)
    got = sdg.groupnorm_mx4(x, gamma, beta, 1e-5, False, groups=8)
    y, delta = groupnorm_ref(x, gamma, beta, 1e-5, False, 8)
    assert np.allclose(y[:HW, :8], beta[:8].double().cpu().numpy(), rtol=0, atol=1e-9)
    check_groupnorm(got, y, delta)


def test_operand_of_many_small_images_feeds_the_product(sdg, cuda):
    """GroupNorm of 200 images of 9 pixels and the product that reads it."""
    x = rnd(200, 9, 320, seed=4, dtype=torch.bfloat16)
    gamma, beta = 1 + 0.2 * rnd(320, seed=1), 0.2 * rnd(320, seed=2)
    q = sdg.groupnorm_mx4(x, gamma, beta, 1e-6, True)
    w = weight(sdg, 320, 320, 5)
    ref, d = linear_ref(op64(*q, 320), op64(*w, 320), None, None, 0)
    close(sdg.linear_mx4(q[0], *w, xscale=q[1], dtype=torch.bfloat16), ref, d)
    code, e = O.unpack(q[0].cpu().numpy(), q[1].cpu().numpy())
    assert code.shape == (1800, 320) and e.shape == (1800, 10)
