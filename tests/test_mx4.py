"""MXFP4 operators: quantise, read back, linear, GroupNorm into an operand, against 64 bits.

Tolerances, each derived from the arithmetic:

* quantisation is exact: a block's exponent comes from the bits of its maximum, dividing by a power of two is exact,
  and the rounding to E2M1 is correctly rounded; so codes and scales are compared bit for bit. Reading back rounds
  once, values that fp16 / bf16 / fp32 hold exactly compare equal.
* linear: the operands' values are given, so y64 = act(sum + bias + residual) in 64 bits has one right value. The
  kernel adds at most K/16 + 16 terms in fp32 whatever its split (a block's products are exact sums), each addition off
  by at most 2^-23 of the sum of magnitudes S = sum|x w| + |bias| + |residual| (2^-24 rounded, 2^-23 truncated):
  d = (K/16 + 16) 2^-23 S before the activation. SiLU's slope is at most 1.1 and its own error below 2^-20 |y|; GEGLU
  v gelu(g): |gelu(g)| d_v + 1.13 |v| d_g + 2^-20 |v| |g|. The result is rounded once: eps/2 |y|, and half the smallest
  subnormal where y is subnormal in the output type.
* GroupNorm: the fp32 value before quantisation is off by at most delta (below); the code has to be what some value
  within delta of the 64-bit one rounds to under the exponent that the kernel chose, and that exponent what some
  maximum within delta gives. With n terms per group, a sum is off by (n/128 + 64) 2^-24 relative to the sum of
  magnitudes whatever the split.
"""
import ctypes

import numpy as np
import pytest
import torch

from oracle import mx4 as O

DT = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
SDG_ERR_ARG, SDG_ERR_SHAPE = 2, 3


# ------------------------------------------------------------------ CPU: the format
def test_format_hand_worked():
    x = np.zeros((2, 40))
    x[0, :9] = [6.0, -4.0, 5.0, 2.5, 1.75, 0.25, 0.75, -0.2, 7.9]   # max 7.9: exponent floor(2.98) - 2 = 0
    x[0, 32:34] = [0.375, 0.0625]                                    # max 0.375: exponent -2 - 2 = -4
    code, e = O.quantize(x)
    v = O.values(code, e)
    assert e[0].tolist() == [127, 123] and e[1].tolist() == [0, 0]
    # ties to the even code: 5 -> 4, 2.5 -> 2, 1.75 -> 2, 0.25 -> 0, 0.75 -> 1; saturation: 7.9 -> 6
    assert v[0, :9].tolist() == [6.0, -4.0, 4.0, 2.0, 2.0, 0.0, 1.0, 0.0, 6.0]
    assert v[0, 32:34].tolist() == [0.375, 0.0625]
    assert not v[1].any()


def test_format_special_blocks():
    x = np.ones((3, 32))
    x[0, 3] = np.inf
    x[1, 5] = np.nan
    x[2] = 2.0 ** -140
    code, e = O.quantize(x)
    assert e[:2, 0].tolist() == [255, 255] and not code[:2].any()
    assert np.isnan(O.values(code, e)[:2]).all()
    assert e[2, 0] == 0 and not code[2].any()


def test_pack_round_trip():
    g = np.random.default_rng(0)
    code, e = O.quantize(g.standard_normal((300, 333)))
    codes, scales = O.pack(code, e)
    assert codes.shape == (300, 176) and scales.shape == (3, 3, 512)
    c2, e2 = O.unpack(codes, scales)
    assert np.array_equal(c2, code) and np.array_equal(e2, e)


def test_plain_grid_error_is_half_a_step():
    g = np.random.default_rng(1)
    x = g.standard_normal((64, 256))
    code, e = O.quantize(x)
    s = np.repeat(np.ldexp(1.0, e.astype(int) - 127), 32, axis=1)
    a = np.minimum(np.abs(x) / s, 6.0)
    step = np.where(a < 2, 0.5, np.where(a < 4, 1.0, 2.0))
    assert (np.abs(np.abs(O.values(code, e)) / s - a) <= step / 2).all()


# ------------------------------------------------------------------ CPU: refusals before any launch
def test_sizes(sdg):
    L = sdg.lib()
    assert L.sdg_mx4_code_bytes(3, 33) == 3 * 32 and L.sdg_mx4_scale_bytes(3, 33) == 512
    assert L.sdg_mx4_code_bytes(129, 320) == 129 * 160 and L.sdg_mx4_scale_bytes(129, 320) == 2 * 3 * 512
    assert L.sdg_mx4_code_bytes((1 << 30) + 1, 5) == 0 and L.sdg_mx4_scale_bytes(5, (1 << 23) + 1) == 0
    assert L.sdg_mx4_code_bytes(0, 5) == 0 and L.sdg_mx4_scale_bytes(5, -1) == 0
    need = L.sdg_linear_mx4_scratch_bytes
    assert need(16, 3, 33, 33, 64) == 0 and need(16, 100, 320, 320, 64) == 0   # few rows, small products: no scratch
    assert need(18, 100, 320, 320, 64) == need(16, 100, 320, 323, 64) == 100 * 160 + 384 + 3 * 512  # unaligned rows
    assert need(16, 0, 33, 33, 64) == 0
    assert need(16, 100001, 320, 320, 1280) == 100001 * 160 + 352 + 782 * 3 * 512


def _addr(n=4096):
    buf = ctypes.create_string_buffer(n + 64)
    return buf, (ctypes.addressof(buf) + 15) // 16 * 16


def test_refusals_without_gpu(sdg):
    """Every refused call returns its status before anything is launched (the pointers are host memory)."""
    L = sdg.lib()
    keep, p = _addr()
    q = lambda **k: L.sdg_quantize_mx4(*({"x": p, "dt": 0, "R": 2, "K": 32, "ld": 32, "c": p, "s": p, "st": None} | k).values())
    assert q(x=None) == q(c=None) == q(s=None) == q(R=0) == q(K=0) == q(ld=-1) == q(dt=3) == q(dt=-1) == q(R=(1 << 30) + 1) == SDG_ERR_ARG
    assert q(c=p + 8) == q(s=p + 4) == q(x=p + 1) == SDG_ERR_ARG
    d = lambda **k: L.sdg_dequantize_mx4(*({"c": p, "s": p, "R": 2, "K": 32, "dt": 0, "y": p, "st": None} | k).values())
    assert d(c=None) == d(s=None) == d(y=None) == d(R=0) == d(K=-1) == d(dt=7) == d(y=p + 1) == d(c=p + 2) == SDG_ERR_ARG
    base = {"xc": p, "xs": p, "M": 2, "K": 32, "wc": p, "ws": p, "b": p, "N": 32, "r": None, "act": 0, "dt": 0, "y": p,
            "err": None, "st": None}
    m = lambda **k: L.sdg_linear_mx4(*(base | k).values())
    assert m(xc=None) == m(xs=None) == m(wc=None) == m(ws=None) == m(y=None) == SDG_ERR_ARG
    assert m(M=0) == m(K=0) == m(N=0) == m(act=3) == m(act=-1) == m(dt=2) == SDG_ERR_ARG
    assert m(act=2, r=p) == m(xc=p + 8) == m(wc=p + 8) == m(y=p + 2) == m(r=p + 2) == m(b=p + 2) == SDG_ERR_ARG
    assert m(N=12) == m(N=40, act=2) == SDG_ERR_SHAPE
    bx = {"x": p, "M": 1 << 20, "K": 32, "ld": 32, "wc": p, "ws": p, "b": None, "N": 32, "r": None, "act": 0, "dt": 0, "y": p,
          "scr": p, "nb": 1 << 30, "err": None, "st": None}
    mx = lambda **k: L.sdg_linear_mx4_x(*(bx | k).values())
    assert mx(x=None) == mx(scr=None) == mx(nb=1 << 24) == mx(scr=p + 8) == mx(ld=-2) == mx(dt=2) == SDG_ERR_ARG
    g = lambda **k: L.sdg_groupnorm_mx4(*({"x": p, "dt": 0, "B": 1, "HW": 4, "C": 64, "G": 8, "ga": p, "be": p, "eps": 1e-5,
                                           "silu": 0, "c": p, "s": p, "scr": p, "st": None} | k).values())
    assert g(x=None) == g(ga=None) == g(c=None) == g(scr=None) == g(B=0) == g(HW=0) == g(C=0) == g(G=0) == SDG_ERR_ARG
    assert g(dt=2) == g(x=p + 2) == g(c=p + 8) == g(scr=p + 4) == SDG_ERR_ARG
    assert g(C=60, G=4) == g(C=64, G=7) == g(B=65536) == g(C=4104, G=8) == g(B=2, HW=1 << 30) == SDG_ERR_SHAPE
    assert "groupnorm_mx4" in sdg.last_error()
    del keep


def test_binding_refuses_cpu_tensors(sdg):
    x = torch.zeros(4, 32, dtype=torch.float16)
    c = torch.zeros(4, 16, dtype=torch.uint8)
    s = torch.zeros(1, 1, 512, dtype=torch.uint8)
    for call in (lambda: sdg.quantize_mx4(x), lambda: sdg.dequantize_mx4(c, s), lambda: sdg.linear_mx4(x, c, s),
                 lambda: sdg.groupnorm_mx4(x[None], None, None, 1e-5, False)):
        with pytest.raises(sdg.SdgError) as ei:
            call()
        assert ei.value.code == SDG_ERR_ARG


# ------------------------------------------------------------------ GPU helpers
def rnd(*shape, seed, dtype=torch.float32, spread=0.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(*shape, generator=g)
    if spread:
        x = x * torch.exp2(spread * torch.randn(*shape[:-1], 1, generator=g))
    return x.to(dtype).cuda()


def op64(codes, scales, K):
    """fp64 CUDA values [R, K] of an operand's two arrays."""
    code, e = O.unpack(codes.cpu().numpy(), scales.cpu().numpy())
    return torch.from_numpy(O.values(code, e)[:, :K]).cuda()


def same_operand(got, x64):
    code, e = O.quantize(x64)
    wc, ws = O.pack(code, e)
    assert np.array_equal(got[1].cpu().numpy(), ws)
    assert np.array_equal(got[0].cpu().numpy(), wc)


# ------------------------------------------------------------------ GPU: quantise and read back
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("R,K", [(1, 1), (1, 31), (1, 32), (1, 1280), (2, 33), (7, 40), (31, 64), (33, 96), (127, 128),
                                 (128, 129), (129, 320), (154, 768), (260, 333), (500, 1000), (40, 5120)])
def test_quantize_bits(sdg, cuda, R, K, dtype):
    x = rnd(R, K, seed=R * 7919 + K, dtype=DT[dtype], spread=3.0)
    out = sdg.quantize_mx4(x, out=(torch.full((R, (K + 31) // 32 * 16), 255, dtype=torch.uint8, device=cuda),
                                   torch.full(((R + 127) // 128, (K + 127) // 128, 512), 255, dtype=torch.uint8,
                                              device=cuda)))
    same_operand(out, x.double().cpu().numpy())
    v64 = op64(*out, K)
    for t in DT.values():
        y = sdg.dequantize_mx4(*out, K, dtype=t)
        assert y.shape == (R, K) and torch.equal(y, v64.to(t))
    full = sdg.dequantize_mx4(*out)
    assert full.shape[1] == 2 * out[0].shape[1] and not full[:, K:].any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DT))
def test_quantize_ties_and_specials(sdg, cuda, dtype):
    """Every midpoint and grid point of E2M1 under many exponents, zero blocks, subnormals, infinities and NaNs."""
    t = DT[dtype]
    mids = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, 7.0, 7.75])
    row = torch.cat([mids, -mids])
    lo, hi = {"fp16": (-20, 13), "bf16": (-130, 125), "fp32": (-146, 125)}[dtype]
    x = torch.stack([torch.ldexp(row, torch.tensor(float(p))) for p in range(lo, hi)])
    extra = torch.zeros(8, 32)
    extra[1, 4] = torch.inf
    extra[2, 31] = -torch.inf
    extra[3] = torch.nan
    extra[4, 0] = torch.finfo(t).max
    extra[5] = -torch.finfo(t).max
    extra[6, 7] = torch.finfo(t).smallest_normal / 4
    extra[7] = -0.0
    x = torch.cat([x, extra]).to(t).cuda()
    x = torch.cat([x, x.roll(5, 0), x.roll(9, 0)], 1)
    out = sdg.quantize_mx4(x)
    same_operand(out, x.double().cpu().numpy())
    y = sdg.dequantize_mx4(*out, dtype=torch.float32)
    ref = op64(*out, x.shape[1])
    assert torch.equal(torch.isnan(y), torch.isnan(ref)) and torch.equal(y.nan_to_num(0.0), ref.float().nan_to_num(0.0))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("first,K,ld", [(0, 64, 96), (8, 64, 96), (1, 64, 96), (0, 63, 65), (3, 40, 47)])
def test_quantize_strided_rows(sdg, cuda, first, K, ld, dtype):
    wide = rnd(133, ld, seed=ld, dtype=DT[dtype])
    x = wide[:, first:first + K]
    same_operand(sdg.quantize_mx4(x), x.double().cpu().numpy())
    one = x[2].expand(130, K)            # row stride 0
    same_operand(sdg.quantize_mx4(one), one.double().cpu().numpy())


@pytest.mark.gpu
def test_dequantize_into_unaligned_output(sdg, cuda):
    c, s = sdg.quantize_mx4(rnd(70, 96, seed=1))
    flat = torch.full((70 * 96 + 9,), 5.0, dtype=torch.float16, device=cuda)
    out = flat[3:3 + 70 * 96].view(70, 96)
    sdg.dequantize_mx4(c, s, out=out)
    assert torch.equal(out, op64(c, s, 96).half())
    assert bool((flat[:3] == 5).all()) and bool((flat[3 + 70 * 96:] == 5).all())


@pytest.mark.gpu
def test_quantize_writes_only_its_arrays(sdg, cuda):
    R, K = 131, 65
    buf = torch.full((4096 + R * 48 + 4096,), 170, dtype=torch.uint8, device=cuda)
    sc = torch.full((4096 + 2 * 512 + 4096,), 170, dtype=torch.uint8, device=cuda)
    codes, scales = buf[4096:4096 + R * 48].view(R, 48), sc[4096:4096 + 1024].view(2, 1, 512)
    sdg.quantize_mx4(rnd(R, K, seed=3), out=(codes, scales))
    torch.cuda.synchronize()
    for b, n in ((buf, R * 48), (sc, 1024)):
        assert bool((b[:4096] == 170).all()) and bool((b[4096 + n:] == 170).all())


# ------------------------------------------------------------------ GPU: linear
def linear_ref(xv, wv, bias, res, act):
    """(y64, bound before the output rounding) of the module docstring."""
    y = xv @ wv.T
    S = xv.abs() @ wv.abs().T
    if bias is not None:
        y, S = y + bias.double(), S + bias.double().abs()
    if res is not None:
        y, S = y + res.double(), S + res.double().abs()
    d = (xv.shape[1] / 16 + 16) * 2.0 ** -23 * S
    if act == 1:
        y = y * torch.sigmoid(y)
        d = 1.1 * d + 2.0 ** -20 * y.abs()
    elif act == 2:
        M = y.shape[0]
        v, g = y.view(M, -1, 2, 16).unbind(2)
        dv, dg = d.view(M, -1, 2, 16).unbind(2)
        ge = torch.nn.functional.gelu(g)
        d = (ge.abs() * dv + 1.13 * v.abs() * dg + 1.2 * dv * dg + 2.0 ** -20 * v.abs() * g.abs()).reshape(M, -1)
        y = (v * ge).reshape(M, -1)
    return y, d


def close(y, ref, d):
    t = torch.finfo(y.dtype)
    tol = d + (ref.abs() + d) * (t.eps / 2) + t.smallest_normal * t.eps / 2
    err = (y.double() - ref).abs()
    assert bool((err <= tol).all()), f"off by {float((err / tol).max()):.3g} of the bound"


def weight(sdg, N, K, seed):
    return sdg.quantize_mx4(rnd(N, K, seed=seed) / K ** 0.5)


SHAPES = [(1, 8, 32), (1, 1280, 1280), (2, 320, 33), (3, 72, 96), (4, 2560, 320), (8, 640, 640), (16, 1280, 320),
          (17, 24, 64), (33, 136, 352), (64, 64, 1000), (65, 1280, 5120), (127, 320, 768), (128, 128, 128),
          (129, 136, 160), (154, 2560, 768), (256, 256, 256), (300, 200, 2560), (512, 1280, 1280), (1000, 960, 320),
          (2048, 640, 2560), (5000, 320, 320), (8192, 320, 320), (20001, 320, 64),
          # long rows and many tiles: CTA pairs, with half a row tile and a w tile that one CTA has no row of
          (9985, 520, 2560), (20001, 200, 1800)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_linear(sdg, cuda, M, N, K, dtype):
    t = DT[dtype]
    wc, ws = weight(sdg, N, K, 1)
    x = rnd(M, K, seed=M + N + K, dtype=t, spread=1.0)
    xq = sdg.quantize_mx4(x)
    xv, wv = op64(*xq, K), op64(wc, ws, K)
    bias, res = 0.1 * rnd(N, seed=5), rnd(M, N, seed=6, dtype=t)
    for b, r, act in ((None, None, 0), (bias, None, 1), (bias, res, 0), (None, res, 1)):
        ref, d = linear_ref(xv, wv, b, r, act)
        y = sdg.linear_mx4(x, wc, ws, b, residual=r, act=act)
        assert y.shape == (M, N) and y.dtype == t
        close(y, ref, d)
        assert torch.equal(sdg.linear_mx4(xq[0], wc, ws, b, residual=r, act=act, xscale=xq[1], dtype=t), y)
    if N % 32 == 0:
        ref, d = linear_ref(xv, wv, bias, None, 2)
        y = sdg.linear_mx4(x, wc, ws, bias, act=2)
        assert y.shape == (M, N // 2)
        close(y, ref, d)


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K", [(1, 64, 64), (5, 64, 96), (200, 192, 320), (5000, 320, 320), (19999, 320, 1824)])
def test_linear_output_bounds_and_in_place(sdg, cuda, M, N, K):
    """Nothing is written around y; y may be the residual itself."""
    wc, ws = weight(sdg, N, K, 2)
    x, res = rnd(M, K, seed=3, dtype=torch.float16), rnd(M, N, seed=4, dtype=torch.float16)
    want = sdg.linear_mx4(x, wc, ws, residual=res)
    buf = torch.full((1024 + M * N + 130 * N,), 7.0, dtype=torch.float16, device=cuda)
    y = buf[1024:1024 + M * N].view(M, N)
    y.copy_(res)
    got = sdg.linear_mx4(x, wc, ws, residual=y, out=y)
    torch.cuda.synchronize()
    assert got is y and torch.equal(y, want)
    assert bool((buf[:1024] == 7).all()) and bool((buf[1024 + M * N:] == 7).all())


@pytest.mark.gpu
@pytest.mark.parametrize("M,N", [(1, 64), (3, 64), (200, 128)])
def test_linear_extreme_scales_and_nan(sdg, cuda, M, N):
    """A NaN in x makes its row NaN and no other; a NaN weight row its column; blocks of very unlike size add up."""
    K = 160
    w = rnd(N, K, seed=1)
    w[:, 64:96] *= 2.0 ** 40
    x = rnd(M, K, seed=2, dtype=torch.bfloat16)
    x[:, 64:96] *= 2.0 ** -40
    x[:, 96:128] = 0
    wc, ws = sdg.quantize_mx4(w)
    xq = sdg.quantize_mx4(x)
    ref, d = linear_ref(op64(*xq, K), op64(wc, ws, K), None, None, 0)
    close(sdg.linear_mx4(x, wc, ws), ref, d)
    x[M - 1, 3] = torch.nan
    w[5, 150] = torch.inf
    wc, ws = sdg.quantize_mx4(w)
    y = sdg.linear_mx4(x, wc, ws)
    nan = torch.zeros(M, N, dtype=torch.bool, device=cuda)
    nan[M - 1], nan[:, 5] = True, True
    assert torch.equal(torch.isnan(y), nan)
    close(y[~nan], ref[~nan], d[~nan])


@pytest.mark.gpu
def test_linear_accumulates_in_fp32(sdg, cuda):
    """2^14 + many small terms: an fp16 accumulator would lose them."""
    K, N, M = 4096, 64, 130
    x = torch.full((M, K), 1.0, dtype=torch.bfloat16, device=cuda)
    w = torch.full((N, K), 1.0, device=cuda)
    w[:, 0:32] = 512.0
    wc, ws = sdg.quantize_mx4(w)
    y = sdg.linear_mx4(x, wc, ws)
    assert bool((y.double() == torch.tensor(32 * 512.0 + K - 32).to(torch.bfloat16).double()).all())


@pytest.mark.gpu
def test_binding_refusals(sdg, cuda):
    x = rnd(4, 64, seed=1, dtype=torch.float16)
    wc, ws = weight(sdg, 32, 64, 2)
    gam = torch.ones(64, device=cuda)
    bad = {
        "x columns": lambda: sdg.linear_mx4(rnd(4, 128, seed=1, dtype=torch.float16), wc, ws),
        "fp32 x": lambda: sdg.linear_mx4(x.float(), wc, ws),
        "other dtype": lambda: sdg.linear_mx4(x, wc, ws, dtype=torch.bfloat16),
        "scale shape": lambda: sdg.linear_mx4(x, wc, ws.view(-1)),
        "bias shape": lambda: sdg.linear_mx4(x, wc, ws, gam),
        "bias type": lambda: sdg.linear_mx4(x, wc, ws, gam[:32].half()),
        "residual shape": lambda: sdg.linear_mx4(x, wc, ws, residual=x),
        "residual type": lambda: sdg.linear_mx4(x, wc, ws, residual=x[:, :32].bfloat16()),
        "geglu residual": lambda: sdg.linear_mx4(x, wc, ws, residual=x[:, :32].contiguous(), act=2),
        "act": lambda: sdg.linear_mx4(x, wc, ws, act=3),
        "out type": lambda: sdg.linear_mx4(x, wc, ws, out=torch.empty(4, 32, device=cuda)),
        "N": lambda: sdg.linear_mx4(x, *weight(sdg, 12, 64, 2)),
        "no rows": lambda: sdg.linear_mx4(x[:0], wc, ws),
        "quantise 3-D": lambda: sdg.quantize_mx4(x[None]),
        "quantise columns strided": lambda: sdg.quantize_mx4(x[:, ::2]),
        "quantise int": lambda: sdg.quantize_mx4(x.int()),
        "read back K": lambda: sdg.dequantize_mx4(wc, ws, 32),
        "groupnorm fp32": lambda: sdg.groupnorm_mx4(x.float()[None], gam, gam, 1e-5, False, groups=8),
        "groupnorm groups": lambda: sdg.groupnorm_mx4(x[None], gam, gam, 1e-5, False, groups=7),
        "groupnorm stats": lambda: sdg.groupnorm_mx4(x[None], gam, gam, 1e-5, False, groups=8, stats=gam[:1]),
        "cpu bias": lambda: sdg.linear_mx4(x, wc, ws, torch.zeros(32)),
    }
    for what, call in bad.items():
        with pytest.raises(sdg.SdgError) as ei:
            call()
        assert ei.value.code in (SDG_ERR_ARG, SDG_ERR_SHAPE), what


# ------------------------------------------------------------------ GPU: GroupNorm into an operand
def groupnorm_ref(x, gamma, beta, eps, silu, groups):
    """(y64 [B*HW, C], bound on the fp32 value)."""
    B, HW, C = x.shape
    t = x.double().view(B, HW, groups, -1)
    n = HW * (C // groups)
    var, mu = torch.var_mean(t, dim=(1, 3), correction=0, keepdim=True)
    rs = torch.rsqrt(var + eps)
    steps = n / 128 + 64
    e_mu = steps * 2.0 ** -24 * t.abs().mean((1, 3), keepdim=True)
    z = (t - mu) * rs
    ga, be = gamma.double().view(1, 1, groups, -1), beta.double().view(1, 1, groups, -1)
    y = z * ga + be
    # the variance's own relative error, plus what the mean's error adds to it: (e_mu)^2 and the rounding of x - mu
    rel = steps * 2.0 ** -24 + 2.0 ** -20 + (e_mu * rs) ** 2
    delta = ga.abs() * rs * e_mu + (z * ga).abs() * rel + ga.abs() * rs * 2.0 ** -23 * (t.abs() + mu.abs()) \
        + 2.0 ** -22 * (y.abs() + be.abs())
    if silu:
        y, delta = y * torch.sigmoid(y), 1.1 * delta
        delta = delta + 2.0 ** -20 * y.abs()
    return y.reshape(B * HW, C).cpu().numpy(), delta.reshape(B * HW, C).cpu().numpy()


def check_groupnorm(got, y, delta):
    code, e = O.unpack(got[0].cpu().numpy(), got[1].cpu().numpy())
    R, C = y.shape
    pad = -C % 32
    y, delta = np.pad(y, ((0, 0), (0, pad))), np.pad(delta, ((0, 0), (0, pad)))
    a, da = np.abs(y).reshape(R, -1, 32), delta.reshape(R, -1, 32)
    top_lo, top_hi = np.maximum(a - da, 0).max(-1), (a + da).max(-1)
    exp = lambda t: np.where(t > 0, np.frexp(t)[1] - 3, -127).clip(-127) + 127
    assert ((e >= exp(top_lo)) & (e <= exp(top_hi))).all()
    s = np.repeat(np.ldexp(1.0, e.astype(int) - 127), 32, axis=1)
    v = np.where(code & 8, -1.0, 1.0) * O.GRID[code & 7]

    def rne(u):
        w = np.minimum(np.abs(u), 6.0)
        lo, hi = np.searchsorted(O.MID, w, "left"), np.searchsorted(O.MID, w, "right")
        return np.copysign(O.GRID[np.where(lo % 2 == 0, lo, hi)], u)

    assert ((v >= rne((y - delta) / s)) & (v <= rne((y + delta) / s))).all()
    _, full = O.pack(code, e)
    assert np.array_equal(full, got[1].cpu().numpy())   # bytes of no block are zero
    return float((v != rne(y / s)).mean())


GN = [(1, 1, 32, 4), (2, 1, 64, 8), (1, 3, 8, 1), (1, 5, 40, 5), (3, 7, 72, 9), (2, 64, 1280, 32), (2, 130, 96, 3),
      (2, 256, 320, 32), (5, 77, 640, 32), (1, 1000, 960, 32), (1, 4096, 320, 32), (2, 1024, 640, 32), (3, 300, 2560, 64),
      (1, 16384, 64, 8), (17, 33, 128, 16), (1, 20000, 320, 32)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("silu", [False, True])
@pytest.mark.parametrize("B,HW,C,groups", GN)
def test_groupnorm(sdg, cuda, B, HW, C, groups, silu, dtype):
    x = (1.5 * rnd(B, HW, C, seed=B + HW + C) + rnd(B, 1, C, seed=9)).to(DT[dtype])
    gamma, beta = 1 + 0.2 * rnd(C, seed=1), 0.2 * rnd(C, seed=2)
    eps = 1e-5 if silu else 1e-6
    got = sdg.groupnorm_mx4(x, gamma, beta, eps, silu, groups=groups)
    off = check_groupnorm(got, *groupnorm_ref(x, gamma, beta, eps, silu, groups))
    assert off < 1e-3  # codes that a rounding error moved are rare
    again = sdg.groupnorm_mx4(x, gamma, beta, eps, silu, groups=groups)
    assert torch.equal(got[0], again[0]) and torch.equal(got[1], again[1])


@pytest.mark.gpu
@pytest.mark.parametrize("B,HW,C,groups", [(2, 64, 1280, 32), (2, 4096, 320, 32), (1, 20000, 64, 8)])
def test_groupnorm_large_mean_and_outlier(sdg, cuda, B, HW, C, groups):
    """Groups far from zero, and a first pixel unlike the rest: the variance is centred, not E[x^2] - mean^2."""
    x = rnd(B, HW, C, seed=4) + 30.0
    x[:, 0] -= 400.0
    x = x.half()
    gamma, beta = torch.ones(C, device=cuda), torch.zeros(C, device=cuda)
    check_groupnorm(sdg.groupnorm_mx4(x, gamma, beta, 1e-5, False, groups=groups),
                    *groupnorm_ref(x, gamma, beta, 1e-5, False, groups))


@pytest.mark.gpu
def test_groupnorm_image_does_not_depend_on_batch(sdg, cuda):
    x = rnd(6, 256, 320, seed=8, dtype=torch.float16)
    gamma, beta = 1 + 0.2 * rnd(320, seed=1), 0.2 * rnd(320, seed=2)
    a = sdg.dequantize_mx4(*sdg.groupnorm_mx4(x, gamma, beta, 1e-5, True))
    b = sdg.dequantize_mx4(*sdg.groupnorm_mx4(x[3:4].contiguous(), gamma, beta, 1e-5, True))
    assert torch.equal(a.view(6, 256, 320)[3], b.view(256, 320))


@pytest.mark.gpu
def test_groupnorm_constant_and_nan_groups(sdg, cuda):
    """A constant group has variance 0 (eps carries it); a NaN spoils its own group only."""
    x = rnd(2, 100, 64, seed=1).half()
    x[0, :, 0:8] = 3.0
    x[1, 50, 33] = torch.nan
    gamma, beta = torch.ones(64, device=cuda), torch.full((64,), 0.25, device=cuda)
    y = sdg.dequantize_mx4(*sdg.groupnorm_mx4(x, gamma, beta, 1e-5, False, groups=8), dtype=torch.float32).view(2, 100, 64)
    assert not torch.isnan(y[0]).any()
    # group 4 (channels 32..39) is NaN; it shares its block with groups 5 to 7
    assert bool(torch.isnan(y[1, :, 32:]).all()) and not torch.isnan(y[1, :, :32]).any()


# ------------------------------------------------------------------ GPU: together, streams, graphs
def _block(sdg, x, p):
    """The operators as a transformer's entry and feed-forward use them: norm, projection, GEGLU, projection + residual."""
    q = sdg.groupnorm_mx4(x, p["g"], p["b"], 1e-6, False)
    h = sdg.linear_mx4(q[0], *p["w0"], p["b0"], xscale=q[1])
    f = sdg.linear_mx4(h, *p["w1"], p["b1"], act=2)
    return sdg.linear_mx4(f, *p["w2"], p["b0"], residual=h)


@pytest.fixture(scope="module")
def block(sdg, cuda):
    C = 320
    w1, b1 = sdg.pack_geglu_weight(rnd(8 * C, C, seed=12) / C ** 0.5, 0.1 * rnd(8 * C, seed=13))
    return {"g": 1 + 0.2 * rnd(C, seed=1), "b": 0.2 * rnd(C, seed=2), "w0": weight(sdg, C, C, 11), "b0": 0.1 * rnd(C, seed=3),
            "w1": sdg.quantize_mx4(w1), "b1": b1, "w2": weight(sdg, C, 4 * C, 14)}


def test_chain_names(sdg):
    for name in ("quantize_mx4", "dequantize_mx4", "linear_mx4", "groupnorm_mx4"):
        assert callable(getattr(sdg, name))


@pytest.mark.gpu
@pytest.mark.parametrize("HW", [64, 1024])
def test_chain(sdg, cuda, block, HW):
    """The chain against 64 bits on the same operands, step by step from each step's own input."""
    x = rnd(2, HW, 320, seed=HW, dtype=torch.float16)
    p = block
    q = sdg.groupnorm_mx4(x, p["g"], p["b"], 1e-6, False)
    check_groupnorm(q, *groupnorm_ref(x, p["g"], p["b"], 1e-6, False, 32))
    h = sdg.linear_mx4(q[0], *p["w0"], p["b0"], xscale=q[1])
    close(h, *linear_ref(op64(*q, 320), op64(*p["w0"], 320), p["b0"], None, 0))
    f = sdg.linear_mx4(h, *p["w1"], p["b1"], act=2)
    close(f, *linear_ref(op64(*sdg.quantize_mx4(h), 320), op64(*p["w1"], 320), p["b1"], None, 2))
    y = sdg.linear_mx4(f, *p["w2"], p["b0"], residual=h)
    close(y, *linear_ref(op64(*sdg.quantize_mx4(f), 1280), op64(*p["w2"], 1280), p["b0"], h, 0))
    assert torch.equal(_block(sdg, x, p), y)


@pytest.mark.gpu
def test_graph_replay_and_two_graphs(sdg, cuda, block):
    xs = [rnd(2, 256, 320, seed=20 + i, dtype=torch.float16) for i in range(2)]
    want = [_block(sdg, x, block) for x in xs]
    graphs, outs, ins = [], [], []
    for x in xs:
        buf = x.clone()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(_block(sdg, buf, block))
        graphs.append(g)
        ins.append(buf)
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(3):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for o, w in zip(outs, want))
    ins[0].copy_(xs[1])
    graphs[0].replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want[1])


@pytest.mark.gpu
def test_side_streams(sdg, cuda, block):
    """Calls on the current stream of a context, and on a raw handle, overlap without touching each other."""
    xs = [rnd(2, 1024, 320, seed=30 + i, dtype=torch.float16) for i in range(4)]
    want = [_block(sdg, x, block) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    got = []
    for x, st in zip(xs, streams):
        with torch.cuda.stream(st):
            got.append(_block(sdg, x, block))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    wc, ws = block["w0"]
    base = sdg.linear_mx4(xs[0].view(-1, 320), wc, ws)
    torch.cuda.synchronize()
    for _ in range(20):
        y = sdg.linear_mx4(xs[0].view(-1, 320), wc, ws, stream=streams[0].cuda_stream)
        junk = [torch.full((xs[0].numel(),), 255, dtype=torch.uint8, device=cuda) for _ in range(3)]
        streams[0].synchronize()
        assert torch.equal(y, base)
        del junk


FIRST_CALL = """
import sys, torch
sys.path.insert(0, {root!r})
import importlib
sdg = importlib.import_module({pkg!r})
x = torch.randn(300, 320, device="cuda").half()
big = torch.randn(8192, 320, device="cuda").half()
ga, be = torch.ones(320, device="cuda"), torch.zeros(320, device="cuda")
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    w = sdg.quantize_mx4(big[:2560])
    a = sdg.linear_mx4(x, *w)
    b = sdg.linear_mx4(big, *w, act=2)
    q = sdg.groupnorm_mx4(big.view(2, 4096, 320), ga, be, 1e-5, True)
    c = sdg.linear_mx4(q[0], *w, xscale=q[1])
    d = sdg.dequantize_mx4(*w)
g.replay()
torch.cuda.synchronize()
w2 = sdg.quantize_mx4(big[:2560])
q2 = sdg.groupnorm_mx4(big.view(2, 4096, 320), ga, be, 1e-5, True)
assert torch.equal(w[0], w2[0]) and torch.equal(w[1], w2[1]) and torch.equal(d, sdg.dequantize_mx4(*w2))
assert torch.equal(a, sdg.linear_mx4(x, *w2)) and torch.equal(b, sdg.linear_mx4(big, *w2, act=2))
assert torch.equal(c, sdg.linear_mx4(q2[0], *w2, xscale=q2[1]))
print("captured")
"""


@pytest.mark.gpu
def test_first_calls_inside_a_capture(cuda):
    """In a fresh process the first call of every operator may come while a stream is being captured."""
    import subprocess
    import sys

    from conftest import PKG, ROOT
    out = subprocess.run([sys.executable, "-c", FIRST_CALL.format(root=ROOT, pkg=PKG)], capture_output=True, text=True,
                         timeout=300)
    assert out.returncode == 0 and "captured" in out.stdout, out.stderr[-2000:]


@pytest.mark.gpu
def test_views_of_unaligned_storage(sdg, cuda):
    """x that starts off a 16-byte boundary, or whose rows do, goes another way to the same result."""
    K, N = 320, 256
    wc, ws = weight(sdg, N, K, 3)
    for M in (1, 5, 64, 300):
        flat = rnd(M * (K + 8) + 8, seed=M, dtype=torch.float16)
        want = None
        for first, ld in ((0, K), (1, K), (8, K + 8), (3, K + 3)):
            x = flat[first:first + M * ld].view(M, ld)[:, :K]
            src = rnd(M, K, seed=7, dtype=torch.float16)
            x.copy_(src)
            y = sdg.linear_mx4(x, wc, ws)
            want = y if want is None else want
            assert torch.equal(y, want)
