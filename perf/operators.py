"""The operators of 4-bit microscaled (MXFP4) serving: what is measured, and their plain forms.

An MXFP4 matrix [rows, K] is held as two arrays. ``codes`` [rows, Kp/2] uint8 (Kp = K rounded up to 32): two
E2M1 values a byte, the even column in the low nibble; zero codes behind column K. ``scales``
[ceil(rows/128), ceil(Kp/128), 512] uint8: one E8M0 exponent for each 32 columns of a row, in tiles of 128 rows x
4 blocks; the exponent of row r, block b is byte (r % 32) * 16 + (r // 32 % 4) * 4 + b % 4 of tile (r // 128, b // 4);
bytes that belong to no block are zero. A block's exponent is floor(log2(max|x|)) - 2, at least -127 (OCP
Microscaling Formats 1.0, section 6.3; E2M1's largest exponent is 2), and its codes are x / 2^exponent rounded to
nearest even and saturated at +-6.

Three operators, one ``kind`` of case each:

  quantize   x [M, K] -> codes and scales, and read back to x's type: the values that the operand stands for
  linear     y = act(x4 w4^T + bias + residual): x quantised on the way, w kept in MXFP4 (act: 0, 1 SiLU, 2 GEGLU
             over weight rows interleaved [16 value rows ; their 16 gate rows])
  groupnorm  GroupNorm (+ SiLU) over channels-last x [B, HW, C] straight into an MXFP4 operand, and the product that
             reads it: y [B * HW, N]
"""
import importlib
import math

import torch

own = False
_PKG = "sd-vulkan-pixel10-tensor-g5_b200"
_DT = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
_ES = {"fp16": 2, "bf16": 2, "fp32": 4}


def listed():
    return [
        # the text encoder's 2 x 77 context tokens of one guided image
        {"name": "quantize_context", "kind": "quantize", "M": 154, "K": 768, "dtype": "fp16"},
        # the GEGLU projection's weight of the 1280-channel level, from an fp32 checkpoint
        {"name": "quantize_weight", "kind": "quantize", "M": 10240, "K": 1280, "dtype": "fp32"},
        # odd rows and a K that ends inside a block and off every vector width
        {"name": "quantize_odd", "kind": "quantize", "M": 20001, "K": 333, "dtype": "bf16"},
        # the 64x64-latent tokens of 32 images with guidance
        {"name": "quantize_tokens", "kind": "quantize", "M": 262144, "K": 320, "dtype": "fp16"},
        # the time-embedding MLP of one timestep: a single row
        {"name": "linear_time_row", "kind": "linear", "M": 1, "K": 1280, "N": 1280, "bias": True, "residual": False,
         "act": 1, "dtype": "fp16"},
        # cross-attention keys and values from the context: ragged rows, no bias
        {"name": "linear_context", "kind": "linear", "M": 154, "K": 768, "N": 2560, "bias": False, "residual": False,
         "act": 0, "dtype": "fp16"},
        # an attention out-projection with its residual, one guided image at 64x64
        {"name": "linear_out_proj", "kind": "linear", "M": 8192, "K": 320, "N": 320, "bias": True, "residual": True,
         "act": 0, "dtype": "fp16"},
        # the GEGLU projection of one guided image at 64x64
        {"name": "linear_geglu", "kind": "linear", "M": 8192, "K": 320, "N": 2560, "bias": True, "residual": False,
         "act": 2, "dtype": "fp16"},
        # the feed-forward's second product at 32x32 for 32 guided images
        {"name": "linear_ff_out", "kind": "linear", "M": 65536, "K": 2560, "N": 640, "bias": True, "residual": True,
         "act": 0, "dtype": "bf16"},
        # transformer entry of the 8x8 level: few pixels, many channels
        {"name": "groupnorm_mid", "kind": "groupnorm", "B": 2, "HW": 64, "C": 1280, "groups": 32, "silu": False,
         "N": 1280, "dtype": "fp16"},
        # transformer entry of the 64x64 level
        {"name": "groupnorm_top", "kind": "groupnorm", "B": 2, "HW": 4096, "C": 320, "groups": 32, "silu": False,
         "N": 320, "dtype": "fp16"},
        # norm + SiLU + 1x1 product of the 32x32 level for 32 guided images
        {"name": "groupnorm_batch", "kind": "groupnorm", "B": 64, "HW": 1024, "C": 640, "groups": 32, "silu": True,
         "N": 640, "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["quantize", "linear", "linear", "groupnorm"])
    if kind == "quantize":
        K = _log(rng, 1, 5120)
        K = K if rng.random() < 0.5 else (K + 31) // 32 * 32
        return {"kind": kind, "M": min(_log(rng, 1, 262144), max(1, 262144 * 320 // K)), "K": K,
                "dtype": rng.choice(["fp16", "bf16", "fp32"])}
    if kind == "linear":
        K = _log(rng, 16, 5120)
        K = K if rng.random() < 0.25 else max(32, K // 32 * 32)
        act = rng.choice([0, 0, 1, 2])
        step = 32 if act == 2 else 8
        N = max(step, _log(rng, 8, 10240) // step * step)
        M = min(_log(rng, 1, 65536), 65536 * 2560 * 640 // (K * N), 65536 * 2560 // K, 65536 * 640 // N)
        return {"kind": kind, "M": max(1, M), "K": K, "N": N, "bias": rng.random() < 0.7,
                "residual": act != 2 and rng.random() < 0.5, "act": act, "dtype": rng.choice(["fp16", "bf16"])}
    groups = rng.choice([4, 8, 16, 32, 32])
    C = max(1, _log(rng, 32, 2560) // (8 * groups)) * 8 * groups
    if rng.random() < 0.5:
        C = max(1, _log(rng, 64, 2560) // 320) * 320
    HW = _log(rng, 1, 16384)
    B = max(1, min(_log(rng, 1, 64), 64 * 1024 * 640 // (HW * C)))
    N = C if rng.random() < 0.5 else max(8, _log(rng, 8, 2560) // 8 * 8)
    return {"kind": kind, "B": B, "HW": HW, "C": C, "groups": groups, "silu": rng.random() < 0.5, "N": N,
            "dtype": rng.choice(["fp16", "bf16"])}


# ------------------------------------------------------------------ inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))

    def rn(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    dt = _DT[case["dtype"]]
    s = {"case": case, "dtype": dt}
    if case["kind"] == "quantize":
        x = rn(case["M"], case["K"])
        x *= torch.exp(0.5 * rn(1, case["K"]))  # channels of unlike size, as activations have
        s["x"] = x.to(dt)
        return s
    if case["kind"] == "linear":
        M, K = case["M"], case["K"]
        x = rn(M, K)
        x *= torch.exp(0.5 * rn(1, K))
        s["x"] = x.to(dt)
    else:
        B, HW, K = case["B"], case["HW"], case["C"]
        M = B * HW
        s["x"] = (1.5 * rn(B, HW, K) + 0.5 * rn(B, 1, K)).to(dt)
        s["gamma"] = 1.0 + 0.2 * rn(K)
        s["beta"] = 0.2 * rn(K)
        s["eps"] = 1e-5 if case["silu"] else 1e-6
    N = case["N"]
    s["codes"], s["scales"] = _pack(rn(N, K) / math.sqrt(K))  # the weight, quantised and laid out once
    s["bias"] = 0.1 * rn(N) if case.get("bias", True) else None
    s["residual"] = rn(M, N).to(dt) if case.get("residual", False) else None
    return s


def _pack(w):
    """A matrix in MXFP4: codes and tiled scales as the module's docstring lays them out."""
    y, e = _blocks(w)
    R, KB = e.shape
    a = y.abs()
    code = (a >= 0.5).to(torch.uint8)
    for v in (1.0, 1.5, 2.0, 3.0, 4.0, 6.0):
        code += a >= v
    code += (y < 0).to(torch.uint8) * 8
    code = code.reshape(R, KB * 16, 2)
    codes = code[..., 0] | (code[..., 1] << 4)
    rt, kt = -(-R // 128), -(-KB // 4)
    full = torch.zeros(rt * 128, kt * 4, dtype=torch.uint8, device=w.device)
    full[:R, :KB] = e.to(torch.uint8)
    tiles = full.reshape(rt, 4, 32, kt, 4).permute(0, 3, 2, 1, 4).reshape(rt, kt, 512)
    return codes.contiguous(), tiles.contiguous()


# ------------------------------------------------------------------ plain forms (32 bits)
def _blocks(x):
    """Values on the E2M1 grid [R, KB, 32] and biased block exponents [R, KB] of x [R, K]."""
    R, K = x.shape
    KB = -(-K // 32)
    x = x.float()
    if KB * 32 != K:
        x = torch.cat([x, torch.zeros(R, KB * 32 - K, device=x.device)], 1)
    x = x.reshape(R, KB, 32)
    amax = x.abs().amax(-1)
    e = (((amax.view(torch.int32) >> 23) & 255) - 2).clamp_min(0)
    inv = ((254 - e) << 23).view(torch.float32)
    a = x.abs() * inv[..., None]
    q = 0.5 * ((a > 0.25).float() + (a >= 0.75) + (a > 1.25) + (a >= 1.75)) + (a > 2.5) + (a >= 3.5) + 2.0 * (a > 5.0)
    return torch.where(x < 0, -q, q), e


def _power(e):
    """2^(e - 127) in fp32, from its bits (e = 0 is the subnormal 2^-127)."""
    return torch.where(e > 0, e << 23, 0x00400000).to(torch.int32).view(torch.float32)


def _plain_values(x):
    y, e = _blocks(x)
    return (y * _power(e)[..., None]).reshape(x.shape[0], -1)


def _plain_weight(codes, scales):
    grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=codes.device)
    grid = torch.cat([grid, -grid])
    R, half = codes.shape
    v = torch.stack([grid[(codes & 15).int()], grid[(codes >> 4).int()]], -1).reshape(R, half // 16, 32)
    rt, kt = scales.shape[:2]
    e = scales.reshape(rt, kt, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(rt * 128, kt * 4)[:R, : half // 16].int()
    return (v * _power(e)[..., None]).reshape(R, 2 * half)


def _plain_product(xv, s):
    c = s["case"]
    y = xv @ _plain_weight(s["codes"], s["scales"]).t()
    if s["bias"] is not None:
        y = y + s["bias"]
    if s["residual"] is not None:
        y = y + s["residual"].float()
    act = c.get("act", 0)
    if act == 1:
        y = y / (1.0 + torch.exp(-y))
    elif act == 2:
        y = y.reshape(y.shape[0], -1, 2, 16)
        gate = y[:, :, 1]
        y = (y[:, :, 0] * (0.5 * gate * (1.0 + torch.erf(gate * math.sqrt(0.5))))).reshape(y.shape[0], -1)
    return y.to(s["dtype"])


def _plain(s):
    c = s["case"]
    if c["kind"] == "quantize":
        return _plain_values(s["x"])[:, : c["K"]].to(s["dtype"])
    if c["kind"] == "linear":
        return _plain_product(_plain_values(s["x"]), s)
    B, HW, C, G = c["B"], c["HW"], c["C"], c["groups"]
    x = s["x"].float().reshape(B, HW, G, C // G)
    d = x - x.mean((1, 3), keepdim=True)
    var = (d * d).mean((1, 3), keepdim=True)
    y = (d / torch.sqrt(var + s["eps"])).reshape(B * HW, C) * s["gamma"] + s["beta"]
    if c["silu"]:
        y = y / (1.0 + torch.exp(-y))
    return _plain_product(_plain_values(y), s)


# ------------------------------------------------------------------ one pass
_mod = None


def run(s):
    if not own:
        return _plain(s)
    global _mod
    if _mod is None:
        _mod = importlib.import_module(_PKG)
    c = s["case"]
    if c["kind"] == "quantize":
        codes, scales = _mod.quantize_mx4(s["x"])
        return _mod.dequantize_mx4(codes, scales, c["K"], dtype=s["dtype"])
    if c["kind"] == "linear":
        return _mod.linear_mx4(s["x"], s["codes"], s["scales"], s["bias"], residual=s["residual"], act=c["act"])
    codes, scales = _mod.groupnorm_mx4(s["x"], s["gamma"], s["beta"], s["eps"], c["silu"], groups=c["groups"])
    return _mod.linear_mx4(codes, s["codes"], s["scales"], s["bias"], xscale=scales, dtype=s["dtype"])


def work(case):
    es = _ES[case["dtype"]]
    if case["kind"] == "quantize":
        M, K = case["M"], case["K"]
        return {"bytes": 2 * M * K * es + M * (-(-K // 32)) * 17, "flops": 2 * M * K}
    if case["kind"] == "linear":
        M, K = case["M"], case["K"]
    else:
        M, K = case["B"] * case["HW"], case["C"]
    N, KB = case["N"], -(-K // 32)
    out = N // 2 if case.get("act") == 2 else N
    b = M * K * es + N * KB * 17 + M * out * es
    b += 4 * N if case.get("bias", True) else 0
    b += M * N * es if case.get("residual", False) else 0
    b += 8 * K if case["kind"] == "groupnorm" else 0
    return {"bytes": b, "flops": 2 * M * N * K}


# ------------------------------------------------------------------ the definition in 64 bits
def _exact_values(x):
    """The MXFP4 values of x [R, K] (fp64, K any): exponent by frexp, codes by the nearest grid point."""
    R, K = x.shape
    out = torch.empty_like(x)
    mid = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], dtype=torch.float64, device=x.device)
    grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64, device=x.device)
    rows = max(1, (1 << 24) // max(K, 32))
    for r0 in range(0, R, rows):
        b = torch.nn.functional.pad(x[r0:r0 + rows], (0, -K % 32)).unflatten(1, (-1, 32))
        top = b.abs().amax(-1, keepdim=True)
        p = torch.where(top > 0, torch.frexp(top)[1] - 3, -127).clamp_min(-127).double()
        a = (b * torch.exp2(-p)).abs()
        below = torch.searchsorted(mid, a.contiguous())              # midpoints < a
        reach = torch.searchsorted(mid, a.contiguous(), right=True)  # midpoints <= a
        code = torch.where(below % 2 == 0, below, reach)             # a tie goes to the even code
        v = torch.copysign(grid[code], b) * torch.exp2(p)
        out[r0:r0 + rows] = v.flatten(1)[:, :K]
    return out


def _exact_weight(codes, scales, K):
    R = codes.shape[0]
    col = torch.arange(K, device=codes.device)
    row = torch.arange(R, device=codes.device)[:, None]
    nib = (codes[:, col // 2].int() >> (4 * (col % 2)).int()) & 15
    blk = col // 32
    e = scales[row // 128, blk // 4, (row % 32) * 16 + (row // 32 % 4) * 4 + blk % 4].double()
    m, x = (nib & 1).double(), (nib >> 1 & 3).double()
    mag = torch.where(x > 0, (1 + m / 2) * torch.exp2(x - 1), m / 2)
    return torch.where(nib > 7, -mag, mag) * torch.exp2(e - 127)


def exact(case, seed):
    s = prepare(case, seed)
    x = s["x"].double()
    if case["kind"] == "quantize":
        return _exact_values(x)
    if case["kind"] == "groupnorm":
        B, HW, C = x.shape
        t = x.view(B, HW, case["groups"], -1)
        var, mean = torch.var_mean(t, dim=(1, 3), correction=0, keepdim=True)
        x = ((t - mean) * torch.rsqrt(var + s["eps"])).view(B * HW, C)
        x = torch.addcmul(s["beta"].double(), x, s["gamma"].double())
        if case["silu"]:
            x = x * torch.sigmoid(x)
    y = _exact_values(x) @ _exact_weight(s["codes"], s["scales"], x.shape[1]).T
    if s["bias"] is not None:
        y += s["bias"].double()
    if s["residual"] is not None:
        y += s["residual"].double()
    if case.get("act") == 1:
        y = y * torch.sigmoid(y)
    elif case.get("act") == 2:
        v, gate = y.unflatten(1, (-1, 32)).split(16, dim=-1)
        y = (v * torch.nn.functional.gelu(gate)).flatten(1)
    return y
