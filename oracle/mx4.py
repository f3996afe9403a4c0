"""MXFP4 operands in 64 bits (numpy): the format of ``include/sdg.h``'s 4-bit section restated from the OCP
Microscaling Formats specification 1.0 (E2M1 elements, E8M0 exponents, blocks of 32; conversion of section 6.3).
Test infrastructure only."""
from __future__ import annotations

import numpy as np

GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
MID = (GRID[1:] + GRID[:-1]) / 2
NAN = 255


def quantize(x: np.ndarray):
    """x [R, K] fp64 -> (code [R, Kp] uint8 in 0..15, biased exponent [R, Kp/32] uint8)."""
    R, K = x.shape
    b = np.zeros((R, -(-K // 32) * 32))
    b[:, :K] = x
    b = b.reshape(R, -1, 32)
    bad = ~np.isfinite(b).all(-1)
    b = np.where(bad[..., None], 0.0, b)
    top = np.abs(b).max(-1)
    p = np.where(top > 0, np.frexp(top)[1] - 3, -127).clip(-127)
    a = np.ldexp(np.abs(b), -p[..., None])
    lo, hi = np.searchsorted(MID, a, "left"), np.searchsorted(MID, a, "right")  # they differ on a tie
    code = np.where(lo % 2 == 0, lo, hi) + 8 * np.signbit(b)
    e = np.where(bad, NAN, p + 127)
    code[bad] = 0
    return code.reshape(R, -1).astype(np.uint8), e.astype(np.uint8)


def values(code: np.ndarray, e: np.ndarray) -> np.ndarray:
    v = np.where(code & 8, -1.0, 1.0) * GRID[code & 7]
    s = np.where(e == NAN, np.nan, np.ldexp(1.0, e.astype(int) - 127))
    return v * np.repeat(s, 32, axis=1)


def pack(code: np.ndarray, e: np.ndarray):
    """Codes and exponents -> the two device arrays."""
    R, KB = e.shape
    codes = code[:, 0::2] | (code[:, 1::2] << 4)
    scales = np.zeros((-(-R // 128), -(-KB // 4), 512), np.uint8)
    r, b = np.indices((R, KB))
    scales[r // 128, b // 4, (r % 32) * 16 + (r // 32 % 4) * 4 + b % 4] = e
    return codes, scales


def unpack(codes: np.ndarray, scales: np.ndarray):
    R, half = codes.shape
    code = np.empty((R, 2 * half), np.uint8)
    code[:, 0::2], code[:, 1::2] = codes & 15, codes >> 4
    r, b = np.indices((R, half // 16))
    return code, scales[r // 128, b // 4, (r % 32) * 16 + (r // 32 % 4) * 4 + b % 4]
