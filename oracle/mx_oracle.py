"""Block-scaled formats in 64 bits with numpy: the definitions the kernels are tested against.

nvfp4: e2m1 codes, blocks of 16, e4m3 scales, one tensor scale; mxfp4 and mxfp8: e2m1 / e4m3 codes,
blocks of 32, power-of-two scales 2^(floor(log2 amax) - emax).  Rounding is to nearest, ties to even.
"""
from __future__ import annotations

import numpy as np

BLOCK = {"nvfp4": 16, "mxfp4": 32, "mxfp8": 32}
E2M1 = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6])
_BYTES = np.arange(256)
_E, _F = (_BYTES >> 3) & 15, _BYTES & 7
E4M3 = np.where(_E > 0, np.ldexp(1 + _F / 8, _E - 7), np.ldexp(_F / 8, -6)) * np.where(_BYTES >= 128, -1.0, 1.0)
E4M3 = np.where((_BYTES & 127) == 127, np.nan, E4M3)
with np.errstate(over="ignore"):
    E8M0 = np.where(_BYTES == 255, np.nan, np.ldexp(1.0, _BYTES - 127))


def k_pad(k: int) -> int:
    return -(-k // 128) * 128


def _nearest(v: np.ndarray, values: np.ndarray) -> np.ndarray:
    """Index of the nearest of ``values`` (ascending, index 0 = zero) to each |v|; halfway goes to the
    even index, beyond the last one to the last one."""
    mid = (values[1:] + values[:-1]) / 2  # exact in 64 bits
    a = np.abs(v)
    lo = np.searchsorted(mid, a, side="left")   # midpoints below a
    hi = np.searchsorted(mid, a, side="right")  # midpoints at or below a
    return np.where(lo == hi, lo, np.where(lo % 2 == 0, lo, hi))


def quantize(x: np.ndarray, fmt: str, tensor_scale: float = 1.0):
    """x [M, K] -> (codes [M, K_pad] as the bytes / nibbles of the format, scale bytes [M, blocks])."""
    m, k = x.shape
    b = BLOCK[fmt]
    v = np.zeros((m, k_pad(k)))
    v[:, :k] = x
    v = v.reshape(m, -1, b)
    with np.errstate(all="ignore"):
        amax = np.abs(v).max(-1)
        bad = ~np.isfinite(v).all(-1)
        if fmt == "nvfp4":
            t = amax / (6 * np.float64(tensor_scale))
            if not (np.isfinite(tensor_scale) and tensor_scale > 0):
                bad = np.ones_like(bad)
            byte = _nearest(np.where(bad, 0, t), E4M3[:127]).astype(np.int64)
            unit = E4M3[byte] * np.float64(tensor_scale)
        else:
            emax = 2 if fmt == "mxfp4" else 8
            e = np.frexp(np.where(bad | (amax == 0), 1.0, amax))[1] - 1 - emax
            byte = np.where(amax == 0, 0, np.clip(e + 127, 0, 254))
            unit = np.ldexp(1.0, byte - 127)
        byte = np.where(bad, 127 if fmt == "nvfp4" else 255, byte)
        q = np.where((unit == 0)[..., None] | bad[..., None], 0.0, v / unit[..., None])
    table = E4M3[:127] if fmt == "mxfp8" else E2M1[:8]
    codes = _nearest(q, table) | (np.signbit(q).astype(np.int64) << (7 if fmt == "mxfp8" else 3))
    codes = np.where((bad | (unit == 0))[..., None], 0, codes)
    return codes.reshape(m, -1), byte


def values(codes: np.ndarray, scale_bytes: np.ndarray, fmt: str, tensor_scale: float = 1.0) -> np.ndarray:
    """The values [M, K_pad] that codes and scale bytes stand for."""
    v = (E4M3 if fmt == "mxfp8" else E2M1)[codes]
    s = E4M3[scale_bytes] * np.float64(tensor_scale) if fmt == "nvfp4" else E8M0[scale_bytes]
    return (v.reshape(len(v), -1, BLOCK[fmt]) * s[..., None]).reshape(len(v), -1)


def unpack(codes: np.ndarray, fmt: str) -> np.ndarray:
    """Stored code bytes -> one code per column."""
    if fmt == "mxfp8":
        return codes.astype(np.int64)
    return np.stack((codes & 15, codes >> 4), -1).reshape(len(codes), -1).astype(np.int64)


def scale_index(rows: int, blocks: int) -> np.ndarray:
    """Byte offset of each (row, block) scale in the tile layout."""
    r, c = np.arange(rows)[:, None], np.arange(blocks)[None, :]
    return ((r // 128) * (blocks // 4) + c // 4) * 512 + (r % 32) * 16 + (r // 32 % 4) * 4 + c % 4


def rms_norm(h: np.ndarray, weight: np.ndarray | None, eps: float) -> np.ndarray:
    h = h.astype(np.float64)
    y = h / np.sqrt((h * h).mean(-1, keepdims=True) + eps)
    return y if weight is None else y * weight.astype(np.float64)
