"""Microscaled 4-bit floats in numpy, 64 bits: the format's definition by search over its eight magnitudes."""

import numpy as np

LEVELS = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
SIGNED = np.concatenate([LEVELS, -LEVELS])


def unpack(packed: np.ndarray) -> np.ndarray:
    """Codes [rows, cols] of bytes [rows, cols / 2]."""
    return np.stack([packed & 15, packed >> 4], -1).reshape(packed.shape[0], -1)


def values(packed: np.ndarray, scale: np.ndarray) -> np.ndarray:
    """float64 [rows, cols]."""
    s = np.where(scale == 255, np.nan, np.ldexp(1.0, scale.astype(int) - 127))
    return SIGNED[unpack(packed)] * np.repeat(s, 32, axis=1)


def exponent(most: float, rule: str) -> int:
    """Of a block whose largest magnitude is `most` (finite)."""
    if most == 0:
        return -127
    e = int(np.frexp(most)[1]) - 1 - 2
    if rule == "ceil" and np.ldexp(6.0, e) < most:
        e += 1
    return min(max(e, -127), 127)


def quantize(x: np.ndarray, rule: str = "floor") -> tuple[np.ndarray, np.ndarray]:
    """(packed, scale) of finite and other values, any float type."""
    x = np.asarray(x, dtype=np.float64)
    rows, cols = x.shape
    codes = np.zeros((rows, cols), dtype=np.uint8)
    scale = np.zeros((rows, cols // 32), dtype=np.uint8)
    for i in range(rows):
        for j in range(cols // 32):
            b = x[i, 32 * j:32 * j + 32]
            if not np.isfinite(b).all():
                scale[i, j] = 255
                continue
            e = exponent(np.abs(b).max(), rule)
            a = np.ldexp(np.abs(b), -e)
            d = np.abs(a[:, None] - LEVELS)  # of two as near the even code: the odd ones are put a hair farther off
            best = d.min(1, keepdims=True)
            tie = d == best
            code = np.where(tie.sum(1) == 1, tie.argmax(1), np.where(tie.argmax(1) % 2 == 0, tie.argmax(1), tie.argmax(1) + 1))
            codes[i, 32 * j:32 * j + 32] = code | (np.signbit(b).astype(np.uint8) << 3)
            scale[i, j] = e + 127
    return codes[:, 0::2] | codes[:, 1::2] << 4, scale


def random_mx(rng, rows: int, cols: int, lo: int = 119, hi: int = 125) -> tuple[np.ndarray, np.ndarray]:
    return (rng.integers(0, 256, (rows, cols // 2), dtype=np.uint8), rng.integers(lo, hi + 1, (rows, cols // 32)).astype(np.uint8))
