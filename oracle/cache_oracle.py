"""The paged cache in 4 bits, restated with numpy in 64 bits: quantising,
the rows' layout and back, and attention over the values.  Test
infrastructure only."""
import numpy as np


def row_bytes(head_dim):
    return 16 * next(w for w in (2, 3, 4, 8) if 32 * w >= head_dim)


def to_fp16(x):
    """FP16 values of finite numbers, saturated; others stay."""
    x = np.asarray(x, np.float64)
    with np.errstate(over="ignore", invalid="ignore"):
        y = np.clip(x, -65504, 65504).astype(np.float32).astype(np.float16).astype(np.float64)
    return np.where(np.isfinite(x), y, np.nan)


def quantise(x, group):
    """x [..., D] (any numbers) -> codes [..., D], (scale, low) [..., groups]."""
    x = to_fp16(x)
    shape = x.shape
    x = x.reshape(shape[:-1] + (-1, group))
    low, high = x.min(-1), x.max(-1)
    scale = ((high - low) / 15).astype(np.float32).astype(np.float16)
    over = low + 15 * scale.astype(np.float64) > 65504
    scale = np.where(over, np.nextafter(scale, np.float16(0)), scale)
    s = scale.astype(np.float64)[..., None]
    with np.errstate(divide="ignore", invalid="ignore"):
        u = np.floor((x - low[..., None]) / s + 0.5)
    u = np.where(s > 0, np.clip(u, 0, 15), 0)
    bad = np.isnan(low)
    return (np.where(bad[..., None], 0, u).reshape(shape).astype(np.uint8), np.where(bad, np.float16(np.nan), scale),
            np.where(bad, np.nan, low).astype(np.float16))


def pack(codes):
    D = codes.shape[-1]
    W = row_bytes(D) // 16
    row = np.zeros(codes.shape[:-1] + (16 * W,), np.uint8)
    for d in range(D):
        row[..., d % 16 * W + d // 32] |= codes[..., d] << (4 if d & 16 else 0)
    return row


def unpack(rows, D):
    W = row_bytes(D) // 16
    codes = np.zeros(rows.shape[:-1] + (D,), np.uint8)
    for d in range(D):
        codes[..., d] = rows[..., d % 16 * W + d // 32] >> (4 if d & 16 else 0) & 15
    return codes


def values(rows, scales, D):
    """The numbers that rows [..., row bytes] with scales [..., groups, 2] stand for."""
    s = np.repeat(scales.astype(np.float64), D // scales.shape[-2], axis=-2)
    return s[..., 1] + unpack(rows, D) * s[..., 0]


def turn(x, cos, sin, interleaved):
    """x [T, heads, D] turned by cos, sin [T, rot / 2]."""
    x = np.array(x, np.float64)
    half = cos.shape[-1]
    a = np.arange(half) * 2 if interleaved else np.arange(half)
    b = a + 1 if interleaved else a + half
    c, s = (np.asarray(v, np.float64)[:, None, :] for v in (cos, sin))
    u, w = x[..., a].copy(), x[..., b].copy()
    x[..., a], x[..., b] = u * c - w * s, w * c + u * s
    return x
