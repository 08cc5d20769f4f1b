"""The 4-bit cache format by itself, for tests: packing and values on the CPU."""
import numpy as np
import torch

GRID = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])


def pack(x: torch.Tensor):
    """codes [..., D/2], scales [..., D/32] of bf16 rows, by search over the grid."""
    y = x.double().numpy()
    y = y.reshape(*y.shape[:-1], -1, 32)
    finite = np.isfinite(y).all(-1)
    clean = np.where(finite[..., None], y, 0.0)
    most = np.abs(clean).max(-1)
    # The least e with most <= 7 * 2^e, in 1 - 127 .. 252 - 127.
    _, exponent = np.frexp(np.maximum(most, 1e-300) / 7.0)
    e = np.where(np.ldexp(7.0, exponent - 1) >= most, exponent - 1, exponent)
    e = np.clip(e, -126, 125)
    z = np.abs(clean) / np.ldexp(1.0, e)[..., None]
    distance = np.abs(z[..., None] - GRID)
    nearest = distance.min(-1)
    tie = distance == nearest[..., None]
    even = tie & (np.arange(8) % 2 == 0)
    t = np.where(even.any(-1), even.argmax(-1), tie.argmax(-1))
    t = np.where(np.signbit(clean), t + 8, t)
    t = np.where(finite[..., None], t, 0).astype(np.uint8).reshape(*y.shape[:-2], -1)
    scales = np.where(finite, e + 127, 255).astype(np.uint8)
    return torch.from_numpy(t[..., 0::2] | (t[..., 1::2] << 4)), torch.from_numpy(scales)


def values(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """float64 values of codes and scales (scale 255: NaN)."""
    c = codes.cpu().numpy()
    t = np.stack([c & 15, c >> 4], -1).reshape(*c.shape[:-1], 2 * c.shape[-1])
    v = np.where(t >= 8, -GRID[t % 8], GRID[t % 8])
    s = scales.cpu().numpy().astype(np.int64)
    s = np.where(s == 255, np.nan, np.ldexp(1.0, s - 127))
    return torch.from_numpy(v * np.repeat(s, 32, -1))
