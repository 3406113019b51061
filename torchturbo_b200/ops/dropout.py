"""Dropout masks that are drawn from a counter and never stored.

Philox4x32-10 (Salmon, Moraes, Dror and Shaw, "Parallel random numbers: as easy as 1, 2, 3", 2011) under the key `seed` gives, for the
counter `(g, 0, i mod 2^32, i div 2^32)`, four 32-bit words; their eight 16-bit halves (low half first) belong to columns
`8 g .. 8 g + 7` of row `i`.  A value stays where its half is at least `t = round(65536 p)` and is multiplied by
`65536 / (65536 - t)`: the probability is rounded to a multiple of 2^-16, the mean is kept exactly.  The mask depends on the seed
and the element's place alone, so it is the same on every device, in the backward pass, under activation recomputation and, with
`first_row`, for a shard of the rows as for the whole.
"""
from __future__ import annotations

from dataclasses import dataclass

import torch


@dataclass(frozen=True)
class Dropout:
    """Arguments of a dropout as the kernels take them."""

    t: int
    scale: float
    seed: int
    seed_tensor: torch.Tensor | None
    first_row: int


NONE = Dropout(0, 1.0, 0, None, 0)


def dropout_args(p: float, seed, first_row: int = 0, scale: float = 1.0, device: torch.device | None = None) -> Dropout:
    """Checks a dropout's arguments.  `seed`: an integer in [0, 2^63), an int64 tensor of one value on the `device` of the rows (read
    when the kernel runs: a captured step draws new masks when the tensor is moved on), or None for one drawn from torch's CPU
    generator (so that `torch.manual_seed` and the restored generator state of activation checkpointing apply)."""
    if p == 0.0 and scale == 1.0 and first_row == 0:
        return NONE
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"dropout probability must lie in [0, 1], got {p}")
    if first_row < 0:
        raise ValueError(f"first_row must not be negative, got {first_row}")
    t = round(65536 * p)
    factor = scale * 65536 / (65536 - t) if t < 65536 else 0.0
    if t == 0:
        return Dropout(0, factor, 0, None, first_row)
    tensor = None
    if isinstance(seed, torch.Tensor):
        if seed.dtype != torch.int64 or seed.numel() != 1:
            raise ValueError("a seed tensor is one int64 value")
        if device is not None and seed.device != device:      # as the kernels' launch functions have it
            raise AssertionError(f"a seed tensor is one int64 value on the device of the rows, {device}, got one on {seed.device}")
        seed, tensor = 0, seed.detach()
    elif seed is None:
        if torch.cuda.is_available() and torch.cuda.is_current_stream_capturing():
            raise ValueError("a captured dropout needs a seed: pass an int64 tensor and move it on between replays")
        seed = int(torch.randint(0, 2 ** 62, (1,), device="cpu"))
    elif isinstance(seed, bool) or not isinstance(seed, int) or not 0 <= seed < 2 ** 63:
        raise ValueError(f"a seed is an integer in [0, 2^63), got {seed!r}")
    return Dropout(t, factor, seed, tensor, first_row)


_LOW = 0xFFFFFFFF


def philox(c0, c1, c2, c3, k0, k1):
    """Philox4x32-10 on int64 tensors (or integers) that hold 32-bit words.  A product of two words wraps in 64 bits, which leaves its
    low 64 bits as they are."""
    for _ in range(10):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = ((b >> 32) & _LOW) ^ c1 ^ k0, b & _LOW, ((a >> 32) & _LOW) ^ c3 ^ k1, a & _LOW
        k0, k1 = (k0 + 0x9E3779B9) & _LOW, (k1 + 0xBB67AE85) & _LOW
    return c0, c1, c2, c3


def keep_mask(rows: int, cols: int, drop: Dropout, device) -> torch.Tensor:
    """[rows, cols] booleans: which values stay."""
    if drop.t == 0:
        return torch.ones(rows, cols, dtype=torch.bool, device=device)
    seed = drop.seed if drop.seed_tensor is None else drop.seed_tensor.reshape(()).to(device)
    g = torch.arange((cols + 7) // 8, device=device)[None, :].expand(rows, -1)
    i = (torch.arange(rows, device=device) + drop.first_row)[:, None]
    zero = torch.zeros_like(g)
    words = torch.stack(philox(g, zero, (i & _LOW) + zero, (i >> 32) + zero, seed & _LOW, (seed >> 32) & _LOW), -1)
    return torch.stack((words & 0xFFFF, words >> 16), -1).reshape(rows, 8 * g.shape[1])[:, :cols] >= drop.t


def wide_float(x: torch.Tensor) -> torch.dtype:
    return torch.float64 if x.dtype == torch.float64 else torch.float32


def dropout_ref(x: torch.Tensor, drop: Dropout, residual: torch.Tensor | None = None) -> torch.Tensor:
    """`residual + dropout(x)` over the rows of `x` (all but its last dimension), in fp32 (fp64 for fp64) and rounded once."""
    wide = wide_float(x)
    v = x.to(wide) * drop.scale
    if drop.t:
        keep = keep_mask(x.numel() // max(x.shape[-1], 1), x.shape[-1], drop, x.device).view(x.shape)
        v = torch.where(keep, v, torch.zeros_like(v))
    if residual is not None:
        v = v + residual.to(wide)
    return v.to(x.dtype)
