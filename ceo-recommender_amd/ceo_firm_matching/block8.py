"""Blocks of 128 values in 8 bits with a power-of-two scale, in torch ops.

What the HIP kernels hold (``tt_block8.h``) for tensors on the CPU: e4m3 rows of
the embedding catalogue, and the two 8-bit Adam states.  A block's scale is
2^e with the smallest e >= -100 for which the largest code covers its largest
finite magnitude; it is stored as the byte e + 127.
"""
from __future__ import annotations

import torch

BLOCK = 128
MIN_EXP = -100
M32 = 0xFFFFFFFF
M64 = (1 << 64) - 1
#: (mantissa bits, largest code as a fraction of 2^9, code of NaN)
E4M3 = (3, 0.875, 0x7F)    # signed, largest 448
E4M4 = (4, 0.9375, 0xFF)   # unsigned, largest 480


def blocks_of(n: int) -> int:
    return -(-n // BLOCK)


def _exponents(b: torch.Tensor, top: float) -> torch.Tensor:
    """b [..., 128] float32 -> scale exponents [...]."""
    a = b.abs()
    a = torch.where(torch.isfinite(a), a, torch.zeros_like(a))
    a = a.amax(-1)
    mant, ex = torch.frexp(a)
    e = (ex - 9 + (mant > top).to(ex.dtype)).clamp_min(MIN_EXP)
    return torch.where(a > 0, e, torch.full_like(e, MIN_EXP))


def scale_values(scales: torch.Tensor) -> torch.Tensor:
    """Scale bytes -> 2^(byte - 127) in float32; byte 255 is NaN."""
    v = torch.exp2(scales.to(torch.float64) - 127).to(torch.float32)
    return torch.where(scales == 255, torch.full_like(v, float("nan")), v)


def encode(x: torch.Tensor):
    """[m, d] of any float type -> e4m3 codes [m, kp] and scale bytes [m, kp / 128] (uint8), kp = d rounded up."""
    m, d = x.shape
    b = torch.nn.functional.pad(x.to(torch.float32), (0, -d % BLOCK)).reshape(m, blocks_of(d), BLOCK)
    e = _exponents(b, E4M3[1])
    y = b * torch.exp2(-e.to(torch.float64)).to(torch.float32).unsqueeze(2)
    # under the largest scale the code after 240 stands for 2^128, which no float holds: what would round to it stays there
    most = torch.where(e == 120, 240.0, 448.0).unsqueeze(2)
    y = torch.where(torch.isfinite(b), torch.minimum(torch.maximum(y, -most), most), torch.full_like(y, float("nan")))
    return y.to(torch.float8_e4m3fn).view(torch.uint8).reshape(m, blocks_of(d) * BLOCK), (e + 127).to(torch.uint8)


def decode(codes: torch.Tensor, scales: torch.Tensor, d: int) -> torch.Tensor:
    """Inverse of encode: float32 [m, d]."""
    v = codes.view(torch.float8_e4m3fn).to(torch.float32).reshape(codes.shape[0], blocks_of(d), BLOCK)
    return (v * scale_values(scales).unsqueeze(2)).reshape(codes.shape)[:, :d]


# ---- the Adam states: magnitudes rounded up or down by a counter hash --------
def _perm32(x: torch.Tensor) -> torch.Tensor:
    x = x ^ (x >> 16)
    x = (x * 0x7FEB352D) & M32
    x = x ^ (x >> 15)
    x = (x * 0x846CA68B) & M32
    return x ^ (x >> 16)


def rounding_key(seed: int, step: int) -> int:
    z = (seed * 0x9E3779B97F4A7C15 + step * 0xD1B54A32D192ED03) & M64
    z = ((z ^ (z >> 30)) * 0xBF58476D1CE4E5B9) & M64
    z = ((z ^ (z >> 27)) * 0x94D049BB133111EB) & M64
    return z ^ (z >> 31)


def rounding_bits(block0: int, n_blocks: int, seed: int, step: int, device=None):
    """Two 16-bit integers per value of blocks block0 .. block0 + n_blocks."""
    key = rounding_key(seed, step)
    b = torch.arange(block0, block0 + n_blocks, device=device)
    rk = (_perm32(b ^ (key & M32)) + (key >> 32)) & M32
    el = (torch.arange(BLOCK, device=device) * 0x9E3779B9) & M32
    h = _perm32(rk.unsqueeze(1) ^ el)
    return h & 0xFFFF, h >> 16


def hold(x: torch.Tensor, bits16: torch.Tensor, fmt, keep_positive: bool):
    """x [nb, 128] float32 (magnitudes, or signed for E4M3) -> codes [nb, 128], scale bytes [nb]."""
    mant, top, nan = fmt
    e = _exponents(x, top)
    y = x.abs() * torch.exp2(-e.to(torch.float64)).to(torch.float32).unsqueeze(1)
    sh = 23 - mant
    z = (y * 2.0 ** -120).view(torch.int32).to(torch.int64)
    c = (z + (bits16 << (sh - 16))) >> sh
    if keep_positive:
        c = torch.where((x > 0) & (c == 0), torch.ones_like(c), c)
    c = torch.where(torch.isfinite(x), c, torch.full_like(c, nan))
    if mant == 3:
        c = c | (torch.signbit(x).to(torch.int64) << 7)
    return c.to(torch.uint8), (e + 127).to(torch.uint8)


def held(codes: torch.Tensor, scales: torch.Tensor, fmt) -> torch.Tensor:
    """The values codes [nb, 128] stand for, float32."""
    mant, _, nan = fmt
    c = codes.to(torch.int32)
    mag = c & 0x7F if mant == 3 else c
    v = (mag << (23 - mant)).view(torch.float32) * 2.0 ** 120 * scale_values(scales).unsqueeze(1)
    v = torch.where(mag == nan, torch.full_like(v, float("nan")), v)
    return torch.where(c >= 128, -v, v) if mant == 3 else v
