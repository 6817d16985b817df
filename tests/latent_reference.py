"""The latent cache, attention over it and the rotation in float64 on the CPU, from their definitions."""

from __future__ import annotations

import math
from fractions import Fraction

import torch

F32, BF16, E4M3 = torch.float32, torch.bfloat16, torch.float8_e4m3fn
U = 2.0 ** -24


def half_step(dtype) -> float:
    """The most a rounding to `dtype` is off, relative to the value."""
    return torch.finfo(dtype).eps / 2


def row_bytes(rank: int, rope: int, store) -> int:
    return rank + 2 * rope + 16 if store == E4M3 else 2 * (rank + rope) + 16


def _e4m3_values() -> torch.Tensor:
    code = torch.arange(256)
    exponent, mantissa = (code >> 3) & 15, (code & 7).double()
    size = torch.where(exponent == 0, mantissa / 512, (8 + mantissa) * 2.0 ** (exponent.double() - 10))
    size[(code & 127) == 127] = torch.nan
    return torch.where(code >= 128, -size, size)


E4M3_VALUES = _e4m3_values()


def contents(cache: torch.Tensor, rank: int, rope: int, store):
    """Latents [.., rank] and key parts [.., rope] of cached rows [.., bytes]."""
    cache = cache.cpu()
    if store == BF16:
        both = cache[..., :2 * (rank + rope)].contiguous().view(BF16).double()
        return both[..., :rank], both[..., rank:]
    scale = cache[..., rank + 2 * rope:rank + 2 * rope + 4].contiguous().view(F32).double()
    return E4M3_VALUES[cache[..., :rank].long()] * scale, cache[..., rank:rank + 2 * rope].contiguous().view(BF16).double()


def nearest(x: torch.Tensor, store) -> torch.Tensor:
    """Rows [.., rank] -> the values that the cache keeps of them."""
    x = x.double()
    if store == BF16:
        kept = x.to(F32).to(BF16).double()
        return torch.where(torch.isfinite(kept).all(-1, keepdim=True), kept, torch.nan)
    fine = torch.isfinite(x).all(-1, keepdim=True)
    y = torch.where(fine, x, 0.0)
    most = y.abs().amax(-1, keepdim=True)
    power = torch.full_like(most, -117.0)
    for e in range(-117, 119):
        power = torch.where(448 * 2.0 ** e < most, torch.tensor(e + 1.0, dtype=torch.float64), power)
    grid = E4M3_VALUES[:127]  # ascending; the code's last bit is the value's
    a = (y / 2.0 ** power).abs()
    low = torch.searchsorted(grid, a.contiguous(), right=True) - 1
    up = (low + 1).clamp(max=126)
    to_up, to_low = grid[up] - a, a - grid[low]
    pick = torch.where((to_up < to_low) | ((to_up == to_low) & (up % 2 == 0)), up, low)
    value = grid[pick] * 2.0 ** power * torch.where(torch.signbit(y), -1.0, 1.0)
    return torch.where(fine, value, torch.nan)


def random_cache(g: torch.Generator, pages: int, page_size: int, rank: int, rope: int, store, garbage: bool = False) -> torch.Tensor:
    """Rows of normal latents and key parts; with `garbage` any bytes at all."""
    n = pages * page_size
    if garbage:
        return torch.randint(0, 256, (pages, page_size, row_bytes(rank, rope, store)), generator=g, dtype=torch.uint8)
    cache = torch.zeros(n, row_bytes(rank, rope, store), dtype=torch.uint8)
    latent, words = torch.randn(n, rank, generator=g), torch.randn(n, rope, generator=g)
    first = rank if store == E4M3 else 2 * rank
    if store == E4M3:
        power = torch.randint(-2, 2, (n, 1), generator=g)
        cache[:, :rank] = (latent * 60).to(E4M3).view(torch.uint8)
        cache[:, first + 2 * rope:first + 2 * rope + 4] = (2.0 ** (power - 6).double()).to(F32).view(torch.uint8)
    else:
        cache[:, :first] = latent.to(BF16).view(torch.uint8)
    cache[:, first:first + 2 * rope] = words.to(BF16).view(torch.uint8)
    return cache.view(pages, page_size, -1)


def random_table(g: torch.Generator, batch: int, width: int, pages: int) -> torch.Tensor:
    assert batch * width <= pages
    return torch.randperm(pages, generator=g)[:batch * width].view(batch, width).to(torch.int32)


def seen_places(position: int, index: int, length: int, bits) -> list[int]:
    """The places that token `index` of a call sees; `bits` is its word of ancestors, or None."""
    if position < 0:
        return []
    if bits is None:
        return list(range(position + 1))
    base = position - index
    return list(range(max(base, 0))) + [base + j for j in range(length) if bits >> j & 1 and base + j >= 0]


def attention(q_latent, q_rope, cache, table, positions, scale, store, ancestors=None):
    """(result, sum of weight * |value|, the scores' rounding scale): float64, [B, L, H, R] twice and [B, L, H]."""
    q_latent, q_rope, table = q_latent.double().cpu(), q_rope.double().cpu(), table.cpu().long()
    B, L, H, R = q_latent.shape
    latent, words = contents(cache, R, q_rope.shape[3], store)
    pages, page = latent.shape[:2]
    out, size = torch.zeros(B, L, H, R, dtype=torch.float64), torch.zeros(B, L, H, R, dtype=torch.float64)
    spread = torch.zeros(B, L, H, dtype=torch.float64)
    for b in range(B):
        for i in range(L):
            bits = None if ancestors is None else int(ancestors[b, i]) % 2 ** 64
            at = int(positions[b, i])
            if at >= table.shape[1] * page:
                out[b, i] = torch.nan
                continue
            places = torch.tensor(seen_places(at, i, L, bits), dtype=torch.long)
            if len(places) == 0:
                continue
            if (places // page >= table.shape[1]).any():
                out[b, i] = torch.nan
                continue
            ids = table[b, places // page]
            if ((ids < 0) | (ids >= pages)).any():
                out[b, i] = torch.nan
                continue
            c, r = latent[ids, places % page], words[ids, places % page]
            weight = torch.softmax((q_latent[b, i] @ c.t() + q_rope[b, i] @ r.t()) * scale, -1)
            out[b, i], size[b, i] = weight @ c, weight @ c.abs()
            spread[b, i] = (q_latent[b, i].abs() @ c.abs().t() + q_rope[b, i].abs() @ r.abs().t()).amax(-1) * abs(scale)
    return out, size, spread


def attention_bound(size, spread, out, keys: int, dim: int, dtype) -> torch.Tensor:
    """How far float32 arithmetic may be off, element by element. With u = 2^-24: a score is a sum of dim = R + P products,
    (dim + 5) u of the sum of its magnitudes (its scale and the factor of the exponent among them), its difference to the
    maximum takes as much again and exp2 2 ulp; numerator and denominator are sums of `keys` terms (keys u) with a rescaling
    of 4 u a tile of 64 or a part; the quotient 3 u. bf16 rounds the weights of the numerator and the result."""
    weight = 2 * (dim + 5) * U * spread[..., None] + 8 * U
    sums = (keys + 4 * (keys / 64 + 260)) * U
    rel = 2 * (weight + sums) + 3 * U
    bound = rel * size + U * out.abs()
    if dtype == BF16:
        h = half_step(BF16)
        bound = bound + h * size * (1 + rel) + h * out.abs() * 1.01
    return bound + 1e-37


def rotate(x, frequencies, positions, interleaved: bool, magnitude: float) -> torch.Tensor:
    """x [B, L, H, D] with its last lanes rotated, float64."""
    x = x.double().cpu().clone()
    rope = 2 * len(frequencies)
    for b in range(x.shape[0]):
        for i in range(x.shape[1]):
            at = int(positions[b, i])
            if at < 0:
                x[b, i] = 0
                continue
            for j, f in enumerate(frequencies.double().cpu().tolist()):
                angle = _angle(at, f)
                c, s = math.cos(angle) * magnitude, math.sin(angle) * magnitude
                start = x.shape[3] - rope
                first, second = (start + 2 * j, start + 2 * j + 1) if interleaved else (start + j, start + j + rope // 2)
                a, d = x[b, i, :, first].clone(), x[b, i, :, second].clone()
                x[b, i, :, first], x[b, i, :, second] = a * c - d * s, d * c + a * s
    return x


TWO_PI = Fraction(2 * 31415926535897932384626433832795028841971693993751, 10 ** 49)


def _angle(position: int, frequency: float) -> float:
    """position * frequency less whole turns, from the exact product (a float64 product of 2^31 radians is off by 2^-22)."""
    exact = Fraction(frequency) * position
    return float(exact - TWO_PI * (exact // TWO_PI))


def rope_bound(expect, x, dtype, magnitude: float = 1.0) -> torch.Tensor:
    """One rounding of a float64 result, whose own error (an angle and its sine to 2^-40) counts by the head's magnitudes."""
    return half_step(dtype) * expect.abs() * 1.001 + 2.0 ** -40 * magnitude * x.double().abs().amax(-1, keepdim=True) + 1e-45
