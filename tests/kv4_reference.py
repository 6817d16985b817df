"""The 4-bit values, the cache and attention over it in float64 on the CPU, from their definitions."""

from __future__ import annotations

import torch

_SIZES = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)


def value_of(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """[..., 16 g] packed codes and [..., g] scale bytes -> [..., 32 g] values."""
    codes = codes.long()
    both = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)
    value = _SIZES[both & 7] * torch.where(both >= 8, -1.0, 1.0)
    power = torch.where(scales.long() == 255, torch.nan, 2.0 ** (scales.double() - 127))
    return (value.unflatten(-1, (-1, 32)) * power[..., None]).flatten(-2)


def nearest(x: torch.Tensor) -> torch.Tensor:
    """[..., 32 g] -> the values that quantisation keeps: for each group the smallest power of two (exponents -124 to 125)
    whose six-fold reaches the largest magnitude, the nearest value of that grid, ties to the even code."""
    x = x.double().unflatten(-1, (-1, 32))
    fine = torch.isfinite(x).all(-1, keepdim=True)
    most = torch.where(fine, x, 0.0).abs().amax(-1, keepdim=True)
    exponent = torch.full_like(most, -124.0)
    for e in range(-124, 125):
        exponent = torch.where(6 * 2.0 ** e < most, torch.tensor(e + 1.0, dtype=torch.float64), exponent)
    y = (torch.where(fine, x, 0.0) / 2.0 ** exponent).abs()
    distance = (y[..., None] - _SIZES).abs()
    even_first = torch.tensor([0, 2, 4, 6, 1, 3, 5, 7])  # argmin takes the first of equals
    pick = even_first[distance[..., even_first].argmin(-1)]
    value = _SIZES[pick] * 2.0 ** exponent * torch.where(torch.signbit(x), -1.0, 1.0)
    return torch.where(fine, value, torch.nan).flatten(-2)


def parts(cache: torch.Tensor, page_size: int, dim: int):
    """Views of a cache [pages, heads, bytes]: key codes, value codes, key scales, value scales."""
    a, b = page_size * dim // 2, page_size * dim // 32
    return (cache[..., :a].unflatten(-1, (page_size, dim // 2)), cache[..., a:2 * a].unflatten(-1, (dim // 2, page_size)),
            cache[..., 2 * a:2 * a + b].unflatten(-1, (page_size, dim // 32)), cache[..., 2 * a + b:].unflatten(-1, (dim // 32, page_size)))


def contents(cache: torch.Tensor, page_size: int, dim: int):
    """Keys and values [pages, heads, page_size, dim] of a whole cache."""
    kc, vc, ks, vs = parts(cache.cpu(), page_size, dim)
    return value_of(kc, ks), value_of(vc.transpose(-1, -2), vs.transpose(-1, -2))


def attention(q, keys, values, table, positions, scale):
    """(result, sum of weight * |value|, the scores' rounding scale) [B, L, H, D] / [B, L, H], float64. keys and values as
    ``contents`` gives them. A token whose position is negative gives 0; one whose keys are not all there NaN."""
    q, table, positions = q.double().cpu(), table.cpu(), positions.cpu()
    B, L, H, D = q.shape
    pages, heads, page_size, _ = keys.shape
    out, size, spread = torch.zeros(B, L, H, D, dtype=torch.float64), torch.zeros(B, L, H, D, dtype=torch.float64), torch.zeros(B, L, H, dtype=torch.float64)
    for b in range(B):
        for i in range(L):
            n = int(positions[b, i]) + 1
            if n <= 0:
                continue
            need = -(-n // page_size)
            ids = table[b, :need].long()
            if need > table.shape[1] or (ids < 0).any() or (ids >= pages).any():
                out[b, i] = torch.nan
                continue
            k = keys[ids].transpose(0, 1).flatten(1, 2)[:, :n]  # [heads, n, D]
            v = values[ids].transpose(0, 1).flatten(1, 2)[:, :n]
            rows = q[b, i].unflatten(0, (heads, -1))  # [heads, group, D]
            weight = torch.softmax(rows @ k.transpose(1, 2) * scale, -1)
            out[b, i] = (weight @ v).flatten(0, 1)
            size[b, i] = (weight @ v.abs()).flatten(0, 1)
            spread[b, i] = ((rows.abs() @ k.abs().transpose(1, 2)).amax(-1) * abs(scale)).flatten(0, 1)
    return out, size, spread


def attention_bound(size, spread, out, keys: int, dim: int, dtype) -> torch.Tensor:
    """How far float32 arithmetic may be off, element by element. With u = 2^-24: a score is a sum of dim products
    (dim + 3) u of the sum of its magnitudes, its difference to the maximum takes as much again and exp2 2 ulp; numerator
    and denominator are sums of `keys` terms (n u) with a rescaling of 4 u a tile of 64; the quotient 3 u. bf16 rounds
    the weights of the numerator (2^-8) and the result (2^-8)."""
    u = 2.0 ** -24
    weight = 2 * (dim + 3) * u * spread[..., None] + 8 * u
    sums = (keys + 4 * (keys / 64 + 8)) * u
    rel = 2 * (weight + sums) + 3 * u
    bound = rel * size + u * out.abs()
    if dtype == torch.bfloat16:
        bound = bound + 2.0 ** -8 * size * (1 + rel) + 2.0 ** -8 * out.abs() * 1.01
    return bound + 1e-37


def random_cache(g: torch.Generator, pages: int, heads: int, page_size: int, dim: int) -> torch.Tensor:
    """Random codes, scale bytes of a few powers of two around 1/2."""
    cache = torch.randint(0, 256, (pages, heads, page_size * (dim + dim // 16)), generator=g, dtype=torch.uint8)
    n = page_size * dim
    cache[..., n:] = torch.randint(124, 128, cache[..., n:].shape, generator=g, dtype=torch.uint8)
    return cache


def random_table(g: torch.Generator, batch: int, width: int, pages: int) -> torch.Tensor:
    assert batch * width <= pages
    return torch.randperm(pages, generator=g)[:batch * width].view(batch, width).to(torch.int32)
